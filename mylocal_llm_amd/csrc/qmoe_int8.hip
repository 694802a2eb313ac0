// Row quantisation, weight tiles, and the linear / SwiGLU products of 8-bit codes.
#include "qmoe_int8.hpp"

namespace qmoe {

// ---- rows -> codes + scales ------------------------------------------------------------------------------
template <int DT>
__global__ __launch_bounds__(256) void int8_quantize_kernel(const void* __restrict__ x, int k, uint8_t* __restrict__ codes, int64_t ld,
                                                            int width, float* __restrict__ scales) {
    __shared__ uint32_t tops[4];
    const int64_t row = blockIdx.x;
    const size_t base = (size_t)row * k;
    uint32_t top = 0;
    for (int i = threadIdx.x; i < k; i += 256) {
        const uint32_t b = abs_bits(Elem<DT>::load(x, base + i));
        top = b > top ? b : top;
    }
    top = wave_top(top);
    if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = top;
    __syncthreads();
    for (int i = 0; i < 4; ++i) top = tops[i] > top ? tops[i] : top;
    const RowScale r(top);
    for (int i = threadIdx.x; i < width; i += 256)
        stg<uint8_t>(codes + row * ld + i, i < k ? (uint8_t)int8_code(Elem<DT>::load(x, base + i), r.inv) : (uint8_t)0);
    if (threadIdx.x == 0) stg<float>(scales + row, r.s);
}

int int8_quantize_launch(const void* x, int dt, int64_t rows, int k, uint8_t* codes, int64_t ld, bool pad, float* scales, hipStream_t s) {
    const int width = pad ? (int)int8_cols64(k) : k;
    const dim3 grid((unsigned)rows), block(256);
    if (dt == QMOE_DT_F32) hipLaunchKernelGGL(int8_quantize_kernel<QMOE_DT_F32>, grid, block, 0, s, x, k, codes, ld, width, scales);
    else if (dt == QMOE_DT_F16) hipLaunchKernelGGL(int8_quantize_kernel<QMOE_DT_F16>, grid, block, 0, s, x, k, codes, ld, width, scales);
    else hipLaunchKernelGGL(int8_quantize_kernel<QMOE_DT_BF16>, grid, block, 0, s, x, k, codes, ld, width, scales);
    return check_launch("int8 row quantisation");
}

// codes given by the caller with a row step the products cannot read: copied once, tail zero
__global__ __launch_bounds__(256) void int8_restep_kernel(const uint8_t* __restrict__ in, int k, uint8_t* __restrict__ out, int64_t ld) {
    const int64_t row = blockIdx.x;
    for (int i = threadIdx.x; i < ld; i += 256) stg<uint8_t>(out + row * ld + i, i < k ? ldg<uint8_t>(in + row * k + i) : (uint8_t)0);
}

// ---- weight tiles ----------------------------------------------------------------------------------------
__global__ __launch_bounds__(256) void int8_tiles_kernel(const uint8_t* __restrict__ codes, int64_t n, int64_t k, int64_t pieces,
                                                         uint8_t* __restrict__ tiles) {
    const int64_t kt = (k + 63) / 64;
    for (int64_t p = (int64_t)blockIdx.x * 256 + threadIdx.x; p < pieces; p += (int64_t)gridDim.x * 256) {
        const int lane = (int)(p & 63);
        const int64_t tile = p >> 6, row = tile / kt * 16 + (lane & 15), col = tile % kt * 64 + (lane >> 4) * 16;
        uint32_t v[4] = {0, 0, 0, 0};
        if (row < n) {
#pragma unroll
            for (int j = 0; j < 16; ++j)
                if (col + j < k) v[j >> 2] |= (uint32_t)ldg<uint8_t>(codes + row * k + col + j) << (8 * (j & 3));
        }
        *(QMOE_GLOBAL u32x4_t*)(tiles + p * 16) = u32x4_t{v[0], v[1], v[2], v[3]};
    }
}

// ---- products: one wave per 16 channels x 16 tokens ---------------------------------------------------------
template <bool PAIR>
__global__ __launch_bounds__(64) void int8_product_kernel(const Int8Product a) {
    const int lane = threadIdx.x, col = lane & 15, g = lane >> 4;
    int first = blockIdx.y * 16, count = a.tokens - first, expert = 0;
    if (a.n_chunks) {
        if ((int)blockIdx.y >= *a.n_chunks) return;
        expert = a.chunk_expert[blockIdx.y];
        first = a.chunk_start[blockIdx.y];
        count = a.chunk_count[blockIdx.y];
    }
    const int pos = first + (col < count ? col : 0);
    const int64_t row = a.row_of ? a.row_of[pos] : pos;
    const uint8_t* q = a.q + row * a.ld + g * 16;
    const int64_t at = (int64_t)blockIdx.x * a.kp * 16 + lane * 16 + expert * a.w_step;
    i32x4_t acc = {0, 0, 0, 0}, acc2 = {0, 0, 0, 0};
    for (int k = 0; k < a.kp; k += 64) {
        const i32x4_t b = ldg_i32x4(q + k);
        acc = mfma_i8(ldg_i32x4(a.w + at + (int64_t)k * 16), b, acc);
        if (PAIR) acc2 = mfma_i8(ldg_i32x4(a.w2 + at + (int64_t)k * 16), b, acc2);
    }
    if (col >= count) return;
    const float s = a.s[row];
    for (int i = 0; i < 4; ++i) {
        const int n = blockIdx.x * 16 + 4 * g + i;
        if (n >= a.n) break;
        const double v = int8_value(acc[i], s, a.c[(int64_t)expert * a.n + n]);
        const size_t out = (size_t)(pos * a.ldy + n);
        if (!PAIR) { store_out(a.y, a.ydt, out, (float)v); continue; }
        const double u = int8_value(acc2[i], s, a.c2[(int64_t)expert * a.n + n]);
        store_out(a.y, a.ydt, out, int8_hidden(v, u));
    }
}

int int8_product_launch(const Int8Product& a, bool pair, int chunks, hipStream_t s) {
    const dim3 grid((a.n + 15) / 16, a.n_chunks ? chunks : (a.tokens + 15) / 16);
    if (pair) hipLaunchKernelGGL(int8_product_kernel<true>, grid, dim3(64), 0, s, a);
    else hipLaunchKernelGGL(int8_product_kernel<false>, grid, dim3(64), 0, s, a);
    return check_launch("int8 product");
}

static size_t round256(size_t v) { return (v + 255) & ~(size_t)255; }

static bool codes_as_they_are(const void* x, int k) { return k % 64 == 0 && (uintptr_t)x % 16 == 0; }

static int dense(const char* who, bool pair, const void* w, const float* c, const void* w2, const float* c2, int n, int k, const void* x,
                 int xdt, const float* xs, int tokens, void* y, int ydt, void* workspace, size_t bytes, hipStream_t st) {
    if (!w || !c || (pair && (!w2 || !c2)) || !x || !y) return fail(QMOE_EINVAL, "%s: null pointer", who);
    if (n < 1 || k < 1 || tokens < 0) return fail(QMOE_EINVAL, "%s: sizes must be positive (n=%d k=%d tokens=%d)", who, n, k, tokens);
    if (k > INT8_MAX_K) return fail(QMOE_EUNSUPPORTED, "%s: K=%d beyond %d, where an int32 sum could overflow", who, k, INT8_MAX_K);
    if (xdt != QMOE_DT_I8 && !dtype_size(xdt)) return fail(QMOE_EINVAL, "%s: unknown activation type %d", who, xdt);
    if (!dtype_size(ydt)) return fail(QMOE_EINVAL, "%s: unknown output type %d", who, ydt);
    if (xdt == QMOE_DT_I8 && !xs) return fail(QMOE_EINVAL, "%s: codes need their scales", who);
    if ((uintptr_t)w % 16 || (pair && (uintptr_t)w2 % 16) || (uintptr_t)c % 4 || (pair && (uintptr_t)c2 % 4) || (uintptr_t)xs % 4 ||
        (xdt != QMOE_DT_I8 && (uintptr_t)x % dtype_size(xdt)) || (uintptr_t)y % dtype_size(ydt))
        return fail(QMOE_EINVAL, "%s: misaligned pointer", who);
    if (tokens == 0) return QMOE_OK;
    const size_t need = qmoe_int8_workspace_bytes(n, k, tokens);
    const bool direct = xdt == QMOE_DT_I8 && codes_as_they_are(x, k);
    if (!direct && (!workspace || (uintptr_t)workspace % 256 || bytes < need))
        return fail(QMOE_EWORKSPACE, "%s: workspace must be 256-byte aligned and hold %zu bytes (got %zu)", who, need, bytes);
    Int8Product a{};
    a.w = (const uint8_t*)w; a.w2 = (const uint8_t*)w2; a.c = c; a.c2 = c2;
    a.n = n; a.kp = (int)int8_cols64(k); a.tokens = tokens; a.y = y; a.ydt = ydt; a.ldy = n; a.ld = a.kp;
    a.q = (const uint8_t*)x; a.s = xs;
    if (!direct) {
        uint8_t* q = (uint8_t*)workspace;
        a.q = q;
        if (xdt == QMOE_DT_I8) {
            hipLaunchKernelGGL(int8_restep_kernel, dim3(tokens), dim3(256), 0, st, (const uint8_t*)x, k, q, a.ld);
            if (const int rc = check_launch(who)) return rc;
        } else {
            float* s = (float*)(q + round256((size_t)tokens * a.ld));
            a.s = s;
            if (const int rc = int8_quantize_launch(x, xdt, tokens, k, q, a.ld, true, s, st)) return rc;
        }
    }
    return int8_product_launch(a, pair, 0, st);
}

}  // namespace qmoe

using namespace qmoe;

extern "C" {

size_t qmoe_int8_matrix_bytes(int n, int k) { return n < 1 || k < 1 ? 0 : (size_t)int8_matrix_bytes(n, k); }

int qmoe_int8_quantize(const void* x, int x_dtype, int64_t rows, int k, void* codes, float* scales, void* stream) {
    const char* who = "qmoe_int8_quantize";
    if (!x || !codes || !scales) return fail(QMOE_EINVAL, "%s: null pointer", who);
    if (!dtype_size(x_dtype)) return fail(QMOE_EINVAL, "%s: unknown activation type %d", who, x_dtype);
    if (rows < 0 || k < 1) return fail(QMOE_EINVAL, "%s: rows=%lld k=%d", who, (long long)rows, k);
    if (rows > INT32_MAX) return fail(QMOE_EUNSUPPORTED, "%s: more than 2^31 - 1 rows", who);
    if ((uintptr_t)x % dtype_size(x_dtype) || (uintptr_t)scales % 4) return fail(QMOE_EINVAL, "%s: misaligned pointer", who);
    if (rows == 0) return QMOE_OK;
    return int8_quantize_launch(x, x_dtype, rows, k, (uint8_t*)codes, k, false, scales, (hipStream_t)stream);
}

int qmoe_int8_tiles(const void* codes, int64_t matrices, int n, int k, void* tiles, void* stream) {
    const char* who = "qmoe_int8_tiles";
    if (!codes || !tiles) return fail(QMOE_EINVAL, "%s: null pointer", who);
    if (matrices < 1 || n < 1 || k < 1) return fail(QMOE_EINVAL, "%s: matrices=%lld n=%d k=%d", who, (long long)matrices, n, k);
    if (k > INT8_MAX_K) return fail(QMOE_EUNSUPPORTED, "%s: K=%d beyond %d, where an int32 sum could overflow", who, k, INT8_MAX_K);
    if ((uintptr_t)tiles % 16) return fail(QMOE_EINVAL, "%s: tiles must be 16-byte aligned", who);
    const int64_t pieces = int8_matrix_bytes(n, k) / 16;
    const int64_t blocks = (pieces + 255) / 256;
    for (int64_t m = 0; m < matrices; ++m)
        hipLaunchKernelGGL(int8_tiles_kernel, dim3((unsigned)(blocks < 4096 ? blocks : 4096)), dim3(256), 0, (hipStream_t)stream,
                           (const uint8_t*)codes + m * n * (int64_t)k, (int64_t)n, (int64_t)k, pieces, (uint8_t*)tiles + m * pieces * 16);
    return check_launch(who);
}

size_t qmoe_int8_workspace_bytes(int n, int k, int tokens) {
    if (n < 1 || k < 1 || tokens < 1) return 0;
    return round256((size_t)tokens * (size_t)int8_cols64(k)) + round256((size_t)tokens * 4);
}

int qmoe_int8_linear(const void* tiles, const float* channel_scales, int n, int k, const void* x, int x_dtype, const float* x_scales,
                     int tokens, void* y, int y_dtype, void* workspace, size_t workspace_bytes, void* stream) {
    return dense("qmoe_int8_linear", false, tiles, channel_scales, nullptr, nullptr, n, k, x, x_dtype, x_scales, tokens, y, y_dtype,
                 workspace, workspace_bytes, (hipStream_t)stream);
}

int qmoe_int8_swiglu(const void* gate, const float* gate_scales, const void* up, const float* up_scales, int f, int k, const void* x,
                     int x_dtype, const float* x_scales, int tokens, void* h, int h_dtype, void* workspace, size_t workspace_bytes,
                     void* stream) {
    return dense("qmoe_int8_swiglu", true, gate, gate_scales, up, up_scales, f, k, x, x_dtype, x_scales, tokens, h, h_dtype, workspace,
                 workspace_bytes, (hipStream_t)stream);
}

}  // extern "C"
