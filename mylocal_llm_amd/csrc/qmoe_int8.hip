// Row quantisation, weight tiles, and the linear / SwiGLU products of 8-bit codes.
#include "qmoe_int8.hpp"

namespace qmoe {

// ---- rows -> codes + scales ------------------------------------------------------------------------------
// One workgroup a row, NX pieces of eight values a thread in registers between the search for the largest and the
// codes: a row is read once.  Bound by the memory for many rows (4096 x 4096, a dozen inputs in turn: fp32 15.1 us, 5.6 TB/s of
// reads and writes; bf16 11.2 us, 4.5 TB/s, or 13.2 where half the waves hold a value next to a half), by one round trip and one meeting for a few (1 x 4096 2.0 - 2.4 us, launch included).
//   vec   a row starts 16-byte aligned and ends on a multiple of eight values: 16-byte loads, 8-byte stores
//   else  neighbouring threads take neighbouring values: whole lines still, 2 or 4 bytes a thread
template <int DT, int NX, bool VEC>
__global__ __launch_bounds__(1024) void int8_quantize_kernel(const void* __restrict__ x, int k, uint8_t* __restrict__ codes, int64_t ld,
                                                             int width, float* __restrict__ scales) {
    __shared__ uint32_t tops[16];
    const int tid = threadIdx.x, threads = blockDim.x;
    const int64_t row = blockIdx.x;
    const size_t base = (size_t)row * k;
    float v[NX][8];
    uint32_t top = 0;
#pragma unroll
    for (int p = 0; p < NX; ++p) {
        if (VEC) {
            const int i = (p * threads + tid) * 8;
            int8_load8<DT>(x, i < k ? base + i : base, k - i, true, v[p]);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int i = (p * 8 + j) * threads + tid;
                const float f = Elem<DT>::load(x, i < k ? base + i : base);
                v[p][j] = i < k ? f : 0.0f;
            }
        }
    }
#pragma unroll
    for (int p = 0; p < NX; ++p)
#pragma unroll
        for (int j = 0; j < 8; ++j) { const uint32_t b = abs_bits(v[p][j]); top = b > top ? b : top; }
    top = wave_max_u32(top);
    if (threads > 64) {
        if ((tid & 63) == 0) tops[tid >> 6] = top;
        __syncthreads();
        for (int i = 0; i < threads / 64; ++i) top = tops[i] > top ? tops[i] : top;
    }
    const RowScale r(top);
    uint8_t* const out = codes + row * ld;
#pragma unroll
    for (int p = 0; p < NX; ++p) {
        if (VEC) {
            const int i = (p * threads + tid) * 8;
            if (i < width) *(QMOE_GLOBAL u32x2_t*)(out + i) = int8_code8(v[p], r);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int i = (p * 8 + j) * threads + tid;
                if (i < width) stg<uint8_t>(out + i, int8_code(v[p][j], r));
            }
        }
    }
    if (tid == 0) stg<float>(scales + row, r.s);
}

// Rows longer than the registers of a workgroup (65536 values, 32768 at odd addresses): read twice, the second time from L2.
// (As they are rare, values one by one: 1024 rows of 20000 would take 38.9 us here, 16.4 above.)
template <int DT>
__global__ __launch_bounds__(1024) void int8_quantize_long_kernel(const void* __restrict__ x, int64_t k, uint8_t* __restrict__ codes,
                                                                  int64_t ld, int64_t width, float* __restrict__ scales) {
    __shared__ uint32_t tops[16];
    const int tid = threadIdx.x;
    const int64_t row = blockIdx.x;
    const size_t base = (size_t)row * k;
    uint32_t top = 0;
    for (int64_t i = tid; i < k; i += 1024) {
        const uint32_t b = abs_bits(Elem<DT>::load(x, base + i));
        top = b > top ? b : top;
    }
    top = wave_max_u32(top);
    if ((tid & 63) == 0) tops[tid >> 6] = top;
    __syncthreads();
    for (int i = 0; i < 16; ++i) top = tops[i] > top ? tops[i] : top;
    const RowScale r(top);
    for (int64_t i = tid; i < width; i += 1024)
        stg<uint8_t>(codes + row * ld + i, i < k ? int8_code(Elem<DT>::load(x, base + i), r) : (uint8_t)0);
    if (tid == 0) stg<float>(scales + row, r.s);
}

template <int DT> static int quantize_as(const void* x, int64_t rows, int k, uint8_t* codes, int64_t ld, int width, float* scales, hipStream_t s) {
    constexpr int64_t MOST = 4000000;      // rows of a launch: its threads are counted in 32 bits
    if (rows > MOST) {
        if (const int rc = quantize_as<DT>(x, MOST, k, codes, ld, width, scales, s)) return rc;
        return quantize_as<DT>((const char*)x + MOST * k * (int64_t)sizeof(typename Elem<DT>::T), rows - MOST, k, codes + MOST * ld, ld, width, scales + MOST, s);
    }
    const dim3 grid((unsigned)rows);
    const int64_t eights = ((int64_t)width + 7) / 8;      // (width + 7 of the longest rows passes 32 bits)
    const bool vec = k % 8 == 0 && (uintptr_t)x % 16 == 0 && (uintptr_t)codes % 8 == 0 && ld % 8 == 0;
    if (eights > (vec ? 8192 : 4096)) {
        hipLaunchKernelGGL(int8_quantize_long_kernel<DT>, grid, dim3(1024), 0, s, x, (int64_t)k, codes, ld, (int64_t)width, scales);
        return check_launch("int8 row quantisation");
    }
    // Few rows are a chain of latencies: as many threads as there are pieces (one row of 4096 bf16 2.4 us, with two pieces a
    // thread 2.7).  Many rows: more in flight with two (4096 x 4096 bf16 15.1 -> 12.9 us; rows of 512 values 4.5 -> 4.8).
    const int nx = eights > 4096 ? 8 : eights > 2048 ? 4 : eights > 1024 || (rows >= 1024 && eights >= 128) ? 2 : 1;
    const dim3 block((unsigned)(((eights + nx - 1) / nx + 63) / 64 * 64));
#define QMOE_QUANTIZE(NX, VEC) hipLaunchKernelGGL((int8_quantize_kernel<DT, NX, VEC>), grid, block, 0, s, x, k, codes, ld, width, scales)
    if (nx == 1) { if (vec) QMOE_QUANTIZE(1, true); else QMOE_QUANTIZE(1, false); }
    else if (nx == 2) { if (vec) QMOE_QUANTIZE(2, true); else QMOE_QUANTIZE(2, false); }
    else if (nx == 4) { if (vec) QMOE_QUANTIZE(4, true); else QMOE_QUANTIZE(4, false); }
    else QMOE_QUANTIZE(8, true);
#undef QMOE_QUANTIZE
    return check_launch("int8 row quantisation");
}

int int8_quantize_launch(const void* x, int dt, int64_t rows, int k, uint8_t* codes, int64_t ld, bool pad, float* scales, hipStream_t s) {
    const int width = pad ? (int)int8_cols256(k) : k;
    if (dt == QMOE_DT_F32) return quantize_as<QMOE_DT_F32>(x, rows, k, codes, ld, width, scales, s);
    if (dt == QMOE_DT_F16) return quantize_as<QMOE_DT_F16>(x, rows, k, codes, ld, width, scales, s);
    return quantize_as<QMOE_DT_BF16>(x, rows, k, codes, ld, width, scales, s);
}

// Codes given by the caller with a row step the tiles of many tokens cannot read: copied once, tail zero.  (4096 x 4096 x 1000
// with the copy 36.4 us, from fp32 rows quantised on the way 35.6.)
__global__ __launch_bounds__(256) void int8_restep_kernel(const uint8_t* __restrict__ in, int k, uint8_t* __restrict__ out, int64_t ld) {
    const int64_t row = blockIdx.x;
    for (int i = threadIdx.x; i < ld; i += 256) stg<uint8_t>(out + row * ld + i, i < k ? ldg<uint8_t>(in + row * k + i) : (uint8_t)0);
}

// ---- weight tiles ----------------------------------------------------------------------------------------
// A workgroup a row of tiles: 16 rows of codes.  Every row of tiles of all matrices, one behind the other.  Done once a weight,
// bound by the memory: 512 matrices of 512 x 2048 in 192 us, 5.6 TB/s of reads and writes.
__global__ __launch_bounds__(256) void int8_tiles_kernel(const uint8_t* __restrict__ all_codes, int n, int k, int row_tiles,
                                                         uint8_t* __restrict__ all_tiles) {
    const int64_t matrix = blockIdx.x / row_tiles;
    const int rt = (int)(blockIdx.x % row_tiles), kt = (k + 63) / 64;
    const uint8_t* const codes = all_codes + matrix * n * (int64_t)k;
    uint8_t* const tiles = all_tiles + (int64_t)blockIdx.x * kt * 1024;
    for (int p = threadIdx.x; p < kt * 64; p += 256) {
        const int lane = p & 63, row = rt * 16 + (lane & 15), col = (p >> 6) * 64 + (lane >> 4) * 16;
        uint32_t v[4] = {0, 0, 0, 0};
        if (row < n && col + 16 <= k) {
            const i32x4_t w = *(const QMOE_GLOBAL i32x4_unaligned_t*)(codes + (int64_t)row * k + col);
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = (uint32_t)w[j];
        } else if (row < n) {
#pragma unroll
            for (int j = 0; j < 16; ++j)
                if (col + j < k) v[j >> 2] |= (uint32_t)ldg<uint8_t>(codes + (int64_t)row * k + col + j) << (8 * (j & 3));
        }
        *(QMOE_GLOBAL u32x4_t*)(tiles + (int64_t)p * 16) = u32x4_t{v[0], v[1], v[2], v[3]};
    }
}

static size_t round256(size_t v) { return (v + 255) & ~(size_t)255; }

static bool codes_as_they_are(const void* x, int k) { return k % 256 == 0 && (uintptr_t)x % 16 == 0; }

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
    if (n > (1 << 26) || tokens > (1 << 22)) return fail(QMOE_EUNSUPPORTED, "%s: more than 2^26 channels or 2^22 tokens; split the call", who);
    if (tokens == 0) return QMOE_OK;
    const size_t need = qmoe_int8_workspace_bytes(n, k, tokens, xdt);
    const bool direct = xdt == QMOE_DT_I8 && codes_as_they_are(x, k);
    if (!direct && need && (!workspace || (uintptr_t)workspace % 256 || bytes < need))
        return fail(QMOE_EWORKSPACE, "%s: workspace must be 256-byte aligned and hold %zu bytes (got %zu)", who, need, bytes);
    Int8Product a{};
    a.w = (const uint8_t*)w; a.w2 = (const uint8_t*)w2; a.c = c; a.c2 = c2;
    a.n = n; a.kp = (int)int8_cols64(k); a.tokens = tokens; a.y = y; a.ydt = ydt; a.ldy = n; a.ld = int8_cols256(k);
    a.q = (const uint8_t*)x; a.s = xs;
    if (xdt != QMOE_DT_I8 && int8_few_fuses(tokens, k)) return int8_few_launch(a, pair, x, xdt, k, st);
    const bool few = int8_few_takes(n, tokens, pair);
    if (xdt != QMOE_DT_I8) {
        uint8_t* const q = (uint8_t*)workspace;
        float* const s = (float*)(q + round256((size_t)tokens * a.ld));
        a.q = q;
        a.s = s;
        if (const int rc = int8_quantize_launch(x, xdt, tokens, k, q, a.ld, true, s, st)) return rc;
    } else if (few) a.ld = k;            // (read as they are, at any alignment)
    else if (!direct) {
        a.q = (const uint8_t*)workspace;
        hipLaunchKernelGGL(int8_restep_kernel, dim3(tokens), dim3(256), 0, st, (const uint8_t*)x, k, (uint8_t*)workspace, a.ld);
        if (const int rc = check_launch(who)) return rc;
    }
    return few ? int8_few_launch(a, pair, nullptr, 0, k, st) : int8_gemm_launch(a, pair, st);
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
    const int row_tiles = (int)(int8_rows16(n) / 16);
    if (matrices > ((1 << 24) - 1) / row_tiles) return fail(QMOE_EUNSUPPORTED, "%s: 2^24 or more rows of tiles; lay the matrices out in parts", who);
    hipLaunchKernelGGL(int8_tiles_kernel, dim3((unsigned)(matrices * row_tiles)), dim3(256), 0, (hipStream_t)stream, (const uint8_t*)codes, n, k,
                       row_tiles, (uint8_t*)tiles);
    return check_launch(who);
}

size_t qmoe_int8_workspace_bytes(int n, int k, int tokens, int x_dtype) {
    if (n < 1 || k < 1 || tokens < 1) return 0;
    if (x_dtype == QMOE_DT_INT8 ? int8_few_takes(n, tokens, false) : int8_few_fuses(tokens, k)) return 0;
    return round256((size_t)tokens * (size_t)int8_cols256(k)) + round256((size_t)tokens * 4);
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
