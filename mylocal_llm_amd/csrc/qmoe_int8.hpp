// 8-bit integer operators: codes with a scale for each token (activations) and for each output
// channel (weights).
//
//   q[t, k] = rint(x[t, k] / s[t]),  s[t] = fl32(max_k |x[t, k]| / 127)      (halves to even, |q| <= 127)
//   y[t, n] = (sum_k q[t, k] w[n, k]) * s[t] * c[n]                            (int32 sum: exact)
//
// Weight layout ("tiles"): [N/16][K/64][lane][16] bytes, lane l of a 1 KB tile holding columns
// 16 (l / 16) .. + 15 of row l % 16 -- the A operand of v_mfma_i32_16x16x64_i8 as a wave reads it,
// 1 KB of consecutive memory an instruction.  Rows are padded to 16 and columns to 64 with zero
// codes.  Activation codes are row-major with a row step that is a multiple of 16 bytes; behind its K
// columns a row holds zeros up to a multiple of 256 (the products of many tokens read that far).  Lane l
// reads the B operand as the 16 bytes at column 16 (l / 16) of token l % 16.  D[i] of lane l is the
// sum of weight row 4 (l / 16) + i and token l % 16: four neighbouring outputs of one token.
#pragma once
#include "qmoe_router.hpp"

namespace qmoe {

typedef int i32x4_t __attribute__((ext_vector_type(4)));
typedef i32x4_t i32x4_unaligned_t __attribute__((aligned(1)));      // (one request all the same)
typedef i32x4_t i32x4_dword_t __attribute__((aligned(4)));

static constexpr int INT8_MAX_K = 131071;     // 128 * 128 * K stays inside int32
static constexpr int QMOE_DT_I8 = QMOE_DT_INT8;

__host__ __device__ inline int64_t int8_rows16(int64_t n) { return (n + 15) / 16 * 16; }
__host__ __device__ inline int64_t int8_cols64(int64_t k) { return (k + 63) / 64 * 64; }
__host__ __device__ inline int64_t int8_cols256(int64_t k) { return (k + 255) / 256 * 256; }
inline int64_t int8_matrix_bytes(int64_t n, int64_t k) { return int8_rows16(n) * int8_cols64(k); }

__device__ __forceinline__ i32x4_t mfma_i8(i32x4_t a, i32x4_t b, i32x4_t c) {
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ i32x4_t ldg_i32x4(const void* p) { return *(const QMOE_GLOBAL i32x4_t*)p; }

// The scale of a row.  `top` is the largest |x| of the row as bits (NaN and infinity compare above every finite value).  A
// row that is not finite gets the scale NaN and codes of zero, so that every product of that row is NaN instead of a
// plausible number.
struct RowScale {
    float s, inv;        // inv: fl(1 / s), used where `plain`
    bool finite, plain;  // plain: s is a normal number
    __device__ __forceinline__ explicit RowScale(uint32_t top) {
        finite = top < 0x7F800000u;
        s = finite ? __fdiv_rn(__uint_as_float(top), 127.0f) : __uint_as_float(0x7FC00000u);
        plain = s >= 1.17549435e-38f;
        inv = plain ? __fdiv_rn(1.0f, s) : 0.0f;
    }
};

__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }

// rint(x / s), halves to even, as if the quotient were exact; inv is 1 / s in 64 bits.  x * inv is off by less than 2^-44; a
// quotient of two fp32 values that is not exactly n + 1/2 is at least 2^-25 away from it (x / s - (2n + 1) / 2
// = (2x - (2n + 1) s) / 2s, and the numerator is a multiple of the smaller of the two last places).  Rounding to multiples of
// 2^-40 first therefore puts every tie on the tie and moves nothing across it.  (inv = 0: every code is 0)
__device__ __forceinline__ int int8_code_slow(float x, double inv) {
    const double snap = 6144.0;      // 1.5 * 2^12: the last place of a sum is 2^-40
    const double q = __builtin_rint(((double)x * inv + snap) - snap);
    return inv > 0.0 ? (int)(q < 127.0 ? (q > -127.0 ? q : -127.0) : 127.0) : 0;
}
// N values' codes as bytes.  u = x * inv + 1.5 * 2^23 in one fma holds the nearest whole number in its low bits; x * inv is
// within 127 * 2^-24 < 2^-17 of x / s, so wherever it is no closer than 2^-16 to a half that number is the code.  The rest,
// one wave of 512 values in 64 of fp32 rows, is decided in 64 bits; of 16-bit rows about half the waves if they are N(0, 1): half
// the largest is 63.5 s, and there are few values to fall on.  (4096 x 4096 bf16: 13.2 us so, 11.2 where a few loud channels hold
// the largest.  The sign of x - (n + 1/2) s, one fp32 fma, decides as well and was no faster: 12.9 / 13.0 us.)
template <int N> __device__ __forceinline__ void int8_codes(const float* v, const RowScale& r, uint32_t* out) {
    const float magic = 12582912.0f;
    uint32_t u[N];
    float off = 0.0f;
#pragma unroll
    for (int j = 0; j < N; ++j) {
        const float m = __builtin_fmaf(v[j], r.inv, magic);
        off = fmaxf(off, fabsf(__builtin_fmaf(v[j], r.inv, magic - m)));
        u[j] = __float_as_uint(m);
    }
    if (__builtin_expect(__any(!r.plain || !(off <= 0.5f - 0x1p-16f)), 0)) {
        const double inv = r.finite && r.s > 0.0f ? 1.0 / (double)r.s : 0.0;
#pragma unroll
        for (int j = 0; j < N; ++j) u[j] = (uint32_t)int8_code_slow(v[j], inv);
    }
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
        const uint32_t lo = __builtin_amdgcn_perm(u[4 * i + 1], u[4 * i], 0x0c0c0400u), hi = __builtin_amdgcn_perm(u[4 * i + 3], u[4 * i + 2], 0x04000c0cu);
        out[i] = lo | hi;
    }
    if (N < 4) out[0] = u[0] & 255u;
}
__device__ __forceinline__ u32x2_t int8_code8(const float* v, const RowScale& r) {
    uint32_t w[2];
    int8_codes<8>(v, r, w);
    return u32x2_t{w[0], w[1]};
}
__device__ __forceinline__ uint8_t int8_code(float v, const RowScale& r) {
    uint32_t w;
    int8_codes<1>(&v, r, &w);
    return (uint8_t)w;
}

// Eight values of a row from element i (in bounds with left <= 0 too); those behind the `left` that it still has are zero.
// fast: the address is 16-byte aligned, left is not cut within the eight and eight values are there to be read.
template <int DT> __device__ __forceinline__ void int8_load8(const void* x, size_t i, int left, bool fast, float* v) {
    if (fast && DT != QMOE_DT_F32) {      // one request
        const u32x4_t w = *(const QMOE_GLOBAL u32x4_t*)((const uint16_t*)x + i);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const uint16_t b = (uint16_t)(w[j >> 1] >> (16 * (j & 1)));
            const float f = DT == QMOE_DT_F16 ? (float)__builtin_bit_cast(_Float16, b) : __uint_as_float((uint32_t)b << 16);
            v[j] = left > 0 ? f : 0.0f;
        }
    } else if (fast) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const float4 f = Elem<DT>::load4(x, i + 4 * h);
            v[4 * h] = left > 0 ? f.x : 0.0f; v[4 * h + 1] = left > 0 ? f.y : 0.0f;
            v[4 * h + 2] = left > 0 ? f.z : 0.0f; v[4 * h + 3] = left > 0 ? f.w : 0.0f;
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) { const float f = Elem<DT>::load(x, j < left ? i + j : i); v[j] = j < left ? f : 0.0f; }
    }
}

// acc * s * c with one rounding that counts: the sum has up to 31 bits, the scales 24 each.
__device__ __forceinline__ double int8_value(int acc, float s, float c) { return (double)acc * ((double)s * (double)c); }

// v rounded to fp32, and to nothing else: a conversion of the result to 16 bits must not be joined with this one (the compiler
// contracts the two to one rounding, in software for fp16, on one path and not on another).
__device__ __forceinline__ float to_fp32(double v) {
    float f = (float)v;
    asm("" : "+v"(f));
    return f;
}

// silu(g) * u = g u / (1 + 2^y), y = -g log2 e, in 64 bits and rounded to fp32: the one formula of every kernel.  The activation
// that an expert hands to its down projection is cut into codes: a value next to the border of two codes gets the same code
// however many tokens share the step, and a SwiGLU's value the same bits.
//   2^y = 2^n 2^r, n = rint(y), |r| <= 1/2;  2^r = 1 + r P(r), P of degree 9 through (2^r - 1) / r at ten Chebyshev nodes: 2^-50.6
//   1 / (1 + 2^y): the instruction's 2^-24, one Newton step
// y's own rounding counts |y| 2^-53 ln 2, so silu is off by 2^-46 at most for |g| up to 110, beyond which |silu| is below 2^-150.
// y below -1000 adds nothing to 1, and 2^n is cut at 2^1000, where silu(g) u is far below fp32 (|g u| < 2^574); g = -infinity and
// NaN give NaN.  Half the instructions of exp and a division in 64 bits: SwiGLU 4096 x 14336 x 64 bf16 from codes 94 us instead of 128
// (silu in fp32: 91), 4096 x 4096 x 512 39 instead of 51.
__device__ __forceinline__ float int8_hidden(double g, double u) {
    const double y = fmax(g * -0x1.71547652b82fep+0, -1000.0), n = __builtin_rint(y), r = y - n;
    double p = 0x1.e5e9f548e5726p-28;
    p = __builtin_fma(p, r, 0x1.b6571de2f2351p-24);
    p = __builtin_fma(p, r, 0x1.62bfe46117445p-20);
    p = __builtin_fma(p, r, 0x1.ffcb76789860fp-17);
    p = __builtin_fma(p, r, 0x1.4309130378460p-13);
    p = __builtin_fma(p, r, 0x1.5d87fe908f88ap-10);
    p = __builtin_fma(p, r, 0x1.3b2ab6fba385fp-7);
    p = __builtin_fma(p, r, 0x1.c6b08d7044119p-5);
    p = __builtin_fma(p, r, 0x1.ebfbdff82c590p-3);
    p = __builtin_fma(p, r, 0x1.62e42fefa39f7p-1);
    p = __builtin_fma(p, r, 1.0);
    const double d = 1.0 + ldexp(p, (int)fmin(n, 1000.0));
    double i = __builtin_amdgcn_rcp(d);
    i = __builtin_fma(__builtin_fma(-d, i, 1.0), i, i);
    return to_fp32(g * i * u);
}

// sigmoid(x . w) of a token's row by one wave: what admits the shared expert.  In fp32, and in one order of additions whichever
// kernel asks, so that a token's step has the same bits in every batch.
template <int XDT> __device__ __forceinline__ float int8_admission(const void* x, size_t row, bool fast, const float* w, bool w_fast, int d) {
    float sum = 0.0f;
#pragma unroll 4
    for (int i = (int)(threadIdx.x & 63) * 8; i < d; i += 512) {
        float a[8], b[8], t[4];
        int8_load8<XDT>(x, row + i, d - i, fast, a);
        int8_load8<QMOE_DT_F32>(w, i, d - i, w_fast, b);
#pragma unroll
        for (int j = 0; j < 4; ++j) t[j] = __builtin_fmaf(a[2 * j + 1], b[2 * j + 1], __fmul_rn(a[2 * j], b[2 * j]));
        sum += (t[0] + t[1]) + (t[2] + t[3]);
    }
    sum = wave_sum(sum);
    return sum >= 0.0f ? 1.0f / (1.0f + expf(-sum)) : expf(sum) / (1.0f + expf(sum));
}

// LDS operations of this workgroup's waves before and after; requests for memory stay in flight.
__device__ __forceinline__ void meet_lds() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// ---- launches shared by the linear and the expert step ------------------------------------------------
// x rows -> codes (row step ld bytes; pad: zeros up to the next multiple of 256 columns) + scales
int int8_quantize_launch(const void* x, int dt, int64_t rows, int k, uint8_t* codes, int64_t ld, bool pad, float* scales, hipStream_t s);

// Whether a product of these rows quantises them in its own workgroups, whether it is one of few tokens, and its launch (x: rows
// to quantise, NULL: p.q holds codes, any alignment).
bool int8_few_fuses(int tokens, int k);
bool int8_few_takes(int n, int tokens, bool pair);
struct Int8Product;
int int8_few_launch(const Int8Product& p, bool pair, const void* x, int xdt, int k, hipStream_t s);
int int8_gemm_launch(const Int8Product& a, bool pair, hipStream_t s);
int int8_plan_rows(int64_t assignments, int n_experts);
int int8_plan_launch(const Int8Product& a, bool pair, int rows, int max_chunks, const Int8Product* side, hipStream_t s);

// One product or one gate/up pair; dense, or over the chunks of a plan (experts' own rows).
struct Int8Product {
    const uint8_t *w, *w2;            // tiles (w2: the up projection of a pair)
    const float *c, *c2;              // channel scales
    int n, kp;                        // output channels, padded columns
    const uint8_t* q;                 // activation codes
    int64_t ld;
    const float* s;                   // their scales
    int tokens;
    void* y;
    int ydt;
    int64_t ldy;
    // over a plan: chunk i covers sorted positions start .. start + count - 1 of expert `expert`
    const int *chunk_expert, *chunk_start, *chunk_count, *n_chunks;
    int64_t w_step;                   // bytes of one expert's matrix
    const int* row_of;                // sorted position -> row of q (NULL: the position itself)
};

}  // namespace qmoe
