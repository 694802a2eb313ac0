// Products of 8-bit codes for a few tokens: the weights are streamed once.
//
// A workgroup of eight waves owns RT tiles of 16 channels (of both matrices of a pair) and the whole of K;
// wave w takes the w-th eighth of the 64-column steps (neighbouring ones: it uses the activation lines it
// fetches whole).  A step is one 1 KB request for each tile, already the A operand of the matrix instruction,
// and one B operand for each 16 tokens; the eight partial sums meet in LDS once, as integers, so the split
// changes no bit of the result.  What bounds it is the memory: an instruction multiplies
// 1 KB of weights in 16 cycles where a CU receives 1 KB in about 100, so the idle token columns cost nothing and
// 1..16 tokens take the same time.  Up to U requests a wave and tile are outstanding while the previous U are
// multiplied: four.  (Eight, with one tile: 16 x 4096 x 4096 7.3 instead of 6.7 us, 1 x 512 x 512 2.6 instead of 2.2,
// 77 x 1001 x 1234 7.8 instead of 5.4: a short wave requests what it does not need.  Two, with two tiles at one token:
// 1 x 151936 x 2048 54 instead of 49 us.)
// From codes in memory, us: 1 x 4096 x 4096 5.5 (16.8 MB: 3.1 TB/s, the launch and its end are half of it),
// 1 x 14336 x 4096 12.1 (4.9 TB/s), 16 x 14336 x 4096 13.6, 1 x 151936 x 2048 49 (6.3 TB/s).
#include "qmoe_int8.hpp"

namespace qmoe {

struct Few8Args {
    const uint8_t *w, *w2;
    const float *c, *c2;
    int n, kp, steps;       // steps = kp / 64
    const void* x;          // fused: rows to quantise
    int k, fast;            // columns; rows of x may be read 16 bytes at a time
    const uint8_t* q;       // otherwise: codes, their row step and scales (any alignment; k of them may be read in a row)
    int64_t ld;
    const float* s;
    int tokens;
    void* y;
    int ydt;
};

// NX < 0   rows of codes at any address
// NX = 0   at multiples of four bytes
// NX > 0   every workgroup quantises the token itself: NX pieces of eight values a thread, kept in registers between the
//          search for the largest and the codes.  They are requested before the first weights, so that waiting for them
//          does not wait for the weights.
template <int XDT, bool PAIR, int NX, int TT, int RT, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void int8_few_kernel(const Few8Args a) {
    constexpr bool FUSED = NX > 0, SHIFT = NX < 0;
    constexpr int THREADS = 64 * WAVES;
    constexpr int NP = PAIR ? 2 : 1, NW = RT * NP, U = NW == 1 ? 4 : (TT == 1 ? 8 : 4) / NW;
    extern __shared__ __align__(16) uint8_t lds[];       // [codes] and, over them at the end, [waves][NW][TT][64] partial sums
    __shared__ uint32_t tops[WAVES];
    __shared__ float srow[16 * TT];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 15, g = lane >> 4;
    const int row_tiles = (a.n + 15) / 16;
    const int first = FUSED ? 0 : (int)blockIdx.y * 16 * TT, tokens = a.tokens - first < 16 * TT ? a.tokens - first : 16 * TT;

    float v[FUSED ? NX : 1][8];
    if (FUSED) {
#pragma unroll
        for (int p = 0; p < NX; ++p) {
            const int i = (p * THREADS + tid) * 8;
            int8_load8<XDT>(a.x, i < a.k ? i : 0, a.k - i, a.fast, v[p]);
        }
    }

    const uint8_t* wp[NW];
#pragma unroll
    for (int r = 0; r < RT; ++r) {
        int tile = blockIdx.x * RT + r;
        tile = tile < row_tiles ? tile : row_tiles - 1;
        wp[r * NP] = a.w + (int64_t)tile * a.kp * 16 + lane * 16;
        if (PAIR) wp[r * NP + 1] = a.w2 + (int64_t)tile * a.kp * 16 + lane * 16;
    }
    // this wave's steps; one without a step of its own (K below 512) requests its neighbour's and multiplies none
    // (codes read as they are: a last step that is not whole is left to the end)
    const int whole = FUSED ? a.steps : a.k / 64, lo = a.steps * wave / WAVES, end = a.steps * (wave + 1) / WAVES, hi = end < whole ? end : whole;
    const int last = hi > lo ? hi - 1 : lo < a.steps ? lo : a.steps - 1;
    i32x4_t wr[U][NW];
    auto request = [&](int chunk) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int step = lo + chunk * U + u < last ? lo + chunk * U + u : last;
#pragma unroll
            for (int i = 0; i < NW; ++i) wr[u][i] = ldg_i32x4(wp[i] + (int64_t)step * 1024);
        }
    };
    request(0);

    const uint8_t* qp[TT];
    uint32_t shift[TT];
#pragma unroll
    for (int t = 0; t < TT; ++t) shift[t] = 0;
    if (FUSED) {
        uint32_t top = 0;
#pragma unroll
        for (int p = 0; p < NX; ++p)
#pragma unroll
            for (int j = 0; j < 8; ++j) { const uint32_t b = abs_bits(v[p][j]); top = b > top ? b : top; }
        top = wave_max_u32(top);
        if (lane == 0) tops[wave] = top;
        __syncthreads();
#pragma unroll
        for (int j = 0; j < WAVES; ++j) top = tops[j] > top ? tops[j] : top;
        const RowScale rs(top);
        if (tid == 0) srow[0] = rs.s;
#pragma unroll
        for (int p = 0; p < NX; ++p) {
            const int i = (p * THREADS + tid) * 8;
            if (i < a.kp) *(u32x2_t*)(lds + i) = int8_code8(v[p], rs);
        }
        __syncthreads();
    } else {
#pragma unroll
        for (int t = 0; t < TT; ++t) {
            const int row = t * 16 + col;
            qp[t] = a.q + (int64_t)(first + (row < tokens ? row : tokens - 1)) * a.ld + g * 16;
            if (SHIFT) shift[t] = (uint32_t)(uintptr_t)qp[t] & 3u;
        }
        if (tid < 16 * TT) srow[tid] = tid < tokens ? a.s[first + tid] : 0.0f;
    }

    i32x4_t acc[NW][TT];
#pragma unroll
    for (int i = 0; i < NW; ++i)
#pragma unroll
        for (int t = 0; t < TT; ++t) acc[i][t] = i32x4_t{0, 0, 0, 0};
    if (!FUSED && end > hi && end > lo) {      // the row's end: bytes, zeros behind it
        const int c = whole * 64 + g * 16;
        i32x4_t w[NW];
#pragma unroll
        for (int i = 0; i < NW; ++i) w[i] = ldg_i32x4(wp[i] + (int64_t)whole * 1024);
#pragma unroll
        for (int t = 0; t < TT; ++t) {
            uint32_t v[16];
            i32x4_t b;
#pragma unroll
            for (int i = 0; i < 16; ++i) v[i] = ldg<uint8_t>(qp[t] + (c + i < a.k ? c + i : a.k - 1) - g * 16);
#pragma unroll
            for (int i = 0; i < 16; ++i) v[i] = c + i < a.k ? v[i] << (8 * (i & 3)) : 0u;
#pragma unroll
            for (int j = 0; j < 4; ++j) b[j] = (int)(v[4 * j] | v[4 * j + 1] | v[4 * j + 2] | v[4 * j + 3]);
#pragma unroll
            for (int i = 0; i < NW; ++i) acc[i][t] = mfma_i8(w[i], b, acc[i][t]);
        }
    }
    const int chunks = hi > lo ? (hi - lo + U - 1) / U : 0;
    const uint8_t* const mine = lds + g * 16;        // (the one token, in every column)
    for (int chunk = 0; chunk < chunks; ++chunk) {
        i32x4_t now[U][NW], b[U][TT];
        int next[SHIFT ? U : 1][TT];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int step = lo + chunk * U + u < hi - 1 ? lo + chunk * U + u : hi - 1;
#pragma unroll
            for (int t = 0; t < TT; ++t) {
                b[u][t] = FUSED ? *(const i32x4_t*)(mine + step * 64) : *(const QMOE_GLOBAL i32x4_dword_t*)(qp[t] - shift[t] + (int64_t)step * 64);
                if (SHIFT) next[u][t] = ldg<int>(qp[t] - shift[t] + (int64_t)step * 64 + (shift[t] ? 16 : 12));
            }
#pragma unroll
            for (int i = 0; i < NW; ++i) now[u][i] = wr[u][i];
        }
        if (chunk + 1 < chunks) request(chunk + 1);
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (lo + chunk * U + u < hi) {
                if (SHIFT) {
#pragma unroll
                    for (int t = 0; t < TT; ++t) {
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            b[u][t][j] = (int)__builtin_amdgcn_alignbyte(j < 3 ? (uint32_t)b[u][t][(j + 1) & 3] : (uint32_t)next[u][t], (uint32_t)b[u][t][j], shift[t]);
                    }
                }
#pragma unroll
                for (int i = 0; i < NW; ++i)
#pragma unroll
                    for (int t = 0; t < TT; ++t) acc[i][t] = mfma_i8(now[u][i], b[u][t], acc[i][t]);
            }
    }
    if (FUSED) __syncthreads();          // the codes' place is taken by the partial sums
    int* const part = (int*)lds;
#pragma unroll
    for (int i = 0; i < NW; ++i)
#pragma unroll
        for (int t = 0; t < TT; ++t) *(i32x4_t*)(part + ((size_t)(wave * NW + i) * TT + t) * 256 + lane * 4) = acc[i][t];
    __syncthreads();
    // (token, channel) of this thread: channel fastest; the sum of channel 4 g + i and token c is value i of lane 16 g + c
    for (int o = tid; o < tokens * RT * 16; o += THREADS) {
        const int ch = o % (RT * 16), t = o / (RT * 16), r = ch >> 4, in = ch & 15;
        const int n = blockIdx.x * RT * 16 + ch;
        if (n >= a.n) continue;
        const int at = (t >> 4) * 256 + ((in >> 2) * 16 + (t & 15)) * 4 + (in & 3);
        int s0 = 0, s1 = 0;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
            s0 += part[(size_t)(w * NW + r * NP) * TT * 256 + at];
            if (PAIR) s1 += part[(size_t)(w * NW + r * NP + 1) * TT * 256 + at];
        }
        const double v = int8_value(s0, srow[t], a.c[n]);
        const float out = PAIR ? int8_hidden(v, int8_value(s1, srow[t], a.c2[n])) : to_fp32(v);
        store_out(a.y, a.ydt, (size_t)(first + t) * a.n + n, out);
    }
}

template <int XDT, bool PAIR, int NX, int TT, int RT, int WAVES>
static int few8_as(const Few8Args& a, hipStream_t s) {
    constexpr int NW = RT * (PAIR ? 2 : 1);
    const size_t partial = (size_t)WAVES * NW * TT * 1024, codes = NX > 0 ? (size_t)a.kp : 0;
    const size_t lds = partial > codes ? partial : codes;            // (at most 32 KB)
    hipLaunchKernelGGL((int8_few_kernel<XDT, PAIR, NX, TT, RT, WAVES>), dim3((a.n + 16 * RT - 1) / (16 * RT), NX > 0 ? 1 : (a.tokens + 16 * TT - 1) / (16 * TT)), dim3(64 * WAVES), lds, s, a);
    return check_launch("int8 product of a few tokens");
}

// Rows quantised by every workgroup: one token of up to four pieces of 4096 columns.  (Two to four tokens on the way cost
// 20.4 us where their own launch and the product take 14.1 + 2.6 us, 4 x 14336 x 4096.)
static int few8_pieces(int k) { return (k + 4095) / 4096; }
bool int8_few_fuses(int tokens, int k) { return tokens == 1 && few8_pieces(k) <= 4; }

// Up to 16 tokens, and more where blocks of 16 channels x 32 tokens are few: there the waves' cut of K beats tiles that walk K as
// a whole (us, cold; this kernel / tiles: 17 x 4096 x 4096 7.5 / 8.2, 32 x 4096 x 4096 8.8 / 8.4, 32 x 4096 x 14336 23.8 / 20.3,
// 64 x 4096 x 4096 12.8 / 8.7; pairs 32 x 4096 x 4096 10.6 / 12.2, 128 x 1024 x 4096 8.6 / 11.0, 128 x 4096 x 4096 27 / 15).
bool int8_few_takes(int n, int tokens, bool pair) {
    const int64_t blocks = (n + 15ll) / 16 * ((tokens + 31ll) / 32);
    return tokens <= 16 || blocks <= 192 || (blocks <= 256 && (pair || tokens <= 24));
}

template <int XDT, bool PAIR, int RT> static int few8_fused(const Few8Args& a, int waves, hipStream_t s) {
    if (waves == 16) return few8_pieces(a.k) <= 2 ? few8_as<XDT, PAIR, 1, 1, 1, 16>(a, s) : few8_as<XDT, PAIR, 2, 1, 1, 16>(a, s);
    return few8_pieces(a.k) == 1 ? few8_as<XDT, PAIR, 1, 1, RT, 8>(a, s) : few8_as<XDT, PAIR, 4, 1, RT, 8>(a, s);
}
template <bool PAIR> static int few8_codes(const Few8Args& a, int rt, hipStream_t s) {
    // rows at odd addresses: whole dwords and a shift (77 x 1001 x 1234: 5.5 us, its neighbour of 1236 columns, at multiples of four, 4.4)
    if (((uintptr_t)a.q | (uintptr_t)a.ld) % 4) return a.tokens <= 16 ? few8_as<0, PAIR, -1, 1, 1, 8>(a, s) : few8_as<0, PAIR, -1, 2, 1, 8>(a, s);
    if (a.tokens > 16) return few8_as<0, PAIR, 0, 2, 1, 8>(a, s);      // blocks of 32 tokens
    return rt == 1 ? few8_as<0, PAIR, 0, 1, 1, 8>(a, s) : few8_as<0, PAIR, 0, 1, 2, 8>(a, s);
}

int int8_few_launch(const Int8Product& p, bool pair, const void* x, int xdt, int k, hipStream_t s) {
    Few8Args a{};
    a.w = p.w; a.w2 = p.w2; a.c = p.c; a.c2 = p.c2; a.n = p.n; a.kp = p.kp; a.steps = p.kp / 64;
    a.q = p.q; a.ld = p.ld; a.s = p.s; a.tokens = p.tokens; a.y = p.y; a.ydt = p.ydt;
    // Two tiles a workgroup once they still make two workgroups a CU: fewer prologues and half the activation reads for the
    // same weights (8192 x 4096 even, 14336 x 4096 13.4 -> 12.2 us, 151936 x 2048 67.5 -> 49.8 us at one token; 4096 x 4096
    // 5.6 -> 6.8 us).
    // Sixteen waves where one token's row is long and the workgroups are few (4096 x 14336: 15.9 -> 14.4 us).
    const int tiles = (p.n + 15) / 16;
    const int rt = tiles < 512 ? 1 : 2;
    const int waves = x && k > 4096 && tiles < 512 ? 16 : 8;
    a.k = x ? k : (int)(p.ld < p.kp ? k : p.kp);
    if (!x) return pair ? few8_codes<true>(a, rt, s) : few8_codes<false>(a, rt, s);
    a.x = x;
    a.fast = (uintptr_t)x % 16 == 0 && k % 8 == 0;
#define QMOE_FUSED(DT) (pair ? few8_fused<DT, true, 1>(a, waves, s) : rt == 1 ? few8_fused<DT, false, 1>(a, waves, s) : few8_fused<DT, false, 2>(a, waves, s))
    if (xdt == QMOE_DT_F32) return QMOE_FUSED(QMOE_DT_F32);
    if (xdt == QMOE_DT_F16) return QMOE_FUSED(QMOE_DT_F16);
    return QMOE_FUSED(QMOE_DT_BF16);
#undef QMOE_FUSED
}

}  // namespace qmoe
