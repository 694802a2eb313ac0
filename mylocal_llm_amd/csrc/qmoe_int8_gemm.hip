// Products of 8-bit codes for many tokens, dense or over the chunks of a plan.
//
// A workgroup owns WN x RT tiles of 16 channels (of both matrices of a pair) by WT x TT tiles of 16 tokens; a wave RT x TT
// of them, accumulated in registers.  The weights go from memory straight to the registers that the matrix instruction
// reads -- their layout is the A operand, 1 KB of consecutive memory a request -- one chunk of KC columns ahead.  The
// activations are shared by the waves: a chunk of every token's codes travels through registers to LDS, two buffers,
// one meeting a chunk, and lies there as B operands, so that an operand is one 16-byte read a lane.  Slots are XORed
// with the piece's number: a row's pieces, written by neighbouring lanes, fall into eight bank groups, and so do the
// rows that neighbouring lanes read.
#include "qmoe_int8.hpp"
#include <type_traits>

namespace qmoe {

// R: steps of 64 columns that the weights' requests run ahead; XR: chunks that the activations' requests run ahead.
template <bool PAIR, bool PLAN, int WN, int WT, int RT, int TT, int KC, int R, int XR>
__global__ __launch_bounds__(64 * WN * WT) __attribute__((amdgpu_waves_per_eu(2))) void int8_gemm_kernel(const Int8Product main_args, int n_blocks, int t_blocks,
                                                                 const Int8Product side_args, int side_n, int side_t) {
    constexpr int THREADS = 64 * WN * WT, NP = PAIR ? 2 : 1, NW = RT * NP;
    constexpr int ROWS = 16 * TT * WT, PIECES = KC / 16, KK = KC / 64, LOADS = ROWS * PIECES / THREADS;
    auto swap = [](int pc) { return pc & 7; };
    static_assert(ROWS * PIECES % THREADS == 0 && LOADS > 0, "whole pieces a thread");
    __shared__ __align__(16) uint8_t lds[2 * ROWS * KC];
    __shared__ float srow[ROWS];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wn = wave % WN, wt = wave / WN, col = lane & 15, g = lane >> 4;

    // workgroups go round the eight XCDs: each XCD takes a run of neighbours in the order below, for its L2
    // (a launch over a plan may carry a dense product of the same kind, the shared expert's, in front)
    const bool aside = PLAN && (int)blockIdx.x < side_n * side_t;
    const Int8Product a = aside ? side_args : main_args;
    const int raw = PLAN && !aside ? (int)blockIdx.x - side_n * side_t : (int)blockIdx.x;
    const int nb = aside ? side_n : n_blocks;
    const int total = aside ? side_n * side_t : n_blocks * t_blocks;
    const int xcd = raw % 8, share = total / 8, over = total % 8;
    const int id = xcd * share + (xcd < over ? xcd : over) + raw / 8;
    int bn, bt;
    if (aside) { bn = id % nb; bt = id / nb; }
    else if (PLAN) {
        // runs of four chunks an XCD, whatever their number turns out to be: it is not waited for to find the chunk
        const int c = raw / 8 / nb;
        bn = raw / 8 % nb;
        bt = c / 4 * 32 + xcd * 4 + c % 4;
        if (bt >= t_blocks) return;
    } else {
        // bands of up to eight token blocks, channel blocks one after the other inside a band
        const int band = id / (8 * n_blocks), in = id % (8 * n_blocks), left = t_blocks - band * 8, high = left < 8 ? left : 8;
        bt = band * 8 + in % high;
        bn = in / high;
    }
    int first = bt * ROWS, count = a.tokens - first, expert = 0;
    if (PLAN && !aside) {
        expert = a.chunk_expert[bt];
        first = a.chunk_start[bt];
        count = a.chunk_count[bt];
        if (bt >= *(const QMOE_GLOBAL int*)a.n_chunks) return;      // (what lies behind the last chunk was loaded, not used)
    }

    const int row_tiles = (a.n + 15) / 16, steps = a.kp / 64, chunks = (a.kp + KC - 1) / KC;
    // one uniform base a matrix, 32-bit offsets behind it (a wave's tiles lie within RT * 2 MB)
    int tile0 = (bn * WN + wn) * RT;
    tile0 = tile0 < row_tiles ? tile0 : row_tiles - 1;
    const uint8_t* const w0 = a.w + (int64_t)expert * a.w_step + (int64_t)tile0 * a.kp * 16;
    const uint8_t* const w1 = PAIR ? a.w2 + (int64_t)expert * a.w_step + (int64_t)tile0 * a.kp * 16 : nullptr;
    uint32_t w_at[RT];
#pragma unroll
    for (int r = 0; r < RT; ++r) w_at[r] = (uint32_t)(tile0 + r < row_tiles ? r : 0) * (uint32_t)a.kp * 16u;
    const uint8_t* const x0 = PLAN ? a.q : a.q + (int64_t)first * a.ld;
    typename std::conditional<PLAN, int64_t, uint32_t>::type xp[LOADS];
    int slot[LOADS];
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
        const int p = tid + i * THREADS, r = p / PIECES, pc = p % PIECES;
        const int at = r < count ? r : 0;
        if (PLAN) xp[i] = (int64_t)(a.row_of ? a.row_of[first + at] : first + at) * a.ld + pc * 16;
        else xp[i] = (uint32_t)at * (uint32_t)a.ld + pc * 16u;
        slot[i] = ((r / 16 * KK + pc / 4) * 64 + pc % 4 * 16 + (r % 16 ^ swap(pc))) * 16;
    }
    for (int i = tid; i < ROWS; i += THREADS) {
        const int pos = first + (i < count ? i : 0);
        srow[i] = a.s[PLAN && a.row_of ? a.row_of[pos] : pos];
    }
    constexpr int ROUND = R / KK > 2 ? R / KK : 2;       // chunks after which rings and buffers are back where they were
    static_assert(ROUND % 2 == 0 && ROUND * KK % R == 0 && ROUND % XR == 0, "a round turns all rings whole");
    const int end = chunks - 1;
    i32x4_t xr[XR][LOADS], wr[R][NW];
    auto request_x = [&](int chunk, i32x4_t (&x)[LOADS]) {
        const int c = chunk < end ? chunk : end;
#pragma unroll
        for (int i = 0; i < LOADS; ++i) x[i] = ldg_i32x4(x0 + (xp[i] + c * KC));
    };
    auto keep_x = [&](int buffer, const i32x4_t (&x)[LOADS]) {
#pragma unroll
        for (int i = 0; i < LOADS; ++i) *(i32x4_t*)(lds + buffer * (ROWS * KC) + slot[i]) = x[i];
    };
    // (steps behind the last repeat it: they meet activations of zero, or nothing; what is in flight never depends on a
    // condition)
    auto request_w = [&](int step, i32x4_t (&w)[NW]) {
        const int64_t at = (int64_t)(step < steps ? step : steps - 1) * 1024;
#pragma unroll
        for (int r = 0; r < RT; ++r) {
            w[r * NP] = ldg_i32x4(w0 + at + (w_at[r] + lane * 16u));
            if (PAIR) w[r * NP + 1] = ldg_i32x4(w1 + at + (w_at[r] + lane * 16u));
        }
    };
    i32x4_t acc[NW][TT];
#pragma unroll
    for (int i = 0; i < NW; ++i)
#pragma unroll
        for (int t = 0; t < TT; ++t) acc[i][t] = i32x4_t{0, 0, 0, 0};
    // a lane's place in an operand for even and odd steps; everything else is a constant offset
    const uint8_t* const mine0 = lds + wt * (TT * 16 * KC) + (g * 16 + (col ^ swap(g))) * 16;
    const uint8_t* const mine1 = lds + wt * (TT * 16 * KC) + (g * 16 + (col ^ swap(g | 4))) * 16;
    constexpr int TH = TT / 2;        // tokens' tiles of half a step
    constexpr int D = TT <= 4 ? 4 : 2, HALVES = 2 * KK;
    static_assert(HALVES % D == 0, "a chunk turns the operands' ring whole");
    i32x4_t b[D][TH];
    auto read_b = [&](int buffer, int half, i32x4_t (&to)[TH]) {
        const int kk = half / 2;
#pragma unroll
        for (int t = 0; t < TH; ++t)
            to[t] = *(const i32x4_t*)((kk & 1 ? mine1 : mine0) + (buffer * (ROWS * KC) + ((half % 2 * TH + t) * KK + kk) * 1024));
    };
    // A chunk in halves of a step: while one half is multiplied the operands of the next D - 1 are on their way from LDS, and
    // the last D - 1 halves of a chunk are multiplied behind the meeting that opens the next one.  (Small tiles multiply a half
    // in less time than LDS answers in: D = 4 instead of 2 takes 512 x 2048 x 2048 from 7.9 to 7.1 us, 64 x 4096 x 4096 from 8.8 to
    // 8.5.)  A step's weights are requested again into the registers they leave, R steps ahead; activations are requested XR + 1
    // chunks ahead of their use.
    auto turn = [&](int c, int h) {
        keep_x((h + 1) & 1, xr[(h + 1) % XR]);
        request_x(c + 1 + XR, xr[(h + 1) % XR]);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int j = 0; j < HALVES; ++j) {
            const int ahead = j + D - 1;
            if (ahead == HALVES) meet_lds();
            read_b((ahead < HALVES ? h : h + 1) & 1, ahead % HALVES, b[ahead % D]);
            i32x4_t(&w)[NW] = wr[(h * KK + j / 2) % R];
#pragma unroll
            for (int t = 0; t < TH; ++t)
#pragma unroll
                for (int i = 0; i < NW; ++i) acc[i][j % 2 * TH + t] = mfma_i8(w[i], b[j % D][t], acc[i][j % 2 * TH + t]);
            if (j & 1) request_w(c * KK + j / 2 + R, w);
            __builtin_amdgcn_sched_barrier(0);     // (the scheduler would gather the requests behind the products)
        }
    };
    request_x(0, xr[0]);
    keep_x(0, xr[0]);
#pragma unroll
    for (int i = 1; i <= XR; ++i) request_x(i, xr[i % XR]);
    __builtin_amdgcn_sched_barrier(0);      // (requests come back in order, and the loop waits for these first)
#pragma unroll
    for (int r = 0; r < R; ++r) request_w(r, wr[r]);
    meet_lds();
#pragma unroll
    for (int j = 0; j + 1 < D; ++j) read_b(0, j, b[j]);
    // whole rounds without a condition inside: one would make the compiler move registers that are still on their way, and
    // wait for them
    int c0 = 0;
    for (; c0 + ROUND <= chunks; c0 += ROUND)
#pragma unroll
        for (int h = 0; h < ROUND; ++h) turn(c0 + h, h);
#pragma unroll
    for (int h = 0; h + 1 < ROUND; ++h)
        if (c0 + h < chunks) turn(c0 + h, h);
    // D[j] of a lane: channel 4 g + j of the tile, token col.  One formula for every value, whatever its type, its place and its
    // neighbours: scaled in 64 bits and rounded to fp32, then to the type, as for a few tokens.  (Scaling 16-bit results in fp32 saves
    // nothing: from codes, 4096 x 14336 x 4096 bf16 212 us so, 209 in 64 bits.)  The type is decided once, not for each value: the
    // unrolled code runs once a workgroup, and its size is its time.
    auto value = [&](int i, int t, int j, float s, double c, double c2) -> float {
        const double y = (double)acc[i * NP][t][j] * ((double)s * c);
        if (!PAIR) return to_fp32(y);
        const double u = (double)acc[i * NP + 1][t][j] * ((double)s * c2);
        return int8_hidden(y, u);
    };
    const int n0 = (bn * WN + wn) * RT * 16 + 4 * g;
    double c[RT][4], c2[RT][4];
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int n = n0 + i * 16 + j;
            const int64_t ch = (int64_t)expert * a.n + (n < a.n ? n : a.n - 1);
            c[i][j] = ldg<float>(a.c + ch);
            if (PAIR) c2[i][j] = ldg<float>(a.c2 + ch);
        }
    auto store16 = [&](auto bits) {
#pragma unroll
        for (int t = 0; t < TT; ++t) {
            const int r = (wt * TT + t) * 16 + col;
            const float s = srow[r];
            uint16_t* const y = (uint16_t*)a.y + (size_t)(first + r) * a.ldy + n0;
            if (r < count) {
#pragma unroll
                for (int i = 0; i < RT; ++i)
                    *(QMOE_GLOBAL u32x2_t*)(y + i * 16) =
                        u32x2_t{bits(value(i, t, 0, s, c[i][0], c2[i][0])) | bits(value(i, t, 1, s, c[i][1], c2[i][1])) << 16,
                                bits(value(i, t, 2, s, c[i][2], c2[i][2])) | bits(value(i, t, 3, s, c[i][3], c2[i][3])) << 16};
            }
        }
    };
    const bool whole = ((bn * WN + wn) * RT + RT) * 16 <= a.n && a.ldy % 4 == 0 && (uintptr_t)a.y % 16 == 0;
    if (whole && a.ydt == QMOE_DT_F32) {
#pragma unroll
        for (int t = 0; t < TT; ++t) {
            const int r = (wt * TT + t) * 16 + col;
            const float s = srow[r];
            float* const y = (float*)a.y + (size_t)(first + r) * a.ldy + n0;
            if (r < count) {
#pragma unroll
                for (int i = 0; i < RT; ++i)
                    stg<float4>(y + i * 16, make_float4(value(i, t, 0, s, c[i][0], c2[i][0]), value(i, t, 1, s, c[i][1], c2[i][1]),
                                                        value(i, t, 2, s, c[i][2], c2[i][2]), value(i, t, 3, s, c[i][3], c2[i][3])));
            }
        }
    } else if (whole && a.ydt == QMOE_DT_BF16) {
        store16([](float v) -> uint32_t { return __builtin_bit_cast(uint16_t, (__bf16)v); });
    } else if (whole) {
        store16([](float v) -> uint32_t { return __half_as_ushort(__float2half_rn(v)); });
    } else {
#pragma unroll
        for (int t = 0; t < TT; ++t) {
            const int r = (wt * TT + t) * 16 + col;
            if (r >= count) continue;
            const float s = srow[r];
#pragma unroll
            for (int i = 0; i < RT; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (n0 + i * 16 + j < a.n) store_out(a.y, a.ydt, (size_t)(first + r) * a.ldy + n0 + i * 16 + j, value(i, t, j, s, c[i][j], c2[i][j]));
        }
    }
}

template <bool PAIR, bool PLAN, int WN, int WT, int RT, int TT, int KC, int R, int XR>
static int gemm8_as(const Int8Product& a, int chunks, hipStream_t s, const Int8Product* side = nullptr) {
    const int nb = (a.n + 16 * WN * RT - 1) / (16 * WN * RT), tb = PLAN ? (chunks + 31) / 32 * 32 : (a.tokens + 16 * WT * TT - 1) / (16 * WT * TT);
    const int sn = side ? (side->n + 16 * WN * RT - 1) / (16 * WN * RT) : 0, st = side ? (side->tokens + 16 * WT * TT - 1) / (16 * WT * TT) : 0;
    if (((int64_t)nb * tb + (int64_t)sn * st) * (64 * WN * WT) > 0xFFFFFFFFll)      // (a launch's threads are counted in 32 bits)
        return fail(QMOE_EUNSUPPORTED, "int8 product: %d x %d blocks exceed a launch; split the tokens", nb, tb);
    hipLaunchKernelGGL((int8_gemm_kernel<PAIR, PLAN, WN, WT, RT, TT, KC, R, XR>), dim3(nb * tb + sn * st), dim3(64 * WN * WT), 0, s, a, nb, PLAN ? chunks : tb,
                       side ? *side : a, sn, st);
    return check_launch("int8 product");
}

// A chunk of a plan holds up to `rows` sorted positions of one expert: 32, 64 or 128, by the average (us of a whole step with
// 32 / 64 / 128; 64 experts of width 1024, 128 of 512, 2048 columns): average 20 105 / 107 / 106 and 108 / 110 / 114, average 40
// 133 / 117 / 116 and 138 / 125 / 129, average 90 190 / 168 / 142 and 208 / 183 / 171, average 256 399 / 315 / 271 and 490 / 405 / 352.
int int8_plan_rows(int64_t assignments, int n_experts) {
    const int64_t average = assignments / n_experts;
    return average < 28 ? 32 : average <= 72 ? 64 : 128;
}
// side: NULL, or a dense product of the same kind (pair or plain) that rides in front.
int int8_plan_launch(const Int8Product& a, bool pair, int rows, int max_chunks, const Int8Product* side, hipStream_t s) {
    if (pair) {
        if (rows == 32) return gemm8_as<true, true, 4, 1, 1, 2, 256, 8, 2>(a, max_chunks, s, side);
        if (rows == 64) return gemm8_as<true, true, 4, 1, 1, 4, 256, 8, 1>(a, max_chunks, s, side);
        return gemm8_as<true, true, 4, 1, 2, 8, 128, 4, 1>(a, max_chunks, s, side);
    }
    if (rows == 32) return gemm8_as<false, true, 4, 1, 2, 2, 256, 4, 2>(a, max_chunks, s, side);
    if (rows == 64) return gemm8_as<false, true, 4, 1, 2, 4, 256, 8, 1>(a, max_chunks, s, side);
    return gemm8_as<false, true, 4, 1, 4, 8, 128, 4, 1>(a, max_chunks, s, side);
}

// The largest tile that still gives nearly every CU a workgroup (us from codes; 256 x 256 of eight waves / 256 channels x
// 128 tokens of four, two workgroups a CU / 256 x 64 / 128 x 64 / 64 x 64 / 64 x 32 / 32 x 32): 4096 tokens x 4096 x 14336
// 184 / 184 / 220 / - / 351, 4096 x 14336 x 4096 225 / 213 / 268 / - / 380, 512 x 14336 x 4096 49 / 33 / 36 / - / 48,
// 1024 x 4096 x 4096 47 / 30 / 22 / 25 / 29, 128 x 14336 x 4096 - / - / 29 / 20 / 22 / 28, 512 x 2048 x 2048 - / - / 12 / 9.2 / 7.1 /
// 7.7, 128 x 4096 x 4096 - / - / 18 / 13 / 12.4 / 10.0 / 12.2, 64 x 4096 x 14336 - / - / - / - / 35 / 27 / 20.
// One workgroup a CU loses what the last round leaves empty, and nothing hides its start and its end: the largest tile is
// taken where the rounds come out nearly even.
// (Measured when the rule was made; the kernels have gained 2 - 10 % since, alike.)
// What bounds it: large sizes the matrix instructions and what feeds them (4096 x 4096 x 14336 173 - 187 us from run to
// run, 2.6 - 2.8 POP/s, of 4.8 that the instruction alone reaches), small ones the way from one chunk to the next, 0.2 - 0.4 us of meeting and latencies.
int int8_gemm_launch(const Int8Product& a, bool pair, hipStream_t s) {
    auto blocks = [&](int channels, int tokens) {
        return (int64_t)((a.n + channels - 1) / channels) * ((a.tokens + tokens - 1) / tokens);
    };
    static constexpr int CUS = 256, ENOUGH = 224;
    const int wide = pair ? 128 : 256;
    const int64_t large = blocks(wide, 256), rounds = (large + CUS - 1) / CUS * CUS;
    if (large >= ENOUGH && large * 20 >= rounds * 19)
        return pair ? gemm8_as<true, false, 4, 2, 2, 8, 128, 4, 1>(a, 0, s) : gemm8_as<false, false, 4, 2, 4, 8, 128, 4, 1>(a, 0, s);
    if (blocks(wide, 128) >= ENOUGH)
        return pair ? gemm8_as<true, false, 4, 1, 2, 8, 128, 4, 1>(a, 0, s) : gemm8_as<false, false, 4, 1, 4, 8, 128, 4, 1>(a, 0, s);
    if (blocks(wide, 64) >= ENOUGH)
        return pair ? gemm8_as<true, false, 4, 1, 2, 4, 128, 4, 1>(a, 0, s) : gemm8_as<false, false, 4, 1, 4, 4, 128, 4, 1>(a, 0, s);
    if (!pair && blocks(128, 64) >= ENOUGH) return gemm8_as<false, false, 4, 1, 2, 4, 256, 8, 1>(a, 0, s);
    if (blocks(64, 64) >= ENOUGH)
        return pair ? gemm8_as<true, false, 4, 1, 1, 4, 256, 8, 2>(a, 0, s) : gemm8_as<false, false, 4, 1, 1, 4, 256, 8, 1>(a, 0, s);
    if (blocks(64, 32) >= 192)
        return pair ? gemm8_as<true, false, 4, 1, 1, 2, 256, 8, 2>(a, 0, s) : gemm8_as<false, false, 4, 1, 1, 2, 256, 8, 2>(a, 0, s);
    return pair ? gemm8_as<true, false, 2, 1, 1, 2, 256, 16, 4>(a, 0, s) : gemm8_as<false, false, 2, 1, 1, 2, 256, 16, 4>(a, 0, s);
}

}  // namespace qmoe
