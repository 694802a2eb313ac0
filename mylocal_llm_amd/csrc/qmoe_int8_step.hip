// The expert step for up to 16 tokens: routing + gate/up in front, down + combine behind.  The back kernel holds the codes of
// every (token, expert) row in LDS at once, 140 KB of them: int8_step_covers.  That is 16 tokens of 10 x 512 and a shared expert of
// 2048 (3.5 KB to spare) or of 8 x 768, 11 of 6 x 1408 and 2816, 10 of 8 x 1536, 4 of 2 x 14336; more tokens take the prompt's step.
//
//   front   Every workgroup routes the tokens and quantises their rows itself (nothing waits for another workgroup), then
//           streams its items: 16 channels of the gate and the up matrix of one expert, shared expert's first.
//   back    A workgroup owns 16 output channels, cuts all hidden activations into codes and streams these channels' rows of
//           every expert that a token chose, then adds each token's terms in ascending expert id.
// Beyond STEP8_FUSED tokens what every workgroup would make again is made by launches of its own: routing and codes of the rows
// in front of the front kernel, codes of the hidden activations between the two (16 tokens: 109 us without the first, 107 with).
//
// Both take each selected expert's bytes once for all tokens that chose it: the 16 token columns of the matrix instruction
// are free (a CU receives 1 KB of weights in about 100 cycles, an instruction multiplies it in 16).  A workgroup's steps of
// 64 columns are one list, cut evenly over its waves whatever expert they belong to; where a wave leaves an expert it adds
// its partial sums to LDS as integers, so neither the cut nor the order of the waves changes a bit, and no wave waits for
// another inside the stream.  Requests run R steps ahead through a ring of registers.
//
// Measured at 512 experts, ten a token, 2048 columns, width 512, shared expert of 2048, weights from memory:
//   1 token    front 13.3 us, back 9.3 us for 44 MB: two launches, each a chain of latencies (launch 2, logits and rows 2,
//              selection 1, first weights 2 us) around 4 - 5 us of streaming
//   16 tokens  routing 6.1, front 62.3 (300 MB, 4.8 TB/s), codes 4.7, back 34.8 us (150 MB, 4.3 TB/s)
#include "qmoe_int8_route.hpp"

namespace qmoe {

// Up to this many tokens every workgroup makes what it needs itself, beyond them launches of their own do it once.
static constexpr int STEP8_FUSED = 4;
static constexpr int STEP8_TOKENS = 16, STEP8_EXPERTS = 1024, STEP8_PAIRS = STEP8_TOKENS * 32;
static constexpr int FRONT8_RING = 4;
static constexpr int BACK8_WAVES = 16, BACK8_THREADS = 64 * BACK8_WAVES, BACK8_RING = 8;
static constexpr int STEP8_LDS = 140 * 1024;         // dynamic; the tables beside it take up to 18 KB of the CU's 160

// what the front kernel leaves for the back kernel
struct Step8Between {
    float* h;            // [tokens * k][f] hidden activations, rows of dropped pairs unwritten
    uint32_t* h_top;     // [tokens * k][f tiles] largest |h| of 16 channels, as bits
    float* sh;           // [tokens][fs], of the shared expert
    uint32_t* sh_top;
    float* admit;        // [tokens] sigmoid of the admission gate
    float* weight;       // [tokens * k]
    int* kept;           // [tokens * k] expert id, -1 for a pair that does not count
    int* n_active;
    int* active;         // experts that some token chose, ascending
    uint8_t* slot;       // [n_active][16] the token's slot that names the expert, 255: none
    uint8_t* row_codes;  // more than STEP8_FUSED tokens: the rows' codes, [tokens * k][fp] and [tokens][fsp], and their scales
    float* row_scale;
};

struct Front8Args {
    const void* x;
    const uint8_t* q;        // [tokens][kp] codes of x and their scales, where they are made beforehand
    const float* q_scale;
    int tokens, k, n_experts, fast;
    const float* logits;
    float floor_value;
    int renorm;
    const float* in_weights;
    const int64_t* in_ids;
    const uint8_t *gate, *up, *s_gate, *s_up;
    const float *gate_c, *up_c, *s_gate_c, *s_up_c;
    const float* admit_w;
    int d, kp, steps, f, f_tiles, fs, fs_tiles, held;      // held: items whose sums fit LDS at a time
    int admit_fast;
    uint32_t per_magic, step_magic, tile_magic, token_magic, k_magic;      // of kp / 8, steps, f_tiles, tokens, k
    Step8Between o;
    float* out_weights;
    int64_t* out_ids;
    int* status;
};

// x / d for x * d < 2^32; magic = floor(2^32 / d) + 1 (d > 1), 0 for d = 1
__host__ __device__ __forceinline__ int over(int x, uint32_t magic) { return magic ? (int)(((uint64_t)(uint32_t)x * magic) >> 32) : x; }

// CODED: routing and codes of the rows are there (int8_route_launch); in_ids and in_weights hold them.
template <int XDT, int WAVES, bool CODED>
__global__ __launch_bounds__(64 * WAVES) void int8_front_kernel(const Front8Args a) {
    extern __shared__ __align__(16) uint8_t dynamic[];      // [tokens][kp + 16] codes | [held][tokens][32] sums | [held][32] scales
    __shared__ uint32_t chosen[STEP8_EXPERTS];              // bit t: token t chose the expert
    __shared__ uint16_t index_of[STEP8_EXPERTS], active[STEP8_PAIRS];
    __shared__ __align__(16) uint8_t slot_of[STEP8_PAIRS * STEP8_TOKENS];     // (scratch of the routing until the lists are made)
    __shared__ int pair_id[STEP8_PAIRS];
    __shared__ uint32_t tops[STEP8_TOKENS];
    __shared__ float srow[STEP8_TOKENS];
    __shared__ int n_found;
    constexpr int THREADS = 64 * WAVES;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), col = lane & 15, g = lane >> 4;
    const int tokens = a.tokens, k = a.k, pairs = tokens * k, stride = a.kp + 16, G = (int)gridDim.x;
    const bool publisher = (int)blockIdx.x == G - 1;        // of the workgroups with the fewest items
    uint8_t* const codes = dynamic;
    int* const sums = (int*)(dynamic + (size_t)tokens * stride);
    float* const scales = (float*)(sums + (size_t)a.held * tokens * 32);

    // ---- requests: a wave's row of logits, eight values of x a thread and turn, up to NX turns in registers ----
    RowIds<8> narrow;
    if (!CODED && a.logits && wave < tokens) narrow.load(a.logits + (size_t)wave * a.n_experts, a.n_experts);
    const int per = a.kp / 8, groups = tokens * per;
    constexpr int NX = 4;
    float v[NX][8];
    auto load = [&](int gi, float* to) {
        const int t = gi < groups ? over(gi, a.per_magic) : 0, i = (gi - t * per) * 8, left = gi < groups ? a.d - i : 0;
        int8_load8<XDT>(a.x, left > 0 ? (size_t)t * a.d + i : 0, left, a.fast, to);
    };
    i32x4_t piece[NX];
    const int pieces = tokens * per / 2;
    auto fetch = [&](int p0) {
#pragma unroll
        for (int j = 0; j < NX; ++j) {
            const int p = p0 + j * THREADS + tid;
            piece[j] = ldg_i32x4(a.q + (int64_t)(p < pieces ? p : 0) * 16);
        }
    };
    if (CODED) fetch(0);
    else {
#pragma unroll
        for (int p = 0; p < NX; ++p)
            if (p * THREADS < groups) load(p * THREADS + tid, v[p]);
    }
    for (int i = tid; i < a.n_experts; i += THREADS) chosen[i] = 0u;
    if (tid < STEP8_TOKENS) tops[tid] = 0u;
    for (int i = tid; i < a.held * tokens * 32; i += THREADS) sums[i] = 0;
    meet_lds();

    // ---- the rows' largest values ----
    const bool wave_row = per % 64 == 0;           // a wave's values belong to one token
    auto raise = [&](int gi, const float* w) {
        uint32_t top = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) { const uint32_t b = abs_bits(w[j]); top = b > top ? b : top; }
        if (wave_row) top = wave_max_u32(top);
        if (gi < groups && (!wave_row || lane == 0)) atomicMax(&tops[over(gi, a.per_magic)], top);
    };
    auto turns = [&](auto&& f) {                   // every turn of eight values: the first ones from registers
#pragma unroll
        for (int p = 0; p < NX; ++p)
            if (p * THREADS < groups) f(p * THREADS + tid, v[p]);
        for (int g0 = NX * THREADS; g0 < groups; g0 += THREADS) {
            float w[8];
            load(g0 + tid, w);
            f(g0 + tid, w);
        }
    };
    if (!CODED) {
        turns(raise);
        meet_lds();
    }

    // ---- codes ----
    if (tid < tokens) srow[tid] = CODED ? ldg<float>(a.q_scale + tid) : RowScale(tops[tid]).s;
    if (CODED) {
        for (int p0 = 0; p0 < pieces; p0 += NX * THREADS) {
#pragma unroll
            for (int j = 0; j < NX; ++j) {
                const int p = p0 + j * THREADS + tid, t = over(2 * p, a.per_magic);
                if (p < pieces) *(i32x4_t*)(codes + t * stride + (2 * p - t * per) * 8) = piece[j];
            }
            if (p0 + NX * THREADS < pieces) fetch(p0 + NX * THREADS);
        }
    } else {
        turns([&](int gi, const float* w) {
            const int t = gi < groups ? over(gi, a.per_magic) : 0, i = (gi - t * per) * 8;
            const u32x2_t q = int8_code8(w, RowScale(tops[t]));
            if (gi < groups) *(u32x2_t*)(codes + t * stride + i) = q;
        });
    }
    // ---- routing: a wave a token ----
    int bad = 0;
    for (int t = wave; t < tokens; t += WAVES) {
        const float* const z = a.logits + (size_t)t * a.n_experts;
        float weight = 0.0f;
        int64_t id = -1;
        uint2* const scratch = (uint2*)slot_of + wave * 64;
        // (nothing but the ids is needed to stream: one workgroup makes the weights)
        if (!CODED && a.logits && a.n_experts <= 512) {
            if (t != wave) narrow.load(z, a.n_experts);
            if (publisher) narrow.route(z, a.n_experts, k, a.floor_value, a.renorm, scratch, weight, id);
            else id = narrow.select(a.n_experts, k, scratch);
        } else if (!CODED && a.logits) {
            RowIds<16> wide;
            wide.load(z, a.n_experts);
            if (publisher) wide.route(z, a.n_experts, k, a.floor_value, a.renorm, scratch, weight, id);
            else id = wide.select(a.n_experts, k, scratch);
        } else if (lane < k) {
            weight = ldg<float>(a.in_weights + (size_t)t * k + lane);
            id = ldg<int64_t>(a.in_ids + (size_t)t * k + lane);
        }
        const bool inside = lane < k && id >= 0 && id < a.n_experts;
        int e = inside ? (int)id : -1;
        int same = 0, below = 0, kept = 0;        // earlier slots with the same id; kept ids smaller than this one
        for (int j = 0; j < k; ++j) same += __builtin_amdgcn_readlane(e, j) == e && j < lane;
        if (inside && same) e = -1;
        if (tokens == 1) {
            for (int j = 0; j < k; ++j) {
                const int o = __builtin_amdgcn_readlane(e, j);
                below += o >= 0 && o < e;
                kept += o >= 0;
            }
        }
        if (lane < k) {
            bad |= (inside ? 0 : 1) | (inside && same ? 2 : 0);
            pair_id[t * k + lane] = e;
            if (e >= 0) {
                atomicOr(&chosen[e], 1u << t);
                if (tokens == 1) { active[below] = (uint16_t)e; index_of[e] = (uint16_t)below; }
            }
            if (tokens == 1 && lane == 0) n_found = kept;
            if (publisher) {
                a.o.weight[t * k + lane] = weight;
                a.o.kept[t * k + lane] = e;
                if (a.out_weights) a.out_weights[t * k + lane] = weight;
                if (a.out_ids) a.out_ids[t * k + lane] = id;
            }
        }
    }
    if (publisher && a.status && bad) atomicOr(a.status, bad);

    meet_lds();
    // the experts that several tokens chose, ascending
    if (tokens > 1) {
        if (wave == 0) {
            int n = 0;
    #pragma unroll
            for (int j = 0; j < STEP8_EXPERTS / 64; ++j) {
                const int e = j * 64 + lane;
                const bool c = e < a.n_experts && chosen[e];
                const unsigned long long m = __ballot(c);
                const int at = n + __popcll(m & ((1ull << lane) - 1));
                if (c) { active[at] = (uint16_t)e; index_of[e] = (uint16_t)at; }
                n += __popcll(m);
            }
            if (lane == 0) n_found = n;
        }
        meet_lds();
    }
    const int n_active = __builtin_amdgcn_readfirstlane(n_found);

    // ---- stream ----
    const int items = a.fs_tiles + n_active * a.f_tiles, first = blockIdx.x;
    const int mine = first < items ? (items - first + G - 1) / G : 0;
    const uint8_t* const row = codes + (col < tokens ? col : tokens - 1) * stride + g * 16;
    // item -> expert (-1: shared) and tile of 16 channels
    auto place = [&](int it, int& e, int& tile) {
        const int gi = first + it * G, ri = gi - a.fs_tiles;
        const int ai = over(ri < 0 ? 0 : ri, a.tile_magic);
        e = ri < 0 ? -1 : active[ai];
        tile = ri < 0 ? gi : ri - ai * a.f_tiles;
    };
    for (int r0 = 0; r0 < mine; r0 += a.held) {
        const int n = mine - r0 < a.held ? mine - r0 : a.held;
        if (r0) {
            meet_lds();            // the last round's sums are read
            for (int i = tid; i < n * tokens * 32; i += THREADS) sums[i] = 0;
            meet_lds();
        }
        // the items' channel scales travel while the stream starts
        auto scale = [&](int i) -> float {
            int e, tile;
            place(r0 + (i >> 5), e, tile);
            const int ch = tile * 16 + (i & 15), wide = e < 0 ? a.fs : a.f, in = ch < wide ? ch : wide - 1;
            const float* const c = i & 16 ? (e < 0 ? a.s_up_c : a.up_c) : (e < 0 ? a.s_gate_c : a.gate_c);
            return ldg<float>(c + (e < 0 ? 0 : (int64_t)e * a.f) + in);
        };
        const float own = scale(tid < n * 32 ? tid : 0);
        const int total = n * a.steps, lo = (int)((int64_t)total * wave / WAVES), hi = (int)((int64_t)total * (wave + 1) / WAVES);
        if (lo < hi) {
            // the fetching end
            int f_it = over(lo, a.step_magic), f_k = lo - f_it * a.steps, left = hi - lo;
            const uint8_t *pg, *pu;
            auto point = [&]() {
                int e, tile;
                place(r0 + f_it, e, tile);
                e = __builtin_amdgcn_readfirstlane(e);
                tile = __builtin_amdgcn_readfirstlane(tile);
                const int64_t off = (int64_t)(e < 0 ? tile : e * a.f_tiles + tile) * a.kp * 16 + (int64_t)f_k * 1024;
                pg = (e < 0 ? a.s_gate : a.gate) + off;
                pu = (e < 0 ? a.s_up : a.up) + off;
            };
            point();
            i32x4_t wg[FRONT8_RING], wu[FRONT8_RING];
            auto request = [&](int u) {
                wg[u] = ldg_i32x4(pg + lane * 16);
                wu[u] = ldg_i32x4(pu + lane * 16);
                if (--left > 0) {              // (past the end the last step is requested again)
                    pg += 1024;
                    pu += 1024;
                    if (++f_k == a.steps) { f_k = 0; ++f_it; point(); }
                }
            };
#pragma unroll
            for (int u = 0; u < FRONT8_RING; ++u) request(u);
            if (tid < n * 32) scales[tid] = own;
            // the multiplying end
            int c_it = over(lo, a.step_magic), c_k = lo - c_it * a.steps;
            i32x4_t ag = {0, 0, 0, 0}, au = {0, 0, 0, 0};
            auto flush = [&]() {
                int e, tile;
                place(r0 + c_it, e, tile);
                if (col < tokens && (e < 0 || chosen[e < 0 ? 0 : e] >> col & 1u)) {
                    int* const s = sums + ((size_t)c_it * tokens + col) * 32 + 4 * g;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        atomicAdd(s + i, ag[i]);
                        atomicAdd(s + 16 + i, au[i]);
                    }
                }
                ag = i32x4_t{0, 0, 0, 0};
                au = i32x4_t{0, 0, 0, 0};
            };
            auto multiply = [&](int u) {
                const i32x4_t b = *(const i32x4_t*)(row + c_k * 64);
                ag = mfma_i8(wg[u], b, ag);
                au = mfma_i8(wu[u], b, au);
                if (++c_k == a.steps) { flush(); c_k = 0; ++c_it; }
            };
            int s = lo;
            for (; s + FRONT8_RING <= hi; s += FRONT8_RING)
#pragma unroll
                for (int u = 0; u < FRONT8_RING; ++u) { multiply(u); request(u); }
#pragma unroll
            for (int u = 0; u + 1 < FRONT8_RING; ++u)
                if (s + u < hi) multiply(u);
            if (c_k) flush();
        } else if (tid < n * 32) scales[tid] = own;
        for (int i = tid + THREADS; i < n * 32; i += THREADS) scales[i] = scale(i);
        if (!r0)
            for (int p = tid; p < pairs; p += THREADS) {
                const int t = over(p, a.k_magic);
                if (pair_id[p] >= 0) slot_of[index_of[pair_id[p]] * STEP8_TOKENS + t] = (uint8_t)(p - t * k);
            }
        meet_lds();
        // 16 neighbouring threads hold the 16 channels of one (item, token)
        for (int o = tid; o < n * tokens * 16; o += THREADS) {
            const int it = over(o >> 4, a.token_magic), t = (o >> 4) - it * tokens, ch = o & 15;
            int e, tile;
            place(r0 + it, e, tile);
            const int wide = e < 0 ? a.fs : a.f, nn = tile * 16 + ch;
            const bool live = e < 0 || (chosen[e < 0 ? 0 : e] >> t & 1u);
            float h = 0.0f;
            if (live) {
                const int* const s = sums + ((size_t)it * tokens + t) * 32 + ch;
                h = int8_hidden(int8_value(s[0], srow[t], scales[it * 32 + ch]), int8_value(s[16], srow[t], scales[it * 32 + 16 + ch]));
            }
            uint32_t top = live && nn < wide ? abs_bits(h) : 0u;
            top = dpp_max_u32<0xB1, 0xf>(top);
            top = dpp_max_u32<0x4E, 0xf>(top);
            top = dpp_max_u32<0x141, 0xf>(top);
            top = dpp_max_u32<0x140, 0xf>(top);
            if (live) {
                const int64_t p = e < 0 ? t : t * k + slot_of[index_of[e] * STEP8_TOKENS + t];
                if (nn < wide) stg<float>((e < 0 ? a.o.sh + p * a.fs : a.o.h + p * a.f) + nn, h);
                if (ch == 0) stg<uint32_t>((e < 0 ? a.o.sh_top + p * a.fs_tiles : a.o.h_top + p * a.f_tiles) + tile, top);
            }
        }
    }
    // ---- what the back kernel reads besides: the plan, and the admission gates from the workgroups in front of this one ----
    if (publisher) {
        if (!mine) {
            for (int p = tid; p < pairs; p += THREADS) {
                const int t = over(p, a.k_magic);
                if (pair_id[p] >= 0) slot_of[index_of[pair_id[p]] * STEP8_TOKENS + t] = (uint8_t)(p - t * k);
            }
            meet_lds();
        }
        if (tid == 0) *a.o.n_active = n_active;
        for (int i = tid; i < n_active; i += THREADS) a.o.active[i] = active[i];
        for (int i = tid; i < n_active * STEP8_TOKENS; i += THREADS)
            a.o.slot[i] = chosen[active[i / STEP8_TOKENS]] >> (i % STEP8_TOKENS) & 1u ? slot_of[i] : (uint8_t)255;
    }
    if (a.admit_w && wave == WAVES - 1) {
        for (int t = (G + G - 2 - (int)blockIdx.x) % G; t < tokens; t += G) {
            const float admit = int8_admission<XDT>(a.x, (size_t)t * a.d, a.fast, a.admit_w, a.fast && a.admit_fast, a.d);
            if (lane == 0) a.o.admit[t] = admit;
        }
    }
}

struct Back8Args {
    Step8Between in;
    int tokens, k, d, f, fp, f_tiles, f_steps, fs, fsp, fs_tiles, fs_steps;
    const uint8_t *down, *s_down;
    const float *down_c, *s_down_c;
    const float* residual;
    void* out;
    int odt, gated;
    uint32_t h_magic, s_magic, hp_magic, sp_magic;      // of the turns and of the 16-byte pieces of a row
};

// The hidden activations' codes for more than STEP8_FUSED tokens, a workgroup a row: a workgroup of the back kernel that makes
// them itself needs 15 us for 16 tokens (every one makes all of them), this launch 4.7 us.
__global__ __launch_bounds__(256) void int8_hidden_codes_kernel(const Back8Args a) {
    __shared__ uint32_t tops[4];
    const int pairs = a.tokens * a.k, r = blockIdx.x, tid = threadIdx.x;
    const bool sh = r >= pairs;
    const int64_t at = sh ? r - pairs : r;
    const int wide = sh ? a.fs : a.f, padded = sh ? a.fsp : a.fp, tiles = sh ? a.fs_tiles : a.f_tiles;
    if (!sh && ldg<int>(a.in.kept + r) < 0) return;        // not read by any result
    const float* const h = (sh ? a.in.sh : a.in.h) + at * wide;
    float v[8];
    int8_load8<QMOE_DT_F32>(h, tid * 8 < wide ? tid * 8 : 0, wide - tid * 8, wide % 8 == 0, v);
    uint32_t top = 0;
    for (int i = tid; i < tiles; i += 256) { const uint32_t b = ldg<uint32_t>((sh ? a.in.sh_top : a.in.h_top) + at * tiles + i); top = b > top ? b : top; }
    top = wave_max_u32(top);
    if ((tid & 63) == 0) tops[tid >> 6] = top;
    __syncthreads();
    for (int i = 0; i < 4; ++i) top = tops[i] > top ? tops[i] : top;
    const RowScale rs(top);
    if (tid == 0) a.in.row_scale[r] = rs.s;
    uint8_t* const to = a.in.row_codes + (sh ? (int64_t)pairs * a.fp + at * a.fsp : at * a.fp);
    for (int i0 = 0; i0 < padded; i0 += 2048) {
        const int i = i0 + tid * 8;
        if (i0) int8_load8<QMOE_DT_F32>(h, i < wide ? i : 0, wide - i, wide % 8 == 0, v);
        const u32x2_t q = int8_code8(v, rs);
        if (i < padded) *(QMOE_GLOBAL u32x2_t*)(to + i) = q;
    }
}

// CODES: they are there; otherwise every workgroup makes them.
template <bool CODES> __global__ __launch_bounds__(BACK8_THREADS) void int8_back_kernel(const Back8Args a) {
    // [pairs][fp + 16] codes | [tokens][fsp + 16] codes | [pairs + tokens][16] sums | [pairs + 1][16] channel scales | [pairs + tokens] row scales
    extern __shared__ __align__(16) uint8_t dynamic[];
    __shared__ int pair_id[STEP8_PAIRS];
    __shared__ float pair_weight[STEP8_PAIRS];
    __shared__ uint16_t active[STEP8_PAIRS];
    __shared__ __align__(4) uint8_t slot_of[STEP8_PAIRS * STEP8_TOKENS];
    __shared__ uint8_t order[STEP8_PAIRS], count[STEP8_TOKENS];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), col = lane & 15, g = lane >> 4;
    const int tokens = a.tokens, k = a.k, pairs = tokens * k, tile = blockIdx.x;
    const int hst = a.fp + 16, sst = a.fsp + 16, srows = a.fs ? tokens : 0;
    uint8_t* const hq = dynamic;
    uint8_t* const sq = hq + (size_t)pairs * hst;
    int* const sums = (int*)(sq + (size_t)srows * sst);
    float* const scales = (float*)(sums + (size_t)(pairs + srows) * 16);
    float* const srow = scales + (size_t)(pairs + 1) * 16;

    const int n_active = __builtin_amdgcn_readfirstlane(ldg<int>(a.in.n_active));
    i32x4_t ring[BACK8_RING];
    // Codes: a wave a row, 512 values a turn.  A row's scale comes from the largest of each 16 channels, which the front kernel
    // left; four turns are requested at a time.  (Rows of pairs that do not count hold anything and are read by no result.)
    const int rows = pairs + srows, h_turns = (a.fp + 511) / 512, s_turns = (a.fsp + 511) / 512;
    const int h_all = pairs * h_turns, all = h_all + srows * s_turns;
    struct Turn { int r, i; bool sh; };
    auto turn = [&](int n) {
        Turn c;
        c.sh = n >= h_all;
        c.r = c.sh ? over(n - h_all, a.s_magic) : over(n, a.h_magic);
        c.i = (c.sh ? n - h_all - c.r * s_turns : n - c.r * h_turns) * 512;
        return c;
    };
    constexpr int NX = 4;
    float v[NX][8];
    uint32_t part[NX];
    auto load = [&](int n, float* x, uint32_t& top) {
        const Turn c = turn(n < all ? n : 0);
        const int wide = c.sh ? a.fs : a.f, tiles = c.sh ? a.fs_tiles : a.f_tiles, i = c.i + lane * 8;
        const float* const h = (c.sh ? a.in.sh : a.in.h) + (int64_t)c.r * wide;
        const uint32_t* const p = (c.sh ? a.in.sh_top : a.in.h_top) + (int64_t)c.r * tiles;
        int8_load8<QMOE_DT_F32>(h, i < wide ? i : 0, wide - i, wide % 8 == 0, x);
        top = ldg<uint32_t>(p + (lane < tiles ? lane : 0));
        for (int j = lane + 64; j < tiles; j += 64) { const uint32_t b = ldg<uint32_t>(p + j); top = b > top ? b : top; }
    };
    // with CODES: pieces of 16 bytes, first the pairs' rows, then the shared expert's
    const int h_pieces = pairs * a.f_steps * 4, pieces = h_pieces + srows * a.fs_steps * 4;
    constexpr int NC = 8;
    i32x4_t piece[NC];
    auto fetch = [&](int p0) {
#pragma unroll
        for (int j = 0; j < NC; ++j) {
            const int p = p0 + j * BACK8_THREADS + tid;
            piece[j] = ldg_i32x4(a.in.row_codes + (int64_t)(p < pieces ? p : 0) * 16);
        }
    };
    if (CODES) fetch(0);
    else {
#pragma unroll
        for (int p = 0; p < NX; ++p) load(wave + p * BACK8_WAVES, v[p], part[p]);
    }
    for (int i = tid; i < pairs; i += BACK8_THREADS) {
        pair_id[i] = ldg<int>(a.in.kept + i);
        pair_weight[i] = ldg<float>(a.in.weight + i);
        // (entries behind the last active expert are not read; the arrays hold one for each pair)
        active[i] = (uint16_t)ldg<int>(a.in.active + i);
    }
    for (int i = tid; i < pairs * 4; i += BACK8_THREADS) ((uint32_t*)slot_of)[i] = ldg<uint32_t>((const uint32_t*)a.in.slot + i);
    // The list of steps: the shared expert's (item -1), then every chosen expert's.  The first requests leave before the codes are
    // made; they come back in order, so that nothing above waits for them.
    const int total = a.fs_steps + n_active * a.f_steps, lo = (int)((int64_t)total * wave / BACK8_WAVES), hi = (int)((int64_t)total * (wave + 1) / BACK8_WAVES);
    const int64_t expert_bytes = (int64_t)((a.d + 15) / 16) * a.fp * 16;
    const int lo_ai = lo < a.fs_steps ? -1 : (lo - a.fs_steps) / a.f_steps, lo_k = lo_ai < 0 ? lo : lo - a.fs_steps - lo_ai * a.f_steps;
    int f_ai = lo_ai, f_k = lo_k, f_end = lo_ai < 0 ? a.fs_steps : a.f_steps, left = hi - lo;
    const uint8_t* pw = nullptr;
    auto point = [&](int e) {
        pw = (f_ai < 0 ? a.s_down + (int64_t)tile * a.fsp * 16 : a.down + e * expert_bytes + (int64_t)tile * a.fp * 16) + (int64_t)f_k * 1024;
    };
    auto request = [&](int u, auto&& expert_at) {
        ring[u] = ldg_i32x4(pw + lane * 16);
        if (--left > 0) {                      // (past the end the last step is requested again)
            pw += 1024;
            if (++f_k == f_end) { f_k = 0; ++f_ai; f_end = a.f_steps; point(expert_at(f_ai)); }
        }
    };
    if (lo < hi) {
        auto listed = [&](int ai) { return __builtin_amdgcn_readfirstlane(ldg<int>(a.in.active + ai)); };
        point(f_ai < 0 ? 0 : listed(f_ai));
#pragma unroll
        for (int u = 0; u < BACK8_RING; ++u) request(u, listed);
    }
    for (int i = tid; i < rows * 16; i += BACK8_THREADS) sums[i] = 0;
    if (CODES) {
        for (int i = tid; i < rows; i += BACK8_THREADS) srow[i] = ldg<float>(a.in.row_scale + i);
        for (int p0 = 0; p0 < pieces; p0 += NC * BACK8_THREADS) {
#pragma unroll
            for (int j = 0; j < NC; ++j) {
                const int p = p0 + j * BACK8_THREADS + tid, sp0 = p - h_pieces;
                const int r = sp0 < 0 ? over(p, a.hp_magic) : over(sp0, a.sp_magic);
                uint8_t* const to = sp0 < 0 ? hq + (size_t)r * hst + (p - r * a.f_steps * 4) * 16 : sq + (size_t)r * sst + (sp0 - r * a.fs_steps * 4) * 16;
                if (p < pieces) *(i32x4_t*)to = piece[j];
            }
            if (p0 + NC * BACK8_THREADS < pieces) fetch(p0 + NC * BACK8_THREADS);
        }
    } else {
        for (int n = wave; n < all; n += NX * BACK8_WAVES) {
#pragma unroll
            for (int p = 0; p < NX; ++p) {
                if (n + p * BACK8_WAVES < all) {
                    const Turn c = turn(n + p * BACK8_WAVES);
                    const RowScale rs(wave_max_u32(part[p]));
                    if (lane == 0 && c.i == 0) srow[(c.sh ? pairs : 0) + c.r] = rs.s;
                    const int i = c.i + lane * 8;
                    const u32x2_t q = int8_code8(v[p], rs);
                    if (i < (c.sh ? a.fsp : a.fp)) *(u32x2_t*)((c.sh ? sq + (size_t)c.r * sst : hq + (size_t)c.r * hst) + i) = q;
                }
            }
            if (n + NX * BACK8_WAVES < all) {
#pragma unroll
                for (int p = 0; p < NX; ++p) load(n + (p + NX) * BACK8_WAVES, v[p], part[p]);
            }
        }
    }
    meet_lds();
    // channel scales, and every token's kept slots in ascending expert id
    for (int i = tid; i < (pairs + 1) * 16; i += BACK8_THREADS) {
        const int p = i >> 4, n = tile * 16 + (i & 15), in = n < a.d ? n : a.d - 1;
        if (p == pairs) scales[i] = a.fs ? ldg<float>(a.s_down_c + in) : 0.0f;
        else scales[i] = pair_id[p] >= 0 ? ldg<float>(a.down_c + (int64_t)pair_id[p] * a.d + in) : 0.0f;
    }
    for (int p = tid; p < pairs; p += BACK8_THREADS) {
        const int t = p / k;
        int rank = 0, n = 0;
        for (int j = 0; j < k; ++j) {
            const int o = pair_id[t * k + j];
            rank += o >= 0 && o < pair_id[p];
            n += o >= 0;
        }
        if (pair_id[p] >= 0) order[t * k + rank] = (uint8_t)(p - t * k);
        if (p == t * k) count[t] = (uint8_t)n;
    }
    auto add = [&](int p, i32x4_t acc) {
        int* const s = sums + p * 16 + 4 * g;
#pragma unroll
        for (int i = 0; i < 4; ++i) atomicAdd(s + i, acc[i]);
    };
    // ---- stream ----
    if (lo < hi) {
        auto listed = [&](int ai) { return __builtin_amdgcn_readfirstlane((int)active[ai]); };
        int c_ai = lo_ai, c_k = lo_k, c_end = lo_ai < 0 ? a.fs_steps : a.f_steps, p = -1;
        const uint8_t* b0 = hq;
        auto enter = [&]() {       // this lane's token's row of codes, a valid one where the token did not choose the expert
            if (c_ai < 0) {
                p = col < tokens ? pairs + col : -1;
                b0 = sq + (size_t)(col < tokens ? col : 0) * sst + g * 16;
                return;
            }
            const int s = col < tokens ? slot_of[c_ai * STEP8_TOKENS + col] : 255;
            p = s < 255 ? col * k + s : -1;
            b0 = hq + (size_t)(p < 0 ? 0 : p) * hst + g * 16;
        };
        enter();
        i32x4_t acc = {0, 0, 0, 0};
        auto multiply = [&](int u) {
            acc = mfma_i8(ring[u], *(const i32x4_t*)(b0 + c_k * 64), acc);
            if (++c_k == c_end) {
                if (p >= 0) add(p, acc);
                acc = i32x4_t{0, 0, 0, 0};
                c_k = 0;
                c_end = a.f_steps;
                if (++c_ai < n_active) enter();
            }
        };
        int s = lo;
        for (; s + BACK8_RING <= hi; s += BACK8_RING)
#pragma unroll
            for (int u = 0; u < BACK8_RING; ++u) { multiply(u); request(u, listed); }
#pragma unroll
        for (int u = 0; u + 1 < BACK8_RING; ++u)
            if (s + u < hi) multiply(u);
        if (c_k && p >= 0) add(p, acc);
    }
    meet_lds();
    for (int o = tid; o < tokens * 16; o += BACK8_THREADS) {
        const int t = o >> 4, ch = o & 15, n = tile * 16 + ch;
        if (n >= a.d) continue;
        float sum = 0.0f;
        for (int j = 0; j < count[t]; ++j) {
            const int p = t * k + order[t * k + j];
            sum = add_product(sum, (float)int8_value(sums[p * 16 + ch], srow[p], scales[p * 16 + ch]), pair_weight[p]);
        }
        if (a.fs) {
            const float y = (float)int8_value(sums[(pairs + t) * 16 + ch], srow[pairs + t], scales[pairs * 16 + ch]);
            sum = add_product(sum, y, a.gated ? ldg<float>(a.in.admit + t) : 1.0f);
        }
        if (a.residual) sum = __fadd_rn(ldg<float>(a.residual + (size_t)t * a.d + n), sum);
        store_out(a.out, a.odt, (size_t)t * a.d + n, sum);
    }
}

// ---- host --------------------------------------------------------------------------------------------------
struct Step8Layout { size_t h, h_top, sh, sh_top, admit, weight, kept, n_active, active, slot, row_codes, row_scale, q, q_scale, ids, total; };
static Step8Layout step8_layout(int tokens, int k, int d, int f, int fs) {
    Step8Layout w;
    size_t at = 0;
    const size_t pairs = (size_t)tokens * k;
    auto take = [&](size_t bytes) { const size_t here = at; at = (at + bytes + 255) & ~(size_t)255; return here; };
    w.h = take(pairs * f * 4);
    w.h_top = take(pairs * ((f + 15) / 16) * 4);
    w.sh = take((size_t)tokens * fs * 4);
    w.sh_top = take((size_t)tokens * ((fs + 15) / 16) * 4);
    w.admit = take(tokens * 4);
    w.weight = take(pairs * 4);
    w.kept = take(pairs * 4);
    w.n_active = take(4);
    w.active = take(pairs * 4);
    w.slot = take(pairs * STEP8_TOKENS);
    w.row_codes = take(pairs * int8_cols64(f) + (size_t)tokens * (fs ? int8_cols64(fs) : 0));
    w.row_scale = take((pairs + tokens) * 4);
    w.q = take(tokens * int8_cols64(d));
    w.q_scale = take(tokens * 4);
    w.ids = take(pairs * 8);
    w.total = at;
    return w;
}

static size_t back8_lds(int tokens, int k, int f, int fs) {
    const size_t pairs = (size_t)tokens * k, srows = fs ? tokens : 0;
    return pairs * (int8_cols64(f) + 16) + srows * (int8_cols64(fs) + 16) + (pairs + srows) * 64 + (pairs + 1) * 64 + (pairs + srows) * 4;
}
static size_t front8_codes(int tokens, int d) { return (size_t)tokens * (int8_cols64(d) + 16); }
static size_t front8_item(int tokens) { return (size_t)tokens * 128 + 128; }

// Whether the two kernels cover a step: their tables, and the rows of codes that they hold in LDS.
bool int8_step_covers(int tokens, int k, int n_experts, int d, int f, int fs) {
    // (the multiply-high divisions are exact while dividend x divisor < 2^32)
    const int64_t f_tiles = (f + 15) / 16, items = (fs + 15) / 16 + f_tiles * ((int64_t)tokens * k < n_experts ? tokens * k : n_experts);
    const int64_t steps = int8_cols64(d) / 64;
    if (items * f_tiles >= (1ll << 31) || items * steps * steps >= (1ll << 31) || n_experts * f_tiles >= (1ll << 31)) return false;
    return tokens <= STEP8_TOKENS && k <= 32 && n_experts <= STEP8_EXPERTS && back8_lds(tokens, k, f, fs) <= STEP8_LDS &&
           front8_codes(tokens, d) + 4 * front8_item(tokens) <= STEP8_LDS;
}
size_t int8_step_bytes(int tokens, int k, int d, int f, int fs) { return step8_layout(tokens, k, d, f, fs).total; }

static int raise_lds(const void* fn, bool (&raised)[64]) {
    int dev = 0;
    (void)hipGetDevice(&dev);
    if (dev >= 0 && dev < 64 && raised[dev]) return QMOE_OK;
    if (hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize, STEP8_LDS) != hipSuccess)
        return fail(QMOE_ELAUNCH, "int8 expert step: the device refuses %d bytes of LDS", STEP8_LDS);
    if (dev >= 0 && dev < 64) raised[dev] = true;
    return QMOE_OK;
}

template <int XDT, int WAVES, bool CODED> static int front8_as(const Front8Args& a, int grid, size_t lds, hipStream_t s) {
    static bool raised[64];
    if (const int rc = raise_lds((const void*)&int8_front_kernel<XDT, WAVES, CODED>, raised)) return rc;
    hipLaunchKernelGGL((int8_front_kernel<XDT, WAVES, CODED>), dim3(grid), dim3(64 * WAVES), lds, s, a);
    return check_launch("int8 expert step (front)");
}
template <int XDT> static int front8_waves(const Front8Args& a, int grid, size_t lds, hipStream_t s) {
    return a.tokens <= STEP8_FUSED ? front8_as<XDT, 8, false>(a, grid, lds, s) : front8_as<XDT, 16, true>(a, grid, lds, s);
}
static uint32_t magic_of(int d) { return d <= 1 ? 0u : (uint32_t)(0x100000000ull / (uint32_t)d) + 1u; }

template <bool CODES> static int back8_as(const Back8Args& a, hipStream_t s) {
    static bool raised[64];
    if (const int rc = raise_lds((const void*)&int8_back_kernel<CODES>, raised)) return rc;
    hipLaunchKernelGGL(int8_back_kernel<CODES>, dim3((a.d + 15) / 16), dim3(BACK8_THREADS), back8_lds(a.tokens, a.k, a.f, a.fs), s, a);
    return check_launch("int8 expert step (back)");
}

int stream_grid();
int int8_route_launch(const qmoe_int8_moe_args& m, float* weights, int64_t* ids, uint8_t* codes, int64_t ld, float* scales, hipStream_t s);

int int8_step_launch(const qmoe_int8_moe_args& m, char* ws, hipStream_t s) {
    const int t = m.tokens, k = m.top_k, d = m.d_model, f = m.d_ff, fs = m.d_ff_shared;
    const Step8Layout L = step8_layout(t, k, d, f, fs);
    Step8Between b{(float*)(ws + L.h), (uint32_t*)(ws + L.h_top), (float*)(ws + L.sh), (uint32_t*)(ws + L.sh_top), (float*)(ws + L.admit),
                   (float*)(ws + L.weight), (int*)(ws + L.kept), (int*)(ws + L.n_active), (int*)(ws + L.active), (uint8_t*)(ws + L.slot),
                   (uint8_t*)(ws + L.row_codes), (float*)(ws + L.row_scale)};
    Front8Args a{};
    a.x = m.hidden; a.tokens = t; a.k = k; a.n_experts = m.n_experts;
    a.fast = (uintptr_t)m.hidden % 16 == 0 && d % 8 == 0;
    a.logits = m.logits; a.floor_value = m.floor_value; a.renorm = m.renormalize; a.in_weights = m.in_weights; a.in_ids = m.in_ids;
    a.gate = (const uint8_t*)m.gate; a.up = (const uint8_t*)m.up; a.gate_c = m.gate_scales; a.up_c = m.up_scales;
    a.s_gate = (const uint8_t*)m.shared_gate_w; a.s_up = (const uint8_t*)m.shared_up_w; a.s_gate_c = m.shared_gate_scales; a.s_up_c = m.shared_up_scales;
    a.admit_w = fs ? m.shared_gate : nullptr;
    a.d = d; a.kp = (int)int8_cols64(d); a.steps = a.kp / 64; a.f = f; a.f_tiles = (f + 15) / 16; a.fs = fs; a.fs_tiles = (fs + 15) / 16;
    a.admit_fast = (uintptr_t)m.shared_gate % 16 == 0;
    a.per_magic = magic_of(a.kp / 8); a.step_magic = magic_of(a.steps); a.tile_magic = magic_of(a.f_tiles); a.token_magic = magic_of(t); a.k_magic = magic_of(k);
    a.o = b; a.out_weights = m.out_weights; a.out_ids = m.out_ids; a.status = m.status_out;
    const int64_t most = (int64_t)t * k < m.n_experts ? (int64_t)t * k : m.n_experts;
    const int64_t items = a.fs_tiles + most * a.f_tiles;
    const int cus = stream_grid() / 2;
    const int grid = (int)(items + 1 < cus ? items + 1 : cus);
    // the sums of as many items as a workgroup has, or as the codes leave room for
    const size_t codes = front8_codes(t, d), room = (size_t)STEP8_LDS - codes;
    const int64_t need = (items + grid - 1) / grid, fits = (int64_t)(room / front8_item(t));
    a.held = (int)(need < fits ? need : fits);
    const size_t lds = codes + a.held * front8_item(t);
    int rc;
    if (t > STEP8_FUSED) {
        a.q = (const uint8_t*)(ws + L.q);
        a.q_scale = (const float*)(ws + L.q_scale);
        a.in_ids = (const int64_t*)(ws + L.ids);
        a.in_weights = b.weight;
        if ((rc = int8_route_launch(m, b.weight, (int64_t*)(ws + L.ids), (uint8_t*)(ws + L.q), a.kp, (float*)(ws + L.q_scale), s))) return rc;
        a.logits = nullptr;
        a.out_weights = nullptr;
        a.out_ids = nullptr;
    }
    if (m.hidden_dtype == QMOE_DT_F32) rc = front8_waves<QMOE_DT_F32>(a, grid, lds, s);
    else if (m.hidden_dtype == QMOE_DT_F16) rc = front8_waves<QMOE_DT_F16>(a, grid, lds, s);
    else rc = front8_waves<QMOE_DT_BF16>(a, grid, lds, s);
    if (rc) return rc;
    Back8Args q{};
    q.in = b; q.tokens = t; q.k = k; q.d = d; q.f = f; q.fp = (int)int8_cols64(f); q.f_tiles = a.f_tiles; q.f_steps = q.fp / 64;
    q.fs = fs; q.fsp = (int)int8_cols64(fs); q.fs_tiles = a.fs_tiles; q.fs_steps = fs ? q.fsp / 64 : 0;
    q.down = (const uint8_t*)m.down; q.down_c = m.down_scales; q.s_down = (const uint8_t*)m.shared_down_w; q.s_down_c = m.shared_down_scales;
    q.residual = m.residual; q.out = m.out; q.odt = m.out_dtype; q.gated = a.admit_w != nullptr;
    q.h_magic = magic_of((q.fp + 511) / 512); q.s_magic = magic_of((q.fsp + 511) / 512);
    q.hp_magic = magic_of(q.f_steps * 4); q.sp_magic = magic_of(q.fs_steps * 4);
    if (t <= STEP8_FUSED) return back8_as<false>(q, s);
    hipLaunchKernelGGL(int8_hidden_codes_kernel, dim3(t * k + (fs ? t : 0)), dim3(256), 0, s, q);
    if ((rc = check_launch("int8 expert step (codes)"))) return rc;
    return back8_as<true>(q, s);
}

}  // namespace qmoe
