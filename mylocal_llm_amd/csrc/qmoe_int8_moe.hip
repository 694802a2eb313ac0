// Mixture-of-experts step on 8-bit integer weights: router, token->expert plan, gate/up + SwiGLU, down projection,
// shared expert and the ordered combine.
//
// A step over T tokens, k experts each (A = T k assignments):
//   (q, s) = codes of the hidden rows;  h = fl32(silu(g) u) per assignment;  (hq, hs) = codes of h;
//   term = down;  out[t] = residual + (((0 + w_1 term_1) + w_2 term_2) + ... + sigmoid(x . gate) shared), experts
//   in ascending id, each product rounded before it is added.
#include "qmoe_int8_route.hpp"

namespace qmoe {

bool int8_step_covers(int tokens, int k, int n_experts, int d, int f, int fs);
size_t int8_step_bytes(int tokens, int k, int d, int f, int fs);
int int8_step_launch(const qmoe_int8_moe_args& m, char* ws, hipStream_t s);

static constexpr int PLAN8_THREADS = 1024;
static constexpr int PLAN8_MIN_ROWS = 32;     // of a chunk (the workspace is laid out for the most chunks there can be)

// ---- routing and codes of a prompt: a workgroup a token, its first wave routes ---------------------------------
// The other four waves cut the token's row into codes meanwhile: one launch, one round trip each.  512 tokens, 512 experts,
// 2048 fp32 columns: 6.8 us (logits 1 MB, rows 4 MB: what the routing's chain of selections takes, not the bytes).
template <int XDT, int NV>
__global__ __launch_bounds__(320) void int8_route_kernel(const void* __restrict__ x, int d, int fast, const float* __restrict__ logits,
                                                         int n_experts, int k, float floor_value, int renorm,
                                                         const float* __restrict__ in_weights, const int64_t* __restrict__ in_ids,
                                                         float* __restrict__ weights, int64_t* __restrict__ ids, float* __restrict__ out_weights,
                                                         int64_t* __restrict__ out_ids, uint8_t* __restrict__ codes, int64_t ld,
                                                         float* __restrict__ scales) {
    __shared__ uint32_t tops[4];
    const int64_t t = blockIdx.x;
    const int lane = threadIdx.x & 63, tid = (int)threadIdx.x - 64;
    float v[8];
    uint32_t top = 0;
    if (tid < 0) {
        float w = 0.0f;
        int64_t id = 0;
        const float* const z = logits + t * n_experts;
        if (logits && NV <= 16) {
            __shared__ uint2 scratch[64];
            RowIds<NV <= 16 ? NV : 16> row;
            row.load(z, n_experts);
            row.route(z, n_experts, k, floor_value, renorm, scratch, w, id);
        } else if (logits) router_row<NV>(z, n_experts, k, floor_value, renorm, w, id, [] {});
        else if (lane < k) {
            w = ldg<float>(in_weights + t * k + lane);
            id = ldg<int64_t>(in_ids + t * k + lane);
        }
        if (lane < k) {
            stg<float>(weights + t * k + lane, w);
            stg<int64_t>(ids + t * k + lane, id);
            if (out_weights) stg<float>(out_weights + t * k + lane, w);
            if (out_ids) stg<int64_t>(out_ids + t * k + lane, id);
        }
    } else {
        for (int i = tid * 8; i < d; i += 2048) {       // (the first 2048 columns stay in registers)
            float u[8];
            int8_load8<XDT>(x, (size_t)t * d + i, d - i, fast, u);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const uint32_t b = abs_bits(u[j]);
                top = b > top ? b : top;
                if (i < 2048) v[j] = u[j];
            }
        }
        top = wave_max_u32(top);
        if (lane == 0) tops[tid >> 6] = top;
    }
    __syncthreads();
    if (tid < 0) return;
#pragma unroll
    for (int i = 0; i < 4; ++i) top = tops[i] > top ? tops[i] : top;
    const RowScale r(top);
    if (tid == 0) stg<float>(scales + t, r.s);
    for (int i = tid * 8; i < ld; i += 2048) {
        float u[8];
        if (i >= 2048 || i >= d) int8_load8<XDT>(x, i < d ? (size_t)t * d + i : (size_t)t * d, d - i, fast, u);
        else {
#pragma unroll
            for (int j = 0; j < 8; ++j) u[j] = v[j];
        }
        *(QMOE_GLOBAL u32x2_t*)(codes + t * ld + i) = int8_code8(u, r);
    }
}

// weights / ids of every token (also to the caller's arrays), codes with row step ld (a multiple of 8, the tail zero) + scales
int int8_route_launch(const qmoe_int8_moe_args& m, float* weights, int64_t* ids, uint8_t* codes, int64_t ld, float* scales, hipStream_t s) {
    const int t = m.tokens, k = m.top_k, e = m.n_experts, d = m.d_model;
    const int fast = (uintptr_t)m.hidden % 16 == 0 && d % 8 == 0;
#define QMOE_INT8_ROUTE(DT)                                                                                                              \
    hipLaunchKernelGGL((e <= 512 ? int8_route_kernel<DT, 8> : e <= 1024 ? int8_route_kernel<DT, 16> : int8_route_kernel<DT, 64>), dim3(t), dim3(320), 0, s, m.hidden, d, fast, \
                       m.logits, e, k, m.floor_value, m.renormalize, m.in_weights, m.in_ids, weights, ids, m.out_weights, m.out_ids,     \
                       codes, ld, scales)
    if (m.hidden_dtype == QMOE_DT_F32) QMOE_INT8_ROUTE(QMOE_DT_F32);
    else if (m.hidden_dtype == QMOE_DT_F16) QMOE_INT8_ROUTE(QMOE_DT_F16);
    else QMOE_INT8_ROUTE(QMOE_DT_BF16);
#undef QMOE_INT8_ROUTE
    return check_launch("int8 expert step (routing)");
}

// ---- plan ------------------------------------------------------------------------------------------------
// One workgroup groups the assignments by expert.  The place of an assignment inside its expert is the order in which the
// adds to the expert's counter happened: it may differ from run to run, and no result depends on it, since a row's
// products do not depend on its neighbours.  An assignment counts if its id lies in the bank and no earlier slot of its token
// names it; the others get the position -1 and are reported.  Bound by its chain of steps (adds in LDS, prefix, places), one
// workgroup: 5120 assignments to 512 experts 7.0 us.
__global__ __launch_bounds__(PLAN8_THREADS) void int8_plan_kernel(const int64_t* __restrict__ ids, int assignments, int k, int n_experts,
                                                                  int rows, int check, int* __restrict__ row_of, int* __restrict__ pos_of,
                                                                  int* __restrict__ chunk_expert, int* __restrict__ chunk_start,
                                                                  int* __restrict__ chunk_count, int* __restrict__ n_chunks,
                                                                  int* __restrict__ status_out) {
    extern __shared__ int count[];               // [experts] counts, [experts] starts
    __shared__ int part[2][PLAN8_THREADS / 64];
    int* const start = count + n_experts;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    for (int e = tid; e < n_experts; e += PLAN8_THREADS) count[e] = 0;
    __syncthreads();
    int bad = 0;
    // the expert and the rank of this thread's first assignments stay in registers, the others' ranks lie in pos_of meanwhile
    constexpr int NR = 8;
    int mine[NR], rank[NR];
    auto count_in = [&](int a, int64_t e) -> int {
        int fault = 0;
        if (check) {                             // (the router's own ids are in the bank and no token has one twice)
            fault = e < 0 || e >= n_experts ? 1 : 0;
            for (int j = a / k * k; j < a; ++j) fault |= ldg<int64_t>(ids + j) == e ? 2 : 0;
            if (fault & 1) fault = 1;
            bad |= fault;
        }
        return fault ? -1 : atomicAdd(&count[e], 1);
    };
#pragma unroll
    for (int j = 0; j < NR; ++j) {
        const int a = tid + j * PLAN8_THREADS;
        mine[j] = 0;
        rank[j] = -1;
        if (j * PLAN8_THREADS < assignments) {
            const int64_t e = ldg<int64_t>(ids + (a < assignments ? a : 0));
            if (a < assignments) rank[j] = count_in(a, e);
            mine[j] = rank[j] < 0 ? 0 : (int)e;
        }
    }
    for (int a = tid + NR * PLAN8_THREADS; a < assignments; a += PLAN8_THREADS) pos_of[a] = count_in(a, ldg<int64_t>(ids + a));
    if (bad && status_out) atomicOr(status_out, bad);
    __syncthreads();
    const int per = (n_experts + PLAN8_THREADS - 1) / PLAN8_THREADS, e0 = tid * per;
    int sum = 0, chunks = 0;
    for (int e = e0; e < e0 + per && e < n_experts; ++e) { sum += count[e]; chunks += (count[e] + rows - 1) / rows; }
    int upto = sum, cupto = chunks;              // inclusive, then exclusive prefix
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const int o = __shfl_up(upto, off, 64), c = __shfl_up(cupto, off, 64);
        if (lane >= off) { upto += o; cupto += c; }
    }
    if (lane == 63) { part[0][wave] = upto; part[1][wave] = cupto; }
    __syncthreads();
    upto -= sum;
    cupto -= chunks;
    for (int w = 0; w < wave; ++w) { upto += part[0][w]; cupto += part[1][w]; }
    if (tid == PLAN8_THREADS - 1) *n_chunks = cupto + chunks;
    for (int e = e0; e < e0 + per && e < n_experts; ++e) {
        start[e] = upto;
        for (int at = 0; at < count[e]; at += rows) {
            chunk_expert[cupto] = e;
            chunk_start[cupto] = upto + at;
            chunk_count[cupto++] = count[e] - at < rows ? count[e] - at : rows;
        }
        upto += count[e];
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < NR; ++j) {
        const int a = tid + j * PLAN8_THREADS;
        if (a >= assignments) break;
        const int p = rank[j] < 0 ? -1 : start[mine[j]] + rank[j];
        pos_of[a] = p;
        if (p >= 0) row_of[p] = a / k;
    }
    for (int a = tid + NR * PLAN8_THREADS; a < assignments; a += PLAN8_THREADS) {
        const int r = pos_of[a];                 // (written by this thread)
        if (r < 0) continue;
        const int p = start[ldg<int64_t>(ids + a)] + r;
        pos_of[a] = p;
        row_of[p] = a / k;
    }
}

// ---- hidden activations -> codes, the routed rows and the shared expert's in one launch, a workgroup a row ------------
// 5120 rows of 512 + 512 rows of 2048 fp32: 8.0 us, 2.2 TB/s -- short workgroups, of which a fifth only is traffic.
struct Int8Rows { const float* x; int wide; int64_t ld; uint8_t* codes; float* scales; };
__global__ __launch_bounds__(256) void int8_hidden_rows_kernel(const Int8Rows routed, int routed_rows, const Int8Rows shared) {
    __shared__ uint32_t tops[4];
    const bool sh = (int)blockIdx.x >= routed_rows;
    const Int8Rows& a = sh ? shared : routed;
    const int64_t r = sh ? (int)blockIdx.x - routed_rows : (int)blockIdx.x;
    const float* const x = a.x + r * a.wide;
    const int tid = threadIdx.x, wide = a.wide;
    const bool fast = wide % 8 == 0;
    float v[8];
    uint32_t top = 0;
    for (int i0 = 0; i0 < wide; i0 += 2048) {           // (the first 2048 values stay in registers)
        const int i = i0 + tid * 8;
        float u[8];
        int8_load8<QMOE_DT_F32>(x, i < wide ? i : 0, wide - i, fast, u);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const uint32_t b = abs_bits(u[j]);
            top = b > top ? b : top;
            if (!i0) v[j] = u[j];
        }
    }
    top = wave_max_u32(top);
    if ((tid & 63) == 0) tops[tid >> 6] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) top = tops[i] > top ? tops[i] : top;
    const RowScale rs(top);
    if (tid == 0) stg<float>(a.scales + r, rs.s);
    for (int i0 = 0; i0 < a.ld; i0 += 2048) {
        const int i = i0 + tid * 8;
        if (i0) int8_load8<QMOE_DT_F32>(x, i < wide ? i : 0, wide - i, fast, v);
        const u32x2_t q = int8_code8(v, rs);
        if (i < a.ld) *(QMOE_GLOBAL u32x2_t*)(a.codes + r * a.ld + i) = q;
    }
}

// ---- combine ----------------------------------------------------------------------------------------------
// A workgroup a token: terms in ascending position, which is ascending expert id, each product rounded before it is added.
// Bound by the memory: 512 tokens, ten terms of 2048 fp32, shared expert and residual in 15.9 us (54 MB, 3.4 TB/s; the admission
// gate's dot product goes in front of the first term).
template <int XDT>
__global__ __launch_bounds__(256) void int8_combine_kernel(const float* __restrict__ terms, const int* __restrict__ pos_of,
                                                           const float* __restrict__ weights, int k, int d,
                                                           const float* __restrict__ shared_out, const float* __restrict__ shared_gate,
                                                           const void* __restrict__ x, const float* __restrict__ residual,
                                                           void* __restrict__ out, int odt) {
    __shared__ int pos[32];
    __shared__ float weight[32], admitted;
    __shared__ int kept;
    const int64_t t = blockIdx.x;
    const int tid = threadIdx.x;
    if (tid < 64) {
        // ascending position is ascending expert id
        const int p = tid < k ? pos_of[t * k + tid] : -1;
        int rank = 0, n = 0;
        for (int j = 0; j < k; ++j) {
            const int o = __builtin_amdgcn_readlane(p, j);
            rank += o >= 0 && o < p;
            n += o >= 0;
        }
        if (p >= 0) { pos[rank] = p; weight[rank] = weights[t * k + tid]; }
        if (tid == 0) kept = n;
    }
    else if (tid < 128) {        // the second wave: the shared expert's admission
        const bool eights = d % 8 == 0;
        const float a = shared_out && shared_gate ? int8_admission<XDT>(x, (size_t)t * d, eights && (uintptr_t)x % 16 == 0, shared_gate,
                                                                          eights && (uintptr_t)shared_gate % 16 == 0, d) : 1.0f;
        if (tid == 64) admitted = a;
    }
    __syncthreads();
    const float admit = admitted;
    const bool wide = d % 4 == 0 && ((uintptr_t)x | (uintptr_t)shared_gate | (uintptr_t)residual | (uintptr_t)out) % 16 == 0;
    if (wide) {
        // four columns a thread; eight terms' requests leave together, the adds follow in order
        for (int i = 4 * tid; i < d; i += 1024) {
            float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int j0 = 0; j0 < kept; j0 += 8) {
                float4 v[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = ldg<float4>(terms + (size_t)pos[j0 + j < kept ? j0 + j : 0] * d + i);
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (j0 + j < kept) {
                        const float w = weight[j0 + j];
                        acc.x = add_product(acc.x, v[j].x, w); acc.y = add_product(acc.y, v[j].y, w);
                        acc.z = add_product(acc.z, v[j].z, w); acc.w = add_product(acc.w, v[j].w, w);
                    }
            }
            if (shared_out) {
                const float4 v = ldg<float4>(shared_out + (size_t)t * d + i);
                acc.x = add_product(acc.x, v.x, admit); acc.y = add_product(acc.y, v.y, admit);
                acc.z = add_product(acc.z, v.z, admit); acc.w = add_product(acc.w, v.w, admit);
            }
            if (residual) {
                const float4 r = ldg<float4>(residual + (size_t)t * d + i);
                acc.x = __fadd_rn(r.x, acc.x); acc.y = __fadd_rn(r.y, acc.y); acc.z = __fadd_rn(r.z, acc.z); acc.w = __fadd_rn(r.w, acc.w);
            }
            const float o[4] = {acc.x, acc.y, acc.z, acc.w};
            if (odt == QMOE_DT_F32) stg<float4>((float*)out + (size_t)t * d + i, acc);
            else
                for (int j = 0; j < 4; ++j) store_out(out, odt, (size_t)t * d + i + j, o[j]);
        }
        return;
    }
    for (int i = tid; i < d; i += 256) {
        float acc = 0.0f;
        for (int j = 0; j < kept; ++j) acc = add_product(acc, terms[(size_t)pos[j] * d + i], weight[j]);
        if (shared_out) acc = add_product(acc, shared_out[(size_t)t * d + i], admit);
        if (residual) acc = __fadd_rn(residual[(size_t)t * d + i], acc);
        store_out(out, odt, (size_t)t * d + i, acc);
    }
}

// ---- the step ----------------------------------------------------------------------------------------------
struct Int8MoeLayout {
    size_t weights, ids, row_of, pos_of, chunk_expert, chunk_start, chunk_count, n_chunks, q, s, h, hq, hs, terms, sh, shq, shs, shared_out, total;
    int max_chunks;
};
static Int8MoeLayout int8_moe_layout(int tokens, int k, int n_experts, int d, int f, int fs) {
    Int8MoeLayout w;
    size_t at = 0;
    const size_t a = (size_t)tokens * k, t = (size_t)tokens;
    auto take = [&](size_t bytes) { const size_t here = at; at = (at + bytes + 255) & ~(size_t)255; return here; };
    w.max_chunks = (int)(a / PLAN8_MIN_ROWS + (a < (size_t)n_experts ? a : (size_t)n_experts));
    w.weights = take(a * 4);
    w.ids = take(a * 8);
    w.row_of = take(a * 4);
    w.pos_of = take(a * 4);
    w.chunk_expert = take((size_t)w.max_chunks * 4);
    w.chunk_start = take((size_t)w.max_chunks * 4);
    w.chunk_count = take((size_t)w.max_chunks * 4);
    w.n_chunks = take(4);
    w.q = take(t * int8_cols256(d));
    w.s = take(t * 4);
    w.h = take(a * f * 4);
    w.hq = take(a * int8_cols256(f));
    w.hs = take(a * 4);
    w.terms = take(a * d * 4);
    w.sh = take(fs ? t * fs * 4 : 0);
    w.shq = take(fs ? t * int8_cols256(fs) : 0);
    w.shs = take(fs ? t * 4 : 0);
    w.shared_out = take(fs ? t * d * 4 : 0);
    w.total = at;
    return w;
}

static size_t int8_moe_bytes(int tokens, int k, int n_experts, int d, int f, int fs) {
    return int8_step_covers(tokens, k, n_experts, d, f, fs) ? int8_step_bytes(tokens, k, d, f, fs)
                                                             : int8_moe_layout(tokens, k, n_experts, d, f, fs).total;
}

static int int8_moe_impl(const qmoe_int8_moe_args& m, char* ws, const Int8MoeLayout& L, hipStream_t s) {
    const int t = m.tokens, k = m.top_k, e = m.n_experts, d = m.d_model, f = m.d_ff, fs = m.d_ff_shared;
    const int a = t * k;
    int rc;
    float* const weights = (float*)(ws + L.weights);
    int64_t* const ids = (int64_t*)(ws + L.ids);
    const int64_t dp = int8_cols256(d), fp = int8_cols256(f);
    if ((rc = int8_route_launch(m, weights, ids, (uint8_t*)(ws + L.q), dp, (float*)(ws + L.s), s))) return rc;
    const int rows = int8_plan_rows(a, e);
    hipLaunchKernelGGL(int8_plan_kernel, dim3(1), dim3(PLAN8_THREADS), (size_t)e * 8, s, ids, a, k, e, rows, m.logits ? 0 : 1, (int*)(ws + L.row_of),
                       (int*)(ws + L.pos_of), (int*)(ws + L.chunk_expert), (int*)(ws + L.chunk_start), (int*)(ws + L.chunk_count),
                       (int*)(ws + L.n_chunks), m.status_out);
    if ((rc = check_launch("int8 expert step (plan)"))) return rc;
    const int max_chunks = (int)(a / rows + (a < e ? a : e));
    Int8Product p{};
    p.w = (const uint8_t*)m.gate; p.w2 = (const uint8_t*)m.up; p.c = m.gate_scales; p.c2 = m.up_scales;
    p.n = f; p.kp = (int)int8_cols64(d); p.w_step = int8_matrix_bytes(f, d);
    p.q = (const uint8_t*)(ws + L.q); p.ld = dp; p.s = (const float*)(ws + L.s);
    p.y = ws + L.h; p.ydt = QMOE_DT_F32; p.ldy = f; p.tokens = t;
    p.chunk_expert = (const int*)(ws + L.chunk_expert); p.chunk_start = (const int*)(ws + L.chunk_start);
    p.chunk_count = (const int*)(ws + L.chunk_count); p.n_chunks = (const int*)(ws + L.n_chunks);
    p.row_of = (const int*)(ws + L.row_of);
    const int64_t fsp = int8_cols256(fs);
    Int8Product g{};
    if (fs) {
        g.w = (const uint8_t*)m.shared_gate_w; g.w2 = (const uint8_t*)m.shared_up_w; g.c = m.shared_gate_scales; g.c2 = m.shared_up_scales;
        g.n = fs; g.kp = p.kp; g.q = p.q; g.ld = dp; g.s = p.s; g.tokens = t; g.y = ws + L.sh; g.ydt = QMOE_DT_F32; g.ldy = fs;
    }
    if ((rc = int8_plan_launch(p, true, rows, max_chunks, fs ? &g : nullptr, s))) return rc;
    const Int8Rows routed{(const float*)(ws + L.h), f, fp, (uint8_t*)(ws + L.hq), (float*)(ws + L.hs)};
    const Int8Rows shared{(const float*)(ws + L.sh), fs, fsp, (uint8_t*)(ws + L.shq), (float*)(ws + L.shs)};
    hipLaunchKernelGGL(int8_hidden_rows_kernel, dim3(a + (fs ? t : 0)), dim3(256), 0, s, routed, a, shared);
    if ((rc = check_launch("int8 expert step (codes)"))) return rc;
    Int8Product q = p;
    q.w = (const uint8_t*)m.down; q.c = m.down_scales; q.n = d; q.kp = (int)int8_cols64(f); q.w_step = int8_matrix_bytes(d, f);
    q.q = (const uint8_t*)(ws + L.hq); q.ld = fp; q.s = (const float*)(ws + L.hs); q.y = ws + L.terms; q.ldy = d;
    q.row_of = nullptr;
    Int8Product o{};
    if (fs) {
        o.w = (const uint8_t*)m.shared_down_w; o.c = m.shared_down_scales; o.n = d; o.kp = (int)int8_cols64(fs);
        o.q = (const uint8_t*)(ws + L.shq); o.ld = fsp; o.s = (const float*)(ws + L.shs); o.tokens = t; o.y = ws + L.shared_out;
        o.ydt = QMOE_DT_F32; o.ldy = d;
    }
    if ((rc = int8_plan_launch(q, false, rows, max_chunks, fs ? &o : nullptr, s))) return rc;
#define QMOE_INT8_COMBINE(DT)                                                                                                       \
    hipLaunchKernelGGL(int8_combine_kernel<DT>, dim3(t), dim3(256), 0, s, (const float*)(ws + L.terms), (const int*)(ws + L.pos_of), \
                       weights, k, d, fs ? (const float*)(ws + L.shared_out) : nullptr, m.shared_gate, m.hidden, m.residual, m.out,  \
                       m.out_dtype)
    if (m.hidden_dtype == QMOE_DT_F32) QMOE_INT8_COMBINE(QMOE_DT_F32);
    else if (m.hidden_dtype == QMOE_DT_F16) QMOE_INT8_COMBINE(QMOE_DT_F16);
    else QMOE_INT8_COMBINE(QMOE_DT_BF16);
#undef QMOE_INT8_COMBINE
    return check_launch("int8 combine");
}

static int int8_moe_check(const qmoe_int8_moe_args& m) {
    const char* who = "qmoe_int8_moe_forward";
    if (!m.hidden || !m.out) return fail(QMOE_EINVAL, "%s: null hidden or output pointer", who);
    if (m.tokens < 0) return fail(QMOE_EINVAL, "%s: negative token count", who);
    if (!dtype_size(m.hidden_dtype) || !dtype_size(m.out_dtype)) return fail(QMOE_EINVAL, "%s: bad element type", who);
    if (m.n_experts < 1 || m.n_experts > 4096) return fail(QMOE_EUNSUPPORTED, "%s: expert count %d outside 1..4096", who, m.n_experts);
    if (m.top_k < 1 || m.top_k > 32 || m.top_k > m.n_experts)
        return fail(QMOE_EUNSUPPORTED, "%s: top_k=%d outside 1..min(32, experts)", who, m.top_k);
    if (m.d_model < 1 || m.d_ff < 1 || m.d_ff_shared < 0) return fail(QMOE_EINVAL, "%s: bank dimensions must be positive", who);
    if (m.d_model > INT8_MAX_K || m.d_ff > INT8_MAX_K || m.d_ff_shared > INT8_MAX_K)
        return fail(QMOE_EUNSUPPORTED, "%s: a width beyond %d, where an int32 sum could overflow", who, INT8_MAX_K);
    if ((int64_t)m.tokens * m.top_k > (1 << 22)) return fail(QMOE_EUNSUPPORTED, "%s: more than 2^22 assignments; split the tokens", who);
    const void* tiles[6] = {m.gate, m.up, m.down, m.shared_gate_w, m.shared_up_w, m.shared_down_w};
    const float* scales[6] = {m.gate_scales, m.up_scales, m.down_scales, m.shared_gate_scales, m.shared_up_scales, m.shared_down_scales};
    bool any = false;
    for (int i = 3; i < 6; ++i) any |= tiles[i] || scales[i];
    if (any != (m.d_ff_shared > 0)) return fail(QMOE_EINVAL, "%s: a shared expert needs its three matrices, their scales and d_ff_shared > 0", who);
    for (int i = 0; i < (any ? 6 : 3); ++i) {
        if (!tiles[i] || !scales[i]) return fail(QMOE_EINVAL, "%s: null weight or scale pointer", who);
        if ((uintptr_t)tiles[i] % 16 || (uintptr_t)scales[i] % 4) return fail(QMOE_EINVAL, "%s: misaligned weight or scale pointer", who);
    }
    if (!m.logits && !(m.in_weights && m.in_ids)) return fail(QMOE_EINVAL, "%s: need router logits or weights+ids", who);
    if (m.logits && m.renormalize && !(m.floor_value >= 1.17549435e-38f && m.floor_value <= 3.40282347e38f))
        return fail(QMOE_EINVAL, "%s: normalisation floor must be a finite positive normal float", who);
    if ((uintptr_t)m.hidden % dtype_size(m.hidden_dtype) || (uintptr_t)m.out % dtype_size(m.out_dtype) || (uintptr_t)m.logits % 4 ||
        (uintptr_t)m.in_weights % 4 || (uintptr_t)m.in_ids % 8 || (uintptr_t)m.out_weights % 4 || (uintptr_t)m.out_ids % 8 ||
        (uintptr_t)m.residual % 4 || (uintptr_t)m.shared_gate % 4 || (uintptr_t)m.status_out % 4)
        return fail(QMOE_EINVAL, "%s: misaligned pointer", who);
    return QMOE_OK;
}

}  // namespace qmoe

using namespace qmoe;

extern "C" {

size_t qmoe_int8_moe_workspace_bytes(int tokens, int top_k, int n_experts, int d_model, int d_ff, int d_ff_shared) {
    if (tokens < 0 || top_k < 1 || n_experts < 1 || d_model < 1 || d_ff < 1 || d_ff_shared < 0) return 0;
    return int8_moe_bytes(tokens, top_k, n_experts, d_model, d_ff, d_ff_shared);
}

int qmoe_int8_moe_forward(const qmoe_int8_moe_args* args, void* workspace, size_t workspace_bytes, void* stream) {
    const char* who = "qmoe_int8_moe_forward";
    if (!args) return fail(QMOE_EINVAL, "%s: null argument struct", who);
    if (const int rc = int8_moe_check(*args)) return rc;
    if (args->tokens == 0) return QMOE_OK;
    const qmoe_int8_moe_args& m = *args;
    const size_t need = int8_moe_bytes(m.tokens, m.top_k, m.n_experts, m.d_model, m.d_ff, m.d_ff_shared);
    if (!workspace || (uintptr_t)workspace % 256 || workspace_bytes < need)
        return fail(QMOE_EWORKSPACE, "%s: workspace must be 256-byte aligned and hold %zu bytes (got %zu)", who, need, workspace_bytes);
    if (int8_step_covers(m.tokens, m.top_k, m.n_experts, m.d_model, m.d_ff, m.d_ff_shared))
        return int8_step_launch(m, (char*)workspace, (hipStream_t)stream);
    return int8_moe_impl(m, (char*)workspace, int8_moe_layout(m.tokens, m.top_k, m.n_experts, m.d_model, m.d_ff, m.d_ff_shared), (hipStream_t)stream);
}

}  // extern "C"
