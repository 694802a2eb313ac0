// Mixture-of-experts step on 8-bit integer weights: router, token->expert plan, gate/up + SwiGLU, down projection,
// shared expert and the ordered combine.
//
// A step over T tokens, k experts each (A = T k assignments):
//   (q, s) = codes of the hidden rows;  h = fl32(silu(g) u) per assignment;  (hq, hs) = codes of h;
//   term = down;  out[t] = residual + (((0 + w_1 term_1) + w_2 term_2) + ... + sigmoid(x . gate) shared), experts
//   in ascending id, each product rounded before it is added.
#include "qmoe_int8.hpp"

namespace qmoe {

int int8_product_launch(const Int8Product& a, bool pair, int chunks, hipStream_t s);
int router_topk_impl(const float* logits, int tokens, int n, int k, float floor_value, int renorm, float* weights, int64_t* ids,
                     hipStream_t s);

bool int8_step_covers(int tokens, int k, int n_experts, int d, int f, int fs);
size_t int8_step_bytes(int tokens, int k, int f, int fs);
int int8_step_launch(const qmoe_int8_moe_args& m, char* ws, hipStream_t s);

static constexpr int PLAN8_THREADS = 256;
static constexpr int PLAN8_GRID = 64;
static constexpr int INT8_CHUNK = 16;         // sorted positions of one expert that a product takes at a time

// ---- plan ------------------------------------------------------------------------------------------------
// Whether assignment a counts: its id lies in the bank and no earlier slot of its token names it.
__device__ __forceinline__ int plan_fault(const int64_t* ids, int64_t a, int k, int n_experts) {
    const int64_t e = ids[a];
    if (e < 0 || e >= n_experts) return 1;
    for (int64_t j = a - a % k; j < a; ++j)
        if (ids[j] == e) return 2;
    return 0;
}

// Every workgroup counts all assignments (LDS integer adds: the order does not matter), turns the counts into
// positions and chunks, and ranks the assignments of its own experts, one wave an expert: ascending position is
// ascending token.  No workgroup waits for another and the number of tokens is not bounded by a table.
__global__ __launch_bounds__(PLAN8_THREADS) void int8_plan_kernel(const int64_t* __restrict__ ids, int assignments, int k, int n_experts,
                                                                  int* __restrict__ row_of, int* __restrict__ pos_of,
                                                                  int* __restrict__ chunk_expert, int* __restrict__ chunk_start,
                                                                  int* __restrict__ chunk_count, int* __restrict__ n_chunks,
                                                                  int* __restrict__ status_out) {
    extern __shared__ int count[];               // [experts] counts, [experts] starts, [experts] first chunks
    __shared__ int part[2][PLAN8_THREADS];
    int* const start = count + n_experts;
    int* const chunk0 = start + n_experts;
    const int tid = threadIdx.x, lane = tid & 63;
    for (int e = tid; e < n_experts; e += PLAN8_THREADS) count[e] = 0;
    __syncthreads();
    int bad = 0;
    for (int64_t a = tid; a < assignments; a += PLAN8_THREADS) {
        const int f = plan_fault(ids, a, k, n_experts);
        bad |= f;
        if (!f) atomicAdd(&count[ids[a]], 1);
        else if (blockIdx.x == 0) pos_of[a] = -1;
    }
    if (bad && blockIdx.x == 0 && status_out) atomicOr(status_out, bad);
    __syncthreads();
    const int per = (n_experts + PLAN8_THREADS - 1) / PLAN8_THREADS;
    int sum = 0, chunks = 0;
    for (int e = tid * per; e < (tid + 1) * per && e < n_experts; ++e) {
        sum += count[e];
        chunks += (count[e] + INT8_CHUNK - 1) / INT8_CHUNK;
    }
    part[0][tid] = sum;
    part[1][tid] = chunks;
    __syncthreads();
    if (tid < 2) {
        int run = 0;
        for (int i = 0; i < PLAN8_THREADS; ++i) { const int c = part[tid][i]; part[tid][i] = run; run += c; }
        if (tid == 1 && blockIdx.x == 0) *n_chunks = run;
    }
    __syncthreads();
    sum = part[0][tid];
    chunks = part[1][tid];
    for (int e = tid * per; e < (tid + 1) * per && e < n_experts; ++e) {
        start[e] = sum;
        chunk0[e] = chunks;
        sum += count[e];
        chunks += (count[e] + INT8_CHUNK - 1) / INT8_CHUNK;
    }
    __syncthreads();
    for (int e = blockIdx.x * (PLAN8_THREADS / 64) + (tid >> 6); e < n_experts; e += gridDim.x * (PLAN8_THREADS / 64)) {
        const int c = count[e], s0 = start[e];
        if (!c) continue;
        for (int i = lane; i * INT8_CHUNK < c; i += 64) {
            chunk_expert[chunk0[e] + i] = e;
            chunk_start[chunk0[e] + i] = s0 + i * INT8_CHUNK;
            chunk_count[chunk0[e] + i] = c - i * INT8_CHUNK < INT8_CHUNK ? c - i * INT8_CHUNK : INT8_CHUNK;
        }
        int at = s0;
        for (int64_t a0 = 0; a0 < assignments && at < s0 + c; a0 += 64) {
            const int64_t a = a0 + lane;
            const bool mine = a < assignments && ids[a] == e && !plan_fault(ids, a, k, n_experts);
            const unsigned long long m = __ballot(mine);
            if (mine) {
                const int p = at + __popcll(m & ((1ull << lane) - 1));
                row_of[p] = (int)(a / k);
                pos_of[a] = p;
            }
            at += __popcll(m);
        }
    }
}

__global__ __launch_bounds__(256) void int8_routing_copy_kernel(const float* __restrict__ w, const int64_t* __restrict__ ids, int64_t n,
                                                                float* __restrict__ out_w, int64_t* __restrict__ out_ids) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        if (out_w && out_w != w) out_w[i] = w[i];
        if (out_ids && out_ids != ids) out_ids[i] = ids[i];
    }
}

// ---- combine ----------------------------------------------------------------------------------------------
template <int XDT>
__global__ __launch_bounds__(256) void int8_combine_kernel(const float* __restrict__ terms, const int* __restrict__ pos_of,
                                                           const float* __restrict__ weights, int k, int d,
                                                           const float* __restrict__ shared_out, const float* __restrict__ shared_gate,
                                                           const void* __restrict__ x, const float* __restrict__ residual,
                                                           void* __restrict__ out, int odt) {
    __shared__ int pos[32];
    __shared__ float weight[32], partial[4];
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
    float admit = 1.0f;
    if (shared_out && shared_gate) {
        float a = 0.0f;
        for (int i = tid; i < d; i += 256) a += Elem<XDT>::load(x, (size_t)t * d + i) * shared_gate[i];
        a = wave_sum(a);
        if ((tid & 63) == 0) partial[tid >> 6] = a;
        __syncthreads();
        a = (partial[0] + partial[1]) + (partial[2] + partial[3]);
        admit = a >= 0.0f ? 1.0f / (1.0f + expf(-a)) : expf(a) / (1.0f + expf(a));
    }
    __syncthreads();
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
    w.max_chunks = (int)(a / INT8_CHUNK + (a < (size_t)n_experts ? a : (size_t)n_experts));
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
    return int8_step_covers(tokens, k, n_experts, d, f, fs) ? int8_step_bytes(tokens, k, f, fs)
                                                             : int8_moe_layout(tokens, k, n_experts, d, f, fs).total;
}

static int int8_moe_impl(const qmoe_int8_moe_args& m, char* ws, const Int8MoeLayout& L, hipStream_t s) {
    const int t = m.tokens, k = m.top_k, e = m.n_experts, d = m.d_model, f = m.d_ff, fs = m.d_ff_shared;
    const int a = t * k;
    const float* weights = m.in_weights;
    const int64_t* ids = m.in_ids;
    int rc;
    if (m.logits) {
        float* const wout = m.out_weights ? m.out_weights : (float*)(ws + L.weights);
        int64_t* const iout = m.out_ids ? m.out_ids : (int64_t*)(ws + L.ids);
        if ((rc = router_topk_impl(m.logits, t, e, k, m.floor_value, m.renormalize, wout, iout, s))) return rc;
        weights = wout;
        ids = iout;
    } else if (m.out_weights || m.out_ids) {
        hipLaunchKernelGGL(int8_routing_copy_kernel, dim3((a + 255) / 256 < 1024 ? (a + 255) / 256 : 1024), dim3(256), 0, s, weights, ids,
                           (int64_t)a, m.out_weights, m.out_ids);
        if ((rc = check_launch("int8 routing copy"))) return rc;
    }
    // the sorted arrays behind dropped assignments are never read: chunks cover kept positions only
    hipLaunchKernelGGL(int8_plan_kernel, dim3(PLAN8_GRID), dim3(PLAN8_THREADS), (size_t)e * 12, s, ids, a, k, e, (int*)(ws + L.row_of),
                       (int*)(ws + L.pos_of), (int*)(ws + L.chunk_expert), (int*)(ws + L.chunk_start), (int*)(ws + L.chunk_count),
                       (int*)(ws + L.n_chunks), m.status_out);
    if ((rc = check_launch("int8 plan"))) return rc;
    const int64_t dp = int8_cols256(d), fp = int8_cols256(f);
    if ((rc = int8_quantize_launch(m.hidden, m.hidden_dtype, t, d, (uint8_t*)(ws + L.q), dp, true, (float*)(ws + L.s), s))) return rc;
    Int8Product p{};
    p.w = (const uint8_t*)m.gate; p.w2 = (const uint8_t*)m.up; p.c = m.gate_scales; p.c2 = m.up_scales;
    p.n = f; p.kp = (int)int8_cols64(d); p.w_step = int8_matrix_bytes(f, d);
    p.q = (const uint8_t*)(ws + L.q); p.ld = dp; p.s = (const float*)(ws + L.s);
    p.y = ws + L.h; p.ydt = QMOE_DT_F32; p.ldy = f; p.hidden = 1; p.tokens = t;
    p.chunk_expert = (const int*)(ws + L.chunk_expert); p.chunk_start = (const int*)(ws + L.chunk_start);
    p.chunk_count = (const int*)(ws + L.chunk_count); p.n_chunks = (const int*)(ws + L.n_chunks);
    p.row_of = (const int*)(ws + L.row_of);
    if ((rc = int8_product_launch(p, true, L.max_chunks, s))) return rc;
    if ((rc = int8_quantize_launch(ws + L.h, QMOE_DT_F32, a, f, (uint8_t*)(ws + L.hq), fp, true, (float*)(ws + L.hs), s))) return rc;
    Int8Product q = p;
    q.w = (const uint8_t*)m.down; q.c = m.down_scales; q.n = d; q.kp = (int)int8_cols64(f); q.w_step = int8_matrix_bytes(d, f);
    q.q = (const uint8_t*)(ws + L.hq); q.ld = fp; q.s = (const float*)(ws + L.hs); q.y = ws + L.terms; q.ldy = d; q.hidden = 0;
    q.row_of = nullptr;
    if ((rc = int8_product_launch(q, false, L.max_chunks, s))) return rc;
    if (fs) {
        const int64_t fsp = int8_cols256(fs);
        Int8Product g{};
        g.w = (const uint8_t*)m.shared_gate_w; g.w2 = (const uint8_t*)m.shared_up_w; g.c = m.shared_gate_scales; g.c2 = m.shared_up_scales;
        g.n = fs; g.kp = p.kp; g.q = p.q; g.ld = dp; g.s = p.s; g.tokens = t; g.y = ws + L.sh; g.ydt = QMOE_DT_F32; g.ldy = fs; g.hidden = 1;
        if ((rc = int8_product_launch(g, true, 0, s))) return rc;
        if ((rc = int8_quantize_launch(ws + L.sh, QMOE_DT_F32, t, fs, (uint8_t*)(ws + L.shq), fsp, true, (float*)(ws + L.shs), s))) return rc;
        Int8Product o{};
        o.w = (const uint8_t*)m.shared_down_w; o.c = m.shared_down_scales; o.n = d; o.kp = (int)int8_cols64(fs);
        o.q = (const uint8_t*)(ws + L.shq); o.ld = fsp; o.s = (const float*)(ws + L.shs); o.tokens = t; o.y = ws + L.shared_out;
        o.ydt = QMOE_DT_F32; o.ldy = d;
        if ((rc = int8_product_launch(o, false, 0, s))) return rc;
    }
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
    if ((int64_t)m.tokens * m.top_k > INT32_MAX / 2) return fail(QMOE_EUNSUPPORTED, "%s: too many assignments; split the tokens", who);
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
