// tree_attn.hip -- attention of every sequence's drafted tokens over a paged KV cache.
#include <algorithm>

#include "paged.h"

using namespace rl;

namespace {

constexpr int kMaxGroup = 64;  // query heads per kv head

struct TreeArgs {
    const void *q, *gate;
    int64_t q_row, q_head, g_row, g_head;
    const void *k, *v;
    const int *table, *ctx_lens, *row_start;
    const uint64_t* mask;
    int words, width, n_seq, rows, max_rows;
    int nq, nkv, page, n_pages;
    float scale;
    void* out;
};

__device__ inline float sigmoid(float x) { return 1.f / (1.f + expf(-x)); }

// One workgroup per (row, query head); each of its 4 waves takes every fourth position with a
// running maximum and sum, lanes over the head's dims; the waves' parts are joined at the end.
template <class R, int HD>
__global__ __launch_bounds__(256) void tree_attn_simple_kernel(TreeArgs p) {
    using T = typename R::T;
    using C = typename R::C;
    constexpr int E = HD / 64;
    const int row = blockIdx.x, head = blockIdx.y, kv = head / (p.nq / p.nkv);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int b = 0;
    SeqSpan s{};
    for (; b < p.n_seq; ++b) {
        s = seq_span(p.row_start, p.ctx_lens, b, p.rows, static_cast<int64_t>(p.width) * p.page);
        if (row >= s.r0 && row < s.r0 + min(s.n, p.max_rows)) break;
    }
    if (b == p.n_seq) return;
    s.n = min(s.n, p.max_rows);
    const int j = row - s.r0;
    float q[E], o[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
        q[e] = static_cast<float>(static_cast<const T*>(p.q)[row * p.q_row + head * p.q_head + lane * E + e]);
        o[e] = 0.f;
    }
    float m = -INFINITY, l = 0.f;
    for (int pos = wave; pos < s.ctx + s.n; pos += 4) {
        const int i = pos - s.ctx;
        if (i >= 0) {
            const bool sees = p.mask ? i / 64 < p.words && (p.mask[static_cast<size_t>(row) * p.words + i / 64] >> (i & 63) & 1)
                                     : i <= j;
            if (!sees) continue;
        }
        int pg = p.table[static_cast<size_t>(b) * p.width + pos / p.page];
        if (pg < 0 || pg >= p.n_pages) pg = 0;
        const size_t at = ((static_cast<size_t>(pg) * p.nkv + kv) * p.page + pos % p.page) * HD + lane * E;
        const C* kr = static_cast<const C*>(p.k) + at;
        const C* vr = static_cast<const C*>(p.v) + at;
        float x = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) x += q[e] * static_cast<float>(kr[e]);
        x = wave_sum(x) * p.scale;
        const float mn = fmaxf(m, x);
        const float a = m == -INFINITY ? 0.f : expf(m - mn), w = expf(x - mn);
        m = mn;
        l = l * a + w;
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = o[e] * a + w * static_cast<float>(vr[e]);
    }
    __shared__ float ms[4], ls[4], os[4][HD];
    if (lane == 0) {
        ms[wave] = m;
        ls[wave] = l;
    }
#pragma unroll
    for (int e = 0; e < E; ++e) os[wave][lane * E + e] = o[e];
    __syncthreads();
    if (threadIdx.x >= HD) return;
    const int d = threadIdx.x;
    const float M = fmaxf(fmaxf(ms[0], ms[1]), fmaxf(ms[2], ms[3]));
    float L = 0.f, O = 0.f;
    for (int w = 0; w < 4; ++w) {
        if (ls[w] == 0.f) continue;
        const float f = expf(ms[w] - M);
        L += f * ls[w];
        O += f * os[w][d];
    }
    O = L == 0.f ? 0.f : O / L;
    if (p.gate) O *= sigmoid(static_cast<float>(static_cast<const T*>(p.gate)[row * p.g_row + head * p.g_head + d]));
    static_cast<T*>(p.out)[(static_cast<size_t>(row) * p.nq + head) * HD + d] = static_cast<T>(O);
}

size_t tree_attn_workspace_bytes(int nq, int nkv, int hd, int n_seq, int max_rows) {
    (void)nq, (void)nkv, (void)hd, (void)n_seq, (void)max_rows;
    return 256;
}

template <class R>
void launch_simple(const TreeArgs& p, int hd, hipStream_t s) {
    const dim3 grid(p.rows, p.nq);
    switch (hd) {
    case 64: hipLaunchKernelGGL((tree_attn_simple_kernel<R, 64>), grid, dim3(256), 0, s, p); break;
    case 128: hipLaunchKernelGGL((tree_attn_simple_kernel<R, 128>), grid, dim3(256), 0, s, p); break;
    default: hipLaunchKernelGGL((tree_attn_simple_kernel<R, 256>), grid, dim3(256), 0, s, p); break;
    }
    check_launch("tree_attn_simple_kernel");
}

void tree_attn(const RlPagedCache* c, int layer, int dtype, const void* q, int64_t q_row, int64_t q_head, const void* gate,
               int64_t gate_row, int64_t gate_head, const int* table, int width, const int* ctx_lens,
               const int* row_start, int n_seq, int rows, int max_rows, const uint64_t* mask, int words, int nq,
               float scale, void* out, void* ws, size_t ws_bytes, hipStream_t s) {
    check_cache(c, layer, "tree_attn");
    check_rows_type(c, dtype, "tree_attn");
    RL_REQUIRE(rows >= 0 && n_seq >= 0 && max_rows >= 0, RL_ERR_RANGE, "tree_attn: bad sizes");
    RL_REQUIRE(nq >= 1 && nq % c->n_kv == 0 && nq / c->n_kv <= kMaxGroup, RL_ERR_RANGE,
               "tree_attn: n_q must be a multiple of n_kv, at most 64 per kv head");
    RL_REQUIRE(width >= 1 && static_cast<int64_t>(width) * c->page_size <= INT32_MAX, RL_ERR_RANGE,
               "tree_attn: bad table width");
    RL_REQUIRE(!mask || words >= 1, RL_ERR_RANGE, "tree_attn: a mask needs words");
    RL_REQUIRE(scale > -INFINITY && scale < INFINITY, RL_ERR_RANGE, "tree_attn: bad scale");
    if (rows == 0 || n_seq == 0 || max_rows == 0) return;
    RL_REQUIRE(q && table && ctx_lens && row_start && out && ws, RL_ERR_RANGE, "tree_attn: null pointer");
    check_strided(q, q_row, q_head, dtype, "tree_attn");
    if (gate) check_strided(gate, gate_row, gate_head, dtype, "tree_attn");
    RL_REQUIRE(aligned(out, 16), RL_ERR_RANGE, "tree_attn: out must be 16-byte aligned");
    RL_REQUIRE(ws_bytes >= tree_attn_workspace_bytes(nq, c->n_kv, c->head_dim, n_seq, max_rows), RL_ERR_RANGE,
               "tree_attn: workspace too small");
    TreeArgs p{};
    p.q = q, p.gate = gate;
    p.q_row = q_row, p.q_head = q_head, p.g_row = gate_row, p.g_head = gate_head;
    p.k = static_cast<const uint16_t*>(c->k) + layer * c->layer_stride;
    p.v = static_cast<const uint16_t*>(c->v) + layer * c->layer_stride;
    p.table = table, p.ctx_lens = ctx_lens, p.row_start = row_start;
    p.mask = mask, p.words = words, p.width = width;
    p.n_seq = n_seq, p.rows = rows, p.max_rows = max_rows;
    p.nq = nq, p.nkv = c->n_kv, p.page = c->page_size, p.n_pages = c->n_pages;
    p.scale = scale, p.out = out;
    if (dtype == RL_Q_F32)
        launch_simple<RowF32>(p, c->head_dim, s);
    else if (dtype == RL_Q_F16)
        launch_simple<RowF16>(p, c->head_dim, s);
    else
        launch_simple<RowBF16>(p, c->head_dim, s);
}

}  // namespace

extern "C" {

size_t rl_hip_tree_attn_workspace_bytes(int n_q, int n_kv, int head_dim, int n_seq, int max_rows) {
    return tree_attn_workspace_bytes(n_q, n_kv, head_dim, n_seq, max_rows);
}

int rl_hip_tree_attn(const RlPagedCache* cache, int layer, int dtype, const void* q, int64_t q_row, int64_t q_head,
                     const void* gate, int64_t gate_row, int64_t gate_head, const int* table, int table_width,
                     const int* ctx_lens, const int* row_start, int n_seq, int rows, int max_rows,
                     const uint64_t* mask, int mask_words, int n_q, float scale, void* out, void* workspace,
                     size_t workspace_bytes, void* stream) {
    return guard([&] {
        tree_attn(cache, layer, dtype, q, q_row, q_head, gate, gate_row, gate_head, table, table_width, ctx_lens, row_start,
                  n_seq, rows, max_rows, mask, mask_words, n_q, scale, out, workspace, workspace_bytes, S(stream));
    });
}

}  // extern "C"
