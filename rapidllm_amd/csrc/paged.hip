// paged.hip -- what a step writes into a paged KV cache: the append (norms of queries and keys,
// rotation, K / V into pages) and the acceptance of a verified tree.
#include <algorithm>

#include "paged.h"

using namespace rl;

namespace {

struct AppendArgs {
    const void *q, *k, *v;
    int64_t q_row, q_head, k_row, k_head, v_row, v_head;
    const float *q_norm, *k_norm;
    int norm, rot;
    float eps;
    double log2_theta;
    const int* pos;
    const int64_t* slots;
    int nq, nkv, page;
    int64_t n_slots;
    void *q_out, *kc, *vc;
};

// One workgroup per (row, part of its heads), HD / 4 lanes per head, so that the angles are formed once
// for many heads and every access is a run of 4 elements a lane.
// Bound by HBM from a few hundred rows on: 4096 rows of 24 / 4 heads of 256 in 32 bits, 251 MB in
// 55.5 us, 4.5 TB/s (a large copy: 4.8); below by one chain of loads: 1 row 4 us, 1013 rows of 32 / 8 heads
// of 128 in bf16 (25 MB) 12 us.  Asking for a workgroup's next heads ahead changed nothing (56 -> 60 us).
// y = x / sqrt(mean x^2 + eps) * (1 + gamma); (a, b) = dims (i, i + rot/2) turned by pos * theta^(-2i/rot).
template <class R, int HD>
__global__ __launch_bounds__(256) void paged_append_kernel(AppendArgs p) {
    using T = typename R::T;
    using C = typename R::C;
    constexpr int kLanes = HD / 4, kHeads = 256 / kLanes;
    __shared__ float2 cs[HD / 2];
    const int row = blockIdx.x, half = p.rot / 2;
    for (int i = threadIdx.x; i < half; i += 256) {
        // turns of the angle in 64 bits: far positions keep their fraction
        const double turns = p.pos[row] * exp2(-p.log2_theta * i / half) * 0.15915494309189535;
        const float f = static_cast<float>(2.0 * (turns - rint(turns)));
        float s, c;
        sincospif(f, &s, &c);
        cs[i] = make_float2(c, s);
    }
    __syncthreads();
    const int64_t slot = p.slots[row];
    const bool put = slot >= 0 && slot < p.n_slots;
    const size_t page = put ? slot / p.page : 0, in_page = put ? slot % p.page : 0;
    const int l = threadIdx.x % kLanes, d = 4 * l;
    const int items = p.nq + 2 * p.nkv;
    for (int h0 = blockIdx.y * kHeads; h0 < items; h0 += gridDim.y * kHeads) {
        const int item = h0 + threadIdx.x / kLanes;
        const bool on = item < items;
        const int kind = item < p.nq ? 0 : item < p.nq + p.nkv ? 1 : 2;
        const int head = kind == 0 ? item : kind == 1 ? item - p.nq : item - p.nq - p.nkv;
        const T* src = kind == 0 ? static_cast<const T*>(p.q) + row * p.q_row + head * p.q_head
                       : kind == 1 ? static_cast<const T*>(p.k) + row * p.k_row + head * p.k_head
                                   : static_cast<const T*>(p.v) + row * p.v_row + head * p.v_head;
        f32x4 x = f32x4{0.f, 0.f, 0.f, 0.f};
        if (on) x = load4(src + d);
        if (p.norm) {
            float ss = x[0] * x[0] + x[1] * x[1] + x[2] * x[2] + x[3] * x[3];
#pragma unroll
            for (int o = kLanes / 2; o > 0; o >>= 1) ss += __shfl_xor(ss, o, kLanes);
            if (on && kind < 2) {
                const float inv = 1.f / sqrtf(ss / HD + p.eps);
                const float* gamma = kind == 0 ? p.q_norm : p.k_norm;
#pragma unroll
                for (int i = 0; i < 4; ++i) x[i] = x[i] * inv * (gamma ? 1.f + gamma[d + i] : 1.f);
            }
        }
        // the other half of a pair sits half / 4 lanes away
        const bool low = d < half;
        const int other = low ? l + half / 4 : l - half / 4;
        f32x4 y;
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] = __shfl(x[i], other & (kLanes - 1), kLanes);
        if (on && kind < 2 && d < p.rot) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2 t = cs[(low ? d : d - half) + i];
                x[i] = low ? x[i] * t.x - y[i] * t.y : y[i] * t.y + x[i] * t.x;
            }
        }
        if (!on) continue;
        if (kind == 0) {
            store4(static_cast<T*>(p.q_out) + (static_cast<size_t>(row) * p.nq + head) * HD + d, x);
        } else if (put) {
            C* dst = static_cast<C*>(kind == 1 ? p.kc : p.vc);
            store4(dst + ((page * p.nkv + head) * p.page + in_page) * HD + d, x);
        }
    }
}

template <class R>
void launch_append(const AppendArgs& p, int hd, int rows, hipStream_t s) {
    const int heads = 256 / (hd / 4), groups = (p.nq + 2 * p.nkv + heads - 1) / heads;
    const dim3 grid(rows, std::min(groups, std::max(1, 2048 / rows)));
    switch (hd) {
    case 64: hipLaunchKernelGGL((paged_append_kernel<R, 64>), grid, dim3(256), 0, s, p); break;
    case 128: hipLaunchKernelGGL((paged_append_kernel<R, 128>), grid, dim3(256), 0, s, p); break;
    default: hipLaunchKernelGGL((paged_append_kernel<R, 256>), grid, dim3(256), 0, s, p); break;
    }
    check_launch("paged_append_kernel");
}

void paged_append(const RlPagedCache* c, int layer, int dtype, const void* q, int64_t q_row, int64_t q_head,
                  const void* k, int64_t k_row, int64_t k_head, const void* v, int64_t v_row, int64_t v_head,
                  const float* q_norm, const float* k_norm, int norm, float eps, int rot, float theta, const int* pos,
                  const int64_t* slots, int rows, int nq, void* q_out, hipStream_t s) {
    check_cache(c, layer, "paged_append");
    check_rows_type(c, dtype, "paged_append");
    RL_REQUIRE(rows >= 0 && nq >= 0 && nq <= 65535, RL_ERR_RANGE, "paged_append: bad sizes");
    RL_REQUIRE(rot >= 0 && rot % 8 == 0 && rot <= c->head_dim, RL_ERR_RANGE,
               "paged_append: rotary_dim must be a multiple of 8 up to head_dim");
    RL_REQUIRE(rot == 0 || (theta > 0.f && theta < INFINITY), RL_ERR_RANGE, "paged_append: bad theta");
    RL_REQUIRE(!norm || eps >= 0.f, RL_ERR_RANGE, "paged_append: bad eps");
    if (rows == 0) return;
    RL_REQUIRE(k && v && pos && slots && (nq == 0 || (q && q_out)), RL_ERR_RANGE, "paged_append: null pointer");
    if (nq) {
        check_strided(q, q_row, q_head, dtype, "paged_append");
        check_strided(q_out, 0, 0, dtype, "paged_append");
    }
    check_strided(k, k_row, k_head, dtype, "paged_append");
    check_strided(v, v_row, v_head, dtype, "paged_append");
    AppendArgs p{};
    p.q = q, p.k = k, p.v = v;
    p.q_row = q_row, p.q_head = q_head, p.k_row = k_row, p.k_head = k_head, p.v_row = v_row, p.v_head = v_head;
    p.q_norm = q_norm, p.k_norm = k_norm, p.norm = norm, p.eps = eps;
    p.rot = rot, p.log2_theta = rot ? std::log2(static_cast<double>(theta)) : 0.0;
    p.pos = pos, p.slots = slots;
    p.nq = nq, p.nkv = c->n_kv, p.page = c->page_size;
    p.n_slots = static_cast<int64_t>(c->n_pages) * c->page_size;
    p.q_out = q_out;
    p.kc = static_cast<uint16_t*>(c->k) + layer * c->layer_stride;
    p.vc = static_cast<uint16_t*>(c->v) + layer * c->layer_stride;
    if (dtype == RL_Q_F32)
        launch_append<RowF32>(p, c->head_dim, rows, s);
    else if (dtype == RL_Q_F16)
        launch_append<RowF16>(p, c->head_dim, rows, s);
    else
        launch_append<RowBF16>(p, c->head_dim, rows, s);
}

// ---- tree acceptance

constexpr int kPathCap = 4096;

struct AcceptTreeArgs {
    const int *table, *ctx_lens, *row_start, *parents, *toks, *samples;
    int width, rows, cap;
    int *path, *n_accept, *next_tok, *ctx_out;
    // cache
    i32x4 *k, *v;
    int64_t layer_stride;  // 16-byte units
    int layers, n_pages, page, nkv, units;  // units per head row
};

// Workgroup (sequence, share of the cache).  Every workgroup walks the tree by itself (a few
// dependent loads a node; no second launch); share 0 writes the results.  Bound by that walk and the
// launch for one chain (2.9 us), by scattered 512-byte runs for many: 48 trees x 64 rows, 16 layers of 4
// heads of 256 (37 MB moved) 11.5 us.  A path row's number
// is at least its depth, so a thread that moves one unit of every path row, in order, reads
// each before it is overwritten.
__global__ __launch_bounds__(256) void tree_accept_kernel(AcceptTreeArgs p) {
    __shared__ int path_s[kPathCap];
    __shared__ int n_s, cur_s;
    const int b = blockIdx.x;
    const int64_t capacity = p.k ? static_cast<int64_t>(p.width) * p.page : INT32_MAX;
    const SeqSpan s = seq_span(p.row_start, p.ctx_lens, b, p.rows, capacity);
    if (threadIdx.x < 64) {
        const int lane = threadIdx.x;
        int cur = 0, n = 0;
        while (n < p.cap && cur < s.n) {
            if (lane == 0) path_s[n] = cur;
            ++n;
            const int want = p.samples[s.r0 + cur];
            int next = s.n;
            for (int j0 = cur + 1; j0 < s.n; j0 += 64) {
                const int j = j0 + lane;
                const bool fit = j < s.n && p.parents[s.r0 + j] == cur && p.toks[s.r0 + j] == want;
                const unsigned long long m = __ballot(fit);
                if (m) {
                    next = j0 + __ffsll(m) - 1;
                    break;
                }
            }
            if (next >= s.n) break;
            if (n < p.cap) cur = next;
            else break;
        }
        if (lane == 0) {
            n_s = n;
            cur_s = cur;
        }
    }
    __syncthreads();
    const int n = n_s;
    if (blockIdx.y == 0) {
        for (int i = threadIdx.x; i < p.cap; i += 256) p.path[static_cast<size_t>(b) * p.cap + i] = i < n ? path_s[i] : -1;
        if (threadIdx.x == 0) {
            p.n_accept[b] = n;
            p.next_tok[b] = n ? p.samples[s.r0 + cur_s] : -1;
            p.ctx_out[b] = p.ctx_lens[b] + n;
        }
    }
    if (!p.k) return;
    const int* table = p.table + static_cast<size_t>(b) * p.width;
    const int per_layer = 2 * p.nkv * p.units;
    const int64_t total = static_cast<int64_t>(p.layers) * per_layer;
    for (int64_t w = static_cast<int64_t>(blockIdx.y) * 256 + threadIdx.x; w < total;
         w += static_cast<int64_t>(gridDim.y) * 256) {
        const int layer = static_cast<int>(w / per_layer), r = static_cast<int>(w % per_layer);
        const int unit = r % p.units, head = r / p.units % p.nkv;
        i32x4* base = (r / p.units / p.nkv ? p.v : p.k) + layer * p.layer_stride;
        for (int d = 1; d < n; ++d) {
            const int from = s.ctx + path_s[d], to = s.ctx + d;
            if (from == to) continue;
            const int pf = table[from / p.page], pt = table[to / p.page];
            if (pf < 0 || pf >= p.n_pages || pt < 0 || pt >= p.n_pages) continue;
            base[((static_cast<size_t>(pt) * p.nkv + head) * p.page + to % p.page) * p.units + unit] =
                base[((static_cast<size_t>(pf) * p.nkv + head) * p.page + from % p.page) * p.units + unit];
        }
    }
}

void tree_accept(const RlPagedCache* c, const int* table, int width, const int* ctx_lens, const int* row_start, int n_seq,
                 int rows, const int* parents, const int* toks, const int* samples, int* path, int cap, int* n_accept,
                 int* next_tok, int* ctx_out, hipStream_t s) {
    RL_REQUIRE(n_seq >= 0 && rows >= 0, RL_ERR_RANGE, "tree_accept: bad sizes");
    RL_REQUIRE(cap >= 1 && cap <= kPathCap, RL_ERR_RANGE, "tree_accept: path_cap must be in 1..4096");
    if (c) {
        check_cache(c, 0, "tree_accept");
        RL_REQUIRE(width >= 1 && static_cast<int64_t>(width) * c->page_size <= kMaxPositions, RL_ERR_RANGE,
                   "tree_accept: bad table width");
    }
    if (n_seq == 0) return;
    RL_REQUIRE(ctx_lens && row_start && path && n_accept && next_tok && ctx_out && (!c || table) &&
                   (rows == 0 || (parents && toks && samples)),
               RL_ERR_RANGE, "tree_accept: null pointer");
    RL_REQUIRE(ctx_out != ctx_lens, RL_ERR_RANGE, "tree_accept: ctx_out must not be ctx_lens");
    AcceptTreeArgs p{};
    p.table = table, p.ctx_lens = ctx_lens, p.row_start = row_start;
    p.parents = parents, p.toks = toks, p.samples = samples;
    p.width = width, p.rows = rows, p.cap = cap;
    p.path = path, p.n_accept = n_accept, p.next_tok = next_tok, p.ctx_out = ctx_out;
    int shares = 1;
    if (c) {
        p.k = static_cast<i32x4*>(c->k), p.v = static_cast<i32x4*>(c->v);
        p.layer_stride = c->layer_stride / 8;
        p.layers = c->n_layers, p.n_pages = c->n_pages, p.page = c->page_size, p.nkv = c->n_kv;
        p.units = c->head_dim / 8;
        const int64_t work = static_cast<int64_t>(c->n_layers) * 2 * c->n_kv * p.units;
        shares = static_cast<int>(std::min<int64_t>((work + 255) / 256, std::max(1, 4096 / n_seq)));
    }
    hipLaunchKernelGGL(tree_accept_kernel, dim3(n_seq, shares), dim3(256), 0, s, p);
    check_launch("tree_accept_kernel");
}

}  // namespace

extern "C" {

int rl_hip_paged_append(const RlPagedCache* cache, int layer, int dtype, const void* q, int64_t q_row, int64_t q_head,
                        const void* k, int64_t k_row, int64_t k_head, const void* v, int64_t v_row, int64_t v_head,
                        const float* q_norm, const float* k_norm, int use_norm, float eps, int rotary_dim, float theta,
                        const int* pos, const int64_t* slots, int rows, int n_q, void* q_out, void* stream) {
    return guard([&] {
        paged_append(cache, layer, dtype, q, q_row, q_head, k, k_row, k_head, v, v_row, v_head, q_norm, k_norm, use_norm,
                     eps, rotary_dim, theta, pos, slots, rows, n_q, q_out, S(stream));
    });
}

int rl_hip_tree_accept(const RlPagedCache* cache, const int* table, int table_width, const int* ctx_lens,
                       const int* row_start, int n_seq, int rows, const int* parents, const int* toks,
                       const int* samples, int* path, int path_cap, int* n_accept, int* next_tok, int* ctx_out,
                       void* stream) {
    return guard([&] {
        tree_accept(cache, table, table_width, ctx_lens, row_start, n_seq, rows, parents, toks, samples, path, path_cap,
                    n_accept, next_tok, ctx_out, S(stream));
    });
}

}  // extern "C"
