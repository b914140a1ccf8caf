// tree_attn.hip -- attention of every sequence's drafted tokens over a paged KV cache.
//
// The query heads of a kv head and a sequence's rows are its "pairs"; every K and V row serves all
// of them.  Work is counted in units of positions over all sequences and kv heads and dealt in
// equal runs to a fixed number of workgroups, whatever the lengths, which are read on the device;
// a run may end inside a sequence, then its outputs, maxima and sums go to the workspace and
// tree_attn_join_kernel adds them.
// S^T = K . Q^T and O^T = V^T . P^T on 32x32x16 MFMA, K and V copied row by row from the pages into
// shared memory: 32 positions x 32 pairs leave each lane with 16 scores of one pair, at just the
// positions that the transposing LDS reads of V give the second product, so the weights never leave
// their registers.  32-bit rows: q and the weights as two half-precision parts (2^-22), K and V
// exact; sums, maxima and outputs in 32 bits.  Half-precision rows round the weights to their type,
// as their output is rounded anyway.
// Few pairs (up to 32): bound by HBM.  Every wave streams tiles of its own without a barrier; 1 row
// x 131071 positions, 24 / 4 heads of 256: 537 MB in 97 us, 5.5 TB/s.  Many pairs: bound by the matrix cores;
// 128 pairs share each K and V, 8 x 64 rows x 32000 positions of 32-bit rows: 0.81 PFLOP (in two
// parts) in 785 us with the join, calls back to back, 1.03 PFLOP/s where a large fp16 library product reaches
// 1.14 (ten launches under a trace: kernel 765 us at least, 932 median).  Short contexts: bound by the
// chain of dependent loads and the instructions of one round; 1 row x 700 positions 13 + 4 us.  One
// thread per dim and a wave per position, without MFMA: 134 us, 31.4 ms and 57 ms for these three.
#include <algorithm>
#include <type_traits>

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
    int page_log2;
    float scale;
    void* out;
    int q_tiles, workers, unit;
    float* part_o;
    float2* part_ml;
};

__device__ inline float sigmoid(float x) { return 1.f / (1.f + expf(-x)); }

// out = acc / l (a row that saw nothing: 0), times sigmoid(gate)
template <class T>
__device__ inline void finish(const TreeArgs& p, int row, int head, int hd, int d, f32x4 acc, float l) {
    f32x4 r = f32x4{0.f, 0.f, 0.f, 0.f};
    if (l != 0.f) r = acc * (1.f / l);
    if (p.gate) {
        const f32x4 g = load4(static_cast<const T*>(p.gate) + row * p.g_row + head * p.g_head + d);
#pragma unroll
        for (int i = 0; i < 4; ++i) r[i] *= sigmoid(g[i]);
    }
    store4(static_cast<T*>(p.out) + (static_cast<size_t>(row) * p.nq + head) * hd + d, r);
}

// A lane's pair (query row, query head of the kv head) and everything its tile of pairs needs.
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
typedef __attribute__((address_space(3))) void lds_void;
typedef const __attribute__((address_space(1))) void global_void;

// Positions of one round of a workgroup: a tile of 32 per wave where every wave has its own, else 64.
constexpr int unit_of(int wp) { return wp == 1 ? 128 : 64; }
constexpr int kAhead = 4;        // operands read from shared memory ahead of their products
constexpr float kRaise = 4.f;  // log2 units that a score may pass the running maximum by
constexpr float kShift = 10.f; // weights are 2^(score - maximum + kShift): at most 2^14

template <class T>
struct Frag;
template <>
struct Frag<_Float16> {
    typedef f16x8 type;
    static __device__ f32x16 mfma(i32x4 a, i32x4 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    }
    static constexpr uint32_t kInf = 0x7c00u;  // exponent bits
};
template <>
struct Frag<__bf16> {
    typedef bf16x8 type;
    static __device__ f32x16 mfma(i32x4 a, i32x4 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
    static constexpr uint32_t kInf = 0x7f80u;
};

// The units of work of 64 sequences, one per lane: kv heads x rounds over its positions; `end` counts
// all units up to and with the lane's.
struct Lanes {
    int b0;  // first sequence
    SeqSpan s;
    int units, end;  // per kv head; over all kv heads and sequences
};
__device__ inline Lanes lanes_at(const TreeArgs& p, int b0, int before) {
    Lanes f;
    f.b0 = b0;
    f.s = SeqSpan{0, 0, 0};
    const int b = b0 + (threadIdx.x & 63);
    if (b < p.n_seq) {
        f.s = seq_span(p.row_start, p.ctx_lens, b, p.rows, static_cast<int64_t>(p.width) * p.page);
        f.s.n = min(f.s.n, p.max_rows);
    }
    f.units = f.s.n ? (f.s.ctx + f.s.n + p.unit - 1) / p.unit : 0;
    f.end = f.units * p.nkv;
    for (int o = 1; o < 64 && o < p.n_seq; o <<= 1) {  // lanes past the last sequence: any value
        const int x = __shfl_up(f.end, o, 64);
        if ((threadIdx.x & 63) >= o) f.end += x;
    }
    f.end += before;
    return f;
}
__device__ inline int lane_value(int v, int lane) { return __builtin_amdgcn_readlane(v, lane); }
// Units of a workgroup: workgroup c has units c * per up to (c + 1) * per of the first 64 sequences' f and
// the rest.
__device__ inline int total_units(const TreeArgs& p, const Lanes& f) {
    int total = lane_value(f.end, min(p.n_seq, 64) - 1);
    for (int b0 = 64; b0 < p.n_seq; b0 += 64) total = lane_value(lanes_at(p, b0, total).end, min(p.n_seq - b0, 64) - 1);
    return total;
}

// Bits of the 32 positions from base on that row j of the sequence sees.
__device__ inline uint32_t seen32(const TreeArgs& p, const SeqSpan& s, int j, int base) {
    const int i0 = base - s.ctx;  // tree slot of the first
    const int left = s.n - i0;    // positions that exist
    if (left <= 0) return 0;
    uint32_t v;
    if (!p.mask) {
        const int n = j - i0 + 1;
        v = n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1;
    } else {
        const uint64_t* m = p.mask + static_cast<size_t>(s.r0 + j) * p.words;
        if (i0 <= -32) {
            v = ~0u;
        } else if (i0 < 0) {
            v = static_cast<uint32_t>(m[0] << -i0) | ((1u << -i0) - 1);
        } else {
            const int w = i0 >> 6, sh = i0 & 63;
            uint64_t x = w < p.words ? m[w] >> sh : 0;
            if (sh > 32 && w + 1 < p.words) x |= m[w + 1] << (64 - sh);
            v = static_cast<uint32_t>(x);
        }
    }
    return left >= 32 ? v : v & ((1u << left) - 1);
}

template <int HD>
__device__ inline int k_swap(int r) {
    return HD == 64 ? r >> 1 & 7 : r & 15;
}
template <int HD>
__device__ inline int v_swap(int r) {
    return HD == 64 ? (r >> 1 & 1) << 2 : (r & 3) << 2;
}
// the same value, of which the compiler knows nothing
__device__ inline int opaque(int v) {
    asm volatile("" : "+v"(v));
    return v;
}

// Waits for all but the last kVm loads from memory, or all but kLds shared-memory reads (63, 15: for none).
// Builtins, not asm: the compiler then knows what is still on its way, and waits for single reads after it.
template <int kVm, int kLds>
__device__ inline void wait() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt((kVm & 15) | (kVm >> 4) << 14 | 7 << 4 | kLds << 8);
    asm volatile("" ::: "memory");
}
// Keeps a product where it stands among the reads and the vector work (the compiler sinks it to its use).
__device__ inline void pin(f32x16& v) { asm volatile("" : "+v"(v)); }

// One workgroup: 4 waves; WP tiles of 32 pairs (a row and one of the kv head's query heads) and
// 4 / WP shares of the positions.  See the top of the file.
template <class R, int HD, int WP>
__global__ __launch_bounds__(256, HD == 256 ? 1 : 2) void tree_attn_kernel(TreeArgs p) {
    using T = typename R::T;
    using C = typename R::C;
    using F = Frag<C>;
    constexpr bool kTwo = sizeof(T) == 4;  // 32-bit rows: q and the weights in two parts
    constexpr int kUnit = unit_of(WP);
    constexpr int WS = 4 / WP;                                // shares of the positions
    constexpr int NT = kUnit / 32 / WS;                       // tiles of 32 positions per share and round
    constexpr int kTiles = kUnit / 32;                        // tiles of a round
    constexpr int U = HD / 8;                                 // 16-byte units of a row
    constexpr int kTile = 32 * U;                             // units of a tile
    constexpr int kPerLoad = 64 / U, kLoads = 32 / kPerLoad;  // rows of one wave load, loads of a tile
    // WP > 1: two buffers of 64 positions; WP == 1: one of 128, a wave's tile overwritten as soon as it is used
    __shared__ i32x4 K_s[4 * kTile], V_s[4 * kTile];
    __shared__ float2 ml_s[4][32];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int h = lane >> 5, col = lane & 31;
    const int wp = wave % WP, ws = wave / WP;
    const int G = p.nq / p.nkv;
    // the tiles of one range of units sit on one XCD, so that its K and V come through one L2
    const int x = blockIdx.x % 8, y = blockIdx.x / 8;
    const int qt = y % p.q_tiles, c = y / p.q_tiles * 8 + x;

    Lanes f = lanes_at(p, 0, 0);
    const int total = total_units(p, f);
    const int per = (total + p.workers - 1) / p.workers;
    const int t0 = min(c * per, total), t1 = min(t0 + per, total);
    if (t0 >= t1) return;

    // Shared-memory addresses (bytes) are a lane's own part, xor a constant: unit u of K row r sits at
    // u ^ (r & 15), of V row r at u ^ 4 (r & 3), so that neither reads nor rows share banks (64 dims, two
    // rows in 256 bytes: by r / 2).  Kept opaque below: a register each for every constant is too many.
    const int vl = lane & 15, vrow = 4 * h + (vl >> 2);
    const int kaddr = (col * U + (h ^ k_swap<HD>(col))) * 16;
    const int vaddr = (vrow * U + (v_swap<HD>(vrow) | ((lane >> 4) & 1) * 2 | (vl >> 1 & 1))) * 16 + (vl & 1) * 8;
    const float sc = p.scale * 1.44269504f;

    for (int t = t0; t < t1;) {
        unsigned long long after;
        while (!(after = __ballot(f.end > t)) && f.b0 + 64 < p.n_seq) f = lanes_at(p, f.b0 + 64, lane_value(f.end, 63));
        if (!after) break;
        const int fl = __ffsll(after) - 1, seq = f.b0 + fl;
        const SeqSpan s{lane_value(f.s.r0, fl), lane_value(f.s.n, fl), lane_value(f.s.ctx, fl)};
        const int units = lane_value(f.units, fl), at = t - (lane_value(f.end, fl) - units * p.nkv);
        const int kv = at / units, ua = at % units, uz = min(units, ua + (t1 - t));
        const bool whole = ua == 0 && uz == units;
        const int slot = t0 < t - ua ? 1 : 0;
        t += uz - ua;
        const int pairs = s.n * G, pair0 = qt * 32 * WP;
        if (pair0 >= pairs) continue;
        const int mine = min(pair0 + 32 * wp + col, pairs - 1);  // this lane's pair
        const int j = mine / G, head = kv * G + mine % G;
        const int row = s.r0 + j;
        // the rows' own causal limit
        const int last = min(pair0 + 32 * WP, pairs) - 1;
        const int L = s.ctx + (p.mask ? s.n : last / G + 1);
        const int ub = min(uz, (L + kUnit - 1) / kUnit);
        const int* table = p.table + static_cast<size_t>(seq) * p.width;

        // The page of position `col` of tile k of round u as the table has it, and the position's row number
        // within the layer's cache.  (Apart: the load is in flight for a round.)
        auto page_of = [&](int u, int k) { return table[min(u * kUnit + 32 * k + col, L - 1) >> p.page_log2]; };
        auto row_of = [&](int pg, int u, int k) {
            pg = pg < 0 || pg >= p.n_pages ? 0 : pg;
            return ((static_cast<uint32_t>(pg) * static_cast<uint32_t>(p.nkv) + kv) << p.page_log2) +
                   (min(u * kUnit + 32 * k + col, L - 1) & (p.page - 1));
        };
        // Load i of a tile: kPerLoad rows.  Where they lie in one page (`runs`), their address is a scalar (in a
        // buffer resource) and a lane's offset; else, and for rows past the last position, each row's own.
        // Global loads to shared memory count as both kinds of access: while one may be on its way, the compiler
        // waits for every read.  They stay out of the loop that most rounds run in.
        auto load1 = [&]<bool runs>(std::bool_constant<runs>, const void* pool, i32x4* dst, uint32_t rows, bool is_v, int own, int i) {
            if constexpr (runs) {
                const int f = is_v ? v_swap<HD>(i * kPerLoad) : k_swap<HD>(i * kPerLoad);
                const uint32_t r0 = __builtin_amdgcn_readlane(rows, i * kPerLoad);
                char* src = static_cast<char*>(const_cast<void*>(pool)) + static_cast<size_t>(r0) * (U * 16);
                const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(src, 0, 1024, 0x00020000);
                __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_void*)(dst + i * 64), 16, own ^ f * 16, 0, 0, 0);
            } else {
                const int r = i * kPerLoad + own / (U * 16), u = lane % U;
                const int f = is_v ? v_swap<HD>(r) : k_swap<HD>(r);
                const uint32_t at = __shfl(rows, r, 64);
                const char* src = static_cast<const char*>(pool) + (static_cast<size_t>(at) * U + (u ^ f)) * 16;
                __builtin_amdgcn_global_load_lds((global_void*)src, (lds_void*)(dst + i * 64), 16, 0, 0);
            }
        };
        // a lane's offset within a load's rows: the swaps of rows i * kPerLoad + lane / U are those of the two parts, xor
        auto own_offset = [&](bool is_v) {
            const int r = lane / U, f = is_v ? v_swap<HD>(r) : k_swap<HD>(r);
            return opaque(r * U * 16 + ((lane % U) ^ f) * 16);
        };
        auto load_of = [&]<bool runs>(std::bool_constant<runs> r, const void* pool, i32x4* dst, uint32_t rows, bool is_v) {
            const int own = own_offset(is_v);
            rows = opaque(rows);
#pragma unroll
            for (int i = 0; i < kLoads; ++i) load1(r, pool, dst, rows, is_v, own, i);
        };
        auto load = [&](const void* pool, i32x4* dst, uint32_t rows, bool is_v, bool runs) {
            if (runs)
                load_of(std::true_type(), pool, dst, rows, is_v);
            else
                load_of(std::false_type(), pool, dst, rows, is_v);
        };
        const bool page_runs = p.page >= kPerLoad;

        // q: this lane's column of the operand, dims 16 st + 8 h ..  Asked for before everything else, split
        // while K and V come.
        typename Vec4<T>::type qr[HD / 8];
        i32x4 qh[HD / 16], ql[kTwo ? HD / 16 : 1];
        {
            const T* src = static_cast<const T*>(p.q) + row * p.q_row + head * p.q_head + 8 * h;
#pragma unroll
            for (int i = 0; i < HD / 8; ++i) qr[i] = *reinterpret_cast<const typename Vec4<T>::type*>(src + 16 * (i / 2) + 4 * (i % 2));
        }
        auto split_q = [&] {
#pragma unroll
            for (int st = 0; st < HD / 16; ++st) {
                typename F::type hi, lo;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float v = static_cast<float>(qr[2 * st + e / 4][e % 4]);
                    hi[e] = static_cast<C>(v);
                    if constexpr (kTwo) lo[e] = static_cast<C>(v - static_cast<float>(hi[e]));
                }
                qh[st] = __builtin_bit_cast(i32x4, hi);
                if constexpr (kTwo) ql[st] = __builtin_bit_cast(i32x4, lo);
                // 256 dims: q lives in accumulation registers, which the MFMAs read directly
                if constexpr (HD == 256) {
#pragma unroll
                    for (int d = 0; d < 4; ++d) {
                        int a;
                        asm("v_accvgpr_write_b32 %0, %1" : "=a"(a) : "v"(qh[st][d]));
                        qh[st][d] = a;
                        if constexpr (kTwo) {
                            asm("v_accvgpr_write_b32 %0, %1" : "=a"(a) : "v"(ql[st][d]));
                            ql[st][d] = a;
                        }
                    }
                }
            }
        };
        f32x16 o[HD / 32];
#pragma unroll
        for (int dt = 0; dt < HD / 32; ++dt)
#pragma unroll
            for (int v = 0; v < 16; ++v) o[dt][v] = 0.f;
        float m = -INFINITY, l = 0.f;

        // S^T = K . Q^T of a tile, in log2 units; side(i): what is done under product i of HD / 16
        auto scores = [&](const i32x4* Kt, f32x16& sn, auto side) {
            const char* K = reinterpret_cast<const char*>(Kt);
            const int own = opaque(kaddr);
#pragma unroll
            for (int v = 0; v < 16; ++v) sn[v] = 0.f;
            // dims 16 i; their K read kAhead products before
            constexpr int N = HD / 16;
            auto read = [&](int i) { return *reinterpret_cast<const i32x4*>(K + (own ^ 32 * i)); };
            i32x4 kk[kAhead];
#pragma unroll
            for (int i = 0; i < kAhead; ++i) kk[i] = read(i);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                sn = F::mfma(kk[i % kAhead], qh[i], sn);
                if constexpr (kTwo) sn = F::mfma(kk[i % kAhead], ql[i], sn);
                pin(sn);
                if (i + kAhead < N) kk[i % kAhead] = read(i + kAhead);
                side(i);
                __builtin_amdgcn_sched_barrier(0);
            }
            sn *= sc;
        };
        const auto nothing = [](int) {};
        auto hide = [&](f32x16& sn, uint32_t vis) {
#pragma unroll
            for (int v = 0; v < 16; ++v)
                if (!(vis >> (8 * (v >> 2) + 4 * h + (v & 3)) & 1)) sn[v] = -INFINITY;
        };
        // the running maximum follows the scores once one passes it by kRaise; true where it did
        auto raise = [&](const f32x16& sn) {
            float mx = sn[0];
#pragma unroll
            for (int v = 1; v < 16; ++v) mx = fmaxf(mx, sn[v]);
            mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
            if (!__any(mx > m + kRaise)) return false;
            const float mn = fmaxf(m, mx);
            const float alpha = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - mn);
            m = mn;
            l *= alpha;
#pragma unroll
            for (int dt = 0; dt < HD / 32; ++dt) o[dt] *= alpha;
            return true;
        };
        struct Weights {
            typename F::type hi[2], lo[kTwo ? 2 : 1];
        };
        // weights 2 i and 2 i + 1 of a tile
        auto weights2 = [&](const f32x16& sn, Weights& w, float sub, int i) {
#pragma unroll
            for (int e = 2 * i; e < 2 * i + 2; ++e) {
                const float x = __builtin_amdgcn_exp2f(sn[e] - sub);
                l += x;
                const C hi = static_cast<C>(x);
                w.hi[e >> 3][e & 7] = hi;
                if constexpr (kTwo) w.lo[e >> 3][e & 7] = static_cast<C>(x - static_cast<float>(hi));
            }
        };
        auto weights = [&](const f32x16& sn, Weights& w, float sub) {
#pragma unroll
            for (int i = 0; i < 8; ++i) weights2(sn, w, sub, i);
        };
        auto level = [&] { return (m == -INFINITY ? 0.f : m) - kShift; };
        // O^T += V^T . P^T of a tile; an edge tile's infinities and NaN go to the pairs that see them alone.
        // side(i): what is computed under product i
        auto output = [&]<bool edge>(std::bool_constant<edge>, const i32x4* Vt, const Weights& w, uint32_t vis, auto side) {
            const char* V = reinterpret_cast<const char*>(Vt);
            const int own = opaque(vaddr);
            bool bad = false;
            constexpr int N = HD / 16;  // product i: dims 32 (i / 2), positions 16 (i % 2)
            union Frag4 {
                s16x4 q[2];
                i32x4 v;
            } vf[kAhead];
            auto read = [&](int i, int e) {
                return __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                    (lds_s16x4*)(V + (own ^ 64 * (i / 2)) + (16 * (i % 2) + 8 * e) * U * 16));
            };
#pragma unroll
            for (int i = 0; i < kAhead; ++i)
#pragma unroll
                for (int e = 0; e < 2; ++e) vf[i].q[e] = read(i, e);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                i32x4 v = vf[i % kAhead].v;
                if constexpr (edge) {
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const uint32_t z = v[k];
                        const bool lo_bad = (z & F::kInf) == F::kInf, hi_bad = (z >> 16 & F::kInf) == F::kInf;
                        bad |= lo_bad || hi_bad;
                        v[k] = z & (lo_bad ? 0xffff0000u : ~0u) & (hi_bad ? 0xffffu : ~0u);
                    }
                }
                o[i / 2] = F::mfma(v, __builtin_bit_cast(i32x4, w.hi[i % 2]), o[i / 2]);
                if constexpr (kTwo) o[i / 2] = F::mfma(v, __builtin_bit_cast(i32x4, w.lo[i % 2]), o[i / 2]);
                pin(o[i / 2]);
                if (i + kAhead < N)
#pragma unroll
                    for (int e = 0; e < 2; ++e) vf[i % kAhead].q[e] = read(i + kAhead, e);
                side(i);
                __builtin_amdgcn_sched_barrier(0);
            }
            if (edge && __any(bad)) {
                const C* Ve = reinterpret_cast<const C*>(Vt);
#pragma unroll 1
                for (int r = 0; r < 32; ++r) {
                    const bool sees = vis >> r & 1;
#pragma unroll
                    for (int dt = 0; dt < HD / 32; ++dt)
#pragma unroll
                        for (int v = 0; v < 16; ++v) {
                            const int d = 32 * dt + 8 * (v >> 2) + 4 * h + (v & 3);
                            const float z = static_cast<float>(Ve[r * HD + ((d >> 3) ^ v_swap<HD>(r)) * 8 + (d & 7)]);
                            if (sees && !(fabsf(z) < INFINITY)) o[dt][v] += z;
                            if (v % 4 == 3) asm volatile("" ::: "memory");
                        }
                }
            }
        };
        // rounds up to u_edge hold positions of the context alone
        const int u_edge = min(max(s.ctx / kUnit, ua), ub), u_runs = page_runs ? max(u_edge - 1, ua) : ua;
        if constexpr (WP == 1) {
            // every wave by itself: K of its next tile comes while this one's V is used, and the other way round
            i32x4 *K = K_s + wave * kTile, *V = V_s + wave * kTile;
            int next = 0;
            if (ua < ub) {
                const uint32_t rows = row_of(page_of(ua, wave), ua, wave);
                next = page_of(min(ua + 1, ub - 1), wave);
                load(p.k, K, rows, false, page_runs && ua < u_edge);
                asm volatile("" ::: "memory");
                load(p.v, V, rows, true, page_runs && ua < u_edge);
            }
            split_q();
            // runs: the next round's loads are runs of rows, and there is a next round
            auto rounds = [&]<bool edge, bool runs>(std::bool_constant<edge> e, std::bool_constant<runs> r, int from, int to) {
                for (int u = from; u < to; ++u) {
                    const bool more = runs || u + 1 < ub;
                    f32x16 sn;
                    uint32_t vis = ~0u;
                    Weights w;
                    // all but the last kLoads loads, V's
                    wait<kLoads, 15>();
                    const uint32_t rows = row_of(next, min(u + 1, ub - 1), wave);
                    next = page_of(min(u + 2, ub - 1), wave);
                    asm volatile("" ::: "memory");
                    scores(K, sn, nothing);
                    wait<63, 0>();
                    if (more) load_of(r, p.k, K, rows, false);
                    if constexpr (edge) hide(sn, vis = seen32(p, s, j, u * kUnit + 32 * wave));
                    raise(sn);
                    weights(sn, w, level());
                    // all but the next K's
                    if (more)
                        wait<kLoads, 15>();
                    else
                        wait<0, 15>();
                    output(e, V, w, vis, nothing);
                    wait<63, 0>();
                    if (more) load_of(r, p.v, V, rows, true);
                }
            };
            rounds(std::false_type(), std::true_type(), ua, u_runs);
            rounds(std::false_type(), std::false_type(), u_runs, u_edge);
            rounds(std::true_type(), std::false_type(), u_edge, ub);
        } else {
            // wave w brings tile w % 2 of K (w < 2) or V: the next round's while this one is computed
            const bool is_v = wave >= 2;
            const void* pool = is_v ? p.v : p.k;
            i32x4* mem = (is_v ? V_s : K_s) + (wave & 1) * kTile;
            int next = 0;
            if (ua < ub) {
                load(pool, mem + (ua & 1) * 2 * kTile, row_of(page_of(ua, wave & 1), ua, wave & 1), is_v, page_runs && ua < u_edge);
                next = page_of(min(ua + 1, ub - 1), wave & 1);
            }
            split_q();
            auto rounds = [&]<bool edge, bool runs>(std::bool_constant<edge> e, std::bool_constant<runs> r, int from, int to) {
                for (int u = from; u < to; ++u) {
                    wait<0, 0>();
                    __builtin_amdgcn_s_barrier();
                    asm volatile("" ::: "memory");
                    const uint32_t rows = row_of(next, min(u + 1, ub - 1), wave & 1);
                    next = page_of(min(u + 2, ub - 1), wave & 1);
                    const i32x4 *K = K_s + ((u & 1) * 2 + ws * NT) * kTile, *V = V_s + ((u & 1) * 2 + ws * NT) * kTile;
                    i32x4* to = mem + ((u + 1) & 1) * 2 * kTile;
                    f32x16 sn[NT];
                    uint32_t vis[NT];
                    Weights w[NT];
#pragma unroll
                    for (int a = 0; a < NT; ++a) vis[a] = ~0u;
                    // the next round's loads under the first tile's scores
                    if constexpr (runs) {
                        const int own = own_offset(is_v);
                        scores(K, sn[0], [&](int i) {
                            if (i < kLoads) load1(r, pool, to, rows, is_v, own, i);
                        });
                    } else {
                        if (u + 1 < ub) load_of(r, pool, to, rows, is_v);
                        scores(K, sn[0], nothing);
                    }
                    if constexpr (edge) hide(sn[0], vis[0] = seen32(p, s, j, u * kUnit + 32 * ws * NT));
                    raise(sn[0]);
                    if constexpr (NT == 2) {
                        // the first tile's weights under the second one's scores, the second one's under the
                        // first one's output
                        float sub = level();
                        scores(K + kTile, sn[1], [&](int i) {
#pragma unroll
                            for (int k = 8 * i / (HD / 16); k < 8 * (i + 1) / (HD / 16); ++k) weights2(sn[0], w[0], sub, k);
                        });
                        if constexpr (edge) hide(sn[1], vis[1] = seen32(p, s, j, u * kUnit + 32 * (ws * NT + 1)));
                        if (raise(sn[1])) {
                            // rarely: the first tile's weights once more, their sum is in l
                            const float had = l;
                            sub = level();
                            weights(sn[0], w[0], sub);
                            l = had;
                        }
                        output(e, V, w[0], vis[0], [&](int i) {
#pragma unroll
                            for (int k = 8 * i / (HD / 16); k < 8 * (i + 1) / (HD / 16); ++k) weights2(sn[1], w[1], sub, k);
                        });
                        output(e, V + kTile, w[1], vis[1], nothing);
                    } else {
                        weights(sn[0], w[0], level());
                        output(e, V, w[0], vis[0], nothing);
                    }
                }
            };
            rounds(std::false_type(), std::true_type(), ua, u_runs);
            rounds(std::false_type(), std::false_type(), u_runs, u_edge);
            rounds(std::true_type(), std::false_type(), u_edge, ub);
        }
        l += __shfl_xor(l, 32, 64);

        // ---- the waves' outputs to shared memory, [pair][HD] in 16-byte units, and out
        __syncthreads();
        char* O_s = reinterpret_cast<char*>((wave < 2 ? K_s : V_s) + (wave & 1) * (2 * kTile));
        const int oaddr = opaque((col * (HD / 4) + (h ^ (col & 15))) * 16);
        if (h == 0) ml_s[wave][col] = make_float2(m, l);
        if (pair0 + 32 * wp + col < pairs)
#pragma unroll
        for (int dt = 0; dt < HD / 32; ++dt)
#pragma unroll
            for (int v = 0; v < 16; v += 4)
                *reinterpret_cast<f32x4*>(O_s + (oaddr ^ (8 * dt + 2 * (v >> 2)) * 16)) =
                    f32x4{o[dt][v], o[dt][v + 1], o[dt][v + 2], o[dt][v + 3]};
        __syncthreads();
        constexpr int kLanes = HD / 4;
        const int od = threadIdx.x % kLanes;
        for (int q = threadIdx.x / kLanes; q < 32 * WP && pair0 + q < pairs; q += 256 / kLanes) {
            const int tw = q / 32, tc = q % 32;
            float M = -INFINITY, L2 = 0.f;
#pragma unroll
            for (int w = 0; w < WS; ++w) M = fmaxf(M, ml_s[w * WP + tw][tc].x);
            f32x4 acc = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < WS; ++w) {
                const int wv = w * WP + tw;
                const float2 ml = ml_s[wv][tc];
                const float f = ml.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ml.x - M);
                const f32x4 part = reinterpret_cast<const f32x4*>(wv < 2 ? K_s : V_s)[(wv & 1) * (2 * kTile) + tc * kLanes + (od ^ (tc & 15))];
                if (ml.y != 0.f) {
                    L2 += ml.y * f;
                    acc += part * f;
                }
            }
            if (whole) {
                finish<T>(p, s.r0 + (pair0 + q) / G, kv * G + (pair0 + q) % G, HD, 4 * od, acc, L2);
            } else {
                const size_t part = (static_cast<size_t>(c) * p.q_tiles + qt) * 2 + slot;
                if (L2 != 0.f) *reinterpret_cast<f32x4*>(p.part_o + (part * (32 * WP) + q) * HD + 4 * od) = acc;
                if (od == 0) p.part_ml[part * (32 * WP) + q] = make_float2(M, L2);
            }
        }
        if (t < t1) __syncthreads();
    }
}

// Joins the parts of the rows whose positions several workgroups shared.  kWaves waves per (row, query
// head): 4 where there are few of them, each a share of the parts, else 1.
template <class R, int HD, int kWaves>
__global__ __launch_bounds__(256) void tree_attn_join_kernel(TreeArgs p, int tile) {
    using T = typename R::T;
    constexpr int kLanes = HD / 4, kGroups = kWaves * 64 / kLanes;  // lanes of an output, parts side by side
    constexpr int kSets = 4 / kWaves;
    __shared__ f32x4 acc_s[kSets][kGroups][kLanes];
    const int lane = threadIdx.x & 63, set = threadIdx.x / (64 * kWaves);
    const int item = blockIdx.x * kSets + set, row = item / p.nq, head = item % p.nq, G = p.nq / p.nkv;
    Lanes f = lanes_at(p, 0, 0);
    const int total = total_units(p, f);
    const int per = (total + p.workers - 1) / p.workers;
    unsigned long long m;
    while (!(m = __ballot(row >= f.s.r0 && row < f.s.r0 + f.s.n)) && f.b0 + 64 < p.n_seq)
        f = lanes_at(p, f.b0 + 64, lane_value(f.end, 63));
    int wa = 0, wz = 0, q = 0, qt = 0, t0 = 0;
    if (m && row < p.rows) {
        const int fl = __ffsll(m) - 1, units = lane_value(f.units, fl);
        t0 = lane_value(f.end, fl) - units * p.nkv + head / G * units;
        wa = t0 / per, wz = (t0 + units - 1) / per;
        const int pair = (row - lane_value(f.s.r0, fl)) * G + head % G;
        qt = pair / tile, q = pair % tile;
    }
    const int od = threadIdx.x % kLanes, grp = threadIdx.x % (64 * kWaves) / kLanes;
    float M = -INFINITY, L = 0.f;
    f32x4 acc = f32x4{0.f, 0.f, 0.f, 0.f};
    if (wa != wz) {
        for (int w0 = wa; w0 <= wz; w0 += 64) {
            // the parts' weights, one per lane, then their outputs
            const int w = w0 + lane;
            const size_t part = ((static_cast<size_t>(min(w, wz)) * p.q_tiles + qt) * 2 + (min(w, wz) * per < t0)) * tile + q;
            const float2 ml = p.part_ml[part];
            const float mine = w <= wz && ml.y != 0.f ? ml.x : -INFINITY;
            const float mn = fmaxf(M, wave_max(mine));
            const float old = M == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(M - mn);
            const float wt = mine == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mine - mn);
            const float lw = w <= wz && ml.y != 0.f ? ml.y * wt : 0.f;
            M = mn;
            L = L * old + wave_sum(lw);
            acc = acc * old;
            const int n = min(64, wz - w0 + 1);
            for (int i0 = grp; i0 < n; i0 += 8 * kGroups) {
                f32x4 o[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const int w = w0 + min(i0 + k * kGroups, n - 1);
                    const size_t at = ((static_cast<size_t>(w) * p.q_tiles + qt) * 2 + (w * per < t0)) * tile + q;
                    o[k] = *reinterpret_cast<const f32x4*>(p.part_o + at * HD + 4 * od);
                }
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    // a part without weight may hold anything
                    const float fw = __shfl(wt, min(i0 + k * kGroups, n - 1), 64);
                    const bool on = i0 + k * kGroups < n && fw != 0.f;
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[e] = on ? fmaf(o[k][e], fw, acc[e]) : acc[e];
                }
            }
        }
    }
    if constexpr (kGroups > 1) {
        acc_s[set][grp][od] = acc;
        __syncthreads();
        if (grp == 0) {
#pragma unroll
            for (int g = 1; g < kGroups; ++g) acc += acc_s[set][g][od];
        }
    }
    if (wa != wz && grp == 0) finish<T>(p, row, head, HD, 4 * od, acc, L);
}

// Workgroups on the chip at once: 256 dims take 128 KB of shared memory and all registers of a wave slot.
constexpr int kSlots(int hd) { return hd == 256 ? 256 : 512; }

// Tiles of 32 pairs per workgroup: as many as a sequence's rows fill, the positions shared by the other waves.
// 8 sequences x 16000 positions, 24 / 4 heads of 256, f32 / f16 rows: 24 pairs with 1, 2, 4 tiles 122 / 110, 127 / 109,
// 172 / 116 us; 54 pairs with 2 and 4 131 / 118, 164 / 124 us.
int pair_waves(int G, int max_rows) {
    const int64_t pairs = static_cast<int64_t>(G) * max_rows;
    return pairs <= 32 ? 1 : pairs <= 64 ? 2 : 4;
}
struct Split {
    int wp, q_tiles, workers;
};
Split split_of(int nq, int nkv, int hd, int max_rows) {
    Split s;
    const int G = nq / nkv;
    s.wp = pair_waves(G, max_rows);
    s.q_tiles = static_cast<int>((static_cast<int64_t>(G) * max_rows + 32 * s.wp - 1) / (32 * s.wp));
    s.workers = std::max(1, kSlots(hd) / (8 * s.q_tiles)) * 8;
    return s;
}

size_t tree_attn_workspace_bytes(int nq, int nkv, int hd, int n_seq, int max_rows) {
    (void)n_seq;
    if (nq < 1 || nkv < 1 || nq % nkv || hd < 1 || max_rows < 1) return 256;
    // at least what split_of takes, and never less for more rows: a workspace serves every smaller max_rows
    const Split s = split_of(nq, nkv, hd, max_rows);
    return static_cast<size_t>(std::max(kSlots(hd), 8 * s.q_tiles)) * 2 * 32 * s.wp * (hd * 4 + 8) + 256;
}

template <class R, int HD>
void launch_tree(const TreeArgs& p, int wp, hipStream_t s) {
    const dim3 grid(p.workers * p.q_tiles);
    switch (wp) {
    case 1: hipLaunchKernelGGL((tree_attn_kernel<R, HD, 1>), grid, dim3(256), 0, s, p); break;
    case 2: hipLaunchKernelGGL((tree_attn_kernel<R, HD, 2>), grid, dim3(256), 0, s, p); break;
    default: hipLaunchKernelGGL((tree_attn_kernel<R, HD, 4>), grid, dim3(256), 0, s, p); break;
    }
    check_launch("tree_attn_kernel");
    // from 512 outputs on a wave each: 70 rows x 32 heads 10.8 -> 5.9 us; below, four: 1 row x 24 heads with 64
    // parts each 6 us
    const int64_t outs = static_cast<int64_t>(p.rows) * p.nq;
    if (outs < 512)
        hipLaunchKernelGGL((tree_attn_join_kernel<R, HD, 4>), dim3(outs), dim3(256), 0, s, p, 32 * wp);
    else
        hipLaunchKernelGGL((tree_attn_join_kernel<R, HD, 1>), dim3((outs + 3) / 4), dim3(256), 0, s, p, 32 * wp);
    check_launch("tree_attn_join_kernel");
}

template <class R>
void launch_tree(const TreeArgs& p, int hd, int wp, hipStream_t s) {
    switch (hd) {
    case 64: launch_tree<R, 64>(p, wp, s); break;
    case 128: launch_tree<R, 128>(p, wp, s); break;
    default: launch_tree<R, 256>(p, wp, s); break;
    }
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
    RL_REQUIRE(width >= 1 && static_cast<int64_t>(width) * c->page_size <= kMaxPositions, RL_ERR_RANGE,
               "tree_attn: bad table width");
    RL_REQUIRE(!mask || (words >= 1 && aligned(mask, 8)), RL_ERR_RANGE, "tree_attn: a mask needs words, 8-byte aligned");
    RL_REQUIRE(scale > -INFINITY && scale < INFINITY, RL_ERR_RANGE, "tree_attn: bad scale");
    if (rows == 0 || n_seq == 0 || max_rows == 0) return;
    RL_REQUIRE(q && table && ctx_lens && row_start && out && ws, RL_ERR_RANGE, "tree_attn: null pointer");
    check_strided(q, q_row, q_head, dtype, "tree_attn");
    if (gate) check_strided(gate, gate_row, gate_head, dtype, "tree_attn");
    RL_REQUIRE(aligned(out, 16) && aligned(ws, 16), RL_ERR_RANGE, "tree_attn: out and workspace must be 16-byte aligned");
    RL_REQUIRE(static_cast<double>(n_seq) * c->n_kv * (static_cast<double>(width) * c->page_size / 64 + 1) < (1 << 30) &&
                   static_cast<int64_t>(rows) * nq < INT32_MAX,
               RL_ERR_UNSUPPORTED, "tree_attn: more than 2^30 units of work");
    RL_REQUIRE(static_cast<int64_t>(c->n_pages) * c->n_kv * c->page_size <= UINT32_MAX, RL_ERR_UNSUPPORTED,
               "tree_attn: a layer's cache has more than 2^32 rows");
    RL_REQUIRE(ws_bytes >= tree_attn_workspace_bytes(nq, c->n_kv, c->head_dim, n_seq, std::min(max_rows, rows)), RL_ERR_RANGE,
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
    while ((1 << p.page_log2) < c->page_size) ++p.page_log2;
    const Split sp = split_of(nq, c->n_kv, c->head_dim, std::min(max_rows, rows));
    p.q_tiles = sp.q_tiles, p.workers = sp.workers, p.unit = unit_of(sp.wp);
    const size_t parts = static_cast<size_t>(sp.workers) * sp.q_tiles * 2 * 32 * sp.wp;
    p.part_o = static_cast<float*>(ws);
    p.part_ml = reinterpret_cast<float2*>(p.part_o + parts * c->head_dim);
    if (dtype == RL_Q_F32)
        launch_tree<RowF32>(p, c->head_dim, sp.wp, s);
    else if (dtype == RL_Q_F16)
        launch_tree<RowF16>(p, c->head_dim, sp.wp, s);
    else
        launch_tree<RowBF16>(p, c->head_dim, sp.wp, s);
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
