// sampling.hip -- one token per row of logits: temperature, top-k, top-p, min-p, from given random
// numbers.
//
// With M the row's maximum and w = exp((z - M) / T), what top-k and top-p keep is a prefix of the
// order (larger z first, equal z by lower index), so it is told by one element, the last kept.
// That element is found without sorting: a histogram of (M - z) / T gives the bin it is in and
// the count and mass before the bin, and only the bin's own elements are put in order.
// Masses are integers (w in units of 2^-44 of the largest), so that sums are exact in any order
// and every kernel sees the same element the same way.
#include <algorithm>

#include "paged.h"

using namespace rl;

namespace {

constexpr int kBins = 2048;
constexpr double kBinsPerUnit = 64.0;  // bins cover weights down to exp(-32) < 2^-45
constexpr int kList = 2048;            // elements of one bin put in order in shared memory
constexpr int kThreads = 1024;

struct SampleArgs {
    const void* logits;
    int64_t ld;
    int V, shift;  // masses in units of 2^-shift
    const float *temperature, *top_p, *min_p, *u;
    const int* top_k;
    int* idx;
    float* prob;
};

// Larger first, equal ones by index.
__device__ inline uint64_t order_key(float z, int i) {
    const uint32_t b = __float_as_uint(z);
    const uint32_t up = b >> 31 ? ~b : b | 0x80000000u;
    return static_cast<uint64_t>(~up) << 32 | static_cast<uint32_t>(i);
}
__device__ inline float key_value(uint64_t key) {
    const uint32_t up = ~static_cast<uint32_t>(key >> 32);
    return __uint_as_float(up >> 31 ? up & 0x7fffffffu : ~up);
}

template <class T>
__device__ inline float logit(const T* row, int i) {
    const float z = static_cast<float>(row[i]) + 0.f;  // -0 becomes +0: they are equal
    return z != z ? -INFINITY : z;
}

struct Row {
    float M;
    double inv_t, unit, min_p;
    // depth (M - z) / T, >= 0; 1e9 for what has no weight at all
    __device__ double depth(float z) const {
        if (z == M) return 0.0;
        if (z == -INFINITY || M == INFINITY) return 1e9;
        return (static_cast<double>(M) - static_cast<double>(z)) * inv_t;
    }
    __device__ double weight(double depth) const { return depth < 32.0 ? exp(-depth) : 0.0; }
    __device__ unsigned long long mass(double w) const { return static_cast<unsigned long long>(rint(w * unit)); }
    __device__ int bin(double depth) const { return static_cast<int>(depth * kBinsPerUnit); }
};

template <class T>
__device__ inline T wave_scan(T v) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const T x = __shfl_up(v, o, 64);
        if (lane >= o) v += x;
    }
    return v;
}
// inclusive sum over the workgroup; all threads call it
template <class T>
__device__ inline T block_scan(T v, T* part) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    v = wave_scan(v);
    __syncthreads();
    if (lane == 63) part[wave] = v;
    __syncthreads();
    T before = 0;
    for (int w = 0; w < wave; ++w) before += part[w];
    return v + before;
}

typedef unsigned long long u64;

struct Shared {
    unsigned cnt[kBins];
    u64 mass[kBins];
    u64 key[kList];
    u64 w[kList];
    u64 part[kThreads / 64];
    unsigned cpart[kThreads / 64];
    uint64_t best[kThreads / 64];
    int n;
    // what a search found
    int bin;
    unsigned before_n;
    u64 before_m, found_key, found_m;
};

// Which element of the row ends the prefix: the `want_n`th of the order, or the first up to which
// want_m of mass stands; elements past `last` do not count.  Histograms in sh; before the call the
// bin, before_n and before_m are known.  Returns the element's key, its mass included in *upto.
template <class T>
__device__ uint64_t find_in_bin(const SampleArgs& p, const T* row, const Row& r, Shared& sh, uint64_t last, unsigned want_n,
                                double want_m, u64* upto) {
    const int tid = threadIdx.x;
    const int bin = sh.bin;
    const unsigned before_n = sh.before_n;
    const u64 before_m = sh.before_m;
    const unsigned n_bin = sh.cnt[bin];
    if (n_bin <= kList) {
        __syncthreads();
        if (tid == 0) sh.n = 0;
        __syncthreads();
        for (int i = tid; i < p.V; i += kThreads) {
            const float z = logit(row, i);
            const double d = r.depth(z);
            if (d >= 32.0 || r.bin(d) != bin) continue;
            const uint64_t key = order_key(z, i);
            const u64 m = r.mass(r.weight(d));
            if (m == 0 || key > last) continue;
            const int at = atomicAdd(&sh.n, 1);
            sh.key[at] = key;
            sh.w[at] = m;
        }
        __syncthreads();
        const int n = sh.n;
        for (int e = tid; e < n; e += kThreads) {
            const uint64_t key = sh.key[e];
            unsigned rank = before_n;
            u64 m = before_m;
            for (int j = 0; j < n; ++j)
                if (sh.key[j] < key) {
                    ++rank;
                    m += sh.w[j];
                }
            const bool hit = want_n ? rank + 1 == want_n
                                    : static_cast<double>(m) < want_m && static_cast<double>(m + sh.w[e]) >= want_m;
            if (hit) {
                sh.found_key = key;
                sh.found_m = m + sh.w[e];
            }
        }
        __syncthreads();
        *upto = sh.found_m;
        return sh.found_key;
    }
    // many elements in one bin (flat or repeated logits): eight bits of the key at a time
    uint64_t prefix = 0;
    unsigned base_n = before_n;
    u64 base_m = before_m;
    for (int shift = 56; shift >= 0; shift -= 8) {
        __syncthreads();
        for (int i = tid; i < 256; i += kThreads) {
            sh.key[i] = 0;
            sh.w[i] = 0;
        }
        __syncthreads();
        for (int i = tid; i < p.V; i += kThreads) {
            const float z = logit(row, i);
            const double d = r.depth(z);
            if (d >= 32.0 || r.bin(d) != bin) continue;
            const uint64_t key = order_key(z, i);
            const u64 m = r.mass(r.weight(d));
            if (m == 0 || key > last || (shift < 56 && (key ^ prefix) >> (shift + 8))) continue;
            atomicAdd(reinterpret_cast<u64*>(&sh.key[key >> shift & 255]), 1ull);
            atomicAdd(&sh.w[key >> shift & 255], m);
        }
        __syncthreads();
        if (tid == 0) {
            u64 c = base_n, m = base_m;
            int digit = 0;
            for (; digit < 256; ++digit) {
                const bool hit = want_n ? c + sh.key[digit] >= want_n : static_cast<double>(m + sh.w[digit]) >= want_m;
                if (sh.key[digit] && hit) break;
                c += sh.key[digit];
                m += sh.w[digit];
            }
            sh.before_n = static_cast<unsigned>(c);
            sh.before_m = m;
            sh.found_m = m + sh.w[digit & 255];
            sh.n = digit;
        }
        __syncthreads();
        prefix |= static_cast<uint64_t>(sh.n) << shift;
        base_n = sh.before_n;
        base_m = sh.before_m;
    }
    *upto = sh.found_m;
    return prefix;
}

template <class T>
__global__ __launch_bounds__(kThreads) void sample_row_kernel(SampleArgs p) {
    __shared__ Shared sh;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const T* row = static_cast<const T*>(p.logits) + blockIdx.x * p.ld;
    const int V = p.V;
    // the maximum, at its lowest index
    uint64_t best = ~0ull;
    for (int i = tid; i < V; i += kThreads) best = min(best, order_key(logit(row, i), i));
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) best = min(best, static_cast<uint64_t>(__shfl_xor(static_cast<u64>(best), o, 64)));
    if (lane == 0) sh.best[wave] = best;
    __syncthreads();
    for (int w = 0; w < kThreads / 64; ++w) best = min(best, sh.best[w]);
    const float t = p.temperature ? p.temperature[blockIdx.x] : 1.f;
    Row r;
    r.M = key_value(best);
    if (r.M == -INFINITY || !(t > 0.f)) {
        if (tid == 0) {
            p.idx[blockIdx.x] = r.M == -INFINITY ? 0 : static_cast<int>(best & 0xffffffffu);
            if (p.prob) p.prob[blockIdx.x] = r.M == -INFINITY ? 0.f : 1.f;
        }
        return;
    }
    r.inv_t = 1.0 / static_cast<double>(t);
    r.unit = ldexp(1.0, p.shift);
    const float mp = p.min_p ? p.min_p[blockIdx.x] : 0.f;
    r.min_p = mp > 0.f ? fminf(mp, 1.f) : 0.0;
    const int k = p.top_k ? p.top_k[blockIdx.x] : 0;
    const float tp = p.top_p ? p.top_p[blockIdx.x] : 1.f;
    const bool use_k = k > 0 && k < V, use_p = tp < 1.f;
    uint64_t last = ~0ull;
    if (use_k || use_p) {
        for (int i = tid; i < kBins; i += kThreads) {
            sh.cnt[i] = 0;
            sh.mass[i] = 0;
        }
        __syncthreads();
        for (int i = tid; i < V; i += kThreads) {
            const double d = r.depth(logit(row, i));
            if (d >= 32.0) continue;
            const u64 m = r.mass(r.weight(d));
            if (m == 0) continue;
            atomicAdd(&sh.cnt[r.bin(d)], 1u);
            atomicAdd(&sh.mass[r.bin(d)], m);
        }
        __syncthreads();
        unsigned c[2], ci;
        u64 m[2], mi;
        for (int e = 0; e < 2; ++e) {
            c[e] = sh.cnt[2 * tid + e];
            m[e] = sh.mass[2 * tid + e];
        }
        ci = block_scan(c[0] + c[1], sh.cpart);
        mi = block_scan(m[0] + m[1], sh.part);
        unsigned total_n = 0;
        u64 total_m = 0;
        for (int w = 0; w < kThreads / 64; ++w) {
            total_n += sh.cpart[w];
            total_m += sh.part[w];
        }
        int k_bin = kBins;
        if (use_k && static_cast<unsigned>(k) < total_n) {
            unsigned b0 = ci - c[0] - c[1];
            u64 m0 = mi - m[0] - m[1];
            for (int e = 0; e < 2; ++e) {
                if (b0 < static_cast<unsigned>(k) && static_cast<unsigned>(k) <= b0 + c[e]) {
                    sh.bin = 2 * tid + e;
                    sh.before_n = b0;
                    sh.before_m = m0;
                }
                b0 += c[e];
                m0 += m[e];
            }
            __syncthreads();
            k_bin = sh.bin;
            last = find_in_bin(p, row, r, sh, last, k, 0.0, &total_m);
            __syncthreads();
        }
        if (use_p) {
            const double want = fmax(static_cast<double>(tp) * static_cast<double>(total_m), 0.5);
            u64 m0 = mi - m[0] - m[1];
            for (int e = 0; e < 2; ++e) {
                // what top-k cut off the last bin, and the bins behind it, do not count
                const u64 m1 = 2 * tid + e < k_bin ? m0 + m[e] : total_m;
                if (2 * tid + e <= k_bin && static_cast<double>(m0) < want && static_cast<double>(m1) >= want) {
                    sh.bin = 2 * tid + e;
                    sh.before_n = 0;
                    sh.before_m = m0;
                }
                m0 += m[e];
            }
            __syncthreads();
            u64 upto;
            last = find_in_bin(p, row, r, sh, last, 0, want, &upto);
        }
        __syncthreads();
    }
    // mass by blocks of the row, then the block the number falls in
    const auto kept = [&](int i) -> u64 {
        const float z = logit(row, i);
        const double d = r.depth(z);
        if (d >= 32.0 || order_key(z, i) > last) return 0;
        const double w = r.weight(d);
        return w >= r.min_p ? r.mass(w) : 0;
    };
    const int bs = ((V + kThreads - 1) / kThreads + 63) / 64 * 64;
    u64* blk = sh.mass;
    for (int b = wave; b < kThreads; b += kThreads / 64) {
        u64 m = 0;
        for (int i = b * bs + lane; i < min(V, (b + 1) * bs); i += 64) m += kept(i);
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) m += __shfl_xor(m, o, 64);
        if (lane == 0) blk[b] = m;
    }
    __syncthreads();
    const u64 mine = blk[tid], upto = block_scan(mine, sh.part);
    u64 total = 0;
    for (int w = 0; w < kThreads / 64; ++w) total += sh.part[w];
    const float u0 = p.u[blockIdx.x];
    const double target = static_cast<double>(u0 >= 0.f ? fminf(u0, 0.99999994f) : 0.f) * static_cast<double>(total);
    if (mine && static_cast<double>(upto - mine) <= target && static_cast<double>(upto) > target) {
        sh.bin = tid;
        sh.before_m = upto - mine;
    }
    __syncthreads();
    const int b = sh.bin;
    u64 before = sh.before_m;
    for (int i0 = b * bs; i0 < min(V, (b + 1) * bs); i0 += kThreads) {
        const int i = i0 + tid;
        const u64 m = i < min(V, (b + 1) * bs) ? kept(i) : 0;
        const u64 at = before + block_scan(m, sh.part);
        if (m && static_cast<double>(at - m) <= target && static_cast<double>(at) > target) {
            p.idx[blockIdx.x] = i;
            if (p.prob) p.prob[blockIdx.x] = static_cast<float>(static_cast<double>(m) / static_cast<double>(total));
        }
        for (int w = 0; w < kThreads / 64; ++w) before += sh.part[w];
    }
}

size_t sample_workspace_bytes(int rows, int V) {
    (void)rows, (void)V;
    return 256;
}

void sample_rows(int dtype, const void* logits, int64_t ld, int rows, int V, const float* temperature, const int* top_k,
                 const float* top_p, const float* min_p, const float* u, int* idx, float* prob, void* ws, size_t ws_bytes,
                 hipStream_t s) {
    RL_REQUIRE(dtype == RL_Q_F32 || dtype == RL_Q_F16 || dtype == RL_Q_BF16, RL_ERR_UNSUPPORTED,
               "sample_rows: logits must be F32, F16 or BF16");
    RL_REQUIRE(rows >= 0 && V >= 1 && V <= 1 << 24 && ld >= V, RL_ERR_RANGE, "sample_rows: bad sizes");
    if (rows == 0) return;
    RL_REQUIRE(logits && u && idx && ws, RL_ERR_RANGE, "sample_rows: null pointer");
    RL_REQUIRE(aligned(logits, type_bytes(dtype)) && aligned(ws, 16), RL_ERR_RANGE, "sample_rows: misaligned pointer");
    RL_REQUIRE(ws_bytes >= sample_workspace_bytes(rows, V), RL_ERR_RANGE, "sample_rows: workspace too small");
    SampleArgs p{};
    p.logits = logits, p.ld = ld, p.V = V;
    int bits = 0;
    while ((1 << bits) < V) ++bits;
    p.shift = std::min(44, 62 - bits);
    p.temperature = temperature, p.top_k = top_k, p.top_p = top_p, p.min_p = min_p, p.u = u;
    p.idx = idx, p.prob = prob;
    if (dtype == RL_Q_F32)
        hipLaunchKernelGGL(sample_row_kernel<float>, dim3(rows), dim3(kThreads), 0, s, p);
    else if (dtype == RL_Q_F16)
        hipLaunchKernelGGL(sample_row_kernel<_Float16>, dim3(rows), dim3(kThreads), 0, s, p);
    else
        hipLaunchKernelGGL(sample_row_kernel<__bf16>, dim3(rows), dim3(kThreads), 0, s, p);
    check_launch("sample_row_kernel");
}

}  // namespace

extern "C" {

size_t rl_hip_sample_workspace_bytes(int rows, int vocab) { return sample_workspace_bytes(rows, vocab); }

int rl_hip_sample_rows(int dtype, const void* logits, int64_t ld, int rows, int vocab, const float* temperature,
                       const int* top_k, const float* top_p, const float* min_p, const float* u, int* out_idx,
                       float* out_prob, void* workspace, size_t workspace_bytes, void* stream) {
    return guard([&] {
        sample_rows(dtype, logits, ld, rows, vocab, temperature, top_k, top_p, min_p, u, out_idx, out_prob, workspace,
                    workspace_bytes, S(stream));
    });
}

}  // extern "C"
