// sampling.hip -- one token per row of logits: temperature, top-k, top-p, min-p, from given random
// numbers.
//
// With M the row's maximum and w = exp((z - M) / T) = 2^-depth, what top-k and top-p keep is a prefix
// of the order (larger z first, equal z by lower index), so it is told by one element, the last kept.
// That element is found without sorting: a histogram over the depth gives the bin it is in and the
// count and mass before the bin, and only that bin's own elements are put in order.  The token
// follows from the masses of tiles of 512 logits, then from one tile's logits.
// Masses are integers (w in units of 2^-44 of the largest), so that sums are exact in any order and
// every kernel sees the same element the same way.
// Four launches, the first three with many workgroups per row: maxima of the tiles; a histogram (rows
// without top-k and top-p: the tiles' masses already); the tiles' surely kept masses and a list of the
// border bins' elements; the choice.  Up to kSmallK, all that top-k may keep goes to the list and the
// histogram needs no masses; where there are 2 k tiles (or groups of them) it is not needed at all: the k-th
// largest of their maxima is a bound that at least k elements reach, and few others do.  One workgroup per row
// doing all of it took 344 us for one row of 248320 logits, 633 us for 128; now 22 us (the launches and the
// last one's chain of small steps, 10 us) and 102 to 117 us.  128 rows with top-k: 21 us for the one pass
// over 127 MB of logits (6 TB/s), 31 us after it; with top-p alone 150 us, bound by the 64-bit arithmetic
// of the weights (about 24 such instructions a logit, twice for the ones that are kept).
#include <algorithm>
#include <cmath>

#include "paged.h"

using namespace rl;

namespace {

typedef unsigned long long u64;

constexpr int kTile = 512;             // logits of a wave at a time, 8 per lane
constexpr int kBins = 2048;
constexpr double kBinsPerUnit = 44.0;  // bins of depth
constexpr double kDepth = 45.0;        // weights from 2^-45 down are no unit
constexpr int kList = 3000;            // elements of the border bins that are listed
constexpr float kLowest = -3.40282347e38f;
constexpr int kSmallK = 2048;
constexpr int kBound = 512;            // maxima that a wave finds the k-th largest of
constexpr int kRanked = 1024;          // elements that are sorted in shared memory
// ... up to this many are put in order by counting the ones before each.  The whole call, one row of 248320, top-p
// behind a top-k of 20 / 120 / 500 / 1000: with a limit of 1 26 / 37 / 42 / 45 us, of 128 21 / 25 / 32 / 33, of
// 1024 20 / 25 / 44 / 88.
constexpr int kCounted = 128;
constexpr int kPick = 1024;            // threads of the last launch

struct SampleArgs {
    const void* logits;
    int64_t ld;
    int V, shift;  // masses in units of 2^-shift
    int chunk, chunks, tiles;  // logits of a workgroup, workgroups and tiles of a row
    int group, groups;         // tiles of a group, groups of a row: up to kBound
    const float *temperature, *top_p, *min_p, *u;
    const int* top_k;
    int* idx;
    float* prob;
    // workspace, per row
    float* cmax;   // [chunks]
    float* tmax;   // [tiles]
    float* bound;  // [1] at least top_k logits reach it
    unsigned* cnt; // [kBins] + the list's length
    u64* mass;     // [kBins]
    u64* tmass;    // [tiles]
    u64* list;     // [kList] keys
    bool wide;     // rows start at 16 bytes
};

// Larger first, equal ones by index.
__device__ inline u64 order_key(float z, int i) {
    const uint32_t b = __float_as_uint(z);
    const uint32_t up = b >> 31 ? ~b : b | 0x80000000u;
    return static_cast<u64>(~up) << 32 | static_cast<uint32_t>(i);
}
__device__ inline float key_value(u64 key) {
    const uint32_t up = ~static_cast<uint32_t>(key >> 32);
    return __uint_as_float(up >> 31 ? up & 0x7fffffffu : ~up);
}

// -0 becomes +0 (they are equal), NaN -infinity
__device__ inline float clean(float z) {
    z += 0.f;
    return z != z ? -INFINITY : z;
}
// logits i .. i + 7 as they are (NaN passes no comparison), -infinity past the row
template <class T>
__device__ inline void load8(const T* row, int i, int end, bool wide, float (&z)[8]) {
    if (wide && i + 8 <= end) {
        typedef T T8 __attribute__((ext_vector_type(16 / sizeof(T))));
#pragma unroll
        for (int k = 0; k < 8; k += 16 / sizeof(T)) {
            const T8 v = *reinterpret_cast<const T8*>(row + i + k);
#pragma unroll
            for (unsigned e = 0; e < 16 / sizeof(T); ++e) z[k + e] = static_cast<float>(v[e]);
        }
    } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) z[k] = i + k < end ? static_cast<float>(row[i + k]) : -INFINITY;
    }
}

// 2^r for |r| <= 1/2: the series of exp(r ln 2) to the 12th power, to 2^-50
__device__ inline double exp2_small(double r) {
    constexpr double c = 0.693147180559945309417;
    constexpr double c2 = c * c, c3 = c2 * c, c4 = c2 * c2, c5 = c4 * c, c6 = c3 * c3;
    double y = c6 * c6 / 479001600.0;
    y = fma(y, r, c6 * c5 / 39916800.0);
    y = fma(y, r, c5 * c5 / 3628800.0);
    y = fma(y, r, c5 * c4 / 362880.0);
    y = fma(y, r, c4 * c4 / 40320.0);
    y = fma(y, r, c4 * c3 / 5040.0);
    y = fma(y, r, c6 / 720.0);
    y = fma(y, r, c5 / 120.0);
    y = fma(y, r, c4 / 24.0);
    y = fma(y, r, c3 / 6.0);
    y = fma(y, r, c2 / 2.0);
    y = fma(y, r, c);
    return fma(y, r, 1.0);
}

// A row's settings, and what its logits weigh.
struct Row {
    float M;
    double scale, min_p, top_p;
    int shift, top_k;  // 0: off
    bool greedy, use_p;
    __device__ bool filters() const { return top_k || use_p; }
    __device__ bool small_k() const { return top_k && top_k <= kSmallK; }
    __device__ bool bounded(const SampleArgs& p) const { return top_k && top_k <= p.groups / 2; }
    __device__ bool masses() const { return use_p && !small_k(); }  // in the histogram
    // (M - z) / (T ln 2), >= 0; past kDepth for what has no weight at all
    __device__ double depth(float z) const {
        if (z == M) return 0.0;
        if (!(z > -INFINITY) || M == INFINITY) return 1e9;
        return (static_cast<double>(M) - static_cast<double>(z)) * scale;
    }
    // everything below it lies deeper (two steps of z down, for the rounding); never -infinity
    __device__ float below(double depth) const {
        if (M == INFINITY) return M;
        const double z = static_cast<double>(M) - depth / scale;
        return scale > 0.0 && z > -3e38 ? nextafterf(nextafterf(static_cast<float>(z), -INFINITY), -INFINITY) : kLowest;
    }
    // weight 2^-depth = p 2^-n for depths up to kDepth, and in units.  Adding 1.5 2^52 leaves a rounded number in
    // a sum's low bits.
    struct Weight {
        double p;
        int n;
    };
    __device__ static Weight weight(double depth) {
        const double t = depth + 6755399441055744.0;
        return {exp2_small((t - 6755399441055744.0) - depth), static_cast<int>(__double_as_longlong(t))};
    }
    __device__ u64 mass_of(Weight w) const {
        const double unit = __longlong_as_double(static_cast<long long>(1023 + shift - w.n) << 52);
        return static_cast<u64>(__double_as_longlong(fma(w.p, unit, 4503599627370496.0))) & 0xfffffffffffffull;
    }
    __device__ bool enough(Weight w) const {
        return w.p * __longlong_as_double(static_cast<long long>(1023 - w.n) << 52) >= min_p;
    }
    __device__ u64 mass(double depth) const {
        const u64 m = mass_of(weight(fmin(depth, kDepth)));
        return depth < kDepth ? m : 0;
    }
    // with min_p: nothing of what falls under it
    __device__ u64 kept(double depth) const {
        const Weight w = weight(fmin(depth, kDepth));
        const u64 m = mass_of(w);
        return depth < kDepth && (min_p == 0.0 || enough(w)) ? m : 0;
    }
    __device__ static int bin(double depth) { return static_cast<int>(fmin(depth, kDepth) * kBinsPerUnit); }
};

__device__ inline Row settings(const SampleArgs& p, int row, float M) {
    Row r;
    r.M = M;
    const float t = p.temperature ? p.temperature[row] : 1.f;
    r.greedy = !(t > 0.f) || M == -INFINITY;
    r.scale = 1.0 / static_cast<double>(t) * 1.44269504088896340736;
    const float mp = p.min_p ? p.min_p[row] : 0.f;
    r.min_p = mp > 0.f ? fminf(mp, 1.f) : 0.0;
    const int k = p.top_k ? p.top_k[row] : 0;
    r.top_k = k > 0 && k < p.V ? k : 0;
    const float tp = p.top_p ? p.top_p[row] : 1.f;
    r.use_p = tp < 1.f;
    r.top_p = tp;
    r.shift = p.shift;
    return r;
}

// Inclusive sum over the workgroup's kThreads threads, and all of it; every thread calls it.
template <int kThreads, class T>
__device__ inline T block_scan(T v, T* part, T* total = nullptr) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const T x = __shfl_up(v, o, 64);
        if (lane >= o) v += x;
    }
    __syncthreads();
    if (lane == 63) part[wave] = v;
    __syncthreads();
    T before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < kThreads / 64; ++w) {
        const T x = part[w];
        before += w < wave ? x : 0;
        all += x;
    }
    if (total) *total = all;
    return v + before;
}
__device__ inline float block_max(float v, float* part) {
    v = wave_max(v);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    v = part[0];
    for (unsigned w = 1; w < blockDim.x >> 6; ++w) v = fmaxf(v, part[w]);
    return v;
}
__device__ inline float row_max(const SampleArgs& p, int row, float* part) {
    float m = -INFINITY;
    for (int i = threadIdx.x; i < p.chunks; i += blockDim.x) m = fmaxf(m, p.cmax[static_cast<size_t>(row) * p.chunks + i]);
    return block_max(m, part);
}

template <class T>
struct Part {  // a workgroup's part of a row
    int row, chunk, begin, end;
    const T* z;
};
template <class T>
__device__ inline Part<T> part_of(const SampleArgs& p) {
    Part<T> a;
    a.row = blockIdx.x / p.chunks, a.chunk = blockIdx.x % p.chunks;
    a.begin = a.chunk * p.chunk, a.end = min(p.V, a.begin + p.chunk);
    a.z = static_cast<const T*>(p.logits) + a.row * p.ld;
    return a;
}

template <class T>
__global__ __launch_bounds__(256) void sample_max_kernel(SampleArgs p) {
    __shared__ float part_s[4];
    const Part<T> a = part_of<T>(p);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    float m = -INFINITY;
    for (int t = a.begin / kTile + wave; t * kTile < a.end; t += 4) {
        float z[8];
        load8(a.z, t * kTile + 8 * lane, a.end, p.wide, z);
        float x = -INFINITY;  // also of a tile of NaN
#pragma unroll
        for (int e = 0; e < 8; ++e) x = fmaxf(x, z[e]);
        x = wave_max(x);
        m = fmaxf(m, x);
        if (lane == 0) p.tmax[static_cast<size_t>(a.row) * p.tiles + t] = x;
    }
    m = block_max(m, part_s);
    if (threadIdx.x == 0) p.cmax[static_cast<size_t>(a.row) * p.chunks + a.chunk] = m;
    // the next launches' histogram and list start empty
    const size_t row = a.row;
    for (int i = a.chunk * 256 + threadIdx.x; i <= kBins; i += 256 * p.chunks) {
        p.cnt[row * (kBins + 1) + i] = 0;
        if (i < kBins) p.mass[row * kBins + i] = 0;
    }
}

__device__ inline u64 wave_sum64(u64 v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

// The k-th largest of the maxima of groups of tiles, or a little less: at least k logits reach it.  A wave's
// work, bit by bit from the top; 11 bits behind the exponent's are enough.
__device__ float kth_max(const SampleArgs& p, int row, int k) {
    const int lane = threadIdx.x & 63, per = p.group;
    uint32_t v[kBound / 64];
#pragma unroll
    for (int i = 0; i < kBound / 64; ++i) {
        const int g = 64 * i + lane;
        float m = g * per < p.tiles ? p.tmax[static_cast<size_t>(row) * p.tiles + g * per] : -INFINITY;
        for (int t = g * per + 1; per > 1 && t < min(p.tiles, (g + 1) * per); ++t)
            m = fmaxf(m, p.tmax[static_cast<size_t>(row) * p.tiles + t]);
        const uint32_t b = __float_as_uint(m);
        v[i] = b >> 31 ? ~b : b | 0x80000000u;  // ordered as the values
    }
    uint32_t x = 0;
    for (int bit = 31; bit >= 12; --bit) {
        const uint32_t y = x | 1u << bit;
        int n = 0;
#pragma unroll
        for (int i = 0; i < kBound / 64; ++i) n += __popcll(__ballot(v[i] >= y));
        if (n >= k) x = y;
    }
    return __uint_as_float(x >> 31 ? x & 0x7fffffffu : ~x);
}

template <class T>
__global__ __launch_bounds__(256) void sample_hist_kernel(SampleArgs p) {
    __shared__ float part_s[4];
    __shared__ unsigned cnt_s[kBins];
    __shared__ u64 mass_s[kBins];
    const Part<T> a = part_of<T>(p);
    Row r = settings(p, a.row, 0.f);
    if (r.bounded(p)) {
        if (a.chunk == 0 && threadIdx.x < 64) {
            const float x = kth_max(p, a.row, r.top_k);
            if (threadIdx.x == 0) p.bound[a.row] = fmaxf(x, kLowest);
        }
        return;
    }
    r = settings(p, a.row, row_max(p, a.row, part_s));
    if (r.greedy) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const float low = r.below(kDepth);
    if (!r.filters()) {
        for (int t = a.begin / kTile + wave; t * kTile < a.end; t += 4) {
            float z[8];
            load8(a.z, t * kTile + 8 * lane, a.end, p.wide, z);
            u64 m = 0;
#pragma unroll
            for (int e = 0; e < 8; ++e) m += r.kept(r.depth(z[e]));
            m = wave_sum64(m);
            if (lane == 0) p.tmass[static_cast<size_t>(a.row) * p.tiles + t] = m;
        }
        return;
    }
    const bool masses = r.masses();
    for (int i = threadIdx.x; i < kBins; i += 256) {
        cnt_s[i] = 0;
        if (masses) mass_s[i] = 0;
    }
    __syncthreads();
    float z[8], next[8];
    load8(a.z, a.begin + 8 * threadIdx.x, a.end, p.wide, next);
    for (int i = a.begin + 8 * threadIdx.x; i < a.end; i += 8 * 256) {
        bool any = false;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            z[e] = next[e];
            any |= z[e] >= low;
        }
        load8(a.z, i + 8 * 256, a.end, p.wide, next);
        if (!__any(any)) continue;
        // all eight side by side: the series is one long chain
        double d[8];
        u64 m[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) d[e] = fmin(r.depth(z[e]), kDepth);
        if (masses) {
#pragma unroll
            for (int e = 0; e < 8; ++e) m[e] = r.mass_of(r.weight(d[e]));
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            if (d[e] >= kDepth) continue;
            const int bin = r.bin(d[e]);
            if (r.top_k) atomicAdd(&cnt_s[bin], 1u);
            if (masses) atomicAdd(&mass_s[bin], m[e]);
        }
    }
    __syncthreads();
    const size_t row = a.row;
    for (int i = threadIdx.x; i < kBins; i += 256) {
        if (r.top_k && cnt_s[i]) atomicAdd(&p.cnt[row * (kBins + 1) + i], cnt_s[i]);
        if (masses && mass_s[i]) atomicAdd(&p.mass[row * kBins + i], mass_s[i]);
    }
}

// The bins in which top-k and top-p end: everything before `sure` is kept, nothing past `top`, and top-k
// itself ends in k_bin (kBins: it cuts nothing off).
struct Borders {
    int sure, top, k_bin;
    unsigned k_before;  // elements before k_bin
    u64 k_mass, all;    // mass before k_bin (with top-p), of all bins
};
struct BorderShared {
    unsigned cpart[16];
    u64 part[16];
    int k_bin, lo, hi;
    unsigned k_before;
    u64 k_mass, k_own;
};
template <int kThreads>
__device__ Borders borders(const SampleArgs& p, int row_, const Row& r, BorderShared& sh) {
    constexpr int E = kBins / kThreads;
    const int tid = threadIdx.x;
    const size_t row = row_;
    unsigned c[E], cs = 0, ct = 0;
    u64 m[E], ms = 0, mt = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        c[e] = r.top_k ? p.cnt[row * (kBins + 1) + tid * E + e] : 0;
        m[e] = r.masses() ? p.mass[row * kBins + tid * E + e] : 0;
        cs += c[e];
        ms += m[e];
    }
    if (tid == 0) sh.k_bin = kBins, sh.lo = sh.hi = kBins;
    const unsigned c0 = block_scan<kThreads>(cs, sh.cpart, &ct) - cs;
    const u64 m0 = block_scan<kThreads>(ms, sh.part, &mt) - ms;
    if (r.top_k && static_cast<unsigned>(r.top_k) < ct) {
        unsigned cb = c0;
        u64 mb = m0;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            if (cb < static_cast<unsigned>(r.top_k) && static_cast<unsigned>(r.top_k) <= cb + c[e]) {
                sh.k_bin = tid * E + e;
                sh.k_before = cb;
                sh.k_mass = mb;
                sh.k_own = m[e];
            }
            cb += c[e];
            mb += m[e];
        }
    }
    __syncthreads();
    Borders b;
    b.k_bin = sh.k_bin;
    b.k_before = sh.k_before;
    b.k_mass = sh.k_mass;
    b.all = mt;
    b.sure = b.top = b.k_bin;
    if (r.small_k()) {
        b.sure = 0;  // all of it is listed
    } else if (r.use_p) {
        // top-k leaves between k_mass and that with all of its last bin
        const u64 least = b.k_bin < kBins ? b.k_mass : mt, most = b.k_bin < kBins ? b.k_mass + sh.k_own : mt;
        const double lo = fmax(r.top_p * static_cast<double>(least), 0.5), hi = fmax(r.top_p * static_cast<double>(most), 0.5);
        u64 mb = m0;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const double x = static_cast<double>(mb), y = static_cast<double>(mb + m[e]);
            if (x < lo && y >= lo) sh.lo = tid * E + e;
            if (x < hi && y >= hi) sh.hi = tid * E + e;
            mb += m[e];
        }
        __syncthreads();
        b.sure = min(sh.lo, b.k_bin);
        b.top = min(sh.hi, b.k_bin);
    }
    return b;
}

template <class T>
__global__ __launch_bounds__(256) void sample_list_kernel(SampleArgs p) {
    __shared__ float part_s[4];
    __shared__ BorderShared sh;
    __shared__ uint16_t idx_s[kList];  // within the chunk
    __shared__ float2 few_s[4][kTile];  // logit, place in the chunk
    __shared__ int n_s, at_s;
    const Part<T> a = part_of<T>(p);
    Row r = settings(p, a.row, 0.f);
    Borders b{0, kBins, kBins, 0, 0, 0};
    float low;
    if (!r.filters()) return;
    if (r.bounded(p)) {
        if (r.greedy) return;
        low = p.bound[a.row];
    } else {
        r = settings(p, a.row, row_max(p, a.row, part_s));
        if (r.greedy) return;
        b = borders<256>(p, a.row, r, sh);
        const int last = b.k_bin < kBins ? b.k_bin : b.top;  // the last bin looked at
        low = r.below(fmin((last + 1) / kBinsPerUnit, kDepth));
    }
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const size_t row = a.row;
    if (threadIdx.x == 0) n_s = 0;
    __syncthreads();
    // the wave's tiles (at most 32), one per lane: those whose maximum reaches it
    const int t0 = a.begin / kTile + wave, mine = t0 + 4 * lane;
    const bool have = mine * kTile < a.end;
    const bool reach = have && p.tmax[row * p.tiles + mine] >= low;
    if (b.sure && have && !reach) p.tmass[row * p.tiles + mine] = 0;
    unsigned long long todo = __ballot(reach);
    float next[8];
    if (todo) load8(a.z, (t0 + 4 * (__ffsll(todo) - 1)) * kTile + 8 * lane, a.end, p.wide, next);
    while (todo) {
        const int t = t0 + 4 * (__ffsll(todo) - 1), i = t * kTile + 8 * lane;
        todo &= todo - 1;
        float z[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) z[e] = next[e];
        if (todo) load8(a.z, (t0 + 4 * (__ffsll(todo) - 1)) * kTile + 8 * lane, a.end, p.wide, next);
        if (b.sure == 0) {
            // nothing is kept unseen; the list may hold some past the border
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (z[e] >= low) {
                    const int at = atomicAdd(&n_s, 1);
                    if (at < kList) idx_s[at] = static_cast<uint16_t>(i + e - a.begin);
                }
            continue;
        }
        // what reaches it, close together: few of a tile do
        int own = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) own += z[e] >= low;
        int upto = own;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int x = __shfl_up(upto, o, 64);
            upto += lane >= o ? x : 0;
        }
        const int n = __builtin_amdgcn_readlane(upto, 63);
        int at = upto - own;
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (z[e] >= low) few_s[wave][at++] = make_float2(z[e], __int_as_float(i + e - a.begin));
        __builtin_amdgcn_wave_barrier();
        u64 m = 0;
        for (int k = lane; k < n; k += 64) {
            const float2 x = few_s[wave][k];
            const double d = r.depth(x.x);
            const int bin = r.bin(d);
            const u64 w = r.kept(d);
            if (bin < b.sure) {
                m += w;
            } else if (d < kDepth && (bin <= b.top || bin == b.k_bin)) {
                const int to = atomicAdd(&n_s, 1);
                if (to < kList) idx_s[to] = static_cast<uint16_t>(__float_as_int(x.y));
            }
        }
        __builtin_amdgcn_wave_barrier();
        m = wave_sum64(m);
        if (lane == 0) p.tmass[row * p.tiles + t] = m;
    }
    __syncthreads();
    if (threadIdx.x == 0 && n_s) at_s = static_cast<int>(atomicAdd(&p.cnt[row * (kBins + 1) + kBins], static_cast<unsigned>(n_s)));
    __syncthreads();
    for (int i = threadIdx.x; i < min(n_s, kList) && at_s + i < kList; i += 256) {
        const int at = a.begin + idx_s[i];
        p.list[row * kList + at_s + i] = order_key(clean(static_cast<float>(a.z[at])), at);
    }
}

struct PickShared {
    BorderShared b;
    float fpart[kPick / 64];
    unsigned cpart[kPick / 64];
    u64 part[kPick / 64];
    u64 key[kList], w[kList];       // the list and its masses
    unsigned cnt[kBins];
    u64 mass[kBins];
    u64 range[kPick];               // masses of equal shares of the row
    u64 sub[kRanked], sub_w[kRanked];
    u64 dig_n[256], dig_m[256];
    u64 found_key, found_upto, before_m;
    unsigned before_n;
    int digit, n, at, bin;
};

// How many of n keys are less than `key`, and their masses; the arrays are filled up to a multiple of 8 with
// ~0 (eight at a time are read side by side).
__device__ inline void count_less(const u64* keys, const u64* w, int n, u64 key, unsigned* less, u64* mass) {
    for (int j = 0; j < n; j += 8) {
        u64 k[8], m[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) k[e] = keys[j + e], m[e] = w[j + e];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            *less += k[e] < key;
            *mass += k[e] < key ? m[e] : 0;
        }
    }
}

// Which of the elements that `each` hands out ends the prefix: the one with `want_n` up to it (before_n stand
// before all of them), or else the first up to which want_m of mass stands.  The key of it, *upto the mass up to it.
template <class Each, class Mass>
__device__ u64 find_last(PickShared& sh, Mass mass, Each each, unsigned before_n, u64 before_m, unsigned want_n, double want_m, u64* upto) {
    __syncthreads();
    if (threadIdx.x == 0) sh.n = 0;
    __syncthreads();
    each([&](u64 key, u64 m) {
        const int at = atomicAdd(&sh.n, 1);
        if (at < kRanked) sh.sub[at] = key, sh.sub_w[at] = m;
    });
    __syncthreads();
    const int n_sub = sh.n;
    if (n_sub <= kRanked) {
        const int t = threadIdx.x;
        if (n_sub <= kCounted) {
            // few: each against every other
            if (t >= n_sub && t < n_sub + 8) sh.sub[t] = ~0ull, sh.sub_w[t] = 0;
            __syncthreads();
            if (t < n_sub) {
                const u64 key = sh.sub[t], m = sh.sub_w[t];
                unsigned n = before_n;
                u64 before = before_m;
                count_less(sh.sub, sh.sub_w, n_sub, key, &n, &before);
                const bool hit = want_n ? n + 1 == want_n
                                        : static_cast<double>(before) < want_m && static_cast<double>(before + m) >= want_m;
                if (hit) {
                    sh.found_key = key;
                    sh.found_upto = before + m;
                }
            }
            __syncthreads();
            *upto = sh.found_upto;
            return sh.found_key;
        }
        // in order (bitonic sort, a key per thread: partners of the same wave by lane moves), the masses before each
        u64 key = t < n_sub ? sh.sub[t] : ~0ull;
        for (int k = 2; k <= kRanked; k *= 2) {
            for (int j = k / 2; j > 0; j /= 2) {
                u64 other;
                if (j >= 64) {
                    __syncthreads();
                    sh.sub[t] = key;
                    __syncthreads();
                    other = sh.sub[t ^ j];
                } else {
                    other = __shfl_xor(key, j, 64);
                }
                const bool least = ((t & j) == 0) == ((t & k) == 0);
                key = (key < other) == least ? key : other;
            }
        }
        const u64 m = t < n_sub ? mass(key) : 0;
        const u64 upto_t = block_scan<kPick>(m, sh.part) + before_m;
        const bool hit = want_n ? before_n + t + 1 == want_n
                                : static_cast<double>(upto_t - m) < want_m && static_cast<double>(upto_t) >= want_m;
        if (t < n_sub && hit) {
            sh.found_key = key;
            sh.found_upto = upto_t;
        }
        __syncthreads();
        *upto = sh.found_upto;
        return sh.found_key;
    }
    // many (flat or repeated logits): eight bits of the key at a time
    u64 prefix = 0;
    for (int shift = 56; shift >= 0; shift -= 8) {
        __syncthreads();
        if (threadIdx.x < 256) sh.dig_n[threadIdx.x] = sh.dig_m[threadIdx.x] = 0;
        __syncthreads();
        each([&](u64 key, u64 m) {
            if (shift < 56 && (key ^ prefix) >> (shift + 8)) return;
            atomicAdd(&sh.dig_n[key >> shift & 255], 1ull);
            atomicAdd(&sh.dig_m[key >> shift & 255], m);
        });
        __syncthreads();
        u64 n = 0, m = 0;
        if (threadIdx.x < 256) n = sh.dig_n[threadIdx.x], m = sh.dig_m[threadIdx.x];
        const u64 ni = block_scan<kPick>(n, sh.part) + before_n, mi = block_scan<kPick>(m, sh.part) + before_m;
        const bool hit = want_n ? ni - n < want_n && want_n <= ni
                                : static_cast<double>(mi - m) < want_m && static_cast<double>(mi) >= want_m;
        if (n && hit) {
            sh.digit = threadIdx.x;
            sh.before_n = static_cast<unsigned>(ni - n);
            sh.before_m = mi - m;
            sh.found_upto = mi;
        }
        __syncthreads();
        prefix |= static_cast<u64>(sh.digit) << shift;
        before_n = sh.before_n;
        before_m = sh.before_m;
    }
    *upto = sh.found_upto;
    return prefix;
}

template <class T>
__global__ __launch_bounds__(kPick) void sample_pick_kernel(SampleArgs p) {
    __shared__ PickShared sh;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const size_t row = blockIdx.x;
    const T* zr = static_cast<const T*>(p.logits) + row * p.ld;
    // asked for before they are known to be there
    const u64 first = p.list[row * kList + tid];
    const unsigned n_all = p.cnt[row * (kBins + 1) + kBins];
    const float u0 = p.u[row];
    const Row r = settings(p, row, row_max(p, row, sh.fpart));
    if (r.greedy) {
        // the first chunk with the maximum, its first such logit
        if (tid == 0) sh.at = p.chunks, sh.n = p.V;
        __syncthreads();
        for (int c = tid; c < p.chunks; c += kPick)
            if (p.cmax[row * p.chunks + c] == r.M) atomicMin(&sh.at, c);
        __syncthreads();
        const int begin = sh.at * p.chunk, end = min(p.V, begin + p.chunk);
        for (int i = begin + tid; i < end; i += kPick)
            if (clean(static_cast<float>(zr[i])) == r.M) {
                atomicMin(&sh.n, i);
                break;
            }
        __syncthreads();
        if (tid == 0) {
            p.idx[row] = r.M == -INFINITY ? 0 : sh.n;
            if (p.prob) p.prob[row] = r.M == -INFINITY ? 0.f : 1.f;
        }
        return;
    }
    // shares of whole tiles, one per thread
    const int per = (p.tiles + kPick - 1) / kPick, share = per * kTile;
    u64 last = ~0ull;
    bool listed = true;  // the tiles' masses and the list hold everything
    int n_list = 0;
    int sure = kBins;  // bins before it are in the tiles' masses
    if (r.filters()) {
        listed = n_all <= kList;
        n_list = listed ? n_all : 0;
        for (int i = tid; i < n_list; i += kPick) {
            sh.key[i] = i < kPick ? first : p.list[row * kList + i];
            sh.w[i] = r.mass(r.depth(key_value(sh.key[i])));
        }
        const auto mass_of = [&](u64 key) { return r.mass(r.depth(key_value(key))); };
        // the elements of some bins with keys up to one: from the list, or where that is too short from the row
        const auto each_of = [&](int bin_lo, int bin_hi, u64 upto, auto f) {
            if (listed) {
                for (int i = tid; i < n_list; i += kPick) {
                    const u64 key = sh.key[i];
                    const int bin = r.bin(r.depth(key_value(key)));
                    if (bin >= bin_lo && bin <= bin_hi && key <= upto) f(key, sh.w[i]);
                }
            } else {
                const float low = r.below(fmin((bin_hi + 1) / kBinsPerUnit, kDepth));
                for (int i = tid; i < p.V; i += kPick) {
                    const float z = clean(static_cast<float>(zr[i]));
                    if (!(z >= low)) continue;
                    const double d = r.depth(z);
                    if (d >= kDepth || r.bin(d) < bin_lo || r.bin(d) > bin_hi) continue;
                    const u64 key = order_key(z, i);
                    if (key <= upto) f(key, r.mass(d));
                }
            }
        };
        if (r.small_k() && listed && n_list <= kCounted) {
            // few: each against every other gives both borders
            sure = 0;
            if (tid == 0) sh.found_key = 0, sh.found_upto = 0;
            if (tid >= n_list && tid < n_list + 8) sh.key[tid] = ~0ull, sh.w[tid] = 0;
            __syncthreads();
            u64 key = 0, before = 0;
            unsigned rank = 0;
            if (tid < n_list) {
                key = sh.key[tid];
                count_less(sh.key, sh.w, n_list, key, &rank, &before);
                if (rank + 1 == static_cast<unsigned>(min(r.top_k, n_list))) sh.found_upto = before + sh.w[tid];
            }
            __syncthreads();
            const double want = fmax(r.top_p * static_cast<double>(sh.found_upto), 0.5);
            if (tid < n_list && rank < static_cast<unsigned>(r.top_k) && (!r.use_p || static_cast<double>(before) < want)) atomicMax(&sh.found_key, key);
            __syncthreads();
            if (n_list) last = sh.found_key;
        } else if (r.small_k()) {
            // a histogram of the list, top-k's border in it, then top-p's in what that leaves
            sure = 0;
            for (int i = tid; i < kBins; i += kPick) sh.cnt[i] = 0, sh.mass[i] = 0;
            if (tid == 0) sh.bin = kBins;
            __syncthreads();
            each_of(0, kBins, ~0ull, [&](u64 key, u64 m) {
                const int bin = r.bin(r.depth(key_value(key)));
                atomicAdd(&sh.cnt[bin], 1u);
                atomicAdd(&sh.mass[bin], m);
            });
            __syncthreads();
            constexpr int E = kBins / kPick;
            unsigned c[E], cs = 0, ct;
            u64 m[E], ms = 0, left;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                cs += c[e] = sh.cnt[tid * E + e];
                ms += m[e] = sh.mass[tid * E + e];
            }
            const unsigned c0 = block_scan<kPick>(cs, sh.cpart, &ct) - cs;
            const u64 m0 = block_scan<kPick>(ms, sh.part, &left) - ms;
            int k_bin = kBins;
            if (static_cast<unsigned>(r.top_k) <= ct) {  // fewer: the list has all that weighs anything
                unsigned cb = c0;
                u64 mb = m0;
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    if (cb < static_cast<unsigned>(r.top_k) && static_cast<unsigned>(r.top_k) <= cb + c[e]) {
                        sh.bin = tid * E + e;
                        sh.before_n = cb;
                        sh.before_m = mb;
                    }
                    cb += c[e];
                    mb += m[e];
                }
                __syncthreads();
                k_bin = sh.bin;
                last = find_last(sh, mass_of, [&](auto f) { each_of(k_bin, k_bin, ~0ull, f); }, sh.before_n, sh.before_m, r.top_k, 0.0, &left);
            }
            if (r.use_p) {
                const double want = fmax(r.top_p * static_cast<double>(left), 0.5);
                __syncthreads();
                u64 mb = m0;
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const int bin = tid * E + e;
                    const u64 me = bin < k_bin ? mb + m[e] : left;
                    if (bin <= k_bin && static_cast<double>(mb) < want && static_cast<double>(me) >= want) {
                        sh.bin = bin;
                        sh.before_m = mb;
                    }
                    mb += m[e];
                }
                __syncthreads();
                const int p_bin = sh.bin;
                u64 upto;
                last = find_last(sh, mass_of, [&](auto f) { each_of(p_bin, p_bin, last, f); }, 0, sh.before_m, 0, want, &upto);
            }
        } else {
            const Borders b = borders<kPick>(p, row, r, sh.b);
            sure = b.sure;
            u64 left = b.all, before = 0;
            if (b.k_bin < kBins)
                last = find_last(sh, mass_of, [&](auto f) { each_of(b.k_bin, b.k_bin, ~0ull, f); }, b.k_before, b.k_mass, r.top_k, 0.0, &left);
            if (r.use_p) {
                // the bins from b.sure to b.top hold the border; the mass before them
                const double want = fmax(r.top_p * static_cast<double>(left), 0.5);
                u64 m = 0;
                for (int i = tid; i < b.sure; i += kPick) m += p.mass[row * kBins + i];
                block_scan<kPick>(m, sh.part, &before);
                u64 upto;
                last = find_last(sh, mass_of, [&](auto f) { each_of(b.sure, b.top, last, f); }, 0, before, 0, want, &upto);
            }
        }
        __syncthreads();
    }
    sh.range[tid] = 0;
    __syncthreads();
    const auto kept = [&](int i) -> u64 {
        const float z = clean(static_cast<float>(zr[i]));
        return order_key(z, i) <= last ? r.kept(r.depth(z)) : 0;
    };
    if (listed) {
        u64 m = 0;
        if (sure > 0)
            for (int t = tid * per; t < min(p.tiles, (tid + 1) * per); ++t) m += p.tmass[row * p.tiles + t];
        sh.range[tid] = m;
        __syncthreads();
        for (int i = tid; i < n_list; i += kPick) {
            const u64 key = sh.key[i];
            if (key <= last) atomicAdd(&sh.range[static_cast<uint32_t>(key) / share], r.kept(r.depth(key_value(key))));
        }
    } else {
        for (int t = wave; t < p.tiles; t += kPick / 64) {
            u64 m = 0;
            for (int i = t * kTile + lane; i < min(p.V, (t + 1) * kTile); i += 64) m += kept(i);
            m = wave_sum64(m);
            if (lane == 0) atomicAdd(&sh.range[t / per], m);
        }
    }
    __syncthreads();
    const u64 mine = sh.range[tid];
    u64 total;
    const u64 upto = block_scan<kPick>(mine, sh.part, &total);
    const double target = static_cast<double>(u0 >= 0.f ? fminf(u0, 0.99999994f) : 0.f) * static_cast<double>(total);
    if (mine && static_cast<double>(upto - mine) <= target && static_cast<double>(upto) > target) {
        sh.at = tid;
        sh.before_m = upto - mine;
    }
    __syncthreads();
    // the share's logits, a run of them per thread
    const int begin = sh.at * share, run = (share + kPick - 1) / kPick;
    const int i0 = begin + tid * run, i1 = min(p.V, min(begin + share, i0 + run));
    u64 m = 0;
    for (int i = i0; i < i1; ++i) m += kept(i);
    const u64 before = sh.before_m;
    u64 at = block_scan<kPick>(m, sh.part) + before - m;
    if (m && static_cast<double>(at) <= target && static_cast<double>(at + m) > target) {
        for (int i = i0; i < i1; ++i) {
            const u64 w = kept(i);
            at += w;
            if (w && static_cast<double>(at) > target) {
                p.idx[row] = i;
                if (p.prob) p.prob[row] = static_cast<float>(static_cast<double>(w) / static_cast<double>(total));
                break;
            }
        }
    }
}

// Logits of a workgroup: about 2048 workgroups for all rows, whole rounds of 256 threads x 8, up to 65536.
// 128 rows of 248320, mixed settings / top-p / top-k and top-p: 1024 workgroups 142 / 147 / 51 us, 2048 119 / 145 / 57,
// 4096 110 / 156 / 58 (every workgroup adds its bins to the row's histogram).
int chunk_of(int rows, int V) {
    const int64_t want = static_cast<int64_t>(rows) * V / 2048;
    return static_cast<int>(std::min<int64_t>(std::max<int64_t>((want + 2047) / 2048, V / 512 / 2048 + 1), 32)) * 2048;
}
struct SampleSpace {
    size_t cmax, tmax, bound, cnt, mass, tmass, list, bytes;
};
SampleSpace sample_space(int rows, int V, int chunks, int tiles) {
    SampleSpace s;
    const size_t n = rows;
    s.mass = 0;
    s.tmass = s.mass + n * kBins * 8;
    s.list = s.tmass + n * tiles * 8;
    s.cnt = s.list + n * kList * 8;
    s.cmax = s.cnt + n * (kBins + 1) * 4;
    s.tmax = s.cmax + n * chunks * 4;
    s.bound = s.tmax + n * tiles * 4;
    s.bytes = (s.bound + n * 4 + 255) / 256 * 256;
    return s;
}

size_t sample_workspace_bytes(int rows, int V) {
    if (rows < 1 || V < 1) return 256;
    const int chunk = chunk_of(rows, V);
    return sample_space(rows, V, (V + chunk - 1) / chunk, (V + kTile - 1) / kTile).bytes;
}

template <class T>
void launch_sample(const SampleArgs& p, int rows, hipStream_t s) {
    const dim3 grid(rows * p.chunks);
    hipLaunchKernelGGL(sample_max_kernel<T>, grid, dim3(256), 0, s, p);
    check_launch("sample_max_kernel");
    hipLaunchKernelGGL(sample_hist_kernel<T>, grid, dim3(256), 0, s, p);
    check_launch("sample_hist_kernel");
    if (p.top_k || p.top_p) {
        hipLaunchKernelGGL(sample_list_kernel<T>, grid, dim3(256), 0, s, p);
        check_launch("sample_list_kernel");
    }
    hipLaunchKernelGGL(sample_pick_kernel<T>, dim3(rows), dim3(kPick), 0, s, p);
    check_launch("sample_pick_kernel");
}

void sample_rows(int dtype, const void* logits, int64_t ld, int rows, int V, const float* temperature, const int* top_k,
                 const float* top_p, const float* min_p, const float* u, int* idx, float* prob, void* ws, size_t ws_bytes,
                 hipStream_t s) {
    RL_REQUIRE(dtype == RL_Q_F32 || dtype == RL_Q_F16 || dtype == RL_Q_BF16, RL_ERR_UNSUPPORTED,
               "sample_rows: logits must be F32, F16 or BF16");
    RL_REQUIRE(rows >= 0 && rows <= 1 << 20 && V >= 1 && V <= 1 << 24 && ld >= V, RL_ERR_RANGE, "sample_rows: bad sizes");
    if (rows == 0) return;
    RL_REQUIRE(logits && u && idx && ws, RL_ERR_RANGE, "sample_rows: null pointer");
    RL_REQUIRE(aligned(logits, type_bytes(dtype)) && aligned(ws, 16), RL_ERR_RANGE, "sample_rows: misaligned pointer");
    RL_REQUIRE(ws_bytes >= sample_workspace_bytes(rows, V), RL_ERR_RANGE, "sample_rows: workspace too small");
    SampleArgs p{};
    p.logits = logits, p.ld = ld, p.V = V;
    int bits = 0;
    while ((1 << bits) < V) ++bits;
    p.shift = std::min(44, 62 - bits);
    p.chunk = chunk_of(rows, V);
    p.chunks = (V + p.chunk - 1) / p.chunk;
    p.tiles = (V + kTile - 1) / kTile;
    p.group = (p.tiles + kBound - 1) / kBound;
    p.groups = (p.tiles + p.group - 1) / p.group;
    p.wide = aligned(logits, 16) && ld * type_bytes(dtype) % 16 == 0;
    p.temperature = temperature, p.top_k = top_k, p.top_p = top_p, p.min_p = min_p, p.u = u;
    p.idx = idx, p.prob = prob;
    const SampleSpace sp = sample_space(rows, V, p.chunks, p.tiles);
    char* w = static_cast<char*>(ws);
    p.mass = reinterpret_cast<u64*>(w + sp.mass);
    p.tmass = reinterpret_cast<u64*>(w + sp.tmass);
    p.list = reinterpret_cast<u64*>(w + sp.list);
    p.cnt = reinterpret_cast<unsigned*>(w + sp.cnt);
    p.cmax = reinterpret_cast<float*>(w + sp.cmax);
    p.tmax = reinterpret_cast<float*>(w + sp.tmax);
    p.bound = reinterpret_cast<float*>(w + sp.bound);
    if (dtype == RL_Q_F32)
        launch_sample<float>(p, rows, s);
    else if (dtype == RL_Q_F16)
        launch_sample<_Float16>(p, rows, s);
    else
        launch_sample<__bf16>(p, rows, s);
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
