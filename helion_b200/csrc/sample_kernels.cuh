// Drawing tokens from logits with given random numbers.
//
//   weight_j = exp((l_j - max l) / temperature)
//   order    by logit, larger first; of equal logits the lower index first. Every filter keeps a prefix of it:
//     top_k  the k first;
//     top_p  those whose predecessors' weights among the top_k sum to at most top_p of the top_k's sum (the first always);
//     min_p  those with weight_j >= min_p.
//   token    the first index j, in vocabulary order, whose kept weights up to and including j sum to more than
//            u times the kept weights' sum.
//
// Weights and their sums are 64 bits: with 32, a draw that falls within 1e-7 of a boundary between two of 100000 tokens
// - one in a hundred rows - would go to the wrong one. A NaN counts as -inf; a row with nothing above -inf gives
// token -1; among +inf all weight is shared equally; a temperature that is not positive takes the first maximum.
//
// A prefix of the order is a threshold on the logit and a number of ties, and both are found by counting:
//   1. a cluster of 1..8 CTAs takes a row; each keeps its slice in shared memory, so the logits are read once;
//   2. a histogram of (max - l) / temperature brackets the threshold: exactly for top_k, and for top_p between bounds,
//      since a bin's weights are known to the bin's width from its count;
//   3. where the top_k's bracket and all above it hold at most 1024 logits, the first CTA collects and sorts those and
//      draws from the list (sample_listed); else, for top_p, one pass sums all weights, and those above the bracket, in
//      64 bits;
//   4. histograms over the ordered bits of the logits inside the bracket narrow it to a single value;
//      only elements inside the bracket need their weight for that;
//   5. one pass sums the kept weights by warp, the sums find the warp that holds u times the total, and that warp
//      finds the index.
// Histograms are counts (integer atomics in shared memory), lists are sorted and sums have a fixed order: the same tokens
// on every run. Large batches of bf16 rows are drawn by sample_values_kernel, below.
//
// The bytes are nothing: 64 x 128256 fp32 is 33 MB, 5 us. What bounds a row is the chain of its steps, each a scan, a block
// scan and a barrier of the cluster with every CTA reading the others' 4 KB of bins: 3 to 5 us, 33 us in all for one row
// with filters of every kind (51 without the list), 25 with a top_k alone. 64 such rows take 93 us (117 without the list):
// about 200 of the 296 CTAs that would fit are resident, since clusters of 8 do not fill every GPC. CTAs of 1024 threads
// in clusters of 4 took the same; slices re-read from L2 instead of kept in shared memory 13 to 40 % more.
#pragma once

#include "ptx.cuh"
#include "vec.cuh"

namespace lce {

constexpr int kSampleThreads = 512;
constexpr int kSampleWarps = kSampleThreads / 32;
constexpr int kSampleMaxCluster = 8;
constexpr int kSampleTable = 512;

struct SampleParams {
    const float* uniform;      // [rows]
    const float* temperature;  // [rows] or nullptr: the scalar
    const void* top_k;         // [rows] int32 / int64 or nullptr
    const float* top_p;
    const float* min_p;
    float temperature_all, top_p_all, min_p_all;
    long long top_k_all;
    int top_k_i64;
    long long* token;
    float* logprob;  // or nullptr
};

// The order-preserving unsigned form of a logit that is no NaN: the bits of the float, without those that the type
// leaves empty, so that neighbouring logits have neighbouring keys.
template <class T>
struct SampleKey {
    static constexpr int kLow = std::is_same<T, __nv_bfloat16>::value ? 16 : (std::is_same<T, __half>::value ? 13 : 0);
    static constexpr uint32_t kZero = 0x80000000u >> kLow;
    static constexpr uint32_t kNone = 0x007fffffu >> kLow;  // -inf
    static __device__ __forceinline__ uint32_t of(float v) {
        const uint32_t u = __float_as_uint(v + 0.f);  // -0 and +0 are equal logits
        return (u ^ (static_cast<uint32_t>(static_cast<int32_t>(u) >> 31) | 0x80000000u)) >> kLow;
    }
    static __device__ __forceinline__ float value(uint32_t key) {
        const uint32_t k = key << kLow;
        return __uint_as_float(key >= kZero ? k & 0x7fffffffu : ~(k | ((1u << kLow) - 1u)));
    }
    // Bounds for comparing logits as floats: the key below zero's belongs to -0, which no logit has but all zeros equal.
    static __device__ __forceinline__ float at_least(uint32_t key) { return value(key == kZero - 1 ? kZero : key); }
    static __device__ __forceinline__ float at_most(uint32_t key) { return value(key == kZero - 1 ? kZero - 2 : key); }
};

// Bins of a histogram, and how many of them the first one has per unit of (max - l) / temperature (32 units in all).
// Every CTA reads all the others' bins, at some 30 bytes per ns through the cluster: with 2048 bins a round on 8 CTAs
// took 4.8 us, 2.2 of them for that. With 512, logits of 16 bits around zero took more rounds (256 x 128256 bf16: 247 us
// against 217).
constexpr int kSampleBins = 1024;
constexpr int kSampleBinsPerThread = kSampleBins / kSampleThreads;
constexpr float kSampleBinsPerNat = kSampleBins / 32;
constexpr double kSampleBinStep = 0.969233234476344055;  // exp(-1 / kSampleBinsPerNat)

// What a CTA of the cluster tells the others at an exchange.
struct SampleSlot {
    double d[3];
    long long n;
    uint32_t u, pad;
};

struct SampleShared {
    uint32_t hist[2][kSampleBins];
    double table[kSampleTable];  // 2^(i / 512)
    SampleSlot slots[2][kSampleMaxCluster];
    double wd[3][kSampleWarps];
    long long wn[1][kSampleWarps];
    uint32_t wu[kSampleWarps];
    double total_d[2];
    unsigned first_u, first_l;
    unsigned bin;
    unsigned listed;  // entries of the list, in the first CTA
    long long before, count;
};

constexpr int kSampleList = 1024;
static_assert(kSampleList == 2 * kSampleThreads, "two entries a thread");

__device__ __forceinline__ void st_cluster_f64(uint32_t addr, double v) {
    asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(addr), "d"(v) : "memory");
}
__device__ __forceinline__ void st_cluster_s64(uint32_t addr, long long v) {
    asm volatile("st.shared::cluster.s64 [%0], %1;" ::"r"(addr), "l"(v) : "memory");
}
__device__ __forceinline__ void ld_cluster(uint32_t addr, uint32_t (&v)[2]) {
    asm volatile("ld.shared::cluster.v2.u32 {%0, %1}, [%2];" : "=r"(v[0]), "=r"(v[1]) : "r"(addr) : "memory");
}

__device__ __forceinline__ uint32_t atom_cluster_add(uint32_t addr, uint32_t v) {
    uint32_t old;
    asm volatile("atom.relaxed.cluster.shared::cluster.add.u32 %0, [%1], %2;" : "=r"(old) : "r"(addr), "r"(v) : "memory");
    return old;
}

// The weights of one row (whose maximum is finite).
struct SampleWeights {
    double top_d, inv_t;
    float top;
    float inv_t32;
    const double* table;
    __device__ __forceinline__ double exponent(float v) const { return (static_cast<double>(v) - top_d) * inv_t; }
    // exp(x) for -700 < x <= 0 by a table of 2^(i / 512) and a polynomial (Tang, 1989): x = n ln2 / 512 + r,
    // |r| <= ln2 / 1024, exp(x) = 2^(n >> 9) 2^((n & 511) / 512) (1 + r + r^2 / 2 + r^3 / 6): relative error below 1e-14
    __device__ __forceinline__ double exp_below(double x) const {
        constexpr double kMagic = 6755399441055744.0;  // 1.5 * 2^52: adding it rounds to an integer
        const double nm = fma(x, 738.6598609349492420, kMagic);  // 512 / ln 2
        const int n = __double2loint(nm);
        const double r = fma(nm - kMagic, -0.001353803087128736302, x);  // ln 2 / 512
        const double q = fma(r * r, fma(r, 1.0 / 6, 0.5), r);
        double t = table[n & (kSampleTable - 1)];
        t = __hiloint2double(__double2hiint(t) + ((n >> 9) << 20), __double2loint(t));
        return fma(t, q, t);
    }
    __device__ __forceinline__ double operator()(float v) const {
        const double x = exponent(v);
        return x > -700.0 ? exp_below(x) : 0.0;
    }
    // bin of the first histogram, of `bins`; does not increase with v
    __device__ __forceinline__ int bin(float v, int bins) const {
        return static_cast<int>(fminf((top - v) * inv_t32, static_cast<float>(bins - 1)));
    }
};

template <class V>
__device__ __forceinline__ V sample_warp_sum(V v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
template <class V>
__device__ __forceinline__ V sample_warp_scan(V v) {  // inclusive
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const V up = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += up;
    }
    return v;
}

// Sums of the values of the threads before this one, for N values side by side; `tmp` holds one value per warp for each.
template <int N, class V>
__device__ __forceinline__ void sample_block_before(V (&v)[N], V (*tmp)[kSampleWarps]) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    V incl[N];
#pragma unroll
    for (int i = 0; i < N; ++i) incl[i] = sample_warp_scan(v[i]);
    __syncthreads();
    if (lane == 31) {
#pragma unroll
        for (int i = 0; i < N; ++i) tmp[i][warp] = incl[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const V warps = sample_warp_scan(lane < kSampleWarps ? tmp[i][lane] : V(0));
        const V base = __shfl_sync(0xffffffffu, warps, warp == 0 ? 0 : warp - 1);
        const V up = __shfl_up_sync(0xffffffffu, incl[i], 1);
        v[i] = (warp == 0 ? V(0) : base) + (lane == 0 ? V(0) : up);
    }
}

// The index, by one warp: the first kept element of vectors begin .. end - 1 with whose weight the sum passes `target`;
// where rounding left the target behind the last of them (or u is 1), that one. fetch(v, x) gives a vector's VEC values,
// `tie_start` ties lie before `begin`.
template <int VEC, class Fetch, class Weight>
__device__ __forceinline__ void sample_find(int begin, int end, int head, Fetch&& fetch, Weight&& kept_weight, float bound,
                                            double w_tie, long long ties, long long tie_start, double target,
                                            double everything, long long row, const SampleParams& p) {
    const int lane = threadIdx.x & 31;
    // 32 vectors at a time
    double passed = 0;
    long long ties_passed = tie_start;
    long long last = -1;  // of this lane's kept elements
    double last_w = 0;
    for (int base = begin; base < end; base += 32) {
        const int v = base + lane;
        float x[VEC];
        int n_equal = 0;
        if (v < end) {
            fetch(v, x);
        } else {
#pragma unroll
            for (int j = 0; j < VEC; ++j) x[j] = -INFINITY;
        }
#pragma unroll
        for (int j = 0; j < VEC; ++j) n_equal += x[j] == bound && v < end;
        const int equal_incl = sample_warp_scan(n_equal);
        long long tie = ties_passed + equal_incl - n_equal;
        double w[VEC], lane_sum = 0;
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            w[j] = 0;
            if (x[j] > bound) w[j] = kept_weight(x[j]);
            else if (x[j] == bound && v < end && tie++ < ties) w[j] = w_tie;
            lane_sum += w[j];
            if (w[j] > 0) {
                last = static_cast<long long>(v) * VEC + j - head;
                last_w = w[j];
            }
        }
        const double incl = sample_warp_scan(lane_sum);
        const unsigned hit = __ballot_sync(0xffffffffu, lane_sum > 0 && passed + incl > target);
        if (hit) {
            if (lane == __ffs(hit) - 1) {
                double r = passed + (incl - lane_sum);
                bool done = false;
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    r += w[j];
                    if (!done && w[j] > 0 && r > target) {
                        done = true;
                        last = static_cast<long long>(v) * VEC + j - head;
                        last_w = w[j];
                    }
                }
                p.token[row] = last;
                if (p.logprob) p.logprob[row] = static_cast<float>(log(last_w / everything));
            }
            return;
        }
        passed += __shfl_sync(0xffffffffu, incl, 31);
        ties_passed += __shfl_sync(0xffffffffu, equal_incl, 31);
    }
    // rounding left the target behind the last kept element, or u is 1: that element
    const uint32_t best = __reduce_max_sync(0xffffffffu, static_cast<uint32_t>(last + 1));
    if (static_cast<uint32_t>(last + 1) == best) {
        p.token[row] = last;
        if (p.logprob) p.logprob[row] = static_cast<float>(log(last_w / everything));
    }
}

// Sorts 2^log2 entries, larger first.
__device__ __forceinline__ void sample_sort(unsigned long long* list, int log2) {
    const int t = threadIdx.x;
    for (int size = 1; size <= log2; ++size)
        for (int step = size - 1; step >= 0; --step) {
            __syncthreads();
            if (t < 1 << (log2 - 1)) {
                const int i = ((t >> step) << (step + 1)) | (t & ((1 << step) - 1)), j = i | (1 << step);
                const unsigned long long a = list[i], b = list[j];
                if ((a < b) == (((i >> size) & 1) == 0)) {
                    list[i] = b;
                    list[j] = a;
                }
            }
        }
    __syncthreads();
}

// The draw from the top_k alone, by one CTA: `list` holds the n largest logits in any order, as key and inverted index,
// the k first of which are kept by the top_k.
template <class T>
__device__ __noinline__ void sample_listed(unsigned long long* list, int n, int k, const SampleWeights& weight, float top_p,
                                           double min_p, const SampleParams& p, SampleShared& sh, long long row) {
    using Key = SampleKey<T>;
    const int t = threadIdx.x;
    int log2 = 1;
    while (1 << log2 < n) ++log2;
    for (int i = n + t; i < 1 << log2; i += kSampleThreads) list[i] = 0;
    sample_sort(list, log2);
    unsigned long long entry[2];
    double w[2], before[1] = {0};
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        entry[j] = 2 * t + j < k ? list[2 * t + j] : 0;
        w[j] = entry[j] ? weight(Key::value(static_cast<uint32_t>(entry[j] >> 32))) : 0.0;
        before[0] += w[j];
    }
    double sum = before[0];
    sample_block_before<1>(before, sh.wd);
    if (t == kSampleThreads - 1) sh.total_d[0] = before[0] + sum;
    if (t == 0) sh.bin = 0xffffffffu;
    __syncthreads();
    // predecessors within top_p of the sum, the first always; what is left is sorted by index
    const double limit = top_p < 1.f ? (top_p > 0.f ? static_cast<double>(top_p) : 0.0) * sh.total_d[0] : INFINITY;
    double ahead = before[0];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const bool kept = entry[j] != 0 && w[j] > 0 && w[j] >= min_p && (ahead <= limit || 2 * t + j == 0);
        ahead += w[j];
        if (2 * t + j < 1 << log2)
            list[2 * t + j] = kept ? (entry[j] << 32) | (entry[j] >> 32) : 0;  // the inverted index leads
    }
    sample_sort(list, log2);
    double sums[1] = {0};
    int entries = 0;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        entry[j] = 2 * t + j < 1 << log2 ? list[2 * t + j] : 0;
        entries += entry[j] != 0;
        w[j] = entry[j] ? weight(Key::value(static_cast<uint32_t>(entry[j]))) : 0.0;
        sums[0] += w[j];
    }
    sum = sums[0];
    sample_block_before<1>(sums, sh.wd);
    if (t == kSampleThreads - 1) sh.total_d[0] = sums[0] + sum;
    const int last = __syncthreads_count(entries > 0) + __syncthreads_count(entries > 1) - 1;
    const double everything = sh.total_d[0];
    float u = p.uniform[row];
    u = u > 0.f ? u : 0.f;
    const double target = static_cast<double>(u) * everything;
    double run = sums[0];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        run += w[j];
        if (entry[j] && (run > target || 2 * t + j == last)) atomicMin(&sh.bin, static_cast<unsigned>(2 * t + j));
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 2; ++j)
        if (entry[j] && sh.bin == 2 * t + j) {
            p.token[row] = 0xffffffffu - static_cast<uint32_t>(entry[j] >> 32);
            if (p.logprob) p.logprob[row] = static_cast<float>(log(w[j] / everything));
        }
}

// One row, by the CTAs of a cluster. `list` is room for kSampleList entries in shared memory.
template <class T>
__device__ __forceinline__ void sample_row(const T* __restrict__ logits, long long ld, int vocab, int n_ctas,
                                           int vectors_per_warp, int in_smem, const SampleParams& p, SampleShared& sh,
                                           unsigned long long* list, unsigned char* sample_slice, long long row) {
    constexpr int VEC = RmsTile<T>::kVec;
    using Key = SampleKey<T>;
    constexpr int kBins = kSampleBins, PER = kSampleBinsPerThread;
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    const int rank = static_cast<int>(ptx::cluster_ctarank());

    // The row in 16-byte vectors that start on 16-byte boundaries: the first and the last may reach past it.
    const T* l = logits + row * ld;
    const int head = static_cast<int>((reinterpret_cast<uintptr_t>(l) & 15u) / sizeof(T));  // elements before the row
    const T* aligned = l - head;
    const int n_vec = static_cast<int>((static_cast<long long>(vocab) + head + VEC - 1) / VEC);
    const int cta_vec0 = rank * kSampleWarps * vectors_per_warp;
    const int v0 = min(n_vec, cta_vec0 + warp * vectors_per_warp), v1 = min(n_vec, v0 + vectors_per_warp);
    uint4* slice = reinterpret_cast<uint4*>(sample_slice);

    // One vector of the row; what is outside the row, and NaN, as -inf.
    auto read = [&](int v) {
        const long long i0 = static_cast<long long>(v) * VEC - head;
        uint4 raw;
        if (i0 >= 0 && i0 + VEC <= vocab) {
            raw = *reinterpret_cast<const uint4*>(aligned + static_cast<long long>(v) * VEC);
        } else {
            alignas(16) T tmp[VEC];
#pragma unroll
            for (int j = 0; j < VEC; ++j)
                tmp[j] = i0 + j >= 0 && i0 + j < vocab ? l[i0 + j] : Cvt<T>::from_f(-INFINITY);
            raw = *reinterpret_cast<const uint4*>(tmp);
        }
        float x[VEC];
        rms_unpack<T>(raw, x);
        bool nan = false;
#pragma unroll
        for (int j = 0; j < VEC; ++j) nan |= !(x[j] == x[j]);
        if (nan) {
#pragma unroll
            for (int j = 0; j < VEC; ++j) x[j] = x[j] == x[j] ? x[j] : -INFINITY;
            raw = rms_pack<T>(x);
        }
        return raw;
    };
    float top = -INFINITY;
    // A vector as floats. Where the maximum is +inf, all of it is shared among the +inf: they become 0, the rest -inf.
    auto fetch = [&](int v, float (&x)[VEC]) {
        const uint4 raw = in_smem ? slice[v - cta_vec0] : read(v);
        rms_unpack<T>(raw, x);
        if (top == INFINITY) {
#pragma unroll
            for (int j = 0; j < VEC; ++j) x[j] = x[j] == INFINITY ? 0.f : -INFINITY;
        }
    };
    // The vectors of this warp's share.
    auto scan = [&](auto&& f) {
        for (int v = v0 + lane; v < v1; v += 32) {
            float x[VEC];
            fetch(v, x);
            f(x);
        }
    };
    auto largest = [&](const float (&x)[VEC]) {
        float m = x[0];
#pragma unroll
        for (int j = 1; j < VEC; ++j) m = fmaxf(m, x[j]);
        return m;
    };
    int slot_parity = 0;
    // Every CTA's values to every CTA; returns this exchange's slots. Two sets alternate: a CTA writes a set again only
    // behind the next exchange's barrier, which all reach after they have read this one.
    auto exchange = [&](double d0, double d1, double d2, long long n, uint32_t u) -> const SampleSlot* {
        SampleSlot* mine = &sh.slots[slot_parity][rank];
        if (t < n_ctas) {
            const uint32_t a = ptx::map_to_cta(ptx::smem_u32(mine), t);
            st_cluster_f64(a, d0);
            st_cluster_f64(a + 8, d1);
            st_cluster_f64(a + 16, d2);
            st_cluster_s64(a + 24, n);
            ptx::st_shared_cluster_u32(a + 32, u);
        }
        __syncthreads();
        ptx::cluster_sync_all();
        const SampleSlot* all = sh.slots[slot_parity];
        slot_parity ^= 1;
        return all;
    };

    // ---- 1. the slice and the maximum
    for (int v = v0 + lane; v < v1; v += 32) {
        const uint4 raw = read(v);
        if (in_smem) slice[v - cta_vec0] = raw;
        float x[VEC];
        rms_unpack<T>(raw, x);
#pragma unroll
        for (int j = 0; j < VEC; ++j) top = fmaxf(top, x[j]);
    }
    if (t < kSampleTable) sh.table[t] = exp2(t / static_cast<double>(kSampleTable));
    if (t == 0) sh.listed = 0;
    for (int i = t; i < kBins; i += kSampleThreads) sh.hist[0][i] = sh.hist[1][i] = 0;
    {
        uint32_t k = __reduce_max_sync(0xffffffffu, Key::of(top));
        if (lane == 0) sh.wu[warp] = k;
        __syncthreads();
        for (int i = 0; i < kSampleWarps; ++i) k = max(k, sh.wu[i]);
        const SampleSlot* all = exchange(0, 0, 0, 0, k);
        for (int c = 0; c < n_ctas; ++c) k = max(k, all[c].u);
        top = Key::value(k);
    }
    const float temp = p.temperature ? p.temperature[row] : p.temperature_all;
    if (top == -INFINITY || !(temp > 0.f)) {  // the same for the whole cluster
        uint32_t first = 0xffffffffu;
        if (top != -INFINITY) {
            const float largest_value = top == INFINITY ? 0.f : top;
            for (int v = v0 + lane; v < v1; v += 32) {
                float x[VEC];
                fetch(v, x);
#pragma unroll
                for (int j = 0; j < VEC; ++j)
                    if (x[j] == largest_value) first = min(first, static_cast<uint32_t>(v) * VEC + j - head);
            }
        }
        first = __reduce_min_sync(0xffffffffu, first);
        __syncthreads();
        if (lane == 0) sh.wu[warp] = first;
        __syncthreads();
        for (int i = 0; i < kSampleWarps; ++i) first = min(first, sh.wu[i]);
        const SampleSlot* all = exchange(0, 0, 0, 0, first);
        for (int c = 0; c < n_ctas; ++c) first = min(first, all[c].u);
        if (rank == 0 && t == 0) {
            p.token[row] = top == -INFINITY ? -1 : static_cast<long long>(first);
            if (p.logprob) p.logprob[row] = top == -INFINITY ? -INFINITY : 0.f;
        }
        return;
    }
    SampleWeights weight;
    weight.top = top == INFINITY ? 0.f : top;  // fetch() goes by `top` itself
    weight.top_d = weight.top;
    weight.inv_t = 1.0 / static_cast<double>(temp);
    weight.inv_t32 = fminf(kSampleBinsPerNat / temp, 1e30f);
    weight.table = sh.table;

    // ---- histograms
    int hist_parity = 0;
    // The counts of this thread's bins (PER t and on) over the whole cluster, f(value) the bin. Two histograms alternate: one is
    // cleared while the other is in use, a barrier after all CTAs have read it.
    // Only values within [low, high] count.
    auto histogram = [&](float low, float high, uint32_t* sum, auto&& f) {
        uint32_t* h = sh.hist[hist_parity];
        scan([&](const float (&x)[VEC]) {
            if (largest(x) < low) return;
#pragma unroll
            for (int j = 0; j < VEC; ++j)
                if (x[j] >= low && x[j] <= high) atomicAdd(&h[f(x[j])], 1u);
        });
        __syncthreads();
        ptx::cluster_sync_all();
#pragma unroll
        for (int j = 0; j < PER; ++j) sum[j] = 0;
        uint32_t o[kSampleMaxCluster][PER] = {};
#pragma unroll
        for (int c = 0; c < kSampleMaxCluster; ++c)  // all in flight together
            if (c < n_ctas) ld_cluster(ptx::map_to_cta(ptx::smem_u32(&h[PER * t]), c), o[c]);
#pragma unroll
        for (int c = 0; c < kSampleMaxCluster; ++c)
#pragma unroll
            for (int j = 0; j < PER; ++j) sum[j] += o[c][j];
        hist_parity ^= 1;
    };
    auto clear_other = [&]() {  // the histogram after next: read by all before the barrier that has just passed
        uint32_t* h = sh.hist[hist_parity];
        for (int i = t; i < kBins; i += kSampleThreads) h[i] = 0;
        __syncthreads();
    };
    // The smallest key whose value falls in bin b of weight.bin or an earlier one, by 32 points at a time.
    auto first_key_of_bin_at_most = [&](int b) {
        uint32_t lo = Key::kNone, hi = Key::of(weight.top);  // hi does
        while (lo < hi) {
            const uint64_t span = hi - lo;
            const uint32_t at = lo + static_cast<uint32_t>(span * lane / 32);
            const unsigned yes = __ballot_sync(0xffffffffu, weight.bin(Key::value(at), kBins) <= b);
            const int i = yes ? __ffs(yes) - 1 : 32;  // points i .. 31 and hi do
            const uint32_t new_hi = i < 32 ? lo + static_cast<uint32_t>(span * i / 32) : hi;
            if (i > 0) lo = lo + static_cast<uint32_t>(span * (i - 1) / 32) + 1;
            hi = new_hi;
        }
        return hi;
    };
    // The keys of bins b1 .. b2, found by two warps side by side.
    auto bracket_of_bins = [&](int b1, int b2, uint32_t& lo, uint32_t& hi) {
        if (warp == 0) {
            const uint32_t k = b2 == kBins - 1 ? Key::kNone + 1 : first_key_of_bin_at_most(b2);
            if (lane == 0) sh.first_l = k;
        } else if (warp == 1) {
            const uint32_t k = b1 == 0 ? Key::of(weight.top) : first_key_of_bin_at_most(b1 - 1) - 1;
            if (lane == 0) sh.first_u = k;
        }
        __syncthreads();
        lo = sh.first_l;
        hi = sh.first_u;
    };

    const float lowest = Key::value(Key::kNone + 1);  // the smallest finite value
    // What is kept: values above `bound`, and `ties` of those equal to it in index order. -inf: everything.
    float bound = -INFINITY;
    long long ties = 0;
    long long k = p.top_k ? (p.top_k_i64 ? static_cast<const long long*>(p.top_k)[row] : static_cast<const int*>(p.top_k)[row]) : p.top_k_all;

    const float top_p = p.top_p ? p.top_p[row] : p.top_p_all;
    const float min_row = p.min_p ? p.min_p[row] : p.min_p_all;
    const double min_p = min_row > 0.f ? fminf(min_row, 1.f) : 0.0;

    // ---- 2., 4. top_k: the k-th value
    if (k > 0 && k < vocab) {
        uint32_t lo = 0, hi = 0;
        int shift = -1;  // -1: the first histogram
        long long above = 0;  // values above the bracket
        bool all = true;  // fewer than k values above -inf
        for (int round = 0; round < 6; ++round) {  // the first histogram, then the bracket in steps of 10 bits
            uint32_t cs[PER];
            if (shift < 0) histogram(lowest, weight.top, cs, [&](float v) { return weight.bin(v, kBins); });
            else histogram(Key::at_least(lo), Key::at_most(hi), cs, [&](float v) { return static_cast<int>((hi - Key::of(v)) >> shift); });
            clear_other();
            long long before[1] = {0};
#pragma unroll
            for (int j = 0; j < PER; ++j) before[0] += cs[j];
            sample_block_before<1>(before, sh.wn);
            long long run = above + before[0];
            if (t == 0) sh.bin = kBins;
            __syncthreads();
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                if (run < k && k <= run + cs[j]) {
                    sh.bin = PER * t + j;
                    sh.before = run;
                    sh.count = cs[j];
                }
                run += cs[j];
            }
            __syncthreads();
            const uint32_t b = sh.bin;
            above = sh.before;
            const long long reached = above + sh.count;  // values down to the bracket's lowest
            if (b == kBins) break;
            all = false;
            if (shift == 0) {
                lo = hi = hi - b;
                break;
            }
            if (shift < 0) {
                bracket_of_bins(static_cast<int>(b), static_cast<int>(b), lo, hi);
                if (reached <= kSampleList) {
                    // few enough to be listed: the first CTA collects them and draws from the list
                    const float low_end = Key::at_least(lo);
                    const uint32_t listed = ptx::map_to_cta(ptx::smem_u32(&sh.listed), 0);
                    for (int v = v0 + lane; v < v1; v += 32) {
                        float x[VEC];
                        fetch(v, x);
                        if (largest(x) < low_end) continue;
#pragma unroll
                        for (int j = 0; j < VEC; ++j)
                            if (x[j] >= low_end) {
                                const uint32_t index = static_cast<uint32_t>(static_cast<long long>(v) * VEC + j - head);
                                const uint32_t n = atom_cluster_add(listed, 1);  // below `reached`: the histogram has counted them
                                const unsigned long long entry = (static_cast<unsigned long long>(Key::of(x[j])) << 32) | (0xffffffffu - index);
                                if (n < kSampleList) st_cluster_s64(ptx::map_to_cta(ptx::smem_u32(&list[n]), 0), static_cast<long long>(entry));
                            }
                    }
                    __syncthreads();
                    ptx::cluster_sync_all();
                    if (rank == 0) sample_listed<T>(list, static_cast<int>(reached), static_cast<int>(k), weight, top_p, min_p, p, sh, row);
                    return;
                }
            } else {
                hi -= b << shift;
                lo = max(lo, hi - ((1u << shift) - 1u));
            }
            shift = 0;
            while (((hi - lo) >> shift) >= kBins) ++shift;
        }
        if (!all) {
            bound = Key::value(lo);
            ties = k - above;
        }
    }

    // ---- 2., 3., 4. top_p: the smallest value whose predecessors' weights stay within the limit
    bool carry = false;  // whether this thread's weights above the bracket are summed already, as `carried`
    double carried = 0;
    float carry_low = 0, carry_high = 0;  // the bracket
    if (top_p < 1.f) {
        const float floor_value = bound;  // only values above it take part; `extra` is the ties' weight
        const double extra = ties > 0 ? ties * weight(bound) : 0.0;
        const double share = top_p > 0.f ? static_cast<double>(top_p) : 0.0;
        uint32_t lo, hi;      // the bracket
        double above = 0, limit;  // weight above the bracket; the largest sum of predecessors
        bool found = false;   // the threshold is in the bracket
        {
            const float low_end = floor_value == -INFINITY ? lowest : Key::value(Key::of(floor_value) + 1);
            uint32_t cs[PER];
            histogram(low_end, weight.top, cs, [&](float v) { return weight.bin(v, kBins); });
            clear_other();
            double up[PER], low[PER], sums[2] = {0, 0};
            // weights of bin b are within e^-((b + 1) / kPerNat) .. e^-(b / kPerNat), and 1e-4 for the bin's 32-bit arithmetic
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                const double e = weight.exp_below(-(PER * t + j) / static_cast<double>(kSampleBinsPerNat));
                up[j] = cs[j] * e * 1.0001;
                low[j] = PER * t + j == kBins - 1 ? 0.0 : cs[j] * e * (kSampleBinStep * 0.9999);
                sums[0] += up[j];
                sums[1] += low[j];
            }
            const double up_sum = sums[0], low_sum = sums[1];
            sample_block_before<2>(sums, sh.wd);
            if (t == kSampleThreads - 1) {
                sh.total_d[0] = sums[0] + up_sum;
                sh.total_d[1] = sums[1] + low_sum;
                sh.first_u = sh.first_l = kBins - 1;
            }
            __syncthreads();
            const double least = share * (sh.total_d[1] + extra), most = share * (sh.total_d[0] + extra);
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                // the first bin whose upper sum may pass the limit, the first whose lower sum must
                sums[0] += up[j];
                sums[1] += low[j];
                if (cs[j] > 0 && sums[0] >= least) atomicMin(&sh.first_u, static_cast<unsigned>(PER * t + j));
                if (cs[j] > 0 && sums[1] > most) atomicMin(&sh.first_l, static_cast<unsigned>(PER * t + j));
            }
            __syncthreads();
            const int b1 = static_cast<int>(sh.first_u), b2 = max(b1, static_cast<int>(sh.first_l));
            __syncthreads();
            bracket_of_bins(b1, b2, lo, hi);
            double s[3] = {0, 0, 0};  // all, inside and above the bracket, above it
            const float in_low = Key::at_least(lo), in_high = Key::at_most(hi);
            scan([&](const float (&x)[VEC]) {
                const bool reaches = largest(x) >= in_low;
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    const double e = weight.exponent(x[j]);
                    const double w = weight.exp_below(e);
                    if (e > -700.0 && x[j] > floor_value) {
                        s[0] += w;
                        if (reaches) {
                            if (x[j] >= in_low) s[1] += w;
                            if (x[j] > in_high) s[2] += w;
                        }
                    }
                }
            });
            carried = s[2];
            carry_low = in_low;
            carry_high = in_high;
            __syncthreads();
#pragma unroll
            for (int i = 0; i < 3; ++i) {
                s[i] = sample_warp_sum(s[i]);
                if (lane == 0) sh.wd[i][warp] = s[i];
            }
            __syncthreads();
#pragma unroll
            for (int i = 0; i < 3; ++i) {
                s[i] = 0;
                for (int w = 0; w < kSampleWarps; ++w) s[i] += sh.wd[i][w];
            }
            const SampleSlot* all = exchange(s[0], s[1], s[2], 0, 0);
            s[0] = s[1] = s[2] = 0;
            for (int c2 = 0; c2 < n_ctas; ++c2) {
                s[0] += all[c2].d[0];
                s[1] += all[c2].d[1];
                s[2] += all[c2].d[2];
            }
            limit = share * (s[0] + extra);
            const uint32_t floor_key = Key::of(floor_value);
            if (s[0] <= limit) {
                above = s[0];  // every value above the floor is kept
                found = false;
            } else if (s[2] > limit) {  // outside the bounds' bracket (they leave room for rounding, but to be sure)
                found = true;
                lo = hi + 1;
                hi = Key::of(weight.top);
                above = 0;
            } else if (s[1] > limit) {
                found = carry = true;
                lo = max(lo, floor_key + 1);
                above = s[2];
            } else {
                found = true;
                hi = lo - 1;
                lo = floor_key + 1;
                above = s[1];
            }
        }
        if (!found) {
            // the ties of the floor, one after the other
            const double w = ties > 0 ? weight(bound) : 0.0;
            if (w > 0) {
                const double room = (limit - above) / w;
                const long long most = room < 0 ? 0 : static_cast<long long>(fmin(room, 4e9)) + 1;
                ties = most < ties ? most : ties;
            }
        } else {
            // every round narrows the bracket to one bin, or by one bin that has values: a few rounds, thousands at the worst
            for (int round = 0; round < 1 << 16; ++round) {
                int shift = 0;
                while (((hi - lo) >> shift) >= kBins) ++shift;
                uint32_t cs[PER];
                histogram(Key::at_least(lo), Key::at_most(hi), cs, [&](float v) { return static_cast<int>((hi - Key::of(v)) >> shift); });
                clear_other();
                double up[PER], low[PER], sums[2] = {0, 0};
#pragma unroll
                for (int j = 0; j < PER; ++j) {
                    const uint32_t off = static_cast<uint32_t>(PER * t + j) << shift, last = off + ((1u << shift) - 1u);
                    const bool in = off <= hi - lo && cs[j] > 0;
                    up[j] = in ? cs[j] * weight(Key::value(hi - off)) : 0.0;
                    low[j] = in ? (shift == 0 ? up[j] : cs[j] * weight(Key::value(hi - min(last, hi - lo)))) : 0.0;
                    sums[0] += up[j];
                    sums[1] += low[j];
                }
                sample_block_before<2>(sums, sh.wd);
                const double up_run = above + sums[0], low_run = above + sums[1];
                if (t == 0) sh.first_u = sh.first_l = kBins;
                __syncthreads();
                // a hair of room on both sides while the bins hold several values; none once they are single ones
                const double hair = shift == 0 ? 0.0 : 1e-9 * limit;
                unsigned last_full = 0;
                double u = up_run, w = low_run;
#pragma unroll
                for (int j = 0; j < PER; ++j) {
                    u += up[j];
                    w += low[j];
                    if (cs[j] > 0) {
                        last_full = PER * t + j + 1;
                        if (u > limit - hair) atomicMin(&sh.first_u, static_cast<unsigned>(PER * t + j));
                        if (w > limit + hair) atomicMin(&sh.first_l, static_cast<unsigned>(PER * t + j));
                    }
                }
                last_full = __reduce_max_sync(0xffffffffu, last_full);
                if (lane == 0) sh.wu[warp] = last_full;
                __syncthreads();
                for (int i = 0; i < kSampleWarps; ++i) last_full = max(last_full, sh.wu[i]);
                // the bracket holds the threshold, so a bin that no sum passes stands for the last one that has values
                const uint32_t b1 = min(sh.first_u, last_full - 1), b2 = max(b1, min(sh.first_l, last_full - 1));
                if (shift == 0) {
                    // the sums of single values are exact: predecessors of this one stay within the limit
                    __syncthreads();
                    double run = up_run;
#pragma unroll
                    for (int j = 0; j < PER; ++j) {
                        if (static_cast<uint32_t>(PER * t + j) == b1) {
                            sh.total_d[0] = run;
                            sh.count = static_cast<long long>(cs[j]);
                        }
                        run += up[j];
                    }
                    __syncthreads();
                    bound = Key::value(hi - b1);
                    const double w1 = weight(bound), ahead = sh.total_d[0];
                    const long long equal = sh.count;
                    // tie number i (from 0) is kept while ahead + i w <= limit; the very first value always
                    long long most = equal;
                    if (w1 > 0) {
                        const double room = (limit - ahead) / w1;
                        most = room < 0 ? 0 : static_cast<long long>(fmin(room, 4e9)) + 1;
                    }
                    if (bound == weight.top && most < 1) most = 1;
                    ties = most < equal ? most : equal;
                    break;
                }
                // weights of the bins before b1, and of b1, exactly
                const uint32_t b1_hi = hi - (b1 << shift);
                const uint32_t b1_lo = max(lo, b1_hi - ((1u << shift) - 1u));
                const uint32_t b2_hi = hi - (b2 << shift);
                const uint32_t b2_lo = max(lo, b2_hi - ((1u << shift) - 1u));
                double s[2] = {0, 0};
                const float f_hi = Key::at_most(hi), f1_hi = Key::at_most(b1_hi), f1_lo = Key::at_least(b1_lo);
                scan([&](const float (&x)[VEC]) {
                    if (largest(x) < f1_lo) return;
#pragma unroll
                    for (int j = 0; j < VEC; ++j) {
                        if (x[j] <= f_hi && x[j] >= f1_lo) {
                            const double wv = weight(x[j]);
                            if (x[j] > f1_hi) s[0] += wv;
                            else s[1] += wv;
                        }
                    }
                });
                __syncthreads();
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    s[i] = sample_warp_sum(s[i]);
                    if (lane == 0) sh.wd[i][warp] = s[i];
                }
                __syncthreads();
                s[0] = s[1] = 0;
                for (int i = 0; i < kSampleWarps; ++i) {
                    s[0] += sh.wd[0][i];
                    s[1] += sh.wd[1][i];
                }
                const SampleSlot* all = exchange(s[0], s[1], 0, 0, 0);
                s[0] = s[1] = 0;
                for (int c2 = 0; c2 < n_ctas; ++c2) {
                    s[0] += all[c2].d[0];
                    s[1] += all[c2].d[1];
                }
                if (b1 == b2 || above + s[0] + s[1] > limit) {
                    above += s[0];
                    hi = b1_hi;
                    lo = b1_lo;
                } else {
                    above += s[0] + s[1];
                    hi = b1_lo - 1;
                    lo = b2_lo;
                }
            }
        }
    }
    // ---- 5. the kept weights by warp
    auto kept_weight = [&](float v) {
        const double w = weight(v);
        return w >= min_p ? w : 0.0;
    };
    const double w_tie = ties > 0 ? kept_weight(bound) : 0.0;
    double sum = 0;
    long long equal = 0;
    if (carry && min_p == 0.0) {  // what is left to add lies inside the bracket
        sum = carried;
        scan([&](const float (&x)[VEC]) {
            if (largest(x) < carry_low) return;
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                if (x[j] >= carry_low && x[j] <= carry_high) {
                    if (x[j] > bound) sum += weight(x[j]);
                    else if (x[j] == bound) ++equal;
                }
            }
        });
    } else {
        scan([&](const float (&x)[VEC]) {
            if (largest(x) < bound) return;
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                if (x[j] > bound) sum += kept_weight(x[j]);
                else if (x[j] == bound) ++equal;
            }
        });
    }
    sum = sample_warp_sum(sum);
    equal = sample_warp_sum(equal);
    __syncthreads();
    if (lane == 0) {
        sh.wd[0][warp] = sum;
        sh.wn[0][warp] = equal;
    }
    __syncthreads();
    sum = 0;
    equal = 0;
    for (int i = 0; i < kSampleWarps; ++i) {
        sum += sh.wd[0][i];
        equal += sh.wn[0][i];
    }
    const SampleSlot* all = exchange(sum, 0, 0, equal, 0);
    auto ties_kept = [&](long long before, long long n) {
        const long long left = ties - before;
        return left <= 0 ? 0ll : (left < n ? left : n);
    };
    float u = p.uniform[row];
    u = u > 0.f ? u : 0.f;
    double everything = 0;
    {
        long long before = 0;
        for (int c = 0; c < n_ctas; ++c) {
            everything += all[c].d[0] + ties_kept(before, all[c].n) * w_tie;
            before += all[c].n;
        }
    }
    // The CTA whose sum passes the target, then the warp of it; where rounding (or u >= 1) leaves the target behind all
    // sums, the last one that holds anything.
    double target = static_cast<double>(u) * everything, run = 0, start = 0;
    long long before = 0, tie_start = 0;
    int owner = -1;
    for (int c = 0; c < n_ctas; ++c) {
        const double s = all[c].d[0] + ties_kept(before, all[c].n) * w_tie;
        if (s > 0) {
            owner = c;
            start = run;
            tie_start = before;
            if (run + s > target) break;
        }
        run += s;
        before += all[c].n;
    }
    if (rank != owner) return;
    target -= start;
    run = start = 0;
    before = tie_start;
    owner = -1;
    for (int i = 0; i < kSampleWarps; ++i) {
        const double s = sh.wd[0][i] + ties_kept(before, sh.wn[0][i]) * w_tie;
        if (s > 0) {
            owner = i;
            start = run;
            tie_start = before;
            if (run + s > target) break;
        }
        run += s;
        before += sh.wn[0][i];
    }
    if (warp != owner) return;
    target -= start;
    sample_find<VEC>(v0, v1, head, fetch, kept_weight, bound, w_tie, ties, tie_start, target, everything, row, p);
}

template <class T>
__global__ void __launch_bounds__(kSampleThreads, 2)
sample_kernel(const T* __restrict__ logits, long long ld, int vocab, int n_ctas, int vectors_per_warp, int in_smem,
              const SampleParams p) {
    extern __shared__ __align__(16) unsigned char sample_slice[];
    __shared__ SampleShared sh;
    sample_row<T>(logits, ld, vocab, n_ctas, vectors_per_warp, in_smem, p, sh, reinterpret_cast<unsigned long long*>(sample_slice),
                  sample_slice + kSampleList * 8, blockIdx.x / n_ctas);
}

// Batches of bf16 rows, a CTA per row: a histogram with one bin per VALUE. A bin's weights are then known from its count,
// so thresholds cost an exponential per value that occurs, nothing has to be narrowed, and the weights of the kept logits
// are looked up. Two passes over the row: counts, then the kept weights by chunks of 1024 logits, of which one holds the
// token. Values of a magnitude of 2^-32 and more below 1020 have bins, and zero. What is -1020 or less, a mask mostly, has
// none: it weighs nothing in 64 bits where the maximum lies 700 temperatures above it. A row in which it might weigh
// something, or with any other value (one in 100000 of rounded normal ones), is drawn by sample_row: 64 x 128256 with a
// fifth of the logits at -1e4 took 308 us that way and takes 82 now, 78 with -inf in their place. 256 x 128256 with top_p
// 0.95: 94 us where a cluster a row takes 250; 1024 rows 303 against 880. What bounds it is shared memory: one atomic per logit, and one 8-byte lookup
// per kept logit; a lone CTA on an SM (up to 148 rows: 74 us) also waits for its own loads and 64-bit chains. Four vectors of
// a lane in flight: two took 98, eight spilled and took 109. A cluster of 2 for a row, each adding up both's counts,
// took 66 us against 74 at 64 rows and lost from 100 rows on.
constexpr int kValueLow = (127 - 32) << 7;  // the bits of 2^-32
constexpr int kValueSpan = 5375;            // magnitudes with bins: all below kValueFloor
constexpr float kValueFloor = 1020.f;       // the magnitude after them
constexpr int kValueBins = 2 * kValueSpan + 1;  // larger values first: positive ones, zero, negative ones
constexpr int kValuePerThread = 21;
constexpr int kValuePadded = kValuePerThread * kSampleThreads;
static_assert(kValuePadded >= kValueBins, "every bin has a thread");
constexpr int kValueUnroll = 4;                      // vectors of a lane in flight
constexpr int kValueChunk = 32 * kValueUnroll;       // vectors that are summed together
constexpr int kValueMaxChunks = 1024;                // of a row: a sum and a number of ties each
constexpr int kValueBytes = kValuePadded * 8 + kValueMaxChunks * 12;

__device__ __forceinline__ float value_of_bin(int bin) {
    const int d = bin - kValueSpan;
    if (d == 0) return 0.f;
    const uint32_t m = kValueLow + (d < 0 ? -d : d) - 1;
    return __uint_as_float((m << 16) | (d > 0 ? 0x80000000u : 0u));
}

// The index of the bin of a value that has one and is not zero, by its bits.
__device__ __forceinline__ int bin_of_value(uint32_t bits) {
    const int off = static_cast<int>(bits & 0x7fffu) - kValueLow + 1;
    return kValueSpan + (bits & 0x8000u ? off : -off);
}

// sample_row from global memory, out of line.
__device__ __noinline__ void sample_row_alone(const __nv_bfloat16* logits, long long ld, int vocab, int vectors_per_warp,
                                              const SampleParams& p, SampleShared& sh, void* list, long long row) {
    sample_row<__nv_bfloat16>(logits, ld, vocab, 1, vectors_per_warp, 0, p, sh, static_cast<unsigned long long*>(list), nullptr, row);
}

__global__ void __launch_bounds__(kSampleThreads, 2)
sample_values_kernel(const __nv_bfloat16* __restrict__ logits, long long ld, int vocab, int groups, const SampleParams p) {
    using T = __nv_bfloat16;
    using Key = SampleKey<T>;
    constexpr int VEC = RmsTile<T>::kVec, PER = kValuePerThread, U = kValueUnroll;
    extern __shared__ __align__(16) unsigned char sample_slice[];
    __shared__ SampleShared sh;
    uint32_t* hist = reinterpret_cast<uint32_t*>(sample_slice);
    double* table = reinterpret_cast<double*>(sample_slice);  // in its place, later: the kept weight of every value
    double* chunk_sum = table + kValuePadded;
    uint32_t* chunk_equal = reinterpret_cast<uint32_t*>(chunk_sum + kValueMaxChunks);
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    const long long row = blockIdx.x;

    const T* l = logits + row * ld;
    const int head = static_cast<int>((reinterpret_cast<uintptr_t>(l) & 15u) / sizeof(T));
    const T* aligned = l - head;
    const int n_vec = static_cast<int>((static_cast<long long>(vocab) + head + VEC - 1) / VEC);
    const long long share = static_cast<long long>(groups) * kValueChunk;  // vectors of a warp
    const int v0 = static_cast<int>(min(static_cast<long long>(n_vec), warp * share));
    const int v1 = static_cast<int>(min(static_cast<long long>(n_vec), (warp + 1) * share));
    constexpr uint32_t kNothing = 0xff80ff80u;  // -inf twice
    auto read = [&](int v, int end) {  // outside the row, and from `end` on, -inf
        if (v >= end) return make_uint4(kNothing, kNothing, kNothing, kNothing);
        const long long i0 = static_cast<long long>(v) * VEC - head;
        if (i0 >= 0 && i0 + VEC <= vocab) return __ldg(reinterpret_cast<const uint4*>(aligned + static_cast<long long>(v) * VEC));
        alignas(16) T tmp[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) tmp[j] = i0 + j >= 0 && i0 + j < vocab ? l[i0 + j] : Cvt<T>::from_f(-INFINITY);
        return *reinterpret_cast<const uint4*>(tmp);
    };

    float temp = p.temperature ? p.temperature[row] : p.temperature_all;
    long long k = p.top_k ? (p.top_k_i64 ? static_cast<const long long*>(p.top_k)[row] : static_cast<const int*>(p.top_k)[row]) : p.top_k_all;
    float top_p = p.top_p ? p.top_p[row] : p.top_p_all;
    float min_row = p.min_p ? p.min_p[row] : p.min_p_all;
    if (!(temp > 0.f)) {  // the first maximum: the top_k of 1
        temp = 1.f;
        k = 1;
        min_row = 0.f;
    }
    const bool counted = k != 1;  // else only the maximum is asked for

    if (t < kSampleTable) sh.table[t] = exp2(t / static_cast<double>(kSampleTable));
    if (t == 0) {
        sh.first_u = kValuePadded;
        sh.first_l = kSampleThreads;
        sh.bin = kValuePadded;
    }
    // ---- the counts, or the maximum
    bool other = false;  // a value without a bin,
    bool below = false;  // or one of -kValueFloor or less, but -inf
    float top = -INFINITY;
    if (counted) {
        for (int i = t; i < kValuePadded; i += kSampleThreads) hist[i] = 0;
        __syncthreads();
        for (int base = v0 + lane; base < v1; base += kValueChunk) {
            uint4 raw[U];
#pragma unroll
            for (int i = 0; i < U; ++i) raw[i] = read(base + 32 * i, v1);
#pragma unroll
            for (int i = 0; i < U; ++i) {
                const uint32_t words[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    const uint32_t h = j & 1 ? words[j >> 1] >> 16 : words[j >> 1] & 0xffffu;
                    const uint32_t m = h & 0x7fffu;
                    if (m - kValueLow < kValueSpan) atomicAdd(&hist[bin_of_value(h)], 1u);
                    else if (m == 0) atomicAdd(&hist[kValueSpan], 1u);
                    else if (h < 0xff80u) {  // not -inf
                        if (h >= 0x8000u + kValueLow + kValueSpan) below = true;
                        else if (m <= 0x7f80u) other = true;
                    }
                }
            }
        }
    } else {
        for (int base = v0 + lane; base < v1; base += kValueChunk) {
            uint4 raw[U];
#pragma unroll
            for (int i = 0; i < U; ++i) raw[i] = read(base + 32 * i, v1);
#pragma unroll
            for (int i = 0; i < U; ++i) {
                float x[VEC];
                rms_unpack<T>(raw[i], x);
#pragma unroll
                for (int j = 0; j < VEC; ++j) top = fmaxf(top, x[j]);
            }
        }
        const uint32_t key = __reduce_max_sync(0xffffffffu, Key::of(top));
        if (lane == 0) sh.wu[warp] = key;
    }
    if (__syncthreads_or(other)) {
        sample_row_alone(logits, ld, vocab, static_cast<int>(share), p, sh, sample_slice, row);
        return;
    }
    long long members = 0;  // of this thread's bins
    if (counted) {
        below = __syncthreads_or(below);
        unsigned first = kValuePadded;
#pragma unroll
        for (int j = PER - 1; j >= 0; --j) {
            const uint32_t c = hist[PER * t + j];
            members += c;
            if (c > 0) first = PER * t + j;
        }
        first = __reduce_min_sync(0xffffffffu, first);
        if (lane == 0 && first < kValuePadded) atomicMin(&sh.first_u, first);
        __syncthreads();
        if (sh.first_u < kValuePadded) top = value_of_bin(sh.first_u);
    } else {
        uint32_t key = 0;
        for (int i = 0; i < kSampleWarps; ++i) key = max(key, sh.wu[i]);
        top = Key::value(key);
        if (top == INFINITY) {
            __syncthreads();  // all have read sh.wu
            sample_row_alone(logits, ld, vocab, static_cast<int>(share), p, sh, sample_slice, row);
            return;
        }
    }
    if (top == -INFINITY && !below) {
        if (t == 0) {
            p.token[row] = -1;
            if (p.logprob) p.logprob[row] = -INFINITY;
        }
        return;
    }
    SampleWeights weight;
    weight.top = top;
    weight.top_d = top;
    weight.inv_t = 1.0 / static_cast<double>(temp);
    weight.inv_t32 = 0;
    weight.table = sh.table;
    if (below && !(top > -INFINITY && weight(-kValueFloor) == 0.0)) {
        __syncthreads();  // all have read sh.first_u
        sample_row_alone(logits, ld, vocab, static_cast<int>(share), p, sh, sample_slice, row);
        return;
    }

    // ---- what is kept: values above `bound`, and `ties` of those equal to it
    float bound = -INFINITY;
    long long ties = 0;
    if (k == 1) {
        bound = top;
        ties = 1;
    } else if (counted) {
        int last_bin = kValuePadded;  // of the top_k
        if (k > 0 && k < vocab) {
            long long before[1] = {members};
            sample_block_before<1>(before, sh.wn);
            if (before[0] < k && k <= before[0] + members) {
                long long run = before[0];
                for (int j = 0; j < PER; ++j) {
                    const long long c = hist[PER * t + j];
                    if (run < k && k <= run + c) {
                        sh.bin = PER * t + j;
                        sh.count = k - run;
                    }
                    run += c;
                }
            }
            __syncthreads();
            if (sh.bin < kValuePadded) {  // else fewer than k values weigh anything
                last_bin = static_cast<int>(sh.bin);
                bound = value_of_bin(last_bin);
                ties = sh.count;
            }
            __syncthreads();
        }
        if (top_p < 1.f) {
            auto kept = [&](int bin) -> long long {  // the top_k's members in a bin
                const long long c = hist[bin];
                return bin < last_bin ? c : (bin == last_bin ? min(c, ties) : 0);
            };
            double sum = 0;
            for (int j = 0; j < PER; ++j) {
                const long long c = kept(PER * t + j);
                if (c > 0) sum += static_cast<double>(c) * weight(value_of_bin(PER * t + j));
            }
            double before[1] = {sum};
            sample_block_before<1>(before, sh.wd);
            if (t == kSampleThreads - 1) sh.total_d[0] = before[0] + sum;
            __syncthreads();
            const double limit = (top_p > 0.f ? static_cast<double>(top_p) : 0.0) * sh.total_d[0];
            if (sum > 0 && before[0] + sum > limit) atomicMin(&sh.first_l, static_cast<unsigned>(t));
            __syncthreads();
            if (sh.first_l == t) {
                // the first bin whose weights pass the limit; by the rounding of the scan, the last one
                double run = before[0], w = 0, ahead = 0;
                long long n = 0;
                for (int j = 0; j < PER; ++j) {
                    const long long c = kept(PER * t + j);
                    if (c == 0) continue;
                    n = c;
                    w = weight(value_of_bin(PER * t + j));
                    ahead = run;
                    sh.bin = PER * t + j;
                    run += static_cast<double>(c) * w;
                    if (run > limit) break;
                }
                // tie number i (from 0) is kept while ahead + i w <= limit; the very first value always
                const double room = w > 0 ? (limit - ahead) / w : 4e9;
                long long most = room < 0 ? 0 : static_cast<long long>(fmin(room, 4e9)) + 1;
                if (sh.bin == sh.first_u && most < 1) most = 1;
                sh.count = min(most, n);
            }
            __syncthreads();
            if (sh.first_l < kSampleThreads) {
                bound = value_of_bin(static_cast<int>(sh.bin));
                ties = sh.count;
            }
        }
    }
    if (counted && bound == -INFINITY) bound = -kValueFloor;  // nothing from there on is kept, and it has no bins
    const double min_p = min_row > 0.f ? fminf(min_row, 1.f) : 0.0;
    auto kept_weight = [&](float v) {
        const double w = weight(v);
        return w >= min_p ? w : 0.0;
    };
    const double w_tie = ties > 0 ? kept_weight(bound) : 0.0;

    // ---- the kept weights by chunk
    const int n_chunks = groups * kSampleWarps;
    if (counted) {
        __syncthreads();  // all have read the counts
        for (int i = t; i < kValueBins; i += kSampleThreads) {
            const float v = value_of_bin(i);
            table[i] = v > bound && v <= top ? kept_weight(v) : 0.0;
        }
        __syncthreads();
    }
    for (int g = 0; g < groups; ++g) {
        const int base = static_cast<int>(min(static_cast<long long>(v1), v0 + static_cast<long long>(g) * kValueChunk)) + lane;
        uint4 raw[U];
#pragma unroll
        for (int i = 0; i < U; ++i) raw[i] = read(base + 32 * i, v1);
        double sum = 0;
        uint32_t equal = 0;
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const uint32_t words[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
            float x[VEC];
            rms_unpack<T>(raw[i], x);
            float m = x[0];
#pragma unroll
            for (int j = 1; j < VEC; ++j) m = fmaxf(m, x[j]);
            if (m >= bound) {
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    const uint32_t h = j & 1 ? words[j >> 1] >> 16 : words[j >> 1] & 0xffffu;
                    if (x[j] > bound) sum += table[x[j] == 0.f ? kValueSpan : bin_of_value(h)];
                    else if (x[j] == bound) ++equal;
                }
            }
        }
        sum = sample_warp_sum(sum);
        equal = __reduce_add_sync(0xffffffffu, equal);
        if (lane == 0) {
            chunk_sum[warp * groups + g] = sum;
            chunk_equal[warp * groups + g] = equal;
        }
    }
    __syncthreads();
    if (warp != 0) return;

    // ---- the chunk, 32 at a time
    auto chunk = [&](int c, long long& before, long long& n_incl, long long& n) -> double {  // its kept weight
        n = c < n_chunks ? chunk_equal[c] : 0;
        n_incl = sample_warp_scan(n);
        const long long left = ties - (before + n_incl - n);
        const long long tied = left <= 0 ? 0 : min(left, n);
        return c < n_chunks ? chunk_sum[c] + static_cast<double>(tied) * w_tie : 0.0;
    };
    double everything = 0;
    long long before = 0, n_incl, n;
    for (int c = lane; c - lane < n_chunks; c += 32) {
        everything += sample_warp_sum(chunk(c, before, n_incl, n));
        before += __shfl_sync(0xffffffffu, n_incl, 31);
    }
    float u = p.uniform[row];
    u = u > 0.f ? u : 0.f;
    const double target = static_cast<double>(u) * everything;
    double run = 0, start = 0;
    long long tie_start = 0;
    int owner = -1;  // the chunk whose weights pass the target, or the last one that holds any
    before = 0;
    for (int c = lane; c - lane < n_chunks; c += 32) {
        const double s = chunk(c, before, n_incl, n);
        const double incl = sample_warp_scan(s);
        const unsigned any = __ballot_sync(0xffffffffu, s > 0), hit = __ballot_sync(0xffffffffu, s > 0 && run + incl > target);
        if (any) {
            const int at = hit ? __ffs(hit) - 1 : 31 - __clz(any);
            owner = c - lane + at;
            start = run + __shfl_sync(0xffffffffu, incl - s, at);
            tie_start = before + __shfl_sync(0xffffffffu, n_incl - n, at);
            if (hit) break;
        }
        run += __shfl_sync(0xffffffffu, incl, 31);
        before += __shfl_sync(0xffffffffu, n_incl, 31);
    }
    if (owner < 0) return;  // not reached: the maximum is kept
    const int begin = static_cast<int>(min(static_cast<long long>(n_vec), owner / groups * share + static_cast<long long>(owner % groups) * kValueChunk));
    const int end = min(n_vec, begin + kValueChunk);
    auto fetch = [&](int v, float (&x)[VEC]) { rms_unpack<T>(read(v, end), x); };
    sample_find<VEC>(begin, end, head, fetch, kept_weight, bound, w_tie, ties, tie_start, target - start, everything, row, p);
}

}  // namespace lce
