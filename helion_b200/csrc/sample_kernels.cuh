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
#pragma once

#include "ptx.cuh"
#include "vec.cuh"

namespace lce {

constexpr int kSampleThreads = 1024;

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

// The bits of a float in an order-preserving unsigned form; NaN sorts with -inf.
__device__ __forceinline__ uint32_t sample_key(float v) {
    if (!(v == v)) v = -INFINITY;
    v += 0.f;  // -0 and +0 are equal logits
    const uint32_t u = __float_as_uint(v);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float sample_key_value(uint32_t key) {
    return __uint_as_float((key & 0x80000000u) ? (key & 0x7fffffffu) : ~key);
}
constexpr uint32_t kSampleNone = 0x007fffffu;  // the key of -inf

struct SampleRow {
    double inv_t;
    float top;  // the largest logit
    __device__ __forceinline__ double weight(uint32_t key) const {
        if (key == kSampleNone) return 0.0;
        const float v = sample_key_value(key);
        if (v == top) return 1.0;
        if (top == INFINITY) return 0.0;
        return exp((static_cast<double>(v) - static_cast<double>(top)) * inv_t);
    }
};

template <class V>
__device__ __forceinline__ V sample_block_sum(V v, V* red) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    V s = red[0];
    for (int i = 1; i < kSampleThreads / 32; ++i) s += red[i];
    return s;
}

template <class T>
__global__ void __launch_bounds__(kSampleThreads)
sample_kernel(const T* __restrict__ logits, long long ld, int vocab, const SampleParams p) {
    __shared__ double red_d[32];
    __shared__ long long red_i[32];
    __shared__ unsigned long long best;
    __shared__ double part_d[kSampleThreads];
    __shared__ long long part_i[kSampleThreads];
    const long long row = blockIdx.x;
    const T* l = logits + row * ld;
    const int t = threadIdx.x;
    auto key_at = [&](int i) { return sample_key(Cvt<T>::to_f(l[i])); };

    // the first maximum
    unsigned long long mine = 0;
    for (int i = t; i < vocab; i += kSampleThreads) {
        const unsigned long long k = (static_cast<unsigned long long>(key_at(i)) << 32) | (0xffffffffu - static_cast<uint32_t>(i));
        mine = k > mine ? k : mine;
    }
    if (t == 0) best = 0;
    __syncthreads();
    atomicMax(&best, mine);
    __syncthreads();
    const uint32_t top_key = static_cast<uint32_t>(best >> 32);
    const int first = static_cast<int>(0xffffffffu - static_cast<uint32_t>(best));
    const float temp = p.temperature ? p.temperature[row] : p.temperature_all;
    if (top_key == kSampleNone || !(temp > 0.f)) {
        if (t == 0) {
            p.token[row] = top_key == kSampleNone ? -1 : first;
            if (p.logprob) p.logprob[row] = top_key == kSampleNone ? -INFINITY : 0.f;
        }
        return;
    }
    SampleRow r;
    r.inv_t = 1.0 / static_cast<double>(temp);
    r.top = sample_key_value(top_key);

    // the largest key such that at least `k` keys are at or above it; ties of it kept in index order
    uint32_t bound = kSampleNone + 1;  // smallest key that may be kept
    long long ties = vocab;            // how many keys equal to `bound` are kept
    long long k = p.top_k ? (p.top_k_i64 ? static_cast<const long long*>(p.top_k)[row] : static_cast<const int*>(p.top_k)[row]) : p.top_k_all;
    auto count_from = [&](uint32_t key) {
        long long c = 0;
        for (int i = t; i < vocab; i += kSampleThreads) c += key_at(i) >= key;
        return sample_block_sum(c, red_i);
    };
    auto mass_above = [&](uint32_t key) {
        double m = 0;
        for (int i = t; i < vocab; i += kSampleThreads) {
            const uint32_t q = key_at(i);
            if (q > key) m += r.weight(q);
        }
        return sample_block_sum(m, red_d);
    };
    if (k > 0 && k < vocab && count_from(bound) > k) {
        uint32_t lo = bound, hi = top_key;  // count_from(lo) > k
        while (lo < hi) {
            const uint32_t mid = lo + (hi - lo + 1) / 2;
            if (count_from(mid) >= k) lo = mid;
            else hi = mid - 1;
        }
        bound = lo;
        ties = k - (bound == top_key ? 0 : count_from(bound + 1));
    }
    const float top_p = p.top_p ? p.top_p[row] : p.top_p_all;
    if (top_p < 1.f) {
        const long long equal = count_from(bound) - count_from(bound + 1);
        const double z = mass_above(bound) + (equal < ties ? equal : ties) * r.weight(bound);
        const double limit = static_cast<double>(top_p) * z;
        uint32_t lo = bound, hi = top_key;  // the smallest key with mass_above <= limit
        while (lo < hi) {
            const uint32_t mid = lo + (hi - lo) / 2;
            if (mass_above(mid) <= limit) hi = mid;
            else lo = mid + 1;
        }
        const double above = mass_above(lo), w = r.weight(lo);
        if (lo != bound) ties = vocab;
        bound = lo;
        // tie number j (from 0) is kept while above + j w <= limit; the very first always
        long long most = w > 0 ? static_cast<long long>(fmin((limit - above) / w, 4e9)) : vocab;
        while (above + most * w <= limit && most < vocab) ++most;
        while (most > 0 && above + (most - 1) * w > limit) --most;
        if (bound == top_key && most < 1) most = 1;
        ties = most < ties ? most : ties;
    }
    const float min_row = p.min_p ? p.min_p[row] : p.min_p_all;
    const double min_p = min_row > 0.f ? fminf(min_row, 1.f) : 0.0;

    // in vocabulary order: thread t owns a run of indices
    const int per = (vocab + kSampleThreads - 1) / kSampleThreads;
    const int i0 = min(vocab, t * per), i1 = min(vocab, i0 + per);
    long long equal = 0;
    for (int i = i0; i < i1; ++i) equal += key_at(i) == bound;
    part_i[t] = equal;
    __syncthreads();
    long long before = 0;
    for (int j = 0; j < t; ++j) before += part_i[j];
    auto kept = [&](uint32_t q, long long& rank) {
        const bool in = q > bound || (q == bound && rank < ties);
        rank += q == bound;
        const double w = in ? r.weight(q) : 0.0;
        return w >= min_p ? w : 0.0;
    };
    double sum = 0;
    long long rank = before;
    for (int i = i0; i < i1; ++i) sum += kept(key_at(i), rank);
    part_d[t] = sum;
    __syncthreads();
    double ahead = 0, total = 0;
    for (int j = 0; j < kSampleThreads; ++j) {
        if (j == t) ahead = total;
        total += part_d[j];
    }
    float u = p.uniform[row];
    u = u > 0.f ? u : 0.f;
    const double target = static_cast<double>(u) * total;
    // the last kept index stands in where u is 1 or more
    const bool owner = ahead <= target && target < ahead + sum;
    if (t == 0) best = 0;
    __syncthreads();
    if (sum > 0 && (owner || target >= total)) {
        double run = ahead;
        rank = before;
        int pick = -1;
        double wp = 0;
        for (int i = i0; i < i1; ++i) {
            const double w = kept(key_at(i), rank);
            if (w > 0) {
                pick = i;
                wp = w;
                run += w;
                if (run > target) break;
            }
        }
        atomicMax(&best, static_cast<unsigned long long>(pick + 1));
        __syncwarp(__activemask());
        part_d[t] = wp;
    }
    __syncthreads();
    if (t == 0) {
        const int pick = static_cast<int>(best) - 1;
        p.token[row] = pick;
        if (p.logprob) p.logprob[row] = static_cast<float>(log(part_d[pick / per] / total));
    }
}

}  // namespace lce
