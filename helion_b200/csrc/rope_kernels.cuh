// Rotary positions, alone (rope) and behind the RMS norm of every query and key head (qk_norm_rope).
//
//   angle_i   = position * frequency_i                      i < half, rotary_dim = 2 half <= dim
//   rope      (a, b) -> scale * (a cos - b sin, b cos + a sin)  for the pairs (a, b) of the first rotary_dim
//             elements: (x[i], x[half + i]) or, interleaved, (x[2i], x[2i + 1]); the rest passes through
//   norm      n = x * rstd * weight,  rstd = 1 / sqrt(mean(x^2) + eps)   over one head; then rope of n
//   backward  g = rope^T(dy) (the rotation by the negative angle), and for the norm
//             dx = rstd * (g weight - x rstd^2 mean(g weight x)),  dweight = sum over tokens and heads of g x rstd
//
// Angles are formed in 64 bits and reduced to a fraction of a turn before they become 32-bit numbers: at a position
// of a million a 32-bit product is off by a twentieth of a radian. Everything else is 32 bits, rounded once.
//
// What bounds it: the heads are read once and written once, nothing is re-used but the angles of a token and the
// weights, so the bound is the copy bandwidth. A warp owns one token (and, when tokens are few, only some of its
// heads): it forms that token's angles once, a few per lane, shares them through its piece of shared memory, and
// walks the heads with the angles and the weights in registers.
//
// Vector form (rows and pairs in whole 16-byte vectors): a head takes `lanes` lanes, each holding the TWO vectors
// whose elements pair up - (i, i + half) in the half layout, two neighbours when interleaved - so that the rotation
// is local to a thread and the norm needs log2(lanes) shuffles. Row form (anything else: odd halves, unaligned
// rows): a warp stages a few rows in shared memory as floats and lanes take pairs from there.
//
// dweight: every warp keeps sums for its columns in registers (vector form) or shared memory (row form) over all the
// rows that it walks, each CTA adds its warps' sums in a fixed order and writes one partial row, and
// head_dweight_kernel adds the partial rows in a fixed order. No atomics: the same bits on every run.
//
// Measured at 16384 tokens, heads of 128, bf16: rope of 40 heads 54 us a direction for 336 MB (0.95 of the copy bandwidth);
// qk_norm_rope of 32 + 8 heads 65 us forward (0.79) and 103 us backward for 503 MB (0.75), where registers leave too few
// warps for more loads in flight (24 % and 19 % of the warps), and 6 us for dweight.
#pragma once

#include "ptx.cuh"
#include "vec.cuh"

namespace lce {

constexpr int kHeadMaxCtas = 592;   // backward CTAs in all = partial dweight rows (4 per SM on 148 SMs)
constexpr int kHeadMaxDim = 1024;
constexpr int kRowFormWarps = 4;
constexpr int kRowFormRows = 4;     // rows staged at a time

enum HeadMode { kHeadRope = 0, kHeadNorm = 1, kHeadNormBackward = 2 };

// One tensor of heads [batch][seq][heads][dim] and how its rows are dealt out.
template <class T>
struct HeadRows {
    const T* x;
    long long x_b, x_s, x_h;  // element strides of batch, sequence and head; dim is contiguous
    const T* dy;
    long long dy_b, dy_s, dy_h;
    T* out;
    long long o_b, o_s, o_h;
    const T* weight;
    float* partial;   // backward: [ctas][dim] sums of dweight, or nullptr
    int heads;
    int chunks;       // warps that share one token
    int steps;        // steps (of 32 / lanes heads; one head in the row form) per warp
    long long units;  // tokens * chunks, below 2^31
    int ctas;
};

struct RopePlan {
    const void* pos;
    int pos_i64;
    long long pos_b, pos_s;
    const double* freq;
    int half;        // angles
    int dim;
    int items;       // vector form: pairs of vectors in a row
    int lanes;       // vector form: lanes a row takes, a power of two >= items
    int pairs2;      // row form: rows can be read two elements at a time
    long long seq;
    float scale;     // of the rotated part
    float sin_sign;  // -1: the inverse rotation
    float eps;
};

// cos and sin of an angle given as position x turns per position, times scale: the product and its fraction in 64 bits.
// For 16-bit results the hardware's sine and cosine do (within 4.2e-7 for an angle in [-pi, pi]); they save most of a
// token's set-up.
template <bool FAST>
__device__ __forceinline__ float2 rope_angle(double pos, double turns_per_position, float scale, float sin_sign) {
    double turns = pos * turns_per_position;
    turns -= rint(turns);
    float s, c;
    if constexpr (FAST) {
        const float radians = 6.283185307179586f * static_cast<float>(turns);
        s = __sinf(radians);
        c = __cosf(radians);
    } else {
        sincospif(2.f * static_cast<float>(turns), &s, &c);
    }
    return make_float2(c * scale, s * scale * sin_sign);
}
constexpr double kTurnsPerRadian = 0.15915494309189533577;  // 1 / (2 pi)

__device__ __forceinline__ double rope_position(const RopePlan& p, long long b, long long s) {
    const long long i = b * p.pos_b + s * p.pos_s;
    return p.pos_i64 ? static_cast<double>(static_cast<const long long*>(p.pos)[i])
                     : static_cast<double>(static_cast<const int*>(p.pos)[i]);
}

// 1 / sqrt(a): the hardware approximation and one Newton step (relative error ~1e-7), where the step is defined.
__device__ __forceinline__ float head_rstd(float sum, float inv_dim, float eps) {
    const float a = fmaf(sum, inv_dim, eps);
    const float y = rsqrtf(a);
    return (a > 0.f && a < INFINITY) ? y * fmaf(-0.5f * a * y, y, 1.5f) : y;
}

// A lane's two vectors, rotated by the angles whose cosines and sines are c and n. The half layout pairs element j of the
// first with element j of the second; interleaved, neighbours of one vector pair up (the first vector takes the first half
// of the angles). rot0 / rot1: whether the vector is inside the rotated part at all; outside it stays as it is.
template <bool INTERLEAVED, int N>
__device__ __forceinline__ void rope_turn(Pair (&x0)[N], Pair (&x1)[N], const float (&c)[2 * N], const float (&n)[2 * N], bool rot0, bool rot1) {
    if constexpr (INTERLEAVED) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            float x, y;
            if (rot0) {
                split(x0[j], x, y);
                x0[j] = pair(fmaf(-y, n[j], x * c[j]), fmaf(x, n[j], y * c[j]));
            }
            if (rot1) {
                split(x1[j], x, y);
                x1[j] = pair(fmaf(-y, n[N + j], x * c[N + j]), fmaf(x, n[N + j], y * c[N + j]));
            }
        }
    } else if (rot0) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const Pair a = x0[j], cs = pair(c[2 * j], c[2 * j + 1]), sn = pair(n[2 * j], n[2 * j + 1]);
            float b0, b1, t0, t1;
            split(x1[j], b0, b1);
            split(a * cs, t0, t1);
            x1[j] = fma2(a, sn, x1[j] * cs);
            x0[j] = pair(fmaf(-b0, n[2 * j], t0), fmaf(-b1, n[2 * j + 1], t1));  // a pair would need registers for -n
        }
    }
}

// Threads of a CTA, CTAs per SM and steps whose loads are in flight while one is worked on. Registers are what limits
// them (a 16-bit step works on 16 elements a lane, an fp32 one on 8); measured at 16384 tokens of 32 + 8 heads of 128:
// the 16-bit norm 71 us on 2 x 256 threads, 76 on 3 (the registers spill); its backward 111 us on 384, 122 on 2 x 256;
// fp32 at 8192 tokens 62 us on 3 x 256, 68 on 2, the backward 93 on 2 x 256, 101 on 384.
template <class T, int MODE>
struct HeadShape {
    static constexpr bool kWide = sizeof(T) == 2;
    static constexpr int kThreads = MODE == kHeadNormBackward && kWide ? 384 : 256;
    static constexpr int kWarps = kThreads / 32;
    static constexpr int kCtas = MODE == kHeadNormBackward ? (kWide ? 1 : 2) : (MODE == kHeadNorm && kWide ? 2 : 3);
    static constexpr int kAhead = 2;
};

// The backward's CTAs belong to q or to k, whose sums they keep; otherwise a unit of work is a token, or a piece of one,
// with its query heads first and then its key heads.
template <class T, bool INTERLEAVED, int MODE>
__global__ void __launch_bounds__(HeadShape<T, MODE>::kThreads, HeadShape<T, MODE>::kCtas)
heads_vector_kernel(const HeadRows<T> rows_q, const HeadRows<T> rows_k, const RopePlan p) {
    constexpr int VEC = RmsTile<T>::kVec, N = VEC / 2;
    constexpr int U = HeadShape<T, MODE>::kAhead, kWarps = HeadShape<T, MODE>::kWarps;
    constexpr bool kBackward = MODE == kHeadNormBackward;
    extern __shared__ __align__(16) unsigned char head_smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const bool second = kBackward && static_cast<int>(blockIdx.x) >= rows_q.ctas;
    const HeadRows<T>& h = second ? rows_k : rows_q;
    const int cta = static_cast<int>(blockIdx.x) - (second ? rows_q.ctas : 0);
    const int table_len = p.items * VEC;
    float* cos_table = reinterpret_cast<float*>(head_smem) + warp * 2 * table_len;
    float* sin_table = cos_table + table_len;

    const int it = lane & (p.lanes - 1), sub = lane / p.lanes, per_step = 32 / p.lanes;
    const bool on = it < p.items;
    int col0, col1;
    bool rot0, rot1;
    if constexpr (INTERLEAVED) {
        col0 = 2 * it * VEC;
        col1 = col0 + VEC;
        rot0 = col0 < 2 * p.half;
        rot1 = col1 < 2 * p.half;
    } else {
        const int np = p.half / VEC;  // rotated pairs of vectors; what is left over is taken two neighbours at a time
        col0 = it < np ? it * VEC : 2 * (p.half + (it - np) * VEC);
        col1 = it < np ? col0 + p.half : col0 + VEC;
        rot0 = rot1 = it < np;
    }
    const bool on0 = on && col0 < p.dim, on1 = on && col1 < p.dim;
    const float inv_dim = 1.0f / static_cast<float>(p.dim);

    Pair acc0[N], acc1[N];  // dweight of this lane's columns
    if constexpr (kBackward) {
#pragma unroll
        for (int j = 0; j < N; ++j) acc0[j] = acc1[j] = both(0.f);
    }
    const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
    uint4 w0 = zero, w1 = zero;
    auto load_weights = [&](const HeadRows<T>& rows) {
        if (MODE != kHeadRope && on0) w0 = *reinterpret_cast<const uint4*>(rows.weight + col0);
        if (MODE != kHeadRope && on1) w1 = *reinterpret_cast<const uint4*>(rows.weight + col1);
    };
    if constexpr (kBackward) load_weights(h);
    uint4 x0[U], x1[U], d0[U], d1[U];
#pragma unroll
    for (int i = 0; i < U; ++i) x0[i] = x1[i] = d0[i] = d1[i] = zero;  // and so they stay in lanes without columns

    float c[VEC], n[VEC];  // this token's angles, for this lane's columns
    // Within a token offsets take 32 bits (the host sees to it).
    auto fetch = [&](const HeadRows<T>& rows, const T* x, const T* dy, int i, int step, int end) {
        if (step >= end) return;  // the same for the warp
        const int head = min(step * per_step + sub, rows.heads - 1);  // a row that is not there: the last, and not stored
        const int at = head * static_cast<int>(rows.x_h);
        if (on0) x0[i] = *reinterpret_cast<const uint4*>(x + (at + col0));
        if (on1) x1[i] = *reinterpret_cast<const uint4*>(x + (at + col1));
        if constexpr (kBackward) {
            const int dat = head * static_cast<int>(rows.dy_h);
            if (on0) d0[i] = *reinterpret_cast<const uint4*>(dy + (dat + col0));
            if (on1) d1[i] = *reinterpret_cast<const uint4*>(dy + (dat + col1));
        }
    };
    // Steps begin .. end of one tensor's heads; the first U are on their way.
    auto walk = [&](const HeadRows<T>& rows, const T* x, const T* dy, T* out, int begin, int end) {
        for (int step = begin; step < end; step += U) {
#pragma unroll
            for (int i = 0; i < U; ++i) {
                const int head = (step + i) * per_step + sub;
                const bool in = step + i < end && head < rows.heads;
                Pair a[N], b[N], g0[N], g1[N];
                unpack_pairs<T>(x0[i], a);
                unpack_pairs<T>(x1[i], b);
                if constexpr (kBackward) {
                    unpack_pairs<T>(d0[i], g0);
                    unpack_pairs<T>(d1[i], g1);
                }
                fetch(rows, x, dy, i, step + i + U, end);
                if constexpr (MODE == kHeadRope) {
                    rope_turn<INTERLEAVED>(a, b, c, n, rot0, rot1);
                } else {
                    Pair v0[N], v1[N], squares = both(0.f);
                    unpack_pairs<T>(w0, v0);
                    unpack_pairs<T>(w1, v1);
#pragma unroll
                    for (int j = 0; j < N; ++j) squares = fma2(a[j], a[j], fma2(b[j], b[j], squares));
                    float ss = sum(squares);
                    if constexpr (MODE == kHeadNorm) {
                        for (int o = p.lanes >> 1; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
                        const Pair rstd = both(head_rstd(ss, inv_dim, p.eps));
#pragma unroll
                        for (int j = 0; j < N; ++j) {
                            a[j] = a[j] * rstd * v0[j];
                            b[j] = b[j] * rstd * v1[j];
                        }
                        rope_turn<INTERLEAVED>(a, b, c, n, rot0, rot1);
                    } else {
                        rope_turn<INTERLEAVED>(g0, g1, c, n, rot0, rot1);
                        Pair dots = both(0.f);
#pragma unroll
                        for (int j = 0; j < N; ++j) {
                            v0[j] = v0[j] * g0[j];
                            v1[j] = v1[j] * g1[j];
                            dots = fma2(v0[j], a[j], fma2(v1[j], b[j], dots));
                        }
                        float dot = sum(dots);
                        for (int o = p.lanes >> 1; o > 0; o >>= 1) {
                            ss += __shfl_xor_sync(0xffffffffu, ss, o);
                            dot += __shfl_xor_sync(0xffffffffu, dot, o);
                        }
                        const float r = head_rstd(ss, inv_dim, p.eps);
                        const Pair rstd = both(r), k = both(-r * r * dot * inv_dim);  // dx = rstd (g w + k x^)
#pragma unroll
                        for (int j = 0; j < N; ++j) {
                            a[j] = a[j] * rstd;
                            b[j] = b[j] * rstd;
                            if (in) {
                                acc0[j] = fma2(g0[j], a[j], acc0[j]);
                                acc1[j] = fma2(g1[j], b[j], acc1[j]);
                            }
                            a[j] = fma2(a[j], k, v0[j] * rstd);
                            b[j] = fma2(b[j], k, v1[j] * rstd);
                        }
                    }
                }
                const int oat = head * static_cast<int>(rows.o_h);
                if (in && on0) *reinterpret_cast<uint4*>(out + (oat + col0)) = pack_pairs<T>(a);
                if (in && on1) *reinterpret_cast<uint4*>(out + (oat + col1)) = pack_pairs<T>(b);
            }
        }
    };
    auto start = [&](const HeadRows<T>& rows, const T* x, const T* dy, int begin, int end) {
#pragma unroll
        for (int i = 0; i < U; ++i) fetch(rows, x, dy, i, begin + i, end);
    };

    const int steps_q = (h.heads + per_step - 1) / per_step, steps_k = kBackward ? 0 : (rows_k.heads + per_step - 1) / per_step;
    const unsigned units = static_cast<unsigned>(h.units), seq = static_cast<unsigned>(p.seq), chunks = h.chunks;
    const unsigned unit_step = static_cast<unsigned>(h.ctas) * kWarps;
    for (unsigned u = cta * kWarps + warp; u < units; u += unit_step) {
        const unsigned token = chunks == 1 ? u : u / chunks;
        const int begin = static_cast<int>(u - token * chunks) * h.steps, end = min(begin + h.steps, steps_q + steps_k);
        const int end_q = min(end, steps_q), begin_k = max(begin, steps_q) - steps_q, end_k = end - steps_q;
        const unsigned b = token / seq, s = token - b * seq;
        const T* x = h.x + b * h.x_b + s * h.x_s;
        const T* dy = kBackward ? h.dy + b * h.dy_b + s * h.dy_s : nullptr;
        const T* xk = kBackward ? nullptr : rows_k.x + b * rows_k.x_b + s * rows_k.x_s;
        // the first loads are in flight while the angles are formed
        if (begin < end_q) start(h, x, dy, begin, end_q);
        else if (!kBackward) start(rows_k, xk, dy, begin_k, end_k);

        const double pos = rope_position(p, b, s);
        __syncwarp();  // the previous token's table has been read
        for (int i = lane; i < table_len; i += 32) {
            const float2 t = i < p.half ? rope_angle<sizeof(T) == 2>(pos, p.freq[i] * kTurnsPerRadian, p.scale, p.sin_sign) : make_float2(1.f, 0.f);
            cos_table[i] = t.x;
            sin_table[i] = t.y;
        }
        __syncwarp();
#pragma unroll
        for (int j = 0; j < VEC; j += 4) {  // 16-byte aligned: table_len and it * VEC are whole vectors
            *reinterpret_cast<float4*>(c + j) = *reinterpret_cast<const float4*>(cos_table + (on ? it * VEC : 0) + j);
            *reinterpret_cast<float4*>(n + j) = *reinterpret_cast<const float4*>(sin_table + (on ? it * VEC : 0) + j);
        }
        if (begin < end_q) {
            if constexpr (MODE == kHeadNorm) load_weights(h);
            walk(h, x, dy, h.out + b * h.o_b + s * h.o_s, begin, end_q);
        }
        if constexpr (!kBackward) {
            if (begin_k < end_k) {
                if (begin < end_q) start(rows_k, xk, dy, begin_k, end_k);
                load_weights(rows_k);
                walk(rows_k, xk, dy, rows_k.out + b * rows_k.o_b + s * rows_k.o_s, begin_k, end_k);
            }
        }
    }

    if constexpr (MODE == kHeadNormBackward) {
        if (h.partial == nullptr) return;  // the same for the whole CTA
        // lanes that hold the same columns first (a fixed butterfly), then the warps in order
        float sum0[VEC], sum1[VEC];
#pragma unroll
        for (int j = 0; j < N; ++j) {
            split(acc0[j], sum0[2 * j], sum0[2 * j + 1]);
            split(acc1[j], sum1[2 * j], sum1[2 * j + 1]);
        }
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            for (int o = p.lanes; o < 32; o <<= 1) {
                sum0[j] += __shfl_xor_sync(0xffffffffu, sum0[j], o);
                sum1[j] += __shfl_xor_sync(0xffffffffu, sum1[j], o);
            }
        }
        __syncthreads();  // the tables are no longer needed: their space holds the warps' sums, [warps][dim]
        float* sums = reinterpret_cast<float*>(head_smem);
        if (sub == 0) {
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                if (on0) sums[warp * p.dim + col0 + j] = sum0[j];
                if (on1) sums[warp * p.dim + col1 + j] = sum1[j];
            }
        }
        __syncthreads();
        for (int d = threadIdx.x; d < p.dim; d += kWarps * 32) {
            float t = 0.f;
#pragma unroll
            for (int k = 0; k < kWarps; ++k) t += sums[k * p.dim + d];
            h.partial[static_cast<long long>(cta) * p.dim + d] = t;
        }
    }
}

// Row form. Shared memory of a warp, in floats: table [half][2] | x rows [kRowFormRows][dim] | (backward) dy rows
// [kRowFormRows][dim] | dweight sums [dim].
__host__ __device__ inline int row_form_floats(int dim, int half, int mode) {
    const int n = 2 * half + kRowFormRows * dim * (mode == kHeadNormBackward ? 2 : 1) + (mode == kHeadNormBackward ? dim : 0);
    return (n + 1) & ~1;  // the next warp's table starts on 8 bytes
}

template <class T, bool INTERLEAVED, int MODE>
__global__ void __launch_bounds__(kRowFormWarps * 32)
heads_row_kernel(const HeadRows<T> rows_q, const HeadRows<T> rows_k, const RopePlan p) {
    extern __shared__ __align__(16) unsigned char head_smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const bool second = static_cast<int>(blockIdx.x) >= rows_q.ctas;
    const HeadRows<T>& h = second ? rows_k : rows_q;
    const int cta = static_cast<int>(blockIdx.x) - (second ? rows_q.ctas : 0);
    const int dim = p.dim, floats = row_form_floats(dim, p.half, MODE);
    float* mine = reinterpret_cast<float*>(head_smem) + warp * floats;
    float2* table = reinterpret_cast<float2*>(mine);
    float* xs = mine + 2 * p.half;
    float* ds = xs + kRowFormRows * dim;
    float* acc = ds + kRowFormRows * dim;
    const float inv_dim = 1.0f / static_cast<float>(dim);
    if constexpr (MODE == kHeadNormBackward)
        for (int d = lane; d < dim; d += 32) acc[d] = 0.f;

    // rows first .. first + n of one token's heads, as floats
    auto load = [&](float* dst, const T* src, long long stride, int first, int n) {
        if (p.pairs2) {
            struct alignas(2 * sizeof(T)) Two { T v[2]; };
#pragma unroll
            for (int r = 0; r < kRowFormRows; ++r) {
                if (r >= n) break;
                const Two* row = reinterpret_cast<const Two*>(src + (first + r) * stride);
#pragma unroll 4
                for (int d = lane; d < dim / 2; d += 32) {
                    const Two t = row[d];
                    dst[r * dim + 2 * d] = Cvt<T>::to_f(t.v[0]);
                    dst[r * dim + 2 * d + 1] = Cvt<T>::to_f(t.v[1]);
                }
            }
        } else {
            for (int r = 0; r < n; ++r) {
                const T* row = src + (first + r) * stride;
#pragma unroll 4
                for (int d = lane; d < dim; d += 32) dst[r * dim + d] = Cvt<T>::to_f(row[d]);
            }
        }
    };
    // the rotation of one staged row in place; a lane owns its pairs
    auto turn = [&](float* row) {
        for (int i = lane; i < p.half; i += 32) {
            const int i0 = INTERLEAVED ? 2 * i : i, i1 = INTERLEAVED ? 2 * i + 1 : i + p.half;
            const float a = row[i0], b = row[i1];
            const float2 t = table[i];
            row[i0] = a * t.x - b * t.y;
            row[i1] = b * t.x + a * t.y;
        }
    };

    const unsigned units = static_cast<unsigned>(h.units), seq = static_cast<unsigned>(p.seq), chunks = h.chunks;
    const unsigned unit_step = static_cast<unsigned>(h.ctas) * kRowFormWarps;
    for (unsigned u = cta * kRowFormWarps + warp; u < units; u += unit_step) {
        const unsigned token = u / chunks;
        const int head0 = static_cast<int>(u - token * chunks) * h.steps;
        const int head1 = min(head0 + h.steps, h.heads);
        const unsigned b = token / seq, s = token - b * seq;
        const T* x = h.x + b * h.x_b + s * h.x_s;
        const T* dy = MODE == kHeadNormBackward ? h.dy + b * h.dy_b + s * h.dy_s : nullptr;
        T* out = h.out + b * h.o_b + s * h.o_s;
        const double pos = rope_position(p, b, s);
        __syncwarp();
        for (int i = lane; i < p.half; i += 32) table[i] = rope_angle<sizeof(T) == 2>(pos, p.freq[i] * kTurnsPerRadian, p.scale, p.sin_sign);
        for (int head = head0; head < head1; head += kRowFormRows) {
            const int n = min(kRowFormRows, head1 - head);
            __syncwarp();  // the rows of the previous step have been stored
            load(xs, x, h.x_h, head, n);
            if constexpr (MODE == kHeadNormBackward) load(ds, dy, h.dy_h, head, n);
            __syncwarp();
            for (int r = 0; r < n; ++r) {
                float* row = xs + r * dim;
                if constexpr (MODE == kHeadRope) {
                    turn(row);
                } else if constexpr (MODE == kHeadNorm) {
                    float ss = 0.f;
                    for (int d = lane; d < dim; d += 32) ss = fmaf(row[d], row[d], ss);
#pragma unroll
                    for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
                    const float rstd = head_rstd(ss, inv_dim, p.eps);
                    for (int d = lane; d < dim; d += 32) row[d] = row[d] * rstd * Cvt<T>::to_f(h.weight[d]);
                    __syncwarp();
                    turn(row);
                } else {
                    float* g = ds + r * dim;
                    turn(g);
                    __syncwarp();
                    float ss = 0.f, dot = 0.f;
                    for (int d = lane; d < dim; d += 32) {
                        ss = fmaf(row[d], row[d], ss);
                        dot = fmaf(g[d] * Cvt<T>::to_f(h.weight[d]), row[d], dot);
                    }
#pragma unroll
                    for (int o = 16; o > 0; o >>= 1) {
                        ss += __shfl_xor_sync(0xffffffffu, ss, o);
                        dot += __shfl_xor_sync(0xffffffffu, dot, o);
                    }
                    const float rstd = head_rstd(ss, inv_dim, p.eps);
                    const float k = rstd * rstd * dot * inv_dim;
                    for (int d = lane; d < dim; d += 32) {
                        acc[d] = fmaf(g[d], row[d] * rstd, acc[d]);
                        row[d] = rstd * (g[d] * Cvt<T>::to_f(h.weight[d]) - row[d] * k);
                    }
                }
            }
            __syncwarp();
            for (int r = 0; r < n; ++r) {
                T* dst = out + (head + r) * h.o_h;
                for (int d = lane; d < dim; d += 32) dst[d] = Cvt<T>::from_f(xs[r * dim + d]);
            }
        }
    }

    if constexpr (MODE == kHeadNormBackward) {
        if (h.partial == nullptr) return;
        __syncthreads();
        for (int d = threadIdx.x; d < dim; d += kRowFormWarps * 32) {
            float t = 0.f;
#pragma unroll
            for (int k = 0; k < kRowFormWarps; ++k)
                t += reinterpret_cast<float*>(head_smem)[k * floats + (acc - mine) + d];
            h.partial[static_cast<long long>(cta) * dim + d] = t;
        }
    }
}

// dweight[d] = sum of the partial rows in a fixed order; blockIdx.y picks the query's or the key's.
template <class T>
__global__ void __launch_bounds__(1024)
head_dweight_kernel(const float* partial_q, int n_q, T* dweight_q, const float* partial_k, int n_k, T* dweight_k, int dim) {
    __shared__ float sm[32][33];
    ptx::grid_dep_wait();  // the partial rows are the preceding kernel's
    const float* partial = blockIdx.y ? partial_k : partial_q;
    const int n = blockIdx.y ? n_k : n_q;
    T* dweight = blockIdx.y ? dweight_k : dweight_q;
    if (dweight == nullptr) return;
    const int col = blockIdx.x * 32 + threadIdx.x;
    float a = 0.f;
    if (col < dim)
        for (int i = threadIdx.y; i < n; i += 32) a += partial[static_cast<long long>(i) * dim + col];
    sm[threadIdx.y][threadIdx.x] = a;
    __syncthreads();
    if (threadIdx.y == 0 && col < dim) {
        float s = 0.f;
#pragma unroll
        for (int k = 0; k < 32; ++k) s += sm[k][threadIdx.x];
        dweight[col] = Cvt<T>::from_f(s);
    }
}

}  // namespace lce
