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
#pragma once

#include "ptx.cuh"
#include "vec.cuh"

namespace lce {

constexpr int kHeadThreads = 256;
constexpr int kHeadWarps = kHeadThreads / 32;
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
    long long units;  // tokens * chunks
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

// cos and sin of position * frequency, times scale: the product in turns and its fraction in 64 bits.
__device__ __forceinline__ float2 rope_angle(double pos, double freq, float scale, float sin_sign) {
    double turns = pos * (freq * 0.15915494309189533577);  // 1 / (2 pi)
    turns -= rint(turns);
    float s, c;
    sincospif(2.f * static_cast<float>(turns), &s, &c);
    return make_float2(c * scale, s * scale * sin_sign);
}

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

// A lane's two vectors turned by the angles cs / sn (VEC of them). rot0 / rot1: whether the vector is inside the
// rotated part at all (the half layout pairs vectors that are both inside or both outside).
template <class T, bool INTERLEAVED, int VEC = RmsTile<T>::kVec>
__device__ __forceinline__ void rope_turn(float (&a)[VEC], float (&b)[VEC], const float (&cs)[VEC], const float (&sn)[VEC],
                                          bool rot0, bool rot1) {
    if constexpr (INTERLEAVED) {
#pragma unroll
        for (int j = 0; j < VEC / 2; ++j) {
            if (rot0) {
                const float x = a[2 * j], y = a[2 * j + 1];
                a[2 * j] = x * cs[j] - y * sn[j];
                a[2 * j + 1] = y * cs[j] + x * sn[j];
            }
            if (rot1) {
                const float x = b[2 * j], y = b[2 * j + 1];
                b[2 * j] = x * cs[VEC / 2 + j] - y * sn[VEC / 2 + j];
                b[2 * j + 1] = y * cs[VEC / 2 + j] + x * sn[VEC / 2 + j];
            }
        }
    } else if (rot0) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            const float x = a[j], y = b[j];
            a[j] = x * cs[j] - y * sn[j];
            b[j] = y * cs[j] + x * sn[j];
        }
    }
}

template <class T, bool INTERLEAVED, int MODE>
__global__ void __launch_bounds__(kHeadThreads, MODE == kHeadNormBackward ? 2 : 3)
heads_vector_kernel(const HeadRows<T> rows_q, const HeadRows<T> rows_k, const RopePlan p) {
    constexpr int VEC = RmsTile<T>::kVec;
    constexpr int U = 2;  // steps whose loads are in flight together
    extern __shared__ __align__(16) unsigned char head_smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const bool second = static_cast<int>(blockIdx.x) >= rows_q.ctas;
    const HeadRows<T>& h = second ? rows_k : rows_q;
    const int cta = static_cast<int>(blockIdx.x) - (second ? rows_q.ctas : 0);
    const int table_len = p.items * VEC;
    float2* table = reinterpret_cast<float2*>(head_smem) + warp * table_len;

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

    const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
    uint4 w0 = zero, w1 = zero;
    if constexpr (MODE != kHeadRope) {
        if (on0) w0 = *reinterpret_cast<const uint4*>(h.weight + col0);
        if (on1) w1 = *reinterpret_cast<const uint4*>(h.weight + col1);
    }
    float acc0[VEC], acc1[VEC];  // dweight of this lane's columns
    if constexpr (MODE == kHeadNormBackward) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) acc0[j] = acc1[j] = 0.f;
    }

    const int total_steps = (h.heads + per_step - 1) / per_step;
    const long long unit_step = static_cast<long long>(h.ctas) * kHeadWarps;
    for (long long u = static_cast<long long>(cta) * kHeadWarps + warp; u < h.units; u += unit_step) {
        const long long token = u / h.chunks;
        const int step0 = static_cast<int>(u - token * h.chunks) * h.steps;
        const int step1 = min(step0 + h.steps, total_steps);
        const long long b = token / p.seq, s = token - b * p.seq;
        const T* x = h.x + b * h.x_b + s * h.x_s;
        const T* dy = MODE == kHeadNormBackward ? h.dy + b * h.dy_b + s * h.dy_s : nullptr;
        T* out = h.out + b * h.o_b + s * h.o_s;

        uint4 x0[U], x1[U], d0[U], d1[U];
        auto fetch = [&](int step) {
#pragma unroll
            for (int i = 0; i < U; ++i) {
                const int head = (step + i) * per_step + sub;
                const bool in = step + i < step1 && head < h.heads;
                x0[i] = in && on0 ? *reinterpret_cast<const uint4*>(x + head * h.x_h + col0) : zero;
                x1[i] = in && on1 ? *reinterpret_cast<const uint4*>(x + head * h.x_h + col1) : zero;
                if constexpr (MODE == kHeadNormBackward) {
                    d0[i] = in && on0 ? *reinterpret_cast<const uint4*>(dy + head * h.dy_h + col0) : zero;
                    d1[i] = in && on1 ? *reinterpret_cast<const uint4*>(dy + head * h.dy_h + col1) : zero;
                }
            }
        };
        fetch(step0);  // in flight while the angles are formed

        const double pos = rope_position(p, b, s);
        __syncwarp();  // the previous token's table has been read
        for (int i = lane; i < table_len; i += 32)
            table[i] = i < p.half ? rope_angle(pos, p.freq[i], p.scale, p.sin_sign) : make_float2(1.f, 0.f);
        __syncwarp();
        float cs[VEC], sn[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            const float2 t = table[on ? it * VEC + j : j];
            cs[j] = t.x;
            sn[j] = t.y;
        }

        for (int step = step0; step < step1; step += U) {
            if (step != step0) fetch(step);
#pragma unroll
            for (int i = 0; i < U; ++i) {
                const int head = (step + i) * per_step + sub;
                const bool in = step + i < step1 && head < h.heads;
                float a[VEC], c[VEC];
                rms_unpack<T>(x0[i], a);
                rms_unpack<T>(x1[i], c);
                if constexpr (MODE == kHeadRope) {
                    rope_turn<T, INTERLEAVED>(a, c, cs, sn, rot0, rot1);
                } else {
                    float v0[VEC], v1[VEC];
                    rms_unpack<T>(w0, v0);
                    rms_unpack<T>(w1, v1);
                    float ss = 0.f;
#pragma unroll
                    for (int j = 0; j < VEC; ++j) ss = fmaf(a[j], a[j], fmaf(c[j], c[j], ss));
                    if constexpr (MODE == kHeadNorm) {
                        for (int o = p.lanes >> 1; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
                        const float rstd = head_rstd(ss, inv_dim, p.eps);
#pragma unroll
                        for (int j = 0; j < VEC; ++j) {
                            a[j] = a[j] * rstd * v0[j];
                            c[j] = c[j] * rstd * v1[j];
                        }
                        rope_turn<T, INTERLEAVED>(a, c, cs, sn, rot0, rot1);
                    } else {
                        float g0[VEC], g1[VEC];
                        rms_unpack<T>(d0[i], g0);
                        rms_unpack<T>(d1[i], g1);
                        rope_turn<T, INTERLEAVED>(g0, g1, cs, sn, rot0, rot1);
                        float dot = 0.f;
#pragma unroll
                        for (int j = 0; j < VEC; ++j) {
                            v0[j] *= g0[j];
                            v1[j] *= g1[j];
                            dot = fmaf(v0[j], a[j], fmaf(v1[j], c[j], dot));
                        }
                        for (int o = p.lanes >> 1; o > 0; o >>= 1) {
                            ss += __shfl_xor_sync(0xffffffffu, ss, o);
                            dot += __shfl_xor_sync(0xffffffffu, dot, o);
                        }
                        const float rstd = head_rstd(ss, inv_dim, p.eps);
                        const float k = rstd * rstd * dot * inv_dim;
#pragma unroll
                        for (int j = 0; j < VEC; ++j) {
                            if (in) {  // a row that is not there adds nothing, whatever 1 / sqrt(eps) is
                                acc0[j] = fmaf(g0[j], a[j] * rstd, acc0[j]);
                                acc1[j] = fmaf(g1[j], c[j] * rstd, acc1[j]);
                            }
                            a[j] = rstd * (v0[j] - a[j] * k);
                            c[j] = rstd * (v1[j] - c[j] * k);
                        }
                    }
                }
                if (in && on0) *reinterpret_cast<uint4*>(out + head * h.o_h + col0) = rms_pack<T>(a);
                if (in && on1) *reinterpret_cast<uint4*>(out + head * h.o_h + col1) = rms_pack<T>(c);
            }
        }
    }

    if constexpr (MODE == kHeadNormBackward) {
        if (h.partial == nullptr) return;  // the same for the whole CTA
        // lanes that hold the same columns first (a fixed butterfly), then the warps in order
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            for (int o = p.lanes; o < 32; o <<= 1) {
                acc0[j] += __shfl_xor_sync(0xffffffffu, acc0[j], o);
                acc1[j] += __shfl_xor_sync(0xffffffffu, acc1[j], o);
            }
        }
        __syncthreads();  // the tables are no longer needed: their space holds the warps' sums, [warps][dim]
        float* sums = reinterpret_cast<float*>(head_smem);
        if (sub == 0) {
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                if (on0) sums[warp * p.dim + col0 + j] = acc0[j];
                if (on1) sums[warp * p.dim + col1 + j] = acc1[j];
            }
        }
        __syncthreads();
        for (int d = threadIdx.x; d < p.dim; d += kHeadThreads) {
            float t = 0.f;
#pragma unroll
            for (int k = 0; k < kHeadWarps; ++k) t += sums[k * p.dim + d];
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

    const long long unit_step = static_cast<long long>(h.ctas) * kRowFormWarps;
    for (long long u = static_cast<long long>(cta) * kRowFormWarps + warp; u < h.units; u += unit_step) {
        const long long token = u / h.chunks;
        const int head0 = static_cast<int>(u - token * h.chunks) * h.steps;
        const int head1 = min(head0 + h.steps, h.heads);
        const long long b = token / p.seq, s = token - b * p.seq;
        const T* x = h.x + b * h.x_b + s * h.x_s;
        const T* dy = MODE == kHeadNormBackward ? h.dy + b * h.dy_b + s * h.dy_s : nullptr;
        T* out = h.out + b * h.o_b + s * h.o_s;
        const double pos = rope_position(p, b, s);
        __syncwarp();
        for (int i = lane; i < p.half; i += 32) table[i] = rope_angle(pos, p.freq[i], p.scale, p.sin_sign);
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
