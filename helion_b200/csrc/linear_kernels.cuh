// A projection with its epilogue on the GEMM cores, and what its backward pass needs around two matrix products.
//
//   forward    z = x W^T + bias;  y = act(z) + residual          (z in fp32 registers, rounded once, as y)
//   backward   dz = dy * act'(z);  dx = dz W;  dW = dz^T x;  dbias = column sums of dz;  dresidual = dy
//
// The epilogue adds the bias, applies the activation and adds the residual to the accumulator tile while the next
// tile multiplies, so that z never makes a round trip through memory. For a backward pass it also stores what the
// activation's derivative is computed from (`pre`: z in the input type, or for relu the derivative itself, 0 or 1, which a
// z that underflows would lose). dz is rounded to the input type because it is the operand of two tensor-core
// products (the column sums take it unrounded).
#pragma once

#include "epilogues.cuh"

namespace lce {

enum LinearAct { kActNone = 0, kActRelu = 1, kActGelu = 2, kActGeluTanh = 3, kActSilu = 4 };

// sigmoid(t) = r for t >= 0 and e r below, with e = exp(-|t|) and r = 1 / (1 + e) in [1/2, 1]: nothing overflows, and
// sigmoid(-t) is as exact as sigmoid(t). e is the square of exp(-|t| / 2) so that a product with it keeps results that
// e itself would flush to zero. FAST: the hardware's base-2 exponential and reciprocal (relative error ~1e-6, for
// results of 16 bits).
template <bool FAST>
struct Sigmoid {
    float h, r;
    bool positive;
    __device__ __forceinline__ explicit Sigmoid(float t) {
        positive = t >= 0.f;
        h = FAST ? ptx::ex2(-0.5f * kLog2e * fabsf(t)) : expf(-0.5f * fabsf(t));
        r = FAST ? __fdividef(1.f, fmaf(h, h, 1.f)) : 1.f / fmaf(h, h, 1.f);
    }
    __device__ __forceinline__ float times(float z) const { return (positive ? z : z * h * h) * r; }  // z sigmoid(t)
    __device__ __forceinline__ float other() const { return (positive ? h * h : 1.f) * r; }           // 1 - sigmoid(t)
};
constexpr float kGeluC = 0.7978845608028654f;  // sqrt(2 / pi)
constexpr float kGeluA = 0.044715f;

// The normal distribution function: Phi(-a) = exp(-a^2 / 2) g(a) for a >= 0, Phi(a) = 1 - Phi(-a). g falls smoothly from
// 1/2; for 16-bit results it is a polynomial in 1 / (1 + 0.26 a), fitted here by reweighted least squares to 3.4e-7 of
// its value for a up to 14 (with the 32-bit exponential 2e-6 up to a = 6). CUDA's normcdff would cost three times the
// instructions, and the epilogue has to keep up with the tensor cores.
struct NormalFast {
    float h, g;  // exp(-a^2 / 4), g(a)
    bool positive;
    __device__ __forceinline__ explicit NormalFast(float z) {
        const float a = fabsf(z), t = __fdividef(1.f, fmaf(0.26f, a, 1.f));
        positive = z >= 0.f;
        h = ptx::ex2(-0.36067376f * (a * a));
        float p = fmaf(-0.07724009f, t, 0.24633712f);
        p = fmaf(p, t, -0.135466f);
        p = fmaf(p, t, 0.19220619f);
        p = fmaf(p, t, 0.06021739f);
        p = fmaf(p, t, 0.11097057f);
        p = fmaf(p, t, 0.10293892f);
        g = fmaf(p, t, 3.572605e-05f);
    }
    __device__ __forceinline__ float times(float z) const {  // z Phi(z)
        const float tail = (z * h) * (h * g);
        return positive ? z - tail : tail;
    }
    __device__ __forceinline__ float density() const { return 0.3989422804014327f * (h * h); }
};

// act(z) of N values at a time; `act` is the same for the whole launch.
template <bool FAST, int N>
__device__ __forceinline__ void linear_act(float (&z)[N], int act) {
    if (act == kActRelu) {
#pragma unroll
        for (int j = 0; j < N; ++j) z[j] = z[j] <= 0.f ? 0.f : z[j];  // a NaN stays one
    } else if (act == kActGelu) {
#pragma unroll
        for (int j = 0; j < N; ++j) z[j] = FAST ? NormalFast(z[j]).times(z[j]) : z[j] * normcdff(z[j]);
    } else if (act == kActGeluTanh) {  // (1 + tanh(u)) / 2 = sigmoid(2u)
#pragma unroll
        for (int j = 0; j < N; ++j) z[j] = Sigmoid<FAST>(2.f * kGeluC * z[j] * fmaf(kGeluA * z[j], z[j], 1.f)).times(z[j]);
    } else if (act == kActSilu) {
#pragma unroll
        for (int j = 0; j < N; ++j) z[j] = Sigmoid<FAST>(z[j]).times(z[j]);
    }
}

// What the forward saves for act': z, or for relu the derivative itself.
template <int N>
__device__ __forceinline__ void linear_saved(const float (&z)[N], int act, float (&saved)[N]) {
#pragma unroll
    for (int j = 0; j < N; ++j) saved[j] = act == kActRelu ? (z[j] > 0.f ? 1.f : 0.f) : z[j];
}

// g *= act'(.) from what the forward saved.
template <bool FAST, int N>
__device__ __forceinline__ void linear_slope(float (&g)[N], const float (&pre)[N], int act) {
    if (act == kActRelu) {
#pragma unroll
        for (int j = 0; j < N; ++j) g[j] *= pre[j];
    } else if (act == kActGelu) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            if constexpr (FAST) {
                const NormalFast n(pre[j]);
                g[j] *= fmaf(pre[j], n.density(), n.times(1.f));
            } else {
                g[j] *= fmaf(pre[j] * 0.3989422804014327f, expf(-0.5f * pre[j] * pre[j]), normcdff(pre[j]));
            }
        }
    } else if (act == kActGeluTanh) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const Sigmoid<FAST> t(2.f * kGeluC * pre[j] * fmaf(kGeluA * pre[j], pre[j], 1.f));
            const float s = t.times(1.f), both = s * t.other();
            // far out the cubic may overflow against a zero
            g[j] *= both == 0.f ? s : fmaf(2.f * kGeluC * pre[j] * fmaf(3.f * kGeluA * pre[j], pre[j], 1.f), both, s);
        }
    } else if (act == kActSilu) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const Sigmoid<FAST> t(pre[j]);
            const float s = t.times(1.f), both = s * t.other();
            g[j] *= both == 0.f ? s : fmaf(pre[j], both, s);
        }
    }
}

// What follows a finished accumulator value: shared by the GEMM epilogue, the split-K sum and the decode kernel.
template <class T>
struct LinearTail {
    T* out;
    long long ldo;
    T* pre;  // [rows] of ldp elements, or nullptr
    long long ldp;
    const T* bias;      // or nullptr
    const T* residual;  // or nullptr
    long long ldr;
    int rows, cols;
    int act;
    static constexpr bool kFast = sizeof(T) == 2;
};

// `N` (compile-time) consecutive values of one row; `valid` of them exist.
template <class T, int N>
__device__ __forceinline__ void load_row(const T* src, float (&v)[N], int valid) {
    constexpr int kPer = 16 / sizeof(T);
    if (N % kPer == 0 && valid >= N && (reinterpret_cast<uintptr_t>(src) & 15u) == 0) {
#pragma unroll
        for (int i = 0; i < N / kPer; ++i) {
            float e[kPer];
            rms_unpack<T>(*reinterpret_cast<const uint4*>(src + i * kPer), e);
#pragma unroll
            for (int j = 0; j < kPer; ++j) v[i * kPer + j] = e[j];
        }
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] = j < valid ? Cvt<T>::to_f(src[j]) : 0.f;
    }
}

// A warp's 32 rows x 64 columns of 16-bit values in its shared-memory area, in the swizzled layout of store_block64: the
// row-wise side (a thread deposits or reads 32 of its own row's columns) and the line-wise side (whole lines of global
// memory; `wide`: 16 bytes per lane, which needs aligned rows, else two elements per lane).
__device__ __forceinline__ void area_put(float* stage, int lane, int half, const uint4 (&v)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) reinterpret_cast<uint4*>(stage)[lane * 8 + ((half * 4 + i) ^ (lane & 7))] = v[i];
}
__device__ __forceinline__ void area_get(const float* stage, int lane, int half, uint4 (&v)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = reinterpret_cast<const uint4*>(stage)[lane * 8 + ((half * 4 + i) ^ (lane & 7))];
}
template <class T>
__device__ __forceinline__ void area_to_lines(const float* stage, int lane, T* blk, long long ld, int rows, int cols, bool wide) {
    if (wide) {
        const int piece = lane & 7, left = cols - piece * 8;
#pragma unroll
        for (int it = 0; it < 8; ++it) {
            const int r = it * 4 + (lane >> 3);
            const uint4 val = reinterpret_cast<const uint4*>(stage)[r * 8 + (piece ^ (r & 7))];
            if (r < rows && left > 0) {
                T* dst = blk + static_cast<long long>(r) * ld + piece * 8;
                if (left >= 8) {
                    *reinterpret_cast<uint4*>(dst) = val;
                } else {
                    const T* e = reinterpret_cast<const T*>(&val);
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        if (j < left) dst[j] = e[j];
                }
            }
        }
    } else {
        const int left = cols - 2 * lane;
#pragma unroll 8
        for (int r = 0; r < 32; ++r) {
            const uint32_t val = reinterpret_cast<const uint32_t*>(stage)[(r * 8 + ((lane >> 2) ^ (r & 7))) * 4 + (lane & 3)];
            const T* e = reinterpret_cast<const T*>(&val);
            T* dst = blk + static_cast<long long>(r) * ld + 2 * lane;
            if (r < rows && left > 0) dst[0] = e[0];
            if (r < rows && left > 1) dst[1] = e[1];
        }
    }
}
// Lines of global memory into the area; the wide form splits into the loads (early) and the deposit (late).
template <class T>
__device__ __forceinline__ void lines_fetch(int lane, const T* blk, long long ld, int rows, int cols, uint4 (&v)[8]) {
    const int piece = lane & 7, left = cols - piece * 8;
#pragma unroll
    for (int it = 0; it < 8; ++it) {
        const int r = it * 4 + (lane >> 3);
        v[it] = make_uint4(0u, 0u, 0u, 0u);
        if (r < rows && left > 0) {
            const T* src = blk + static_cast<long long>(r) * ld + piece * 8;
            if (left >= 8) {
                v[it] = *reinterpret_cast<const uint4*>(src);
            } else {
                alignas(16) T e[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) e[j] = j < left ? src[j] : Cvt<T>::from_f(0.f);
                v[it] = *reinterpret_cast<const uint4*>(e);
            }
        }
    }
}
__device__ __forceinline__ void lines_put(float* stage, int lane, const uint4 (&v)[8]) {
    const int piece = lane & 7;
#pragma unroll
    for (int it = 0; it < 8; ++it) {
        const int r = it * 4 + (lane >> 3);
        reinterpret_cast<uint4*>(stage)[r * 8 + (piece ^ (r & 7))] = v[it];
    }
}
template <class T>
__device__ __forceinline__ void lines_to_area(float* stage, int lane, const T* blk, long long ld, int rows, int cols) {
    const int left = cols - 2 * lane;
#pragma unroll 8
    for (int r = 0; r < 32; ++r) {
        const T* src = blk + static_cast<long long>(r) * ld + 2 * lane;
        alignas(4) T e[2];
        e[0] = r < rows && left > 0 ? src[0] : Cvt<T>::from_f(0.f);
        e[1] = r < rows && left > 1 ? src[1] : Cvt<T>::from_f(0.f);
        reinterpret_cast<uint32_t*>(stage)[(r * 8 + ((lane >> 2) ^ (r & 7))) * 4 + (lane & 3)] = *reinterpret_cast<const uint32_t*>(e);
    }
}
template <class T>
__device__ __forceinline__ void pack32(const float (&v)[32], uint4 (&raw)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float e[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) e[j] = v[i * 8 + j];
        raw[i] = rms_pack<T>(e);
    }
}

template <class T>
struct EpiLinear {
    static constexpr bool kHasFinish = false;
    struct Params {
        LinearTail<T> t;
        float* scratch;         // split-K: slabs of partial sums (the layout of EpiStore), or nullptr
        long long slab_floats;
        int wide_out, wide_residual;  // rows that 16-byte accesses can take (pre's always are)
    };
    // Besides the row: the residual's next 64 columns in flight, and the first half of a block's saved values, which
    // leave when the second half is there.
    struct State {
        int row;
        uint4 next[sizeof(T) == 2 ? 8 : 1];
        uint4 saved[sizeof(T) == 2 ? 4 : 1];
    };
    static __device__ __forceinline__ void begin(State& st, const Params& p, const TileCtx& tc) {
        st.row = tc.m_tile * kBM + tc.row_in_tile;
        if constexpr (sizeof(T) == 2) {
            if (p.scratch != nullptr || tc.stage == nullptr) return;
            const LinearTail<T>& t = p.t;
            const int lane = tc.row_in_tile & 31, col0 = tc.n_tile * tc.bn, row_base = st.row - lane;
            if (t.bias != nullptr) {  // the tile's slice of the bias, as floats, behind the re-shaping area
                float* bias = tc.stage + kStageBiasOffset;
                __syncwarp();  // the previous tile's has been read
                for (int c = lane * 8; c < tc.bn; c += 256) {
                    float b[8];
                    load_row<T>(t.bias + col0 + c, b, t.cols - col0 - c);
                    *reinterpret_cast<float4*>(bias + c) = make_float4(b[0], b[1], b[2], b[3]);
                    *reinterpret_cast<float4*>(bias + c + 4) = make_float4(b[4], b[5], b[6], b[7]);
                }
                __syncwarp();
            }
            if (t.residual != nullptr && p.wide_residual)
                lines_fetch<T>(lane, t.residual + static_cast<long long>(row_base) * t.ldr + col0, t.ldr, t.rows - row_base, t.cols - col0, st.next);
        }
    }
    static __device__ __forceinline__ void chunk(State& st, const Params& p, const TileCtx& tc, int col0, float (&v)[32]) {
        const LinearTail<T>& t = p.t;
        const int gcol0 = tc.n_tile * tc.bn + col0;
        const int valid = t.cols - gcol0;
        if (p.scratch != nullptr) {
            if (st.row >= t.rows || valid <= 0) return;
            float4* sp = reinterpret_cast<float4*>(p.scratch) + static_cast<long long>(tc.k_slice) * (p.slab_floats / 4) +
                         ((static_cast<long long>(tc.m_tile) * tc.n_tiles + tc.n_tile) * (tc.bn / 4) + col0 / 4) * kBM + tc.row_in_tile;
#pragma unroll
            for (int i = 0; i < 8; ++i) sp[i * kBM] = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
            return;
        }
        if constexpr (sizeof(T) == 2) {
            if (tc.stage != nullptr) {  // all 32 lanes take part, whatever their row and column
                staged(st, p, tc, col0, gcol0, v);
                return;
            }
        }
        if (st.row >= t.rows || valid <= 0) return;
        if (t.bias != nullptr) {
            float b[32];
            load_row<T>(t.bias + gcol0, b, valid);
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] += b[j];
        }
        if (t.pre != nullptr) {
            float saved[32];
            linear_saved(v, t.act, saved);
            store_row32<T>(t.pre + static_cast<long long>(st.row) * t.ldp + gcol0, saved, valid);
        }
        linear_act<LinearTail<T>::kFast>(v, t.act);
        if (t.residual != nullptr) {
            float r[32];
            load_row<T>(t.residual + static_cast<long long>(st.row) * t.ldr + gcol0, r, valid);
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] += r[j];
        }
        store_row32<T>(t.out + static_cast<long long>(st.row) * t.ldo + gcol0, v, valid);
    }
    // The 16-bit form: everything that touches global memory goes through the warp's area as whole lines.
    static __device__ __forceinline__ void staged(State& st, const Params& p, const TileCtx& tc, int col0, int gcol0, float (&v)[32]) {
        const LinearTail<T>& t = p.t;
        const int lane = tc.row_in_tile & 31, half = (col0 >> 5) & 1;
        const int row_base = st.row - lane, blk0 = gcol0 - half * 32;
        const int rows = t.rows - row_base, cols = t.cols - blk0;  // of the 64-column block
        if (t.bias != nullptr) {
            const float4* b = reinterpret_cast<const float4*>(tc.stage + kStageBiasOffset + col0);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float4 x = b[i];
                v[4 * i] += x.x;
                v[4 * i + 1] += x.y;
                v[4 * i + 2] += x.z;
                v[4 * i + 3] += x.w;
            }
        }
        uint4 keep[4];
        if (t.pre != nullptr) {
            float saved[32];
            linear_saved(v, t.act, saved);
            pack32<T>(saved, keep);
        }
        linear_act<true>(v, t.act);
        if (t.residual != nullptr) {
            if (half == 0) {
                const T* src = t.residual + static_cast<long long>(row_base) * t.ldr + blk0;
                if (p.wide_residual) {
                    lines_put(tc.stage, lane, st.next);
                    if (col0 + 64 < tc.bn) lines_fetch<T>(lane, src + 64, t.ldr, rows, cols - 64, st.next);
                } else {
                    lines_to_area<T>(tc.stage, lane, src, t.ldr, rows, cols);
                }
                __syncwarp();
            }
            uint4 r[4];
            area_get(tc.stage, lane, half, r);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float e[8];
                rms_unpack<T>(r[i], e);
#pragma unroll
                for (int j = 0; j < 8; ++j) v[i * 8 + j] += e[j];
            }
        }
        uint4 y[4];
        pack32<T>(v, y);
        area_put(tc.stage, lane, half, y);
        if (half == 0) {
            if (t.pre != nullptr) {
#pragma unroll
                for (int i = 0; i < 4; ++i) st.saved[i] = keep[i];
            }
            return;
        }
        __syncwarp();
        area_to_lines<T>(tc.stage, lane, t.out + static_cast<long long>(row_base) * t.ldo + blk0, t.ldo, rows, cols, p.wide_out != 0);
        __syncwarp();
        if (t.pre != nullptr) {
            area_put(tc.stage, lane, 0, st.saved);
            area_put(tc.stage, lane, 1, keep);
            __syncwarp();
            area_to_lines<T>(tc.stage, lane, t.pre + static_cast<long long>(row_base) * t.ldp + blk0, t.ldp, rows, cols, true);
            __syncwarp();
        }
    }
    static __device__ __forceinline__ void end(State&, const Params&, const TileCtx&) {}
};

// Adds the slices of a split contraction in slice order and finishes the values. One thread = four columns of a row.
template <class T>
__global__ void __launch_bounds__(256)
linear_reduce_kernel(const float* scratch, int slices, long long slab_floats, int n_tiles, int bn, const LinearTail<T> t) {
    ptx::grid_dep_launch();
    ptx::grid_dep_wait();  // `scratch` holds the slices of the preceding GEMM
    const long long quads_per_row = (static_cast<long long>(t.cols) + 3) / 4;
    const long long total = quads_per_row * t.rows;
    for (long long i = blockIdx.x * static_cast<long long>(blockDim.x) + threadIdx.x; i < total;
         i += static_cast<long long>(gridDim.x) * blockDim.x) {
        const int row = static_cast<int>(i / quads_per_row);
        const int col = static_cast<int>(i - row * quads_per_row) * 4;
        const int n_tile = col / bn, c4 = (col - n_tile * bn) / 4, m_tile = row / kBM;
        const float4* sp = reinterpret_cast<const float4*>(scratch) +
                           ((static_cast<long long>(m_tile) * n_tiles + n_tile) * (bn / 4) + c4) * kBM + (row - m_tile * kBM);
        float4 a = sp[0];
        for (int s = 1; s < slices; ++s) {
            const float4 o = sp[static_cast<long long>(s) * (slab_floats / 4)];
            a.x += o.x;
            a.y += o.y;
            a.z += o.z;
            a.w += o.w;
        }
        float z[4] = {a.x, a.y, a.z, a.w};
        const int valid = t.cols - col;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (t.bias != nullptr && j < valid) z[j] += Cvt<T>::to_f(t.bias[col + j]);
        if (t.pre != nullptr) {
            float saved[4];
            linear_saved(z, t.act, saved);
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (j < valid) t.pre[row * t.ldp + col + j] = Cvt<T>::from_f(saved[j]);
        }
        linear_act<LinearTail<T>::kFast>(z, t.act);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (j >= valid) break;
            if (t.residual != nullptr) z[j] += Cvt<T>::to_f(t.residual[row * t.ldr + col + j]);
            t.out[row * t.ldo + col + j] = Cvt<T>::from_f(z[j]);
        }
    }
}

// Rows copied to a pitch that TMA can read (a multiple of 16 bytes): operands whose rows start off 16-byte boundaries.
template <class T>
__global__ void __launch_bounds__(256)
repitch_kernel(const T* __restrict__ src, long long lds, T* __restrict__ dst, long long ldd, long long rows, int cols) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (long long r = blockIdx.x * 8ll + warp; r < rows; r += gridDim.x * 8ll)
        for (int c = lane; c < cols; c += 32) dst[r * ldd + c] = src[r * lds + c];
}

// dz = dy * act'(pre), rounded, and the column sums of the unrounded dz over this CTA's rows.
// A CTA of 256 threads owns 32 x VEC columns and the row slab [slab * rows_per_slab, ...): 32 column groups x 8 rows
// at a time, two of them in flight. Bound by the bytes: dy and pre in, dz out. partial: [slabs][cols] (nullptr: no sums);
// dz nullptr: sums only (no activation, dz = dy). Columns of dz up to its pitch, behind the last, are set to zero.
template <class T, int VEC>
__global__ void __launch_bounds__(256)
linear_dz_kernel(const T* __restrict__ dy, long long ldy, const T* __restrict__ pre, long long ldp, T* __restrict__ dz, long long ldz,
                 float* __restrict__ partial, long long rows, int cols, long long rows_per_slab, int act) {
    constexpr int U = 2;
    __shared__ float sums[8][32 * VEC + 1];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int col = (blockIdx.x * 32 + lane) * VEC;
    const long long row_begin = blockIdx.y * rows_per_slab, row_end = min(rows, row_begin + rows_per_slab);
    const int valid = cols - col;
    float acc[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) acc[j] = 0.f;
    if (valid > 0) {
        for (long long row0 = row_begin + warp; row0 < row_end; row0 += 8 * U) {
            float g[U][VEC], z[U][VEC];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const long long row = row0 + 8 * u;
                if (row < row_end) {
                    load_row<T, VEC>(dy + row * ldy + col, g[u], valid);
                    if (act != kActNone) load_row<T, VEC>(pre + row * ldp + col, z[u], valid);
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const long long row = row0 + 8 * u;
                if (row >= row_end) break;
                linear_slope<LinearTail<T>::kFast>(g[u], z[u], act);
                if (dz != nullptr) *reinterpret_cast<uint4*>(dz + row * ldz + col) = rms_pack<T>(g[u]);
#pragma unroll
                for (int j = 0; j < VEC; ++j) acc[j] += g[u][j];
            }
        }
    }
    if (partial == nullptr) return;
#pragma unroll
    for (int j = 0; j < VEC; ++j) sums[warp][lane * VEC + j] = acc[j];
    __syncthreads();
    for (int c = threadIdx.x; c < 32 * VEC; c += 256) {
        const int gc = blockIdx.x * 32 * VEC + c;
        if (gc >= cols) break;
        float s = 0.f;
#pragma unroll
        for (int k = 0; k < 8; ++k) s += sums[k][c];
        partial[static_cast<long long>(blockIdx.y) * cols + gc] = s;
    }
}

// dbias[c] = sum of the slabs' column sums in a fixed order. 32 columns x 32 slabs at a time.
template <class T>
__global__ void __launch_bounds__(1024)
linear_dbias_kernel(const float* partial, int slabs, int cols, T* __restrict__ dbias) {
    __shared__ float sm[32][33];
    ptx::grid_dep_wait();  // the preceding kernel's partial sums
    const int x = threadIdx.x & 31, y = threadIdx.x >> 5, c = blockIdx.x * 32 + x;
    float s = 0.f;
    if (c < cols)
        for (int k = y; k < slabs; k += 32) s += partial[static_cast<long long>(k) * cols + c];
    sm[y][x] = s;
    __syncthreads();
    if (y == 0 && c < cols) {
        s = 0.f;
#pragma unroll
        for (int k = 0; k < 32; ++k) s += sm[k][x];
        dbias[c] = Cvt<T>::from_f(s);
    }
}

}  // namespace lce
