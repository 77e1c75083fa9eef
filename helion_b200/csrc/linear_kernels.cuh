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

template <bool FAST>
__device__ __forceinline__ float linear_act(float z, int act) {
    switch (act) {
        case kActRelu: return z <= 0.f ? 0.f : z;  // a NaN stays one
        case kActGelu: return z * normcdff(z);
        case kActGeluTanh: return Sigmoid<FAST>(2.f * kGeluC * z * fmaf(kGeluA * z, z, 1.f)).times(z);  // tanh(u) = 2 sigmoid(2u) - 1
        case kActSilu: return Sigmoid<FAST>(z).times(z);
        default: return z;
    }
}

// act'(z) from what the forward saved.
template <bool FAST>
__device__ __forceinline__ float linear_slope(float pre, int act) {
    switch (act) {
        case kActRelu: return pre;
        case kActGelu: return fmaf(pre * 0.3989422804014327f, expf(-0.5f * pre * pre), normcdff(pre));
        case kActGeluTanh: {
            const Sigmoid<FAST> g(2.f * kGeluC * pre * fmaf(kGeluA * pre, pre, 1.f));
            const float s = g.times(1.f), both = s * g.other();
            if (both == 0.f) return s;  // far out, where the cubic may overflow against it
            return fmaf(2.f * kGeluC * pre * fmaf(3.f * kGeluA * pre, pre, 1.f), both, s);
        }
        case kActSilu: {
            const Sigmoid<FAST> g(pre);
            const float s = g.times(1.f), both = s * g.other();
            return both == 0.f ? s : fmaf(pre, both, s);
        }
        default: return 1.f;
    }
}

// What follows a finished accumulator value: shared by the GEMM epilogue and the split-K sum.
template <class T>
struct LinearTail {
    T* out;
    long long ldo;
    T* pre;  // [rows][cols] contiguous, or nullptr
    const T* bias;      // or nullptr
    const T* residual;  // or nullptr
    long long ldr;
    int rows, cols;
    int act;
    static constexpr bool kFast = sizeof(T) == 2;
};

// `n` (compile-time) consecutive values of one row; `valid` of them exist.
template <class T, int N>
__device__ __forceinline__ void load_row(const T* src, float (&v)[N], int valid) {
    constexpr int kPer = 16 / sizeof(T);
    if (N % kPer == 0 && valid >= N && (reinterpret_cast<uintptr_t>(src) & 15u) == 0) {
#pragma unroll
        for (int i = 0; i < N / kPer; ++i) {
            const uint4 raw = *reinterpret_cast<const uint4*>(src + i * kPer);
            const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
            for (int j = 0; j < kPer; ++j) v[i * kPer + j] = Cvt<T>::to_f(e[j]);
        }
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] = j < valid ? Cvt<T>::to_f(src[j]) : 0.f;
    }
}

template <class T>
struct EpiLinear {
    static constexpr bool kHasFinish = false;
    struct Params {
        LinearTail<T> t;
        float* scratch;         // split-K: slabs of partial sums (the layout of EpiStore), or nullptr
        long long slab_floats;
        int wide;  // 16-bit results leave as whole 128-byte lines
    };
    struct State {
        int row;
    };
    static __device__ __forceinline__ void begin(State& st, const Params&, const TileCtx& tc) {
        st.row = tc.m_tile * kBM + tc.row_in_tile;
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
        const bool here = st.row < t.rows && valid > 0;
        if (t.bias != nullptr && valid > 0) {
            float b[32];
            load_row<T>(t.bias + gcol0, b, valid);
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] += b[j];
        }
        if (t.pre != nullptr && here) {
            T* dst = t.pre + static_cast<long long>(st.row) * t.cols + gcol0;
            if (t.act == kActRelu) {
                float step[32];
#pragma unroll
                for (int j = 0; j < 32; ++j) step[j] = v[j] > 0.f ? 1.f : 0.f;
                store_row32<T>(dst, step, valid);
            } else {
                store_row32<T>(dst, v, valid);
            }
        }
        if (t.act != kActNone) {
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] = linear_act<LinearTail<T>::kFast>(v[j], t.act);
        }
        if (t.residual != nullptr && here) {
            float r[32];
            load_row<T>(t.residual + static_cast<long long>(st.row) * t.ldr + gcol0, r, valid);
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] += r[j];
        }
        if constexpr (sizeof(T) == 2) {
            if (p.wide != 0 && tc.stage != nullptr) {  // all 32 lanes take part, whatever their row and column
                const int lane = tc.row_in_tile & 31, half = (col0 >> 5) & 1;
                const int row_base = st.row - lane, blk0 = gcol0 - half * 32;
                store_block64<T>(tc.stage, lane, half, v, t.out + static_cast<long long>(row_base) * t.ldo + blk0, t.ldo,
                                 t.rows - row_base, t.cols - blk0);
                return;
            }
        }
        if (here) store_row32<T>(t.out + static_cast<long long>(st.row) * t.ldo + gcol0, v, valid);
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
        const float acc[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (col + j >= t.cols) break;
            float z = acc[j];
            if (t.bias != nullptr) z += Cvt<T>::to_f(t.bias[col + j]);
            if (t.pre != nullptr)
                t.pre[static_cast<long long>(row) * t.cols + col + j] = Cvt<T>::from_f(t.act == kActRelu ? (z > 0.f ? 1.f : 0.f) : z);
            float y = linear_act<LinearTail<T>::kFast>(z, t.act);
            if (t.residual != nullptr) y += Cvt<T>::to_f(t.residual[row * t.ldr + col + j]);
            t.out[row * t.ldo + col + j] = Cvt<T>::from_f(y);
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
// at a time. partial: [slabs][cols] (nullptr: no sums); dz nullptr: sums only (no activation, dz = dy).
template <class T, int VEC>
__global__ void __launch_bounds__(256)
linear_dz_kernel(const T* __restrict__ dy, long long ldy, const T* __restrict__ pre, T* __restrict__ dz, long long ldz,
                 float* __restrict__ partial, long long rows, int cols, long long rows_per_slab, int act) {
    __shared__ float sums[8][32 * VEC + 1];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int col = (blockIdx.x * 32 + lane) * VEC;
    const long long row_begin = blockIdx.y * rows_per_slab, row_end = min(rows, row_begin + rows_per_slab);
    const int valid = cols - col;
    float acc[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) acc[j] = 0.f;
    if (valid > 0) {
#pragma unroll 2
        for (long long row = row_begin + warp; row < row_end; row += 8) {
            float g[VEC];
            load_row<T, VEC>(dy + row * ldy + col, g, valid);
            if (dz != nullptr) {
                if (act != kActNone) {
                    float z[VEC];
                    load_row<T, VEC>(pre + row * cols + col, z, valid);
#pragma unroll
                    for (int j = 0; j < VEC; ++j) g[j] *= linear_slope<LinearTail<T>::kFast>(z[j], act);
                }
                T* dst = dz + row * ldz + col;
                if (VEC * sizeof(T) == 16 && valid >= VEC) {
                    alignas(16) T tmp[VEC];
#pragma unroll
                    for (int j = 0; j < VEC; ++j) tmp[j] = Cvt<T>::from_f(g[j]);
                    *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(tmp);  // ldz is a whole number of vectors
                } else {
#pragma unroll
                    for (int j = 0; j < VEC; ++j)
                        if (j < valid) dst[j] = Cvt<T>::from_f(g[j]);
                }
            }
#pragma unroll
            for (int j = 0; j < VEC; ++j) acc[j] += g[j];
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

// dbias[c] = sum of the slabs' column sums, in slab order.
template <class T>
__global__ void __launch_bounds__(256)
linear_dbias_kernel(const float* partial, int slabs, int cols, T* __restrict__ dbias) {
    ptx::grid_dep_wait();  // the preceding kernel's partial sums
    const int c = blockIdx.x * 256 + threadIdx.x;
    if (c >= cols) return;
    float s = 0.f;
    for (int k = 0; k < slabs; ++k) s += partial[static_cast<long long>(k) * cols + c];
    dbias[c] = Cvt<T>::from_f(s);
}

}  // namespace lce
