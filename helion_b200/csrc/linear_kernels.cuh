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

constexpr float kGeluC = 0.7978845608028654f;  // sqrt(2 / pi)
constexpr float kGeluA = 0.044715f;

// ---- activations ----------------------------------------------------------------------------------
// All three smooth ones are z times a distribution function F with F(-a) = 1 - F(a), so that with a = |z|
//   act(z)  = max(z, 0) - a F(-a)            nothing overflows, and small results of negative z keep their digits
//   act'(z) = [z >= 0] - sign(z) (F(-a) - a f(a))      f the density
// silu: F the logistic function of z; gelu_tanh: the logistic function of u(z) = 2 sqrt(2/pi) (z + 0.044715 z^3); gelu:
// the normal distribution. exp(-x) enters as the square of exp(-x / 2), so that a product with it keeps results that the
// exponential itself would flush to zero.
//
// For 16-bit results (FAST) the exponential and the reciprocal are the hardware's, 1e-6 relative, and two elements share
// an instruction where the hardware has it (fma and mul of fp32 pairs): at a contraction of 1024 a tile's epilogue
// has to be done in 8000 cycles of its four schedulers. The normal distribution is
//   F(-a) = exp(-a^2 / 2) g(a),  g a polynomial in 1 / (1 + 0.26 a)
// fitted here by reweighted least squares to 3.4e-7 of g for a up to 14 (with the exponential 2e-6 up to a = 6).
__device__ __forceinline__ float fast_reciprocal(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ Pair reciprocal2(Pair x) {
    float a, b;
    split(x, a, b);
    return pair(fast_reciprocal(a), fast_reciprocal(b));
}
__device__ __forceinline__ Pair exp2_2(Pair x) {
    float a, b;
    split(x, a, b);
    return pair(ptx::ex2(a), ptx::ex2(b));
}
// -|z|, an infinity as the largest finite value (whose weight is 0 all the same) and a NaN as it is.
__device__ __forceinline__ float minus_abs(float z) {
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(-fabsf(z)), "f"(-3.402823466e38f));
    return y;
}

// h = exp(-x / 2) and q with F(-a) = h h q, for a pair of -a.
template <int ACT>
__device__ __forceinline__ void distribution2(Pair na, Pair& h, Pair& q) {
    if constexpr (ACT == kActGelu) {
        const Pair t = reciprocal2(fma2(na, both(-0.26f), both(1.f)));
        h = exp2_2((na * both(-0.36067376f)) * na);
        Pair p = fma2(both(-0.07724009f), t, both(0.24633712f));
        p = fma2(p, t, both(-0.135466f));
        p = fma2(p, t, both(0.19220619f));
        p = fma2(p, t, both(0.06021739f));
        p = fma2(p, t, both(0.11097057f));
        p = fma2(p, t, both(0.10293892f));
        q = fma2(p, t, both(3.572605e-05f));
    } else {
        Pair x = na;  // -x
        if constexpr (ACT == kActGeluTanh) x = na * fma2(na * both(2.f * kGeluC * kGeluA), na, both(2.f * kGeluC));
        h = exp2_2(x * both(0.5f * kLog2e));
        q = reciprocal2(fma2(h, h, both(1.f)));
    }
}
// The same for one value of a logistic one in full 32-bit accuracy.
template <int ACT>
__device__ __forceinline__ void distribution(float a, float& h, float& q) {
    static_assert(ACT == kActGeluTanh || ACT == kActSilu, "gelu goes by normcdff");
    const float x = ACT == kActGeluTanh ? 2.f * kGeluC * a * fmaf(kGeluA * a, a, 1.f) : a;
    h = expf(-0.5f * x);
    q = 1.f / fmaf(h, h, 1.f);
}

// act(z) of N values.
template <bool FAST, int ACT, int N>
__device__ __forceinline__ void linear_act(float (&z)[N]) {
    if constexpr (ACT == kActRelu) {
#pragma unroll
        for (int j = 0; j < N; ++j) z[j] = z[j] <= 0.f ? 0.f : z[j];  // a NaN stays one
    } else if constexpr (ACT != kActNone && FAST) {
        static_assert(N % 2 == 0, "pairs");
#pragma unroll
        for (int j = 0; j < N; j += 2) {
            const Pair na = pair(minus_abs(z[j]), minus_abs(z[j + 1]));
            Pair h, q;
            distribution2<ACT>(na, h, q);
            split(fma2(na * h, h * q, pair(fmaxf(z[j], 0.f), fmaxf(z[j + 1], 0.f))), z[j], z[j + 1]);
        }
    } else if constexpr (ACT == kActGelu) {
#pragma unroll
        for (int j = 0; j < N; ++j) z[j] = z[j] * normcdff(z[j]);
    } else if constexpr (ACT != kActNone) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            float h, q;
            distribution<ACT>(fabsf(z[j]), h, q);
            z[j] = (z[j] >= 0.f ? z[j] : z[j] * h * h) * q;
        }
    }
}
template <bool FAST, int N>
__device__ __forceinline__ void linear_act(float (&z)[N], int act) {
    switch (act) {
        case kActRelu: linear_act<FAST, kActRelu>(z); break;
        case kActGelu: linear_act<FAST, kActGelu>(z); break;
        case kActGeluTanh: linear_act<FAST, kActGeluTanh>(z); break;
        case kActSilu: linear_act<FAST, kActSilu>(z); break;
        default: break;
    }
}

// What the forward saves for act': z, or for relu the derivative itself.
template <int N>
__device__ __forceinline__ void linear_saved(const float (&z)[N], int act, float (&saved)[N]) {
#pragma unroll
    for (int j = 0; j < N; ++j) saved[j] = act == kActRelu ? (z[j] > 0.f ? 1.f : 0.f) : z[j];
}

// g *= act'(.) from what the forward saved. a f(a) is 0.3989 a h h for the normal distribution and x' F(-a) F(a) for the
// logistic ones (x' = a for silu; for gelu_tanh a du/da, which may overflow against a zero far out).
template <bool FAST, int ACT, int N>
__device__ __forceinline__ void linear_slope(float (&g)[N], const float (&pre)[N]) {
    if constexpr (ACT == kActRelu) {
#pragma unroll
        for (int j = 0; j < N; ++j) g[j] *= pre[j];
    } else if constexpr (ACT == kActGelu && FAST) {
#pragma unroll
        for (int j = 0; j < N; j += 2) {
            const Pair na = pair(minus_abs(pre[j]), minus_abs(pre[j + 1]));
            Pair h, q;
            distribution2<ACT>(na, h, q);
            float d[2];  // F(-a) - a f(a)
            split((h * h) * fma2(na, both(0.3989422804014327f), q), d[0], d[1]);
#pragma unroll
            for (int i = 0; i < 2; ++i) g[j + i] *= pre[j + i] >= 0.f ? 1.f - d[i] : d[i];
        }
    } else if constexpr (ACT == kActGelu) {
#pragma unroll
        for (int j = 0; j < N; ++j) g[j] *= fmaf(pre[j] * 0.3989422804014327f, expf(-0.5f * pre[j] * pre[j]), normcdff(pre[j]));
    } else if constexpr (ACT != kActNone) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const float a = fabsf(pre[j]);
            float h, q;
            if constexpr (FAST) {
                const float x = ACT == kActGeluTanh ? 2.f * kGeluC * a * fmaf(kGeluA * a, a, 1.f) : a;
                h = ptx::ex2(-0.5f * kLog2e * x);
                q = fast_reciprocal(fmaf(h, h, 1.f));
            } else {
                distribution<ACT>(a, h, q);
            }
            const float low = h * h * q;  // F(-a); F(a) = q
            const float x1 = ACT == kActGeluTanh ? 2.f * kGeluC * a * fmaf(3.f * kGeluA * a, a, 1.f) : a;
            const float d = low == 0.f ? 0.f : fmaf(-x1 * q, low, low);
            g[j] *= pre[j] >= 0.f ? 1.f - d : d;
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

// ACT: the activation, or kActAny to go by the call's (CUDA-core GEMM, split contractions). HEAVY: for calls with a
// bias, an activation or a residual.
constexpr int kActAny = -1;
template <class T, int ACT, bool HEAVY>
struct EpiLinear;
// A heavy epilogue runs on eight warps beside CTA pairs: with four, 8192 x 1024 x 4096 with gelu took 129 us where eight
// take 101 (the product alone 60); without any of it four warps and a sixth stage are faster (60 against 66 us).
template <class T, int ACT>
struct EpiWarps<EpiLinear<T, ACT, true>, 2> {
    static constexpr int value = 8;
};

template <class T, int ACT, bool HEAVY>
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
        uint4 next[sizeof(T) == 2 && HEAVY ? 8 : 1];
        uint4 saved[sizeof(T) == 2 && HEAVY ? 4 : 1];
    };
    template <int N>
    static __device__ __forceinline__ void activate(float (&v)[N], int act) {
        if constexpr (ACT == kActAny) linear_act<LinearTail<T>::kFast>(v, act);
        else linear_act<LinearTail<T>::kFast, ACT>(v);
    }
    static __device__ __forceinline__ void begin(State& st, const Params& p, const TileCtx& tc) {
        st.row = tc.m_tile * kBM + tc.row_in_tile;
        if constexpr (sizeof(T) == 2) {
            if (p.scratch != nullptr || tc.stage == nullptr) return;
            const LinearTail<T>& t = p.t;
            const int lane = tc.row_in_tile & 31, col0 = tc.n_tile * tc.bn + tc.col_begin, row_base = st.row - lane;
            if (t.bias != nullptr) {  // this warp's slice of the bias, as floats, behind the re-shaping area
                float* bias = tc.stage + kStageBiasOffset;
                __syncwarp();  // the previous tile's has been read
                for (int c = lane * 8; c < tc.col_end - tc.col_begin; c += 256) {
                    float b[8];
                    load_row<T>(t.bias + col0 + c, b, t.cols - col0 - c);
                    *reinterpret_cast<float4*>(bias + c) = make_float4(b[0], b[1], b[2], b[3]);
                    *reinterpret_cast<float4*>(bias + c + 4) = make_float4(b[4], b[5], b[6], b[7]);
                }
                __syncwarp();
            }
            if constexpr (HEAVY)
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
        activate(v, t.act);
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
            const float4* b = reinterpret_cast<const float4*>(tc.stage + kStageBiasOffset + col0 - tc.col_begin);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float4 x = b[i];
                v[4 * i] += x.x;
                v[4 * i + 1] += x.y;
                v[4 * i + 2] += x.z;
                v[4 * i + 3] += x.w;
            }
        }
        uint4 y[4];
        if constexpr (!HEAVY) {
            pack32<T>(v, y);
            area_put(tc.stage, lane, half, y);
            if (half == 0) return;
        } else {
            uint4 keep[4];
            if (t.pre != nullptr) {
                float saved[32];
                linear_saved(v, t.act, saved);
                pack32<T>(saved, keep);
            }
            activate(v, t.act);
            if (t.residual != nullptr) {
                if (half == 0) {
                    const T* src = t.residual + static_cast<long long>(row_base) * t.ldr + blk0;
                    if (p.wide_residual) {
                        lines_put(tc.stage, lane, st.next);
                        if (col0 + 64 < tc.col_end) lines_fetch<T>(lane, src + 64, t.ldr, rows, cols - 64, st.next);
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
            pack32<T>(v, y);
            area_put(tc.stage, lane, half, y);
            if (half == 0) {
                if (t.pre != nullptr) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) st.saved[i] = keep[i];
                }
                return;
            }
            if (t.pre != nullptr) {
                __syncwarp();
                area_to_lines<T>(tc.stage, lane, t.out + static_cast<long long>(row_base) * t.ldo + blk0, t.ldo, rows, cols, p.wide_out != 0);
                __syncwarp();
                area_put(tc.stage, lane, 0, st.saved);
                area_put(tc.stage, lane, 1, keep);
                __syncwarp();
                area_to_lines<T>(tc.stage, lane, t.pre + static_cast<long long>(row_base) * t.ldp + blk0, t.ldp, rows, cols, true);
                __syncwarp();
                return;
            }
        }
        __syncwarp();
        area_to_lines<T>(tc.stage, lane, t.out + static_cast<long long>(row_base) * t.ldo + blk0, t.ldo, rows, cols, p.wide_out != 0);
        __syncwarp();
    }
    static __device__ __forceinline__ void end(State&, const Params&, const TileCtx&) {}
};

// Adds the slices of a split contraction in slice order and finishes the values. One thread = four columns of a row; 64
// threads take 16 rows (which lie side by side in a slab) of 4 such quads (side by side in the output).
template <class T>
__global__ void __launch_bounds__(256)
linear_reduce_kernel(const float* scratch, int slices, long long slab_floats, int n_tiles, int bn, const LinearTail<T> t) {
    ptx::grid_dep_launch();
    ptx::grid_dep_wait();  // `scratch` holds the slices of the preceding GEMM
    const long long groups_per_row = (static_cast<long long>(t.cols) + 15) / 16;
    const long long total = groups_per_row * ((t.rows + 15ll) / 16) * 64;
    for (long long i = blockIdx.x * static_cast<long long>(blockDim.x) + threadIdx.x; i < total;
         i += static_cast<long long>(gridDim.x) * blockDim.x) {
        const long long group = i / 64, row_group = group / groups_per_row;
        const int in_group = static_cast<int>(i & 63);
        const int row = static_cast<int>(row_group) * 16 + (in_group & 15);
        const int col = static_cast<int>(group - row_group * groups_per_row) * 16 + (in_group >> 4) * 4;
        if (row >= t.rows || col >= t.cols) continue;
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

// ---------------------------------------------------------------------------------------------
// A handful of tokens (at most 64): the product is bound by reading W once, so W is the operand with 128 rows and the
// tokens are the narrow one:
//   D[n, m] = sum_k W[n, k] x[m, k],  128 x BN tiles, BN = 16, 32 or 64 (tokens beyond M read as zeros)
// With x as the 128-row operand (the core above) a launch moves the same bytes but needs its partial sums in global
// memory and a second launch to add them. Here the contraction is split over the CTAs of a cluster: each streams its
// share of 128 rows of W through a TMA ring, multiplies (tcgen05, one accumulator of BN columns), leaves its partial
// tile in shared memory, and after one cluster barrier every CTA adds BN / S columns of it over the cluster in rank order
// and runs the epilogue on them. A ring of about 100 KB lets two CTAs share an SM, so a whole wave of W is in flight.
// Warp roles: 0 TMA producer, 1 MMA issuer and tensor-memory owner, 2-5 read the accumulator (warp w lanes 32*(w%4)..).
// announce_extra: the test hook of ptx.cuh, as an argument: reading the variable delayed the first copy by 0.5 us.
// ---------------------------------------------------------------------------------------------
template <int BN>
struct DecodeSmem {
    static constexpr int kABytes = kBM * kBK * 2;
    static constexpr int kStageBytes = kABytes + BN * kBK * 2;
    static constexpr int kStages = BN == 16 ? 6 : (BN == 32 ? 5 : 4);
    static constexpr int kTotalBytes = kStages * kStageBytes + 128 + 1024;  // barriers; slack to align the ring by hand
    static_assert(BN * kBM * 4 <= kStages * kStageBytes, "the partial tile takes the ring's place");
};

__device__ __forceinline__ float ld_cluster_f32(uint32_t addr) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
    return v;
}

template <class T, int BN>
__global__ void __launch_bounds__(kGemmThreads, 2)
linear_decode_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_x, int k_blocks, int splits,
                     const LinearTail<T> t, int* __restrict__ status, unsigned announce_extra) {
    using S = DecodeSmem<BN>;
    constexpr int kStages = S::kStages;
    constexpr uint32_t kTmemCols = BN < 32 ? 32 : BN;
    constexpr uint32_t kIdesc = ptx::make_idesc_f16(kBM, BN, std::is_same<T, __nv_bfloat16>::value, false, false);
    extern __shared__ uint8_t smem_raw[];
    const uint32_t base = (ptx::smem_u32(smem_raw) + 1023u) & ~1023u;
    const uint32_t bars = base + kStages * S::kStageBytes;  // full[kStages] | empty[kStages] | done | tmem ptr | abort
    uint8_t* gen = smem_raw + (base - ptx::smem_u32(smem_raw));
    uint8_t* gen_bars = gen + kStages * S::kStageBytes;
    auto full = [&](int s) { return bars + 8u * s; };
    auto empty = [&](int s) { return bars + 8u * (kStages + s); };
    const uint32_t done = bars + 8u * (2 * kStages);
    volatile uint32_t* tmem_ptr = reinterpret_cast<volatile uint32_t*>(gen_bars + 8 * (2 * kStages + 1));
    volatile int* abort_flag = reinterpret_cast<volatile int*>(gen_bars + 8 * (2 * kStages + 1) + 4);
    static_assert(8 * (2 * kStages + 2) <= 128, "barrier block");

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = splits > 1 ? static_cast<int>(ptx::cluster_ctarank()) : 0;
    const int tile = static_cast<int>(blockIdx.x) / splits;
    const int kb0 = static_cast<int>(static_cast<long long>(k_blocks) * rank / splits);
    const int kb1 = static_cast<int>(static_cast<long long>(k_blocks) * (rank + 1) / splits);  // splits <= k_blocks: never empty

    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            ptx::mbar_init(full(s), 1);
            ptx::mbar_init(empty(s), 1);
        }
        ptx::mbar_init(done, 1);
        *abort_flag = 0;
        ptx::fence_mbar_init();
        ptx::prefetch_tensormap(&tm_w);
        ptx::prefetch_tensormap(&tm_x);
    }
    if (warp == 1) {
        ptx::tmem_alloc(ptx::smem_u32(const_cast<uint32_t*>(tmem_ptr)), kTmemCols);
        ptx::tmem_relinquish();
    }
    ptx::tc_fence_before_sync();
    __syncthreads();
    ptx::tc_fence_after_sync();
    const uint32_t tmem = *tmem_ptr;
    ptx::grid_dep_launch();
    ptx::grid_dep_wait();  // nothing above touched global memory

    int issued = 0;  // by the producer's lane
    if (warp == 0) {
        if (ptx::elect_one()) {
            const uint64_t keep = ptx::make_l2_policy(ptx::kL2EvictLast), stream = ptx::make_l2_policy(ptx::kL2EvictFirst);
            for (int kb = kb0; kb < kb1; ++kb, ++issued) {
                const int s = issued % kStages;
                if (!ptx::mbar_wait(empty(s), ((issued / kStages) & 1u) ^ 1u, abort_flag)) {
                    atomicCAS(status, 0, kDevErrProducerTimeout);
                    break;
                }
                const uint32_t sa = base + s * S::kStageBytes;
                ptx::mbar_arrive_expect_tx(full(s), S::kStageBytes + (issued == 0 ? announce_extra : 0u));
                ptx::tma_load_2d_hint(sa, &tm_w, full(s), kb * kBK, tile * kBM, stream);   // W: read once
                ptx::tma_load_2d_hint(sa + S::kABytes, &tm_x, full(s), kb * kBK, 0, keep);  // x: every CTA reads it
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        if (ptx::elect_one()) {
            bool ok = true;
            int used = 0;
            for (int kb = kb0; kb < kb1; ++kb, ++used) {
                const int s = used % kStages;
                if (!ptx::mbar_wait(full(s), (used / kStages) & 1u, abort_flag)) {
                    atomicCAS(status, 0, kDevErrMmaTimeout);
                    ok = false;
                    break;
                }
                ptx::tc_fence_after_sync();
                const uint32_t sa = base + s * S::kStageBytes, sb = sa + S::kABytes;
#pragma unroll
                for (int k = 0; k < kBK / kUmmaK; ++k)
                    ptx::umma_f16(tmem, ptx::make_smem_desc(sa + k * (kUmmaK * 2), 0, 1024),
                                  ptx::make_smem_desc(sb + k * (kUmmaK * 2), 0, 1024), kIdesc, (kb != kb0 || k != 0) ? 1u : 0u);
                ptx::umma_commit(empty(s));
            }
            ptx::umma_commit(done);  // also on the way out of a timeout: what was issued drains before the memory is freed
            if (!ok)
                for (int spin = 0; spin < (1 << 16); ++spin)
                    if (ptx::mbar_try_wait(done, 0)) break;
        }
        __syncwarp();
    }
    // The accumulator: thread = one of 128 features, a column a token.
    float acc[BN < 32 ? 32 : BN];
    const int feature = (warp & 3) * 32 + lane;
    if (warp >= 2) {
        if (!ptx::mbar_wait(done, 0, abort_flag) && lane == 0) atomicCAS(status, 0, kDevErrEpilogueTimeout);
        __syncwarp();
        ptx::tc_fence_after_sync();
        const uint32_t taddr = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
#pragma unroll
        for (int c = 0; c < static_cast<int>(kTmemCols); c += 32) ptx::tmem_ld_32x32(taddr + c, *reinterpret_cast<float(*)[32]>(acc + c));
        ptx::tmem_ld_wait();
        ptx::tc_fence_before_sync();
    }
    __syncthreads();  // every wait on the ring has ended, so the flag holds still
    if (*abort_flag) {
        // a wait ran out: the copies in flight land (or are given the time to) before their space is used and the CTA retires
        const int back = issued < kStages ? issued : kStages;
        for (int j = 1; j <= back; ++j)
            for (int spin = 0; spin < (1 << 16); ++spin)
                if (ptx::mbar_try_wait(full((issued - j) % kStages), ((issued - j) / kStages) & 1u)) break;
        __syncthreads();
    }
    const int n = tile * kBM + feature;
    // G tokens of feature n from token m0 on (those below m1): everything is read before anything is written.
    const float bias = warp >= 2 && n < t.cols && t.bias != nullptr ? Cvt<T>::to_f(t.bias[n]) : 0.f;
    constexpr int G = BN / 8;  // a cluster of 8 leaves this many to each
    auto finish = [&](float* z, int m0, int m1) {
        float r[G];
#pragma unroll
        for (int i = 0; i < G; ++i) {
            r[i] = t.residual != nullptr && m0 + i < m1 ? Cvt<T>::to_f(t.residual[(m0 + i) * t.ldr + n]) : 0.f;
            z[i] += bias;
        }
        float (&v)[G] = *reinterpret_cast<float(*)[G]>(z);
        if (t.pre != nullptr) {
            float saved[G];
            linear_saved(v, t.act, saved);
#pragma unroll
            for (int i = 0; i < G; ++i)
                if (m0 + i < m1) t.pre[(m0 + i) * t.ldp + n] = Cvt<T>::from_f(saved[i]);
        }
        linear_act<true>(v, t.act);
#pragma unroll
        for (int i = 0; i < G; ++i)
            if (m0 + i < m1) t.out[(m0 + i) * t.ldo + n] = Cvt<T>::from_f(v[i] + r[i]);
    };
    if (splits == 1) {
        if (warp >= 2 && n < t.cols) {
#pragma unroll
            for (int m = 0; m < BN; m += G)
                if (m < t.rows) finish(acc + m, m, t.rows);
        }
        __syncthreads();
    } else {
        float* part = reinterpret_cast<float*>(gen);  // [token][feature]: all products that read the ring have finished
        if (warp >= 2) {
#pragma unroll
            for (int m = 0; m < BN; ++m) part[m * kBM + feature] = acc[m];
        }
        __syncthreads();
        ptx::cluster_sync_all();
        if (warp >= 2 && n < t.cols) {
            const int per = BN / splits;
            const int m1 = min((rank + 1) * per, t.rows);
            for (int m0 = rank * per; m0 < m1; m0 += G) {
                const uint32_t at = base + static_cast<uint32_t>(m0 * kBM + feature) * 4u;
                float z[G];
#pragma unroll
                for (int i = 0; i < G; ++i) z[i] = m0 + i < m1 ? ld_cluster_f32(ptx::map_to_cta(at + i * kBM * 4, 0)) : 0.f;
                for (int s = 1; s < splits; ++s) {  // in rank order
#pragma unroll
                    for (int i = 0; i < G; ++i) z[i] += m0 + i < m1 ? ld_cluster_f32(ptx::map_to_cta(at + i * kBM * 4, s)) : 0.f;
                }
                finish(z, m0, m1);
            }
        }
        __syncthreads();
        ptx::cluster_sync_all();  // no CTA leaves while another may still read its part
    }
    if (warp == 1) {
        ptx::tc_fence_after_sync();
        ptx::tmem_dealloc(tmem, kTmemCols);
    }
}

// Rows copied to a pitch of whole 16-byte vectors, zeros behind the last column: operands whose rows start off 16-byte
// boundaries, which TMA cannot read and the CUDA-core GEMM only element by element.
template <class T>
__global__ void __launch_bounds__(256)
repitch_kernel(const T* __restrict__ src, long long lds, T* __restrict__ dst, long long ldd, long long rows, int cols) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (long long r = blockIdx.x * 8ll + warp; r < rows; r += gridDim.x * 8ll)
        for (int c = lane; c < ldd; c += 32) dst[r * ldd + c] = c < cols ? src[r * lds + c] : Cvt<T>::from_f(0.f);
}

// dz = dy * act'(pre), rounded, and the column sums of the unrounded dz over this CTA's rows.
// A CTA of 256 threads owns 32 x VEC columns and the row slab [slab * rows_per_slab, ...): 32 column groups x 8 rows
// at a time, two of them in flight. Bytes: dy and pre in, dz out; 8192 x 4096 bf16, 201 MB, with the bias gradient and on a
// cold cache: 47 us with gelu, 40 with relu (0.77 of the copy bandwidth). Three CTAs an SM with four rows in flight took 52
// and 45, two with four 48 and 42, two with eight (which spill) 69 and 54, five with two (likewise) 56 and 50. partial: [slabs][cols] (nullptr: no sums);
// dz nullptr: sums only (no activation, dz = dy). Columns of dz up to its pitch, behind the last, are set to zero.
template <class T, int ACT>
__global__ void __launch_bounds__(256, 4)
linear_dz_kernel(const T* __restrict__ dy, long long ldy, const T* __restrict__ pre, long long ldp, T* __restrict__ dz, long long ldz,
                 float* __restrict__ partial, long long rows, int cols, long long rows_per_slab) {
    constexpr int U = 2, VEC = 16 / sizeof(T);
    __shared__ float sums[8][32 * VEC + 1];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int col = (blockIdx.x * 32 + lane) * VEC;
    const long long row_begin = blockIdx.y * rows_per_slab, row_end = min(rows, row_begin + rows_per_slab);
    const int valid = cols - col;
    const bool whole = valid >= VEC && ldy % VEC == 0 && (reinterpret_cast<uintptr_t>(dy) & 15u) == 0;
    float acc[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) acc[j] = 0.f;
    if (valid > 0) {
        for (long long row0 = row_begin + warp; row0 < row_end; row0 += 8 * U) {
            uint4 rg[U], rz[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const long long row = row0 + 8 * u;
                rg[u] = rz[u] = make_uint4(0u, 0u, 0u, 0u);
                if (row >= row_end) continue;
                if (whole) {
                    rg[u] = *reinterpret_cast<const uint4*>(dy + row * ldy + col);
                } else {
                    alignas(16) T e[VEC];
#pragma unroll
                    for (int j = 0; j < VEC; ++j) e[j] = j < valid ? dy[row * ldy + col + j] : Cvt<T>::from_f(0.f);
                    rg[u] = *reinterpret_cast<const uint4*>(e);
                }
                if (ACT != kActNone) rz[u] = *reinterpret_cast<const uint4*>(pre + row * ldp + col);  // whole rows by its pitch
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const long long row = row0 + 8 * u;
                if (row >= row_end) continue;
                float g[VEC], z[VEC];
                rms_unpack<T>(rg[u], g);
                rms_unpack<T>(rz[u], z);
                linear_slope<LinearTail<T>::kFast, ACT>(g, z);
                if (valid < VEC) {  // what the saved rows hold behind their last column is anything
#pragma unroll
                    for (int j = 0; j < VEC; ++j) g[j] = j < valid ? g[j] : 0.f;
                }
                if (dz != nullptr) *reinterpret_cast<uint4*>(dz + row * ldz + col) = rms_pack<T>(g);
#pragma unroll
                for (int j = 0; j < VEC; ++j) acc[j] += g[j];
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
