// CUDA-core GEMM core with the same epilogue contract as the tcgen05 core.
//
//   D[m, n] = sum_k A[m, k] * B[n, k]     fp32 FMA, k ascending, no tensor cores
//
// It serves the inputs the tensor-core path cannot take: fp32 tensors (the reference demands
// 1e-5 agreement with fp32 torch there, so TF32 is not an option), hidden sizes that are not a
// multiple of 8 (TMA needs 16-byte row pitches) and unaligned bases. Operands are addressed through
// explicit (row, k) strides, so any majorness works.
//
// One CTA of 256 threads computes a 128 x 128 tile. Thread (ty, tx) of a 16 x 16 grid keeps an 8 x 8
// block of it in registers, as rows {ty*4.., 64 + ty*4..} x columns {tx*4.., 64 + tx*4..}: four
// conflict-free 16-byte shared-memory loads feed 64 FMAs. Tiles of 64 x 64 (TS = 64: 128 threads with 8 x 4
// blocks, rows {ty*4.., 32 + ty*4..}) serve products whose contraction must not be split although large
// tiles would leave SMs idle (fp32 777 x 1003 x 520: 46 us against 82). The operand tiles are double-buffered in
// shared memory and the next ones are fetched into registers while the current ones are multiplied
// (one barrier per step of 16 k, 32 with the small tiles). When the contraction is done the tile goes through
// shared memory in 64-column halves so that the epilogue sees it the way every epilogue expects: one thread = one
// row, 32 columns at a time (threads 0..TS-1).
#pragma once

#include "epilogues.cuh"

namespace lce {

constexpr int kSimtBN = 128;
constexpr int kSimtBK = 16;
template <int TS>
struct SimtTile {
    static constexpr int kThreads = 2 * TS;
    static constexpr int kDepth = TS == 128 ? kSimtBK : 32;  // k of a step: with few warps an SM the steps' latency counts
    static constexpr int kLoads = kDepth / 2;                // elements of each operand per thread and k step
    static constexpr int kVecs = kLoads / 4;                 // the same in 16-byte vectors, for the vector loaders
    static constexpr int kPitch = TS + 4;                    // operand tiles [k][mn] in floats: rows stay 16-byte aligned,
                                                             // the pad spreads a k-contiguous deposit over the banks
};
constexpr int kSimtCPitch = 64 + 4;   // one 64-column half of the C tile
static_assert(kBM == 128, "the thread layout below is written for 128 x 128 tiles");

template <class T>
struct SimtOperand {
    const T* ptr;
    long long stride_mn;  // elements between consecutive m (resp. n)
    long long stride_k;   // elements between consecutive k
    int extent_mn;        // valid m (resp. n)
    int extent_k;         // readable k: at or beyond it the operand counts as zero (a contraction may be longer, when the
                          // other operand has zeros there)
};

// How a thread fetches its share (kLoads elements) of a TS x kDepth operand tile:
//   kSimtGeneric  scalar loads with run-time strides and per-element bounds tests: any dtype,
//                 any alignment, any majorness (consecutive threads walk the contiguous direction);
//   kSimtVecK     fp32, k contiguous: 16-byte loads of 4 consecutive k of one row, each deposited as four
//                 scalar stores (the tile is [k][mn]);
//   kSimtVecMN    fp32, m/n contiguous: 16-byte copies of 4 consecutive m/n at one k, which land as they are.
// The vector modes need a 16-byte aligned base, strides and the vectorised extent in multiples of 4;
// the host picks them (launch_simt). Row validity is settled once per tile, and the pointer just advances.
enum SimtMode { kSimtGeneric = 0, kSimtVecK = 1, kSimtVecMN = 2 };

template <class T, int MODE, int TS>
struct SimtLoader;

template <class T, int TS>
struct SimtLoader<T, kSimtGeneric, TS> {
    static constexpr int kThreads = SimtTile<TS>::kThreads, kPitch = SimtTile<TS>::kPitch, kLoads = SimtTile<TS>::kLoads,
                         kDepth = SimtTile<TS>::kDepth;
    static constexpr bool kAsync = false;
    const T* p;
    long long step, k_adv;
    int mn_t, k_t, mn_step, k_step, mn_left, k_limit;
    __device__ __forceinline__ void init(const SimtOperand<T>& op, int mn0, int k_begin, int t) {
        if (op.stride_k == 1) { k_t = t % kDepth; mn_t = t / kDepth; mn_step = kThreads / kDepth; k_step = 0; }
        else { mn_t = t % TS; k_t = t / TS; mn_step = 0; k_step = kThreads / TS; }
        p = op.ptr + static_cast<long long>(mn0 + mn_t) * op.stride_mn + static_cast<long long>(k_begin + k_t) * op.stride_k;
        step = mn_step * op.stride_mn + k_step * op.stride_k;
        k_adv = kDepth * op.stride_k;
        k_limit = op.extent_k;
        mn_left = op.extent_mn - mn0 - mn_t;  // element i is in range iff i * mn_step < mn_left
    }
    __device__ __forceinline__ void fetch(int k0, int k_end, float (&r)[kLoads], float*) {
        k_end = min(k_end, k_limit);
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            r[i] = 0.f;
            if (i * mn_step < mn_left && k0 + k_t + i * k_step < k_end) r[i] = Cvt<T>::to_f(p[i * step]);
        }
        p += k_adv;
    }
    __device__ __forceinline__ void deposit(float* tile, const float (&r)[kLoads]) const {
#pragma unroll
        for (int i = 0; i < kLoads; ++i) tile[(k_t + i * k_step) * kPitch + mn_t + i * mn_step] = r[i];
    }
};

template <int TS>
struct SimtLoader<float, kSimtVecK, TS> {
    // thread t, vector i: row (t / (BK/4)) + i * (threads / (BK/4)), k offset 4 * (t % (BK/4))
    static constexpr int kPitch = SimtTile<TS>::kPitch, kLoads = SimtTile<TS>::kLoads, kVecs = SimtTile<TS>::kVecs,
                         kDepth = SimtTile<TS>::kDepth;
    static constexpr bool kAsync = false;
    static constexpr int kPerRow = kDepth / 4;
    static constexpr int kRowStep = SimtTile<TS>::kThreads / kPerRow;
    const float* p;
    long long row_adv;
    int row, k4;
    bool valid[kVecs];
    __device__ __forceinline__ void init(const SimtOperand<float>& op, int mn0, int k_begin, int t) {
        row = t / kPerRow;
        k4 = (t % kPerRow) * 4;
#pragma unroll
        for (int i = 0; i < kVecs; ++i) valid[i] = mn0 + row + i * kRowStep < op.extent_mn;
        p = op.ptr + static_cast<long long>(mn0 + row) * op.stride_mn + k_begin + k4;
        row_adv = static_cast<long long>(kRowStep) * op.stride_mn;
    }
    __device__ __forceinline__ void fetch(int k0, int k_end, float (&r)[kLoads], float*) {
#pragma unroll
        for (int i = 0; i < kVecs; ++i) {
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
            if (valid[i] && k0 + k4 < k_end) v = *reinterpret_cast<const float4*>(p + i * row_adv);  // K % 4 == 0: all four or none
            r[4 * i + 0] = v.x; r[4 * i + 1] = v.y; r[4 * i + 2] = v.z; r[4 * i + 3] = v.w;
        }
        p += kDepth;
    }
    __device__ __forceinline__ void deposit(float* tile, const float (&r)[kLoads]) const {
#pragma unroll
        for (int i = 0; i < kVecs; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) tile[(k4 + j) * kPitch + row + i * kRowStep] = r[4 * i + j];
    }
};

template <int TS>
struct SimtLoader<float, kSimtVecMN, TS> {
    // thread t, vector i: k (t / (TS/4)) + i * 8, m/n offset 4 * (t % (TS/4)). The tile in shared memory is [k][mn], so a
    // 16-byte vector of consecutive m/n lands as it is: the copy goes global -> shared with cp.async and needs
    // no registers between fetch and deposit (out-of-range vectors are zero-filled by a source size of 0).
    static constexpr bool kAsync = true;
    static constexpr int kPitch = SimtTile<TS>::kPitch, kLoads = SimtTile<TS>::kLoads, kVecs = SimtTile<TS>::kVecs,
                         kDepth = SimtTile<TS>::kDepth;
    static constexpr int kPerK = TS / 4, kStep = SimtTile<TS>::kThreads / kPerK;
    const float* p;
    long long k_adv, k_half;
    int k, mn4, k_limit;
    bool valid;
    __device__ __forceinline__ void init(const SimtOperand<float>& op, int mn0, int k_begin, int t) {
        k = t / kPerK;
        mn4 = (t % kPerK) * 4;
        k_limit = op.extent_k;
        valid = mn0 + mn4 < op.extent_mn;  // extent % 4 == 0: all four or none
        p = op.ptr + (mn0 + mn4) + static_cast<long long>(k_begin + k) * op.stride_k;
        k_adv = kDepth * op.stride_k;
        k_half = kStep * op.stride_k;
        if (!valid) p = op.ptr;  // never dereferenced (source size 0), but keep the address inside the tensor
    }
    __device__ __forceinline__ void fetch(int k0, int k_end, float (&)[kLoads], float* tile) {
        k_end = min(k_end, k_limit);
#pragma unroll
        for (int i = 0; i < kVecs; ++i) {
            const bool in = valid && k0 + k + i * kStep < k_end;
            const unsigned dst = static_cast<unsigned>(__cvta_generic_to_shared(tile + (k + i * kStep) * kPitch + mn4));
            const float* src = in ? p + i * k_half : p;
            asm volatile("cp.async.ca.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(in ? 16 : 0) : "memory");
        }
        if (valid) p += k_adv;
    }
    __device__ __forceinline__ void deposit(float*, const float (&)[kLoads]) const {}
};

// TS 64: m_tiles and n_tiles count 64 x 64 tiles, and the epilogue is told of the 128 x 128 tile they lie in.
template <class T, class Epi, int AMODE = kSimtGeneric, int BMODE = kSimtGeneric, int TS = 128>
__global__ void __launch_bounds__(SimtTile<TS>::kThreads, TS == 128 ? 2 : 4)
gemm_simt_kernel(SimtOperand<T> A, SimtOperand<T> B, int K, int m_tiles, int n_tiles, int k_splits,
                 const typename Epi::Params ep) {
    // main loop: two buffers of As[k][m] + Bs[k][n]; afterwards the same memory stages half a C tile
    static_assert(TS == 128 || TS == 64, "tile size");
    constexpr int kDepth = SimtTile<TS>::kDepth, kLoads = SimtTile<TS>::kLoads;
    constexpr int kPitch = SimtTile<TS>::kPitch, kTileFloats = kDepth * kPitch, kHalves = TS / 64;
    __shared__ __align__(16) float smem[4 * kTileFloats > TS * kSimtCPitch ? 4 * kTileFloats : TS * kSimtCPitch];

    const int t = threadIdx.x;
    const int ty = t >> 4, tx = t & 15;
    // k_splits > 1: work item = (tile, slice of the contraction); the epilogue stores slices side by side
    // (kStoreSlice) and splitk_reduce_kernel adds them in slice order.
    const int total_tiles = m_tiles * n_tiles;
    const int k_per_slice = ((K + k_splits - 1) / k_splits + kDepth - 1) / kDepth * kDepth;
    for (int work = blockIdx.x; work < total_tiles * k_splits; work += gridDim.x) {
        const int tile = work % total_tiles;
        const int k_slice = work / total_tiles;
        const int k_begin = k_slice * k_per_slice;
        const int k_end = min(K, k_begin + k_per_slice);
        const int n_tile = tile % n_tiles;
        const int m_tile = tile / n_tiles;
        const int m0 = m_tile * TS;
        const int n0 = n_tile * TS;

        float acc[8][4 * kHalves];
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int j = 0; j < 4 * kHalves; ++j) acc[i][j] = 0.f;

        SimtLoader<T, AMODE, TS> la;
        SimtLoader<T, BMODE, TS> lb;
        la.init(A, m0, k_begin, t);
        lb.init(B, n0, k_begin, t);
        constexpr bool kAnyAsync = SimtLoader<T, AMODE, TS>::kAsync || SimtLoader<T, BMODE, TS>::kAsync;
        float ra[kLoads], rb[kLoads];
        la.fetch(k_begin, k_end, ra, smem);
        lb.fetch(k_begin, k_end, rb, smem + kTileFloats);
        la.deposit(smem, ra);
        lb.deposit(smem + kTileFloats, rb);
        if constexpr (kAnyAsync) asm volatile("cp.async.wait_all;" ::: "memory");
        __syncthreads();
        int cur = 0;
        for (int k0 = k_begin; k0 < k_end; k0 += kDepth) {
            const bool more = k0 + kDepth < k_end;
            float* nxt = smem + (cur ^ 1) * 2 * kTileFloats;
            if (more) {  // in flight while this step multiplies (straight into the other buffer where the copy is async)
                la.fetch(k0 + kDepth, k_end, ra, nxt);
                lb.fetch(k0 + kDepth, k_end, rb, nxt + kTileFloats);
            }
            const float* As = smem + cur * 2 * kTileFloats;
            const float* Bs = As + kTileFloats;
#pragma unroll
            for (int k = 0; k < kDepth; ++k) {
                const float4 a0 = *reinterpret_cast<const float4*>(As + k * kPitch + ty * 4);
                const float4 a1 = *reinterpret_cast<const float4*>(As + k * kPitch + TS / 2 + ty * 4);
                const float a[8] = {a0.x, a0.y, a0.z, a0.w, a1.x, a1.y, a1.z, a1.w};
                float b[4 * kHalves];
#pragma unroll
                for (int h = 0; h < kHalves; ++h) {
                    const float4 v = *reinterpret_cast<const float4*>(Bs + k * kPitch + h * 64 + tx * 4);
                    b[4 * h] = v.x;
                    b[4 * h + 1] = v.y;
                    b[4 * h + 2] = v.z;
                    b[4 * h + 3] = v.w;
                }
#pragma unroll
                for (int i = 0; i < 8; ++i)
#pragma unroll
                    for (int j = 0; j < 4 * kHalves; ++j) acc[i][j] = fmaf(a[i], b[j], acc[i][j]);
            }
            if (more) {
                la.deposit(nxt, ra);
                lb.deposit(nxt + kTileFloats, rb);
                if constexpr (kAnyAsync) asm volatile("cp.async.wait_all;" ::: "memory");
            }
            __syncthreads();
            cur ^= 1;
        }

        // C tile through shared memory, one 64-column half at a time: blocked registers -> one row per thread
        constexpr int kPer = 128 / TS;  // of these tiles along each side of the epilogue's
        TileCtx tc{m_tile / kPer, n_tile / kPer, (n_tiles + kPer - 1) / kPer, m_tile % kPer * TS + t % TS, kSimtBN, k_slice, nullptr};
        const int col0 = n_tile % kPer * TS;
        typename Epi::State st;
        if (t < TS) Epi::begin(st, ep, tc);
#pragma unroll
        for (int half = 0; half < kHalves; ++half) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int row = (i < 4 ? 0 : TS / 2) + ty * 4 + (i & 3);
                *reinterpret_cast<float4*>(&smem[row * kSimtCPitch + tx * 4]) =
                    make_float4(acc[i][half * 4 + 0], acc[i][half * 4 + 1], acc[i][half * 4 + 2], acc[i][half * 4 + 3]);
            }
            __syncthreads();
            if (t < TS) {
#pragma unroll 1
                for (int c = 0; c < 2; ++c) {
                    float v[32];
#pragma unroll
                    for (int q = 0; q < 8; ++q) {
                        const float4 x = *reinterpret_cast<const float4*>(&smem[t * kSimtCPitch + c * 32 + q * 4]);
                        v[4 * q + 0] = x.x;
                        v[4 * q + 1] = x.y;
                        v[4 * q + 2] = x.z;
                        v[4 * q + 3] = x.w;
                    }
                    Epi::chunk(st, ep, tc, col0 + half * 64 + c * 32, v);
                }
            }
            __syncthreads();  // the staging area is free again (next half, or operand tiles of the next item)
        }
        if (t < TS) Epi::end(st, ep, tc);
    }
}

}  // namespace lce
