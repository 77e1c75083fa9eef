// Host side of the two GEMM cores (gemm_tc.cuh, gemm_simt.cuh): tensor maps, tile order, split of the contraction and
// the launches. Shared by the files that hold entry points built on a matrix product.
#pragma once

#include <cudaTypedefs.h>

#include <cstdio>
#include <type_traits>

#include "api_common.cuh"
#include "gemm_simt.cuh"
#include "gemm_tc.cuh"

namespace lce {

constexpr int kBN = 256;
constexpr int kStages1 = 4;  // 48 KB stages, one CTA per tile
constexpr int kStages2 = 6;  // 32 KB stages, CTA pair per tile

inline PFN_cuTensorMapEncodeTiled_v12000 g_encode = nullptr;

// The current device with everything that the GEMM cores need (status word, completion counters, tensor-map encoder).
int device_info(DeviceInfo** out);

// Sets the wait limit and the announcement hook (ptx.cuh) of the including source file, whose own they are.
static int set_debug_waits(unsigned long long limit_ns, unsigned announce_extra_bytes) {
    if (cuda_failed(cudaMemcpyToSymbol(ptx::g_wait_limit_ns, &limit_ns, sizeof(limit_ns))) ||
        cuda_failed(cudaMemcpyToSymbol(ptx::g_debug_announce_extra, &announce_extra_bytes, sizeof(announce_extra_bytes))))
        return LCE_ERR_CUDA;
    return LCE_OK;
}
int linear_debug_waits(unsigned long long limit_ns, unsigned announce_extra_bytes);  // linear_api.cu's

// 2-D tensor map over a row-major 16-bit matrix: `inner` contiguous elements per row, `outer`
// rows, `pitch_bytes` between rows; 128-byte swizzle; out-of-range elements read as zero.
// Encoding is host-only work (no driver state is touched), but it costs about a microsecond per map and
// a training step issues the same handful of maps over and over, so finished maps are kept in a small
// per-thread, direct-mapped cache keyed by everything the encoding depends on.
struct TmapKey {
    const void* base;
    long long inner, outer, pitch_bytes;
    unsigned box_inner, box_outer;
    int dtype;
    bool operator==(const TmapKey& o) const {
        return base == o.base && inner == o.inner && outer == o.outer && pitch_bytes == o.pitch_bytes &&
               box_inner == o.box_inner && box_outer == o.box_outer && dtype == o.dtype;
    }
};
struct TmapSlot {
    TmapKey key;
    bool valid = false;
    CUtensorMap map;
};
constexpr int kTmapCacheSlots = 64;

inline int make_tmap(CUtensorMap* tm, const void* base, int dtype, long long inner, long long outer,
              long long pitch_bytes, unsigned box_inner, unsigned box_outer) {
    if ((reinterpret_cast<uintptr_t>(base) & 15u) != 0 || (pitch_bytes & 15) != 0) return LCE_ERR_ALIGN;
    static thread_local TmapSlot cache[kTmapCacheSlots];
    const TmapKey key{base, inner, outer, pitch_bytes, box_inner, box_outer, dtype};
    unsigned long long h = reinterpret_cast<uintptr_t>(base) >> 4;
    h = h * 0x9E3779B97F4A7C15ull ^ static_cast<unsigned long long>(inner) * 0xC2B2AE3D27D4EB4Full ^
        static_cast<unsigned long long>(outer) * 0x165667B19E3779F9ull ^ (static_cast<unsigned long long>(box_outer) << 7) ^
        static_cast<unsigned long long>(pitch_bytes);
    TmapSlot& slot = cache[(h ^ (h >> 29)) % kTmapCacheSlots];
    if (slot.valid && slot.key == key) {
        *tm = slot.map;
        return LCE_OK;
    }
    // The encoder is a DRIVER entry point and wants a context current on the calling thread. A thread that has
    // made no runtime call yet (an autograd worker whose first CUDA call is this one) has none bound, and the
    // encoder then fails with CUDA_ERROR_INVALID_CONTEXT. cudaSetDevice on the thread's current device binds
    // the primary context (and, unlike cudaFree(0), is no stream operation, so it is legal under stream capture).
    {
        static thread_local int bound_device = -1;
        int dev = 0;
        if (cudaGetDevice(&dev) == cudaSuccess && dev != bound_device && cudaSetDevice(dev) == cudaSuccess) bound_device = dev;
    }
    cuuint64_t dims[2] = {static_cast<cuuint64_t>(inner), static_cast<cuuint64_t>(outer)};
    cuuint64_t strides[1] = {static_cast<cuuint64_t>(pitch_bytes)};
    cuuint32_t box[2] = {box_inner, box_outer};
    cuuint32_t estr[2] = {1, 1};
    const CUtensorMapDataType dt =
        dtype == LCE_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    const CUresult r = g_encode(tm, dt, 2, const_cast<void*>(base), dims, strides, box, estr,
                                CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) {
        t_last_cuda_error = static_cast<cudaError_t>(r);  // driver and runtime share the numbering of the common codes
        if (getenv("HELION_B200_DEBUG"))
            fprintf(stderr, "helion_b200: cuTensorMapEncodeTiled failed (%d): base %p inner %lld outer %lld pitch %lld box %u x %u\n",
                    static_cast<int>(r), base, inner, outer, pitch_bytes, box_inner, box_outer);
        return LCE_ERR_CUDA;
    }
    slot.key = key;
    slot.map = *tm;
    slot.valid = true;
    return LCE_OK;
}

// One operand of a GEMM as the host sees it: a row-major matrix [rows, cols] with a pitch.
// As a K-major operand its rows are the m (n) index; as an MN-major operand its rows are k. Columns beyond the
// problem's are readable and hold zeros (only the CUDA-core GEMM looks at them).
struct Mat {
    const void* ptr;
    long long rows, cols, pitch_elems;
};

// Tuning knobs of the tcgen05 launches (environment at load time, lce_set_tuning at run time):
//   band_mb     size of the operand band the tile order keeps resident in L2 (HELION_B200_BAND_MB)
//   hint_mode   L2 eviction hints: 0 none, 1 resident operand evict_last + streaming evict_first,
//               2 evict_last only (HELION_B200_L2_HINTS)
//   dyn_waves   launches of at least this many waves of tiles deal their tiles dynamically, when the caller's
//               workspace has room for the counter; 0 = never (HELION_B200_DYN_WAVES). 32: the long forward
//               launches, where the static deal drifts apart; the backward's launches are capped at about 28
//               waves by the block size and measured 1 % faster on the static deal
struct Tuning {
    std::atomic<int> band_mb, hint_mode, dyn_waves;
    Tuning() {
        const char* e = getenv("HELION_B200_BAND_MB");
        band_mb = (e && atoi(e) > 0) ? atoi(e) : 32;
        e = getenv("HELION_B200_L2_HINTS");
        hint_mode = e ? atoi(e) : 2;
        e = getenv("HELION_B200_DYN_WAVES");
        dyn_waves = e ? atoi(e) : 32;
    }
};
inline Tuning g_tuning;

template <int CG, bool A_MN, bool B_MN, bool IS_BF16, class Epi>
int launch_tc_cg(const DeviceInfo& d, const Mat& a, const Mat& b, long long M, long long Nn, long long K,
                 int m_fastest, int k_splits, const typename Epi::Params& ep, cudaStream_t stream, int* sched,
                 unsigned* done) {
    // Band the tile order so that the panels which co-running CTAs do NOT share stay resident in L2:
    // about 32 MB of them (the two L2 partitions of 63 MB each also hold the streaming operand).
    const long long kBandBytes = static_cast<long long>(g_tuning.band_mb.load(std::memory_order_relaxed)) << 20;
    const int kHintMode = g_tuning.hint_mode.load(std::memory_order_relaxed);
    constexpr int kEpiWarps = EpiWarps<Epi, CG>::value;
    constexpr int kStages = kEpiWarps == 8 ? kStages2 - 1 : (CG == 2 ? kStages2 : kStages1);  // the warps' areas take a stage
    static_assert(kEpiWarps == 4 || CG == 2, "eight epilogue warps beside CTA pairs only");
    const int dtype = IS_BF16 ? LCE_DTYPE_BF16 : LCE_DTYPE_F16;
    CUtensorMap tma, tmb;
    int rc;
    if (A_MN) rc = make_tmap(&tma, a.ptr, dtype, M, K, a.pitch_elems * 2, 64, kBK);
    else rc = make_tmap(&tma, a.ptr, dtype, K, M, a.pitch_elems * 2, kBK, kBM);
    if (rc) return rc;
    // each CTA of a pair stages half of the B tile
    if (B_MN) rc = make_tmap(&tmb, b.ptr, dtype, Nn, K, b.pitch_elems * 2, 64, kBK);
    else rc = make_tmap(&tmb, b.ptr, dtype, K, Nn, b.pitch_elems * 2, kBK, kBN / CG);
    if (rc) return rc;
    const long long m_tiles = cdiv(M, kBM), n_tiles = cdiv(Nn, kBN), k_blocks = cdiv(K, kBK);
    const long long units = cdiv(m_tiles, CG) * n_tiles;
    if (m_tiles * n_tiles > 0x3fffffffll || k_blocks > 0x7fffffffll) return LCE_ERR_TOO_LARGE;
    if (units == 0 || k_blocks == 0) return LCE_OK;
    // every k slice must hold at least one block
    if (k_splits < 1 || (k_splits - 1) * cdiv(k_blocks, k_splits) >= k_blocks) return LCE_ERR_ARG;
    auto kern = gemm_tc_kernel<kBN, kStages, CG, A_MN, B_MN, IS_BF16, Epi>;
    constexpr int smem = GemmSmem<kBN, kStages, CG, kEpiWarps>::kTotalBytes;
    // per kernel instantiation and device; setting the attribute twice from two threads is harmless
    static std::atomic<bool> smem_opted_in[kMaxDevices];
    if (!smem_opted_in[d.index].load(std::memory_order_acquire)) {
        if (cuda_failed(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem)))
            return LCE_ERR_CUDA;
        smem_opted_in[d.index].store(true, std::memory_order_release);
    }
    const long long slots = d.sm_count / CG;  // one CTA per SM; a pair occupies the two SMs of a TPC
    const long long work = units * k_splits;
    const int grid = static_cast<int>(work < slots ? work : slots) * CG;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(64 + 32 * kEpiWarps);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    // The kernel waits for its predecessor in the stream itself (ptx::grid_dep_wait after its set-up), so it may
    // be started under the predecessor's tail; pairs additionally launch as clusters of two.
    cudaLaunchAttribute attr[2];
    int n_attr = 0;
    if (pdl_enabled()) {
        attr[n_attr].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[n_attr].val.programmaticStreamSerializationAllowed = 1;
        ++n_attr;
    }
    if (CG > 1) {
        attr[n_attr].id = cudaLaunchAttributeClusterDimension;
        attr[n_attr].val.clusterDim.x = CG;
        attr[n_attr].val.clusterDim.y = 1;
        attr[n_attr].val.clusterDim.z = 1;
        ++n_attr;
    }
    cfg.attrs = attr;
    cfg.numAttrs = n_attr;
    // the banded operand is re-read by every tile of the band: keep it; the other one streams
    const int stream_hint = kHintMode == 1 ? ptx::kL2EvictFirst : ptx::kL2Normal;
    const int l2_hints = kHintMode == 0 ? 0 : (m_fastest ? (ptx::kL2EvictLast | (stream_hint << 2))
                                                          : (stream_hint | (ptx::kL2EvictLast << 2)));
    int raster;
    if (m_fastest) {  // bands of row units: rows fastest inside
        long long wb = kBandBytes / (static_cast<long long>(CG) * kBM * K * 2);
        const long long m_units = cdiv(m_tiles, CG);
        raster = static_cast<int>(wb < 1 ? 1 : (wb > m_units ? m_units : wb));
    } else {  // bands of tile columns: columns fastest inside
        long long wb = kBandBytes / (static_cast<long long>(kBN) * K * 2);
        raster = -static_cast<int>(wb < 1 ? 1 : (wb > n_tiles ? n_tiles : wb));
    }
    // Long launches deal their tiles from a counter in the caller's workspace, zeroed in stream order here.
    const int dyn_waves = g_tuning.dyn_waves.load(std::memory_order_relaxed);
    int* counter = (sched != nullptr && dyn_waves > 0 && work >= dyn_waves * slots) ? sched : nullptr;
    if (counter != nullptr && cuda_failed(cudaMemsetAsync(counter, 0, sizeof(int), stream))) return LCE_ERR_CUDA;
    const cudaError_t err = cudaLaunchKernelEx(&cfg, kern, tma, tmb, static_cast<int>(m_tiles),
                                               static_cast<int>(n_tiles), static_cast<int>(k_blocks), k_splits,
                                               raster, l2_hints, ep, d.status_ptr, counter, done, NoSecondGemm{});
    LCE_COUNT_LAUNCH();
    return cuda_failed(err) ? LCE_ERR_CUDA : LCE_OK;
}

// Two independent products with the same epilogue kind in ONE launch of single-CTA tiles: the first with a
// K-major A operand, the second with an MN-major one, both with MN-major B (the backward's dX = G W and
// dW = G^T X). Work items of the second follow those of the first in the round-robin deal.
struct GemmProblem {
    Mat a, b;
    long long M, Nn, K;
    int k_splits;
};
template <bool IS_BF16, class Epi>
int launch_tc_two(const DeviceInfo& d, const GemmProblem& p1, const typename Epi::Params& ep1, const GemmProblem& p2,
                  const typename Epi::Params& ep2, cudaStream_t stream) {
    constexpr int dtype = IS_BF16 ? LCE_DTYPE_BF16 : LCE_DTYPE_F16;
    using Second = SecondGemm<Epi, true>;
    CUtensorMap tma1, tmb1;
    Second sec;
    int rc;
    if ((rc = make_tmap(&tma1, p1.a.ptr, dtype, p1.K, p1.M, p1.a.pitch_elems * 2, kBK, kBM))) return rc;      // K-major A
    if ((rc = make_tmap(&tmb1, p1.b.ptr, dtype, p1.Nn, p1.K, p1.b.pitch_elems * 2, 64, kBK))) return rc;       // MN-major B
    if ((rc = make_tmap(&sec.tmA, p2.a.ptr, dtype, p2.M, p2.K, p2.a.pitch_elems * 2, 64, kBK))) return rc;    // MN-major A
    if ((rc = make_tmap(&sec.tmB, p2.b.ptr, dtype, p2.Nn, p2.K, p2.b.pitch_elems * 2, 64, kBK))) return rc;   // MN-major B
    const long long mt1 = cdiv(p1.M, kBM), nt1 = cdiv(p1.Nn, kBN), kb1 = cdiv(p1.K, kBK);
    const long long mt2 = cdiv(p2.M, kBM), nt2 = cdiv(p2.Nn, kBN), kb2 = cdiv(p2.K, kBK);
    if (mt1 * nt1 * p1.k_splits + mt2 * nt2 * p2.k_splits > 0x3fffffffll) return LCE_ERR_TOO_LARGE;
    if (mt1 * nt1 == 0 || mt2 * nt2 == 0 || kb1 == 0 || kb2 == 0) return LCE_ERR_ARG;
    if (p1.k_splits < 1 || (p1.k_splits - 1) * cdiv(kb1, p1.k_splits) >= kb1) return LCE_ERR_ARG;
    if (p2.k_splits < 1 || (p2.k_splits - 1) * cdiv(kb2, p2.k_splits) >= kb2) return LCE_ERR_ARG;
    sec.m_tiles = static_cast<int>(mt2);
    sec.n_tiles = static_cast<int>(nt2);
    sec.k_blocks = static_cast<int>(kb2);
    sec.k_splits = p2.k_splits;
    sec.raster = -static_cast<int>(nt2);  // columns fastest: small problems, everything stays in L2
    sec.ep = ep2;
    auto kern = gemm_tc_kernel<kBN, kStages1, 1, false, true, IS_BF16, Epi, Second>;
    constexpr int smem = GemmSmem<kBN, kStages1, 1>::kTotalBytes;
    static std::atomic<bool> smem_opted_in[kMaxDevices];
    if (!smem_opted_in[d.index].load(std::memory_order_acquire)) {
        if (cuda_failed(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem))) return LCE_ERR_CUDA;
        smem_opted_in[d.index].store(true, std::memory_order_release);
    }
    const long long work = mt1 * nt1 * p1.k_splits + mt2 * nt2 * p2.k_splits;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(work < d.sm_count ? work : d.sm_count));
    cfg.blockDim = dim3(kGemmThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl_enabled() ? 1 : 0;
    const cudaError_t err = cudaLaunchKernelEx(&cfg, kern, tma1, tmb1, static_cast<int>(mt1), static_cast<int>(nt1),
                                               static_cast<int>(kb1), p1.k_splits, -static_cast<int>(nt1), 0, ep1,
                                               d.status_ptr, static_cast<int*>(nullptr),
                                               static_cast<unsigned*>(nullptr), sec);
    LCE_COUNT_LAUNCH();
    return cuda_failed(err) ? LCE_ERR_CUDA : LCE_OK;
}

// CTA pairs cover two 128-row tiles at a time; with an odd, small number of row tiles the second
// half of the last pair would idle, so such problems run on single CTAs.
inline bool use_pair(long long M, int cg) {
    const long long m_tiles = cdiv(M, kBM);
    return cg == 2 && (m_tiles % 2 == 0 || m_tiles >= 16);
}

// Which tcgen05 variant a call asks for: CTA pairs (cta_group::2) unless LCE_FLAG_ONE_CTA is set.
inline int cta_group_of(unsigned flags) { return (flags & LCE_FLAG_ONE_CTA) ? 1 : 2; }

// Kernel family of one call, decided once from the arguments and passed down (no per-thread state).
struct Path {
    bool use_tc;  // tcgen05 GEMM core (else the CUDA-core one)
    int cg;       // cta group asked for: 2 = CTA pairs, 1 = single CTAs
    int* sched = nullptr;  // 4 bytes of the call's workspace for the dynamic tile deal, or nullptr
};

template <bool A_MN, bool B_MN, bool IS_BF16, class Epi>
int launch_tc(const DeviceInfo& d, int cg, const Mat& a, const Mat& b, long long M, long long Nn, long long K,
              int m_fastest, const typename Epi::Params& ep, cudaStream_t stream, int k_splits = 1,
              int* sched = nullptr, unsigned* done = nullptr) {
    if (use_pair(M, cg))
        return launch_tc_cg<2, A_MN, B_MN, IS_BF16, Epi>(d, a, b, M, Nn, K, m_fastest, k_splits, ep, stream, sched, done);
    return launch_tc_cg<1, A_MN, B_MN, IS_BF16, Epi>(d, a, b, M, Nn, K, m_fastest, k_splits, ep, stream, sched, done);
}

// The same for the CUDA-core GEMM (128 x 128 tiles, two CTAs per SM worth of work items).
inline int choose_k_splits_simt(long long M, long long Nn, long long K) {
    const long long units = cdiv(M, kBM) * cdiv(Nn, kSimtBN);
    if (units == 0 || units * 2 > 296) return 1;
    long long s = 296 / units;
    if (s > 32) s = 32;
    while (s > 1 && (K / s < 64 || (s - 1) * (cdiv(cdiv(K, s), kSimtBK) * kSimtBK) >= K)) --s;
    return static_cast<int>(s);
}

// How many slices to cut the contraction of an M x Nn x K GEMM into so that a problem with few output
// tiles still fills the GPU (the deterministic split-K: slices are added in slice order afterwards).
// Uses a fixed SM count so that workspace sizes do not depend on the device.
inline int choose_k_splits(long long M, long long Nn, long long K, int cg) {
    const long long slots = use_pair(M, cg) ? 74 : 148;
    const long long units = cdiv(cdiv(M, kBM), use_pair(M, cg) ? 2 : 1) * cdiv(Nn, kBN);
    const long long k_blocks = cdiv(K, kBK);
    if (units == 0 || units * 2 > slots) return 1;
    long long s = slots / units;
    if (s > 16) s = 16;
    while (s > 1 && (k_blocks / s < 16 || (s - 1) * cdiv(k_blocks, s) >= k_blocks)) --s;
    return static_cast<int>(s);
}

template <class T, class Epi, int TS = 128>
int launch_simt(const DeviceInfo& d, const Mat& a, bool a_mn, const Mat& b, bool b_mn, long long M,
                long long Nn, long long K, const typename Epi::Params& ep, cudaStream_t stream, int k_splits = 1) {
    SimtOperand<T> A, B;
    A.ptr = static_cast<const T*>(a.ptr);
    A.stride_mn = a_mn ? 1 : a.pitch_elems;
    A.stride_k = a_mn ? a.pitch_elems : 1;
    // fp32 rows that are padded with zeros to whole 16-byte vectors are read as whole vectors
    auto up4 = [](long long v) { return (v + 3) / 4 * 4; };
    auto mn_extent = [&](const Mat& x, bool mn, long long v) { return mn && x.cols >= up4(v) ? up4(v) : v; };
    auto k_extent = [&](const Mat& x, bool mn) { return !mn && x.cols >= up4(K) ? up4(K) : K; };
    A.extent_mn = static_cast<int>(mn_extent(a, a_mn, M));
    A.extent_k = static_cast<int>(k_extent(a, a_mn));
    B.ptr = static_cast<const T*>(b.ptr);
    B.stride_mn = b_mn ? 1 : b.pitch_elems;
    B.stride_k = b_mn ? b.pitch_elems : 1;
    B.extent_mn = static_cast<int>(mn_extent(b, b_mn, Nn));
    B.extent_k = static_cast<int>(k_extent(b, b_mn));
    const long long m_tiles = cdiv(M, TS), n_tiles = cdiv(Nn, TS);
    if (m_tiles * n_tiles > 0x7fffffffll) return LCE_ERR_TOO_LARGE;
    if (m_tiles * n_tiles == 0 || K == 0) return LCE_OK;
    constexpr int kThreads = SimtTile<TS>::kThreads;
    const long long cap = static_cast<long long>(d.sm_count) * (4 * 128 / TS);
    const long long work = m_tiles * n_tiles * k_splits;
    const int grid = static_cast<int>(work < cap ? work : cap);
    // one operand's zeros make up for what the other does not have
    const int k = A.extent_k > B.extent_k ? A.extent_k : B.extent_k, mt = static_cast<int>(m_tiles), nt = static_cast<int>(n_tiles);
    bool launched = false;
    if constexpr (std::is_same<T, float>::value) {
        // fp32 operands that allow 16-byte loads along their contiguous direction take the vector loaders
        const auto mode = [&](const SimtOperand<float>& op) {
            if ((reinterpret_cast<uintptr_t>(op.ptr) & 15u) != 0) return static_cast<int>(kSimtGeneric);
            if (op.stride_k == 1 && op.stride_mn % 4 == 0 && op.extent_k % 4 == 0) return static_cast<int>(kSimtVecK);
            if (op.stride_mn == 1 && op.stride_k % 4 == 0 && op.extent_mn % 4 == 0) return static_cast<int>(kSimtVecMN);
            return static_cast<int>(kSimtGeneric);
        };
        const int am = mode(A), bm = mode(B);
#define LCE_SIMT_GO(AM, BM) \
    gemm_simt_kernel<float, Epi, AM, BM, TS><<<grid, kThreads, 0, stream>>>(A, B, k, mt, nt, k_splits, ep), launched = true
        if (am == kSimtVecK && bm == kSimtVecK) LCE_SIMT_GO(kSimtVecK, kSimtVecK);
        else if (am == kSimtVecK && bm == kSimtVecMN) LCE_SIMT_GO(kSimtVecK, kSimtVecMN);
        else if (am == kSimtVecMN && bm == kSimtVecK) LCE_SIMT_GO(kSimtVecMN, kSimtVecK);
        else if (am == kSimtVecMN && bm == kSimtVecMN) LCE_SIMT_GO(kSimtVecMN, kSimtVecMN);
#undef LCE_SIMT_GO
    }
    if (!launched) gemm_simt_kernel<T, Epi, kSimtGeneric, kSimtGeneric, TS><<<grid, kThreads, 0, stream>>>(A, B, k, mt, nt, k_splits, ep);
    LCE_COUNT_LAUNCH();
    return (cuda_failed(cudaGetLastError()) ? LCE_ERR_CUDA : LCE_OK);
}

// The tcgen05 path needs 16-bit inputs, 16-byte aligned bases and row pitches (H % 8 == 0).
inline int choose_path(int dtype, long long H, const void* x, const void* w, unsigned flags, bool* use_tc) {
    const bool can_tc = dtype != LCE_DTYPE_F32 && (H % 8) == 0 && aligned16(x) && aligned16(w);
    if (flags & LCE_FLAG_FORCE_TC) {
        if (flags & LCE_FLAG_FORCE_SIMT) return LCE_ERR_ARG;
        if (dtype == LCE_DTYPE_F32) return LCE_ERR_ARG;
        if (!can_tc) return LCE_ERR_ALIGN;
        *use_tc = true;
        return LCE_OK;
    }
    *use_tc = can_tc && !(flags & LCE_FLAG_FORCE_SIMT);
    return LCE_OK;
}

// Whether a 16-bit result may leave the tcgen05 epilogue as whole 128-byte lines (store_block64): needs 16-byte
// aligned rows. HELION_B200_EPI_WIDE=0 (tuning knob) switches back to per-thread row stores.
inline int wide_stores(const void* out, long long ld) {
    static const int kEnabled = [] { const char* e = getenv("HELION_B200_EPI_WIDE"); return e ? atoi(e) : 1; }();
    return (kEnabled != 0 && aligned16(out) && ld % 8 == 0) ? 1 : 0;
}

}  // namespace lce
