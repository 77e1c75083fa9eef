// extern "C" entry points of the projection with its epilogue (declared in include/helion_lce.h): argument checks, the
// plan of a call (kernel family, split of the contraction, operands that need another pitch) and the launches.
#include "api_common.cuh"
#include "gemm_launch.cuh"
#include "linear_kernels.cuh"

namespace lce {
namespace {

// The row pitch of what a forward saves for its backward: whole 16-byte vectors whatever the type.
inline long long pre_pitch(long long N) { return cdiv(N, 8) * 8; }

std::atomic<unsigned> g_decode_announce_extra{0};  // the decode kernel's test hook

constexpr long long kDzCtas = 592;  // CTAs that the column sums of the backward aim for (4 per SM on 148 SMs, one wave)

// Scratch of one product C[M, N] = A[M, K] B[N, K]^T: slabs of a split contraction.
struct ProductPlan {
    bool use_tc;
    int cg, splits, bn;
    long long slab_floats;
    size_t bytes;
    bool small_tiles;  // CUDA-core GEMM: 64 x 64 tiles
};

ProductPlan plan_product(long long M, long long N, long long K, int dtype, unsigned flags) {
    ProductPlan p;
    p.use_tc = dtype != LCE_DTYPE_F32 && !(flags & LCE_FLAG_FORCE_SIMT);
    p.cg = cta_group_of(flags);
    p.bn = p.use_tc ? kBN : kSimtBN;
    p.splits = p.use_tc ? choose_k_splits(M, N, K, p.cg) : choose_k_splits_simt(M, N, K);
    p.slab_floats = cdiv(M, 2 * kBM) * 2 * cdiv(N, p.bn) * kBM * p.bn;
    p.bytes = p.splits > 1 ? align_up(static_cast<size_t>(p.splits) * p.slab_floats * sizeof(float), 256) : 0;
    p.small_tiles = false;
    return p;
}

// The forward of a call whose relu slopes are saved. A slope is the sign of z, and at a z within its rounding of 0 the order
// of the sum decides it: one such element in 777 x 1003 shifts fp32 gradients by 6e-4 of their norm, thirty times what
// rounding does. So an fp32 z whose sign is saved is one chain of fused multiply-adds over the contraction, whatever the number of
// tokens: a row gets the same slopes in every batch, and those of an unsplit fp32 product elsewhere. Where the contraction would be
// split, tiles of 64 x 64 fill the GPU instead: 777 x 520 x 1003 46 us (split 35, unsplit tiles of 128 x 128 82); a long
// contraction with few tiles pays most, 128 x 4096 x 128 167 us against 26.
ProductPlan plan_forward(long long M, long long N, long long K, int act, const void* pre, int dtype, unsigned flags) {
    ProductPlan p = plan_product(M, N, K, dtype, flags);
    if (p.splits > 1 && act == LCE_ACT_RELU && pre && dtype == LCE_DTYPE_F32) {
        p.splits = 1;
        p.bytes = 0;
        p.small_tiles = true;
    }
    return p;
}

// Few tokens take the decode kernel: one launch that reads W once, 14.3 us at 16 x 4096 x 4096 (cold cache) where the core's
// split contraction and its sum took 23.5. It was the faster one up to its 64 tokens.
constexpr long long kDecodeTokens = 64;
inline bool decodes(long long M, int dtype, unsigned flags) {
    return dtype != LCE_DTYPE_F32 && !(flags & LCE_FLAG_FORCE_SIMT) && M <= kDecodeTokens;
}

// An operand [rows, cols] as the caller has it, and whether the kernels need it at another pitch (a copy in scratch).
struct Operand {
    const void* ptr;
    long long ld, rows, cols;
    long long copy_ld;  // 0: taken as it is
    size_t copy_bytes;
};

Operand plan_operand(const void* ptr, long long ld, long long rows, long long cols, int dtype, unsigned flags) {
    Operand o{ptr, ld, rows, cols, 0, 0};
    const long long vec = 16 / static_cast<long long>(elem_size(dtype));
    const bool vectors = dtype == LCE_DTYPE_F32 || !(flags & LCE_FLAG_FORCE_SIMT);  // forced: element by element anyway
    if (vectors && !(aligned16(ptr) && ld % vec == 0)) {
        o.copy_ld = cdiv(cols, vec) * vec;
        o.copy_bytes = align_up(static_cast<size_t>(rows) * o.copy_ld * elem_size(dtype), 256);
    }
    return o;
}

template <class T>
int place_operand(Operand& o, char*& ws, cudaStream_t s) {
    if (o.copy_ld == 0) return LCE_OK;
    T* dst = reinterpret_cast<T*>(ws);
    ws += o.copy_bytes;
    const long long blocks = cdiv(o.rows, 8);
    repitch_kernel<T><<<static_cast<unsigned>(blocks < 8192 ? blocks : 8192), 256, 0, s>>>(
        static_cast<const T*>(o.ptr), o.ld, dst, o.copy_ld, o.rows, static_cast<int>(o.cols));
    LCE_COUNT_LAUNCH();
    o.ptr = dst;
    o.ld = o.cols = o.copy_ld;
    return cuda_failed(cudaGetLastError()) ? LCE_ERR_CUDA : LCE_OK;
}

template <class Epi, class T>
typename Epi::Params epilogue_params(const ProductPlan& p, const LinearTail<T>& tail, void* scratch) {
    typename Epi::Params ep;
    ep.t = tail;
    ep.scratch = p.splits > 1 ? static_cast<float*>(scratch) : nullptr;
    ep.slab_floats = p.slab_floats;
    ep.wide_out = wide_stores(tail.out, tail.ldo);
    ep.wide_residual = wide_stores(tail.residual, tail.ldr);
    return ep;
}

template <class T, bool A_MN, bool B_MN, int ACT, bool HEAVY>
int product_tc(const DeviceInfo& d, const ProductPlan& p, const Mat& a, const Mat& b, long long M, long long N, long long K,
               const LinearTail<T>& tail, void* scratch, cudaStream_t s) {
    using Epi = EpiLinear<T, ACT, HEAVY>;
    // tiles that run together share a B panel when there are many row tiles, an A panel otherwise
    const int m_fastest = cdiv(M, kBM) >= cdiv(N, kBN) ? 1 : 0;
    return launch_tc<A_MN, B_MN, std::is_same<T, __nv_bfloat16>::value, Epi>(d, p.cg, a, b, M, N, K, m_fastest,
                                                                            epilogue_params<Epi>(p, tail, scratch), s, p.splits);
}

// C = act(A B^T + bias) + residual; an operand is K-major ([mn, K] rows) or MN-major ([K, mn] rows). Only K-major operands
// come with an activation, a residual or saved values (the forward).
template <class T, bool A_MN, bool B_MN>
int product(const DeviceInfo& d, const ProductPlan& p, const Operand& a, const Operand& b, long long M, long long N,
            long long K, const LinearTail<T>& tail, void* scratch, cudaStream_t s) {
    const Mat am{a.ptr, a.rows, a.cols, a.ld}, bm{b.ptr, b.rows, b.cols, b.ld};
    int rc = LCE_ERR_ARG;
    if (p.use_tc) {
        if constexpr (sizeof(T) == 2) {
            // a split contraction leaves as plain sums; linear_reduce_kernel finishes them
            const bool light = (tail.act == kActNone && tail.residual == nullptr && tail.bias == nullptr) || p.splits > 1;
            if constexpr (A_MN || B_MN) {
                rc = product_tc<T, A_MN, B_MN, kActNone, false>(d, p, am, bm, M, N, K, tail, scratch, s);
            } else if (light) {
                rc = product_tc<T, false, false, kActNone, false>(d, p, am, bm, M, N, K, tail, scratch, s);
            } else {
                switch (tail.act) {
                    case kActNone: rc = product_tc<T, false, false, kActNone, true>(d, p, am, bm, M, N, K, tail, scratch, s); break;
                    case kActRelu: rc = product_tc<T, false, false, kActRelu, true>(d, p, am, bm, M, N, K, tail, scratch, s); break;
                    case kActGelu: rc = product_tc<T, false, false, kActGelu, true>(d, p, am, bm, M, N, K, tail, scratch, s); break;
                    case kActGeluTanh: rc = product_tc<T, false, false, kActGeluTanh, true>(d, p, am, bm, M, N, K, tail, scratch, s); break;
                    case kActSilu: rc = product_tc<T, false, false, kActSilu, true>(d, p, am, bm, M, N, K, tail, scratch, s); break;
                    default: break;
                }
            }
        }
    } else {
        using Epi = EpiLinear<T, kActAny, false>;
        const typename Epi::Params ep = epilogue_params<Epi>(p, tail, scratch);
        if constexpr (std::is_same<T, float>::value && !A_MN && !B_MN) {
            rc = p.small_tiles ? launch_simt<T, Epi, 64>(d, am, A_MN, bm, B_MN, M, N, K, ep, s)
                               : launch_simt<T, Epi>(d, am, A_MN, bm, B_MN, M, N, K, ep, s, p.splits);
        } else {
            rc = launch_simt<T, Epi>(d, am, A_MN, bm, B_MN, M, N, K, ep, s, p.splits);
        }
    }
    if (rc == LCE_OK && p.splits > 1) {
        const long long quads = cdiv(N, 16) * cdiv(M, 16) * 64;
        const int blocks = static_cast<int>(cdiv(quads, 256) < 4096 ? cdiv(quads, 256) : 4096);
        const cudaError_t err = launch_dependent(linear_reduce_kernel<T>, blocks, 256, s, static_cast<const float*>(scratch),
                                                 p.splits, p.slab_floats, static_cast<int>(cdiv(N, p.bn)), p.bn, tail);
        LCE_COUNT_LAUNCH();
        if (cuda_failed(err)) rc = LCE_ERR_CUDA;
    }
    return rc;
}

bool linear_args_ok(long long M, long long N, long long K, long long ldx, long long ldw, int act, int dtype) {
    return M >= 0 && N > 0 && K > 0 && ldx >= K && ldw >= K && known_dtype(dtype) && act >= LCE_ACT_NONE && act <= LCE_ACT_SILU;
}
bool linear_too_large(long long M, long long N, long long K) { return M > 0x7fffff00ll || N > 0x7fffff00ll || K > 0x7fffff00ll; }

size_t forward_bytes(const Operand& x, const Operand& w, const ProductPlan& p, bool decode) {
    return x.copy_bytes + w.copy_bytes + (decode ? 0 : p.bytes);
}

template <class T, int BN>
int launch_decode(const DeviceInfo& d, const Operand& x, const Operand& w, long long N, long long K, const LinearTail<T>& tail, cudaStream_t s) {
    const int dtype = std::is_same<T, __nv_bfloat16>::value ? LCE_DTYPE_BF16 : LCE_DTYPE_F16;
    CUtensorMap tm_w, tm_x;
    int rc;
    if ((rc = make_tmap(&tm_w, w.ptr, dtype, K, N, w.ld * 2, kBK, kBM))) return rc;
    if ((rc = make_tmap(&tm_x, x.ptr, dtype, K, x.rows, x.ld * 2, kBK, BN))) return rc;
    // the contraction is cut until the CTAs fill the GPU twice over, as long as a CTA has two blocks of 64 to stream
    const long long tiles = cdiv(N, kBM), k_blocks = cdiv(K, kBK);
    int splits = 1;
    while (splits < 8 && tiles * splits * 2 <= 2 * d.sm_count && k_blocks >= 4 * splits) splits *= 2;
    if (tiles * splits > 0x7fffffffll) return LCE_ERR_TOO_LARGE;
    auto kern = linear_decode_kernel<T, BN>;
    constexpr int smem = DecodeSmem<BN>::kTotalBytes;
    static std::atomic<bool> opted_in[kMaxDevices];  // setting the attribute twice from two threads is harmless
    if (!opted_in[d.index].load(std::memory_order_acquire)) {
        if (cuda_failed(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem))) return LCE_ERR_CUDA;
        opted_in[d.index].store(true, std::memory_order_release);
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(tiles * splits));
    cfg.blockDim = dim3(kGemmThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    int n_attr = 0;
    if (pdl_enabled()) {
        attr[n_attr].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[n_attr].val.programmaticStreamSerializationAllowed = 1;
        ++n_attr;
    }
    if (splits > 1) {
        attr[n_attr].id = cudaLaunchAttributeClusterDimension;
        attr[n_attr].val.clusterDim.x = splits;
        attr[n_attr].val.clusterDim.y = 1;
        attr[n_attr].val.clusterDim.z = 1;
        ++n_attr;
    }
    cfg.attrs = attr;
    cfg.numAttrs = n_attr;
    const cudaError_t err = cudaLaunchKernelEx(&cfg, kern, tm_w, tm_x, static_cast<int>(k_blocks), splits, tail, d.status_ptr,
                                               g_decode_announce_extra.load(std::memory_order_relaxed));
    LCE_COUNT_LAUNCH();
    return cuda_failed(err) ? LCE_ERR_CUDA : LCE_OK;
}

template <class T>
int forward_impl(const DeviceInfo& d, Operand x, Operand w, const ProductPlan& p, bool decode, long long M, long long N, long long K,
                 const LinearTail<T>& tail, char* ws, cudaStream_t s) {
    int rc;
    if ((rc = place_operand<T>(x, ws, s)) || (rc = place_operand<T>(w, ws, s))) return rc;
    if constexpr (sizeof(T) == 2) {
        if (decode) {
            if (M <= 16) return launch_decode<T, 16>(d, x, w, N, K, tail, s);
            if (M <= 32) return launch_decode<T, 32>(d, x, w, N, K, tail, s);
            return launch_decode<T, 64>(d, x, w, N, K, tail, s);
        }
    }
    return product<T, false, false>(d, p, x, w, M, N, K, tail, ws, s);
}

// Scratch of a backward pass: copies of x and W, dz at a pitch that TMA can read, the column sums, and the slabs of the
// two products (which run one after the other and share their space).
struct BackwardPlan {
    Operand x, w;
    bool copy_dz;       // dz is not dy as it stands
    long long ldz, slabs, rows_per_slab;
    size_t dz_bytes, sums_bytes, slab_bytes, total;
    ProductPlan px, pw;
};

BackwardPlan plan_linear_backward(const void* dy, long long ldy, const void* x, long long ldx, const void* w, long long ldw,
                                  long long M, long long N, long long K, int act, int dtype, unsigned flags) {
    BackwardPlan b;
    b.x = plan_operand(x, ldx, M, K, dtype, flags);
    b.w = plan_operand(w, ldw, N, K, dtype, flags);
    b.copy_dz = act != LCE_ACT_NONE || plan_operand(dy, ldy, M, N, dtype, flags).copy_ld != 0;
    const long long vec = 16 / static_cast<long long>(elem_size(dtype));
    b.ldz = cdiv(N, vec) * vec;
    b.dz_bytes = b.copy_dz ? align_up(static_cast<size_t>(M) * b.ldz * elem_size(dtype), 256) : 0;
    const long long strips = cdiv(N, 32 * vec);
    b.slabs = kDzCtas / strips;
    b.slabs = b.slabs < 1 ? 1 : b.slabs;
    b.rows_per_slab = cdiv(M, b.slabs);
    b.rows_per_slab = b.rows_per_slab < 32 ? 32 : b.rows_per_slab;
    b.slabs = cdiv(M, b.rows_per_slab);
    b.sums_bytes = align_up(static_cast<size_t>(b.slabs) * N * sizeof(float), 256);
    b.px = plan_product(M, K, N, dtype, flags);
    b.pw = plan_product(N, K, M, dtype, flags);
    b.slab_bytes = b.px.bytes > b.pw.bytes ? b.px.bytes : b.pw.bytes;
    b.total = b.x.copy_bytes + b.w.copy_bytes + b.dz_bytes + b.sums_bytes + b.slab_bytes;
    return b;
}

template <class T, int ACT>
void launch_dz(const BackwardPlan& b, const void* dy, long long ldy, const void* pre, T* dz, float* sums, long long M, long long N,
               cudaStream_t s) {
    const dim3 grid(static_cast<unsigned>(cdiv(N, 32 * (16 / sizeof(T)))), static_cast<unsigned>(b.slabs));
    linear_dz_kernel<T, ACT><<<grid, 256, 0, s>>>(static_cast<const T*>(dy), ldy, static_cast<const T*>(pre), pre_pitch(N),
                                                  b.copy_dz ? dz : nullptr, b.ldz, sums, M, static_cast<int>(N), b.rows_per_slab);
}

template <class T>
int linear_backward_impl(const DeviceInfo& d, BackwardPlan& b, const void* dy, long long ldy, const void* pre, void* dx, void* dw,
                         void* dbias, long long M, long long N, long long K, int act, char* ws, cudaStream_t s) {
    int rc;
    if (dw && (rc = place_operand<T>(b.x, ws, s))) return rc;
    if (dx && (rc = place_operand<T>(b.w, ws, s))) return rc;
    T* dz = reinterpret_cast<T*>(ws);
    ws += b.dz_bytes;
    float* sums = reinterpret_cast<float*>(ws);
    ws += b.sums_bytes;
    const bool products = dx || dw;
    if (dbias || (products && b.copy_dz)) {
        switch (act) {
            case kActRelu: launch_dz<T, kActRelu>(b, dy, ldy, pre, dz, dbias ? sums : nullptr, M, N, s); break;
            case kActGelu: launch_dz<T, kActGelu>(b, dy, ldy, pre, dz, dbias ? sums : nullptr, M, N, s); break;
            case kActGeluTanh: launch_dz<T, kActGeluTanh>(b, dy, ldy, pre, dz, dbias ? sums : nullptr, M, N, s); break;
            case kActSilu: launch_dz<T, kActSilu>(b, dy, ldy, pre, dz, dbias ? sums : nullptr, M, N, s); break;
            default: launch_dz<T, kActNone>(b, dy, ldy, pre, dz, dbias ? sums : nullptr, M, N, s); break;
        }
        LCE_COUNT_LAUNCH();
        if (cuda_failed(cudaGetLastError())) return LCE_ERR_CUDA;
        if (dbias) {
            const cudaError_t err = launch_dependent(linear_dbias_kernel<T>, static_cast<int>(cdiv(N, 32)), 1024, s,
                                                     static_cast<const float*>(sums), static_cast<int>(b.slabs),
                                                     static_cast<int>(N), static_cast<T*>(dbias));
            LCE_COUNT_LAUNCH();
            if (cuda_failed(err)) return LCE_ERR_CUDA;
        }
    }
    const Operand z{b.copy_dz ? dz : dy, b.copy_dz ? b.ldz : ldy, M, b.copy_dz ? b.ldz : N, 0, 0};
    LinearTail<T> tail = {};
    if (dx) {  // [M, K] = dz [M, N] W [N, K]
        tail.out = static_cast<T*>(dx);
        tail.ldo = K;
        tail.rows = static_cast<int>(M);
        tail.cols = static_cast<int>(K);
        if ((rc = product<T, false, true>(d, b.px, z, b.w, M, K, N, tail, ws, s))) return rc;
    }
    if (dw) {  // [N, K] = dz^T [N, M] x [M, K]
        tail.out = static_cast<T*>(dw);
        tail.ldo = K;
        tail.rows = static_cast<int>(N);
        tail.cols = static_cast<int>(K);
        if ((rc = product<T, true, true>(d, b.pw, z, b.x, N, K, M, tail, ws, s))) return rc;
    }
    return LCE_OK;
}

}  // namespace

int linear_debug_waits(unsigned long long limit_ns, unsigned announce_extra_bytes) {
    g_decode_announce_extra.store(announce_extra_bytes, std::memory_order_relaxed);
    return set_debug_waits(limit_ns, announce_extra_bytes);
}

}  // namespace lce

using namespace lce;

extern "C" {

size_t lce_linear_forward_workspace_bytes(const void* x, int64_t ldx, const void* w, int64_t ldw, int64_t M, int64_t N,
                                          int64_t K, int dtype, unsigned flags) {
    if (!linear_args_ok(M, N, K, ldx, ldw, LCE_ACT_NONE, dtype) || linear_too_large(M, N, K) || M == 0) return 0;
    return forward_bytes(plan_operand(x, ldx, M, K, dtype, flags), plan_operand(w, ldw, N, K, dtype, flags),
                         plan_product(M, N, K, dtype, flags), decodes(M, dtype, flags));
}

int lce_linear_forward(const void* x, int64_t ldx, const void* w, int64_t ldw, const void* bias, const void* residual,
                       int64_t ldr, void* out, int64_t ldo, void* pre, int64_t M, int64_t N, int64_t K, int act, int dtype,
                       void* ws, size_t ws_bytes, unsigned flags, void* stream) {
    if (!linear_args_ok(M, N, K, ldx, ldw, act, dtype) || ldo < N || (residual && ldr < N)) return LCE_ERR_ARG;
    if (linear_too_large(M, N, K)) return LCE_ERR_TOO_LARGE;
    if ((flags & LCE_FLAG_FORCE_TC) && dtype == LCE_DTYPE_F32) return LCE_ERR_ARG;
    if (M == 0) return LCE_OK;
    if (!x || !w || !out) return LCE_ERR_ARG;
    const Operand xo = plan_operand(x, ldx, M, K, dtype, flags), wo = plan_operand(w, ldw, N, K, dtype, flags);
    const ProductPlan p = plan_forward(M, N, K, act, pre, dtype, flags);
    const bool decode = decodes(M, dtype, flags);
    const size_t need = forward_bytes(xo, wo, p, decode);
    if (need > 0 && (!ws || ws_bytes < need)) return LCE_ERR_WS_TOO_SMALL;
    DeviceInfo* d;
    const int rc = device_info(&d);
    if (rc) return rc;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    char* scratch = static_cast<char*>(ws);
#define LCE_LINEAR_FORWARD(T)                                                                                              \
    forward_impl<T>(*d, xo, wo, p, decode, M, N, K,                                                                             \
                    LinearTail<T>{static_cast<T*>(out), ldo, act == LCE_ACT_NONE ? nullptr : static_cast<T*>(pre),         \
                                  pre_pitch(N), static_cast<const T*>(bias), static_cast<const T*>(residual), ldr, static_cast<int>(M),  \
                                  static_cast<int>(N), act},                                                               \
                    scratch, s)
    switch (dtype) {
        case LCE_DTYPE_BF16: return LCE_LINEAR_FORWARD(__nv_bfloat16);
        case LCE_DTYPE_F16: return LCE_LINEAR_FORWARD(__half);
        default: return LCE_LINEAR_FORWARD(float);
    }
#undef LCE_LINEAR_FORWARD
}

size_t lce_linear_backward_workspace_bytes(const void* dy, int64_t ldy, const void* x, int64_t ldx, const void* w, int64_t ldw,
                                           int64_t M, int64_t N, int64_t K, int act, int dtype, unsigned flags) {
    if (!linear_args_ok(M, N, K, ldx, ldw, act, dtype) || ldy < N || linear_too_large(M, N, K) || M == 0) return 0;
    return plan_linear_backward(dy, ldy, x, ldx, w, ldw, M, N, K, act, dtype, flags).total;
}

int lce_linear_backward(const void* dy, int64_t ldy, const void* x, int64_t ldx, const void* w, int64_t ldw, const void* pre,
                        void* dx, void* dw, void* dbias, int64_t M, int64_t N, int64_t K, int act, int dtype, void* ws,
                        size_t ws_bytes, unsigned flags, void* stream) {
    if (!linear_args_ok(M, N, K, ldx, ldw, act, dtype) || ldy < N) return LCE_ERR_ARG;
    if (linear_too_large(M, N, K)) return LCE_ERR_TOO_LARGE;
    if ((flags & LCE_FLAG_FORCE_TC) && dtype == LCE_DTYPE_F32) return LCE_ERR_ARG;
    if (!dx && !dw && !dbias) return LCE_OK;
    if (M > 0 && (!dy || (act != LCE_ACT_NONE && !pre) || (dw && !x) || (dx && !w))) return LCE_ERR_ARG;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    DeviceInfo* d;
    const int rc = device_info(&d);
    if (rc) return rc;
    if (M == 0) {  // sums of nothing
        if (dw && cuda_failed(cudaMemsetAsync(dw, 0, static_cast<size_t>(N) * K * elem_size(dtype), s))) return LCE_ERR_CUDA;
        if (dbias && cuda_failed(cudaMemsetAsync(dbias, 0, static_cast<size_t>(N) * elem_size(dtype), s))) return LCE_ERR_CUDA;
        return LCE_OK;
    }
    BackwardPlan b = plan_linear_backward(dy, ldy, x, ldx, w, ldw, M, N, K, act, dtype, flags);
    if (!ws || ws_bytes < b.total) return LCE_ERR_WS_TOO_SMALL;
    char* scratch = static_cast<char*>(ws);
    switch (dtype) {
        case LCE_DTYPE_BF16: return linear_backward_impl<__nv_bfloat16>(*d, b, dy, ldy, pre, dx, dw, dbias, M, N, K, act, scratch, s);
        case LCE_DTYPE_F16: return linear_backward_impl<__half>(*d, b, dy, ldy, pre, dx, dw, dbias, M, N, K, act, scratch, s);
        default: return linear_backward_impl<float>(*d, b, dy, ldy, pre, dx, dw, dbias, M, N, K, act, scratch, s);
    }
}

}  // extern "C"
