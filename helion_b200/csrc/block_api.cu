// extern "C" entry points of the operators of a decoder block around the head (declared in include/helion_lce.h):
// rotary positions, the query / key norms, and the sampler. Argument checks, the choice of kernel form, the launches.
#include "api_common.cuh"
#include "rope_kernels.cuh"
#include "sample_kernels.cuh"

namespace lce {
namespace {

// ---------------------------------------------------------------------------------------------
// rotary positions, query / key norms
// ---------------------------------------------------------------------------------------------
struct HeadCall {
    long long batch, seq, dim, half;
    int interleaved, mode, dtype, sm_count;
};

// Whether every row, and every pair of vectors that rotate together, is made of whole aligned `vec`-element vectors.
bool head_rows_vectors(const lce_head_rows& r, const HeadCall& c, long long vec, uintptr_t bytes) {
    auto fits = [&](const void* p, const int64_t* stride) {
        return reinterpret_cast<uintptr_t>(p) % bytes == 0 && stride[0] % vec == 0 && stride[1] % vec == 0 && stride[2] % vec == 0;
    };
    if (r.heads == 0) return true;
    if (!fits(r.x, r.x_stride) || !fits(r.out, r.out_stride)) return false;
    if (c.mode == kHeadNormBackward && !fits(r.grad, r.grad_stride)) return false;
    return c.mode == kHeadRope || reinterpret_cast<uintptr_t>(r.weight) % bytes == 0;
}

// Whether the offsets within one token fit 32 bits.
bool head_offsets_32(const lce_head_rows& r, const HeadCall& c) {
    auto fits = [&](const int64_t* stride) {
        const long long s = stride[2] < 0 ? -stride[2] : stride[2];
        return s < (1ll << 31) && s * r.heads + c.dim < (1ll << 31);
    };
    return fits(r.x_stride) && fits(r.out_stride) && fits(r.grad_stride);
}

int check_head_rows(const lce_head_rows* r, const HeadCall& c) {
    if (!r || r->heads < 0) return LCE_ERR_ARG;
    if (r->heads > 0x7fffffll / 32) return LCE_ERR_TOO_LARGE;
    if (r->heads == 0 || c.batch == 0 || c.seq == 0) return LCE_OK;
    if (!r->x || !r->out) return LCE_ERR_ARG;
    if (c.mode != kHeadRope && !r->weight) return LCE_ERR_ARG;
    if (c.mode == kHeadNormBackward && !r->grad) return LCE_ERR_ARG;
    return LCE_OK;
}

// A dimension of one entry has no stride: whatever the caller's tensor says there must not cost it the vector form.
lce_head_rows plain_strides(lce_head_rows r, const HeadCall& c) {
    const int64_t extent[3] = {c.batch, c.seq, r.heads};
    for (int i = 0; i < 3; ++i)
        if (extent[i] == 1) r.x_stride[i] = r.out_stride[i] = r.grad_stride[i] = 0;
    return r;
}

// Deals `tokens` x `heads` rows to warps: whole tokens per warp (their angles are formed once) as long as that gives
// every SM `kWarps` warps, pieces of a token otherwise. `total_steps`: of a token.
template <class T>
HeadRows<T> deal_heads(const lce_head_rows& r, const HeadCall& c, long long total_steps, int warps_per_cta, long long max_ctas) {
    HeadRows<T> h;
    h.x = static_cast<const T*>(r.x);
    h.x_b = r.x_stride[0], h.x_s = r.x_stride[1], h.x_h = r.x_stride[2];
    h.dy = static_cast<const T*>(r.grad);
    h.dy_b = r.grad_stride[0], h.dy_s = r.grad_stride[1], h.dy_h = r.grad_stride[2];
    h.out = static_cast<T*>(r.out);
    h.o_b = r.out_stride[0], h.o_s = r.out_stride[1], h.o_h = r.out_stride[2];
    h.weight = static_cast<const T*>(r.weight);
    h.partial = nullptr;
    h.heads = static_cast<int>(r.heads);
    const long long tokens = c.batch * c.seq;
    if (tokens == 0 || total_steps == 0) {
        h.chunks = h.steps = 1;
        h.units = 0;
        h.ctas = 0;
        return h;
    }
    constexpr long long kWarps = 16;
    long long steps = total_steps * tokens / (kWarps * c.sm_count);
    steps = steps < 1 ? 1 : (steps > total_steps ? total_steps : steps);
    h.steps = static_cast<int>(steps);
    h.chunks = static_cast<int>(cdiv(total_steps, steps));
    h.units = tokens * h.chunks;
    const long long want = cdiv(h.units, warps_per_cta);
    h.ctas = static_cast<int>(want < max_ctas ? want : max_ctas);
    return h;
}

template <class T, bool INTERLEAVED, int MODE>
int launch_heads(const HeadCall& c, const lce_head_rows& q, const lce_head_rows& k, RopePlan p, float* partial, cudaStream_t s) {
    constexpr int VEC = RmsTile<T>::kVec;
    const long long pair = INTERLEAVED ? 2 * c.half : c.half;  // what has to be whole vectors besides the rows
    const long long np = c.half / VEC, nv = c.dim / VEC;
    const int items = static_cast<int>(INTERLEAVED ? cdiv(nv, 2) : np + cdiv(nv - 2 * np, 2));
    const bool vector = c.dim % VEC == 0 && pair % VEC == 0 && items <= 32 && head_rows_vectors(q, c, VEC, 16) &&
                        head_rows_vectors(k, c, VEC, 16) && head_offsets_32(q, c) && head_offsets_32(k, c);
    p.items = items;
    p.lanes = 1;
    while (p.lanes < items) p.lanes <<= 1;
    p.pairs2 = c.dim % 2 == 0 && head_rows_vectors(q, c, 2, 2 * sizeof(T)) && head_rows_vectors(k, c, 2, 2 * sizeof(T));
    const int per_step = vector ? 32 / p.lanes : 1;
    using Shape = HeadShape<T, MODE>;
    const int warps = vector ? Shape::kWarps : kRowFormWarps;
    // The grid is what fits the GPU at once: a warp then walks many tokens, which spreads its set-up, and in the backward
    // its sums. Where q and k have CTAs of their own they share the grid by their steps, a token's set-up counting as two.
    const long long steps_q = cdiv(q.heads, per_step), steps_k = cdiv(k.heads, per_step);
    const long long cost_q = steps_q > 0 ? steps_q + 2 : 0, cost_k = steps_k > 0 ? steps_k + 2 : 0;
    const bool together = vector && MODE != kHeadNormBackward;
    auto share = [&](long long cost) {
        // rotations alone, and fp32 norms, keep up without and are 4 % faster dealt out by the hardware, a token to a warp
        if (MODE == kHeadRope || (MODE == kHeadNorm && sizeof(T) == 4)) return 1ll << 20;
        const long long fit = c.sm_count * (vector ? static_cast<long long>(Shape::kCtas) : 3ll);
        if (together) return fit;
        const long long cap = (fit < kHeadMaxCtas ? fit : kHeadMaxCtas) * cost / (cost_q + cost_k > 0 ? cost_q + cost_k : 1);
        return cap < 1 ? 1ll : cap;
    };
    HeadRows<T> hq = deal_heads<T>(q, c, together ? steps_q + steps_k : steps_q, warps, share(cost_q));
    HeadRows<T> hk = deal_heads<T>(k, c, together ? 0 : steps_k, warps, share(cost_k));
    if (MODE == kHeadNormBackward) {
        // the partial rows have to fit the workspace, whatever the split above comes to
        if (hq.ctas + hk.ctas > kHeadMaxCtas + 1) return LCE_ERR_WS_TOO_SMALL;
        if (q.dweight) hq.partial = partial;
        if (k.dweight) hk.partial = partial + static_cast<long long>(hq.ctas) * c.dim;
    }
    if (hq.ctas + hk.ctas > 0) {
        if (vector) {
            const int smem = Shape::kWarps * items * VEC * static_cast<int>(sizeof(float2));
            heads_vector_kernel<T, INTERLEAVED, MODE><<<hq.ctas + hk.ctas, Shape::kThreads, smem, s>>>(hq, hk, p);
        } else {
            const int smem = kRowFormWarps * row_form_floats(p.dim, p.half, MODE) * 4;
            auto kern = heads_row_kernel<T, INTERLEAVED, MODE>;
            if (smem > 48 * 1024 && cuda_failed(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem)))
                return LCE_ERR_CUDA;
            kern<<<hq.ctas + hk.ctas, kRowFormWarps * 32, smem, s>>>(hq, hk, p);
        }
        LCE_COUNT_LAUNCH();
        if (cuda_failed(cudaGetLastError())) return LCE_ERR_CUDA;
    }
    if (MODE == kHeadNormBackward && (q.dweight || k.dweight)) {
        // cudaLaunchKernelEx takes one grid dimension through launch_dependent; this one has two
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(static_cast<unsigned>(cdiv(c.dim, 32)), 2);
        cfg.blockDim = dim3(32, 32);
        cfg.stream = s;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = attr;
        cfg.numAttrs = pdl_enabled() ? 1 : 0;
        const cudaError_t err = cudaLaunchKernelEx(&cfg, head_dweight_kernel<T>, static_cast<const float*>(hq.partial), hq.ctas,
                                                   static_cast<T*>(q.dweight), static_cast<const float*>(hk.partial), hk.ctas,
                                                   static_cast<T*>(k.dweight), p.dim);
        LCE_COUNT_LAUNCH();
        if (cuda_failed(err)) return LCE_ERR_CUDA;
    }
    return LCE_OK;
}

template <int MODE>
int dispatch_heads(const HeadCall& c, const lce_head_rows& q, const lce_head_rows& k, const RopePlan& p, float* partial, cudaStream_t s) {
    switch (c.dtype) {
        case LCE_DTYPE_BF16:
            return c.interleaved ? launch_heads<__nv_bfloat16, true, MODE>(c, q, k, p, partial, s)
                                 : launch_heads<__nv_bfloat16, false, MODE>(c, q, k, p, partial, s);
        case LCE_DTYPE_F16:
            return c.interleaved ? launch_heads<__half, true, MODE>(c, q, k, p, partial, s)
                                 : launch_heads<__half, false, MODE>(c, q, k, p, partial, s);
        default:
            return c.interleaved ? launch_heads<float, true, MODE>(c, q, k, p, partial, s)
                                 : launch_heads<float, false, MODE>(c, q, k, p, partial, s);
    }
}

template <int MODE>
int heads_call(const lce_head_rows* q, const lce_head_rows* k, int64_t batch, int64_t seq, int64_t dim, const void* positions,
               int pos_i64, int64_t pos_b, int64_t pos_s, const double* freq, int64_t half, int interleaved, float scale,
               int inverse, float eps, int dtype, void* ws, size_t ws_bytes, void* stream) {
    if (!known_dtype(dtype) || batch < 0 || seq < 0 || dim < 1 || half < 0 || 2 * half > dim) return LCE_ERR_ARG;
    // a grid's stride over 2^31 units must not wrap 32 bits
    if (dim > kHeadMaxDim || batch > 0x7fffffffll || seq > 0x7fffffffll || batch * seq > 0x70000000ll) return LCE_ERR_TOO_LARGE;
    HeadCall c{batch, seq, dim, half, interleaved, MODE, dtype, 0};
    int rc = check_head_rows(q, c);
    if (rc) return rc;
    if (k && (rc = check_head_rows(k, c))) return rc;
    const lce_head_rows qr = plain_strides(*q, c), kr = k ? plain_strides(*k, c) : lce_head_rows{};
    const bool work = batch > 0 && seq > 0 && (qr.heads > 0 || kr.heads > 0);
    if (!work && !(MODE == kHeadNormBackward && (qr.dweight || kr.dweight))) return LCE_OK;
    if (work && (!positions || (half > 0 && !freq))) return LCE_ERR_ARG;
    if (MODE == kHeadNormBackward && (qr.dweight || kr.dweight) &&
        (!ws || ws_bytes < lce_qk_norm_rope_backward_workspace_bytes(dim)))
        return LCE_ERR_WS_TOO_SMALL;
    DeviceInfo* d;
    if ((rc = device_basics(&d))) return rc;
    c.sm_count = d->sm_count;
    RopePlan p;
    p.pos = positions;
    p.pos_i64 = pos_i64;
    p.pos_b = pos_b;
    p.pos_s = pos_s;
    p.freq = freq;
    p.half = static_cast<int>(half);
    p.dim = static_cast<int>(dim);
    p.items = p.lanes = 1;
    p.pairs2 = 0;
    p.seq = seq > 0 ? seq : 1;
    p.scale = scale;
    p.sin_sign = inverse ? -1.f : 1.f;
    p.eps = eps;
    return dispatch_heads<MODE>(c, qr, kr, p, static_cast<float*>(ws), static_cast<cudaStream_t>(stream));
}

// ---------------------------------------------------------------------------------------------
// sampler
// ---------------------------------------------------------------------------------------------
constexpr long long kSampleSliceBytes = 64 << 10;       // a CTA's share of a row: two CTAs and more fit an SM
constexpr long long kSampleMaxSliceBytes = 160 << 10;   // beyond it a CTA re-reads its share from L2

// bf16 batches that take sample_values_kernel, a CTA per row. top_p 0.95, sample_kernel against it, us, at 128256 logits:
// 24 rows 52 / 72, 48 rows 84 / 72, 148 rows 160 / 74, 256 rows 250 / 94; at 50257: 24 rows 37 / 49, 48 rows 61 / 49; at
// 8003: 148 rows 27 / 32, 256 rows 47 / 35, 16384 rows 1323 / 1186; below that a row's bins cost as much as they save (4000:
// 1055 / 1110). A top_k of 50: 40 rows of 128256 37 / 41, 64 rows 47 / 41, 256 rows 98 / 53, 256 rows of 8003 36 / 25; of
// 5000: 64 rows of 128256 67 / 59, 256 rows 171 / 80. Parameters of each row, of every kind, count as filters: 40 rows of
// 128256 56 / 72, 64 rows 64 / 72, 148 rows 98 / 71, 256 rows 157 / 93. Rows without filters, of which sample_kernel only
// needs the maximum and the weights: 48 rows of 128256 43 / 63, 256 rows 125 / 88, 256 rows of 50257 64 / 53, 1024 rows of
// 8000 57 / 84.
inline bool takes_values(long long rows, long long vocab, bool filtered) {
    return filtered ? rows >= 40 && vocab >= 8000 && rows * vocab >= 2000000 : rows >= 128 && vocab >= 32768;
}

// A CTA per row, for batches of bf16 rows.
int launch_sample_values(const DeviceInfo& d, const __nv_bfloat16* logits, long long ld, long long rows, long long vocab,
                         int groups, const SampleParams& p, cudaStream_t s) {
    auto kern = sample_values_kernel;
    static std::atomic<bool> opted_in[kMaxDevices];
    if (!opted_in[d.index].load(std::memory_order_acquire)) {
        if (cuda_failed(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kValueBytes))) return LCE_ERR_CUDA;
        opted_in[d.index].store(true, std::memory_order_release);
    }
    kern<<<static_cast<unsigned>(rows), kSampleThreads, kValueBytes, s>>>(logits, ld, static_cast<int>(vocab), groups, p);
    LCE_COUNT_LAUNCH();
    return cuda_failed(cudaGetLastError()) ? LCE_ERR_CUDA : LCE_OK;
}

template <class T>
int launch_sample(const DeviceInfo& d, const void* logits, long long ld, long long rows, long long vocab, const SampleParams& p,
                  cudaStream_t s) {
    constexpr int VEC = RmsTile<T>::kVec;
    const long long n_vec = cdiv(vocab + VEC - 1, VEC);
    if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        const long long groups = cdiv(n_vec, static_cast<long long>(kSampleWarps) * kValueChunk);
        const bool filtered = p.top_k || p.top_p || (p.top_k_all > 0 && p.top_k_all < vocab) || p.top_p_all < 1.f;
        if (takes_values(rows, vocab, filtered) && groups * kSampleWarps <= kValueMaxChunks)
            return launch_sample_values(d, static_cast<const T*>(logits), ld, rows, vocab, static_cast<int>(groups), p, s);
    }
    // CTAs per row: enough that a share fits shared memory well and, for few rows, that the GPU is busy - as long as a share
    // is worth the cluster's barriers.
    int ctas = 1;
    while (ctas < kSampleMaxCluster &&
           (cdiv(n_vec, ctas) * 16 > kSampleSliceBytes || (rows * ctas < 2 * d.sm_count && vocab / (2 * ctas) >= 2048)))
        ctas *= 2;
    if (rows * ctas > 0x7fffffffll) return LCE_ERR_TOO_LARGE;
    const int per_warp = static_cast<int>(cdiv(n_vec, static_cast<long long>(ctas) * kSampleWarps));
    const long long slice = static_cast<long long>(per_warp) * kSampleWarps * 16;
    const int in_smem = slice <= kSampleMaxSliceBytes ? 1 : 0;
    auto kern = sample_kernel<T>;
    static std::atomic<bool> opted_in[kMaxDevices];  // setting the attribute twice from two threads is harmless
    if (!opted_in[d.index].load(std::memory_order_acquire)) {
        if (cuda_failed(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                             static_cast<int>(kSampleList * 8 + kSampleMaxSliceBytes))))
            return LCE_ERR_CUDA;
        opted_in[d.index].store(true, std::memory_order_release);
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(rows * ctas));
    cfg.blockDim = dim3(kSampleThreads);
    cfg.dynamicSmemBytes = kSampleList * 8 + (in_smem ? static_cast<size_t>(slice) : 0);
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = ctas;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t err = cudaLaunchKernelEx(&cfg, kern, static_cast<const T*>(logits), ld, static_cast<int>(vocab), ctas, per_warp,
                                               in_smem, p);
    LCE_COUNT_LAUNCH();
    return cuda_failed(err) ? LCE_ERR_CUDA : LCE_OK;
}

}  // namespace
}  // namespace lce

using namespace lce;

extern "C" {

int lce_rope(const lce_head_rows* rows, int64_t batch, int64_t seq, int64_t dim, const void* positions, int pos_i64,
             int64_t pos_b, int64_t pos_s, const double* freq, int64_t half, int interleaved, float scale, int inverse,
             int dtype, void* stream) {
    return heads_call<kHeadRope>(rows, nullptr, batch, seq, dim, positions, pos_i64, pos_b, pos_s, freq, half, interleaved,
                                 scale, inverse, 0.f, dtype, nullptr, 0, stream);
}

int lce_qk_norm_rope_forward(const lce_head_rows* q, const lce_head_rows* k, int64_t batch, int64_t seq, int64_t dim,
                             const void* positions, int pos_i64, int64_t pos_b, int64_t pos_s, const double* freq,
                             int64_t half, int interleaved, float scale, float eps, int dtype, void* stream) {
    if (!k) return LCE_ERR_ARG;
    return heads_call<kHeadNorm>(q, k, batch, seq, dim, positions, pos_i64, pos_b, pos_s, freq, half, interleaved, scale, 0,
                                 eps, dtype, nullptr, 0, stream);
}

size_t lce_qk_norm_rope_backward_workspace_bytes(int64_t dim) {
    if (dim < 1 || dim > kHeadMaxDim) return 0;
    return static_cast<size_t>(kHeadMaxCtas + 1) * dim * sizeof(float);
}

int lce_qk_norm_rope_backward(const lce_head_rows* q, const lce_head_rows* k, int64_t batch, int64_t seq, int64_t dim,
                              const void* positions, int pos_i64, int64_t pos_b, int64_t pos_s, const double* freq,
                              int64_t half, int interleaved, float scale, float eps, int dtype, void* ws, size_t ws_bytes,
                              void* stream) {
    if (!k) return LCE_ERR_ARG;
    return heads_call<kHeadNormBackward>(q, k, batch, seq, dim, positions, pos_i64, pos_b, pos_s, freq, half, interleaved,
                                         scale, 1, eps, dtype, ws, ws_bytes, stream);
}

size_t lce_sample_logits_workspace_bytes(int64_t rows, int64_t vocab, int dtype) {
    (void)rows, (void)vocab, (void)dtype;
    return 0;
}

int lce_sample_logits(const void* logits, int64_t ld, int64_t rows, int64_t vocab, int dtype, const float* uniform,
                      const float* temperature, float temperature_all, const void* top_k, int top_k_is_i64, int64_t top_k_all,
                      const float* top_p, float top_p_all, const float* min_p, float min_p_all, int64_t* token, float* logprob,
                      void* ws, size_t ws_bytes, void* stream) {
    if (!known_dtype(dtype) || rows < 0 || vocab < 1 || ld < vocab) return LCE_ERR_ARG;
    if (vocab > 0x7fffff00ll || rows > 0x7fffff00ll) return LCE_ERR_TOO_LARGE;
    if (rows == 0) return LCE_OK;
    if (!logits || !uniform || !token) return LCE_ERR_ARG;
    if (ws_bytes < lce_sample_logits_workspace_bytes(rows, vocab, dtype)) return LCE_ERR_WS_TOO_SMALL;
    (void)ws;
    DeviceInfo* d;
    const int rc = device_basics(&d);
    if (rc) return rc;
    SampleParams p;
    p.uniform = uniform;
    p.temperature = temperature;
    p.top_k = top_k;
    p.top_p = top_p;
    p.min_p = min_p;
    p.temperature_all = temperature_all;
    p.top_p_all = top_p_all;
    p.min_p_all = min_p_all;
    p.top_k_all = top_k_all;
    p.top_k_i64 = top_k_is_i64;
    p.token = reinterpret_cast<long long*>(token);
    p.logprob = logprob;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    switch (dtype) {
        case LCE_DTYPE_BF16: return launch_sample<__nv_bfloat16>(*d, logits, ld, rows, vocab, p, s);
        case LCE_DTYPE_F16: return launch_sample<__half>(*d, logits, ld, rows, vocab, p, s);
        default: return launch_sample<float>(*d, logits, ld, rows, vocab, p, s);
    }
}

}  // extern "C"
