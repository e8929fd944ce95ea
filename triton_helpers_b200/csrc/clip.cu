// The norm of a list of gradients as if they were one vector, and what is scaled by it.  Streaming kernels: a CTA takes one chunk of one
// tensor, found by a search in the list, which travels as a kernel parameter.
//
//     norm = sqrt(sum_k scale_k^2 sum_i g_k[i]^2)        factor = min(1, max_norm / (norm + 1e-6))
//
// Partial sums are float64 and added in a fixed order by a second kernel of one CTA, so that results repeat, nothing has to be
// cleared before a call, and calls share no state.  The pair (norm, factor) stays on the device: what follows reads it there.
#include "adam.cuh"
#include "chained.cuh"

#include <algorithm>

namespace th {
namespace {

constexpr int kClipThreads = 256;
constexpr int kNormTensors = 512, kUpdateTensors = 256;  // of one launch: some 13 KB of parameters
constexpr long long kLeastChunk = 4096, kMostChunks = 2368;  // elements; 16 chunks for each of 148 SMs

// Elements of a chunk: a multiple of every packet, so that chunks start as their tensor does
long long chunk_elements(long long total) {
    const long long per = (total + kMostChunks - 1) / kMostChunks;
    return std::max(kLeastChunk, (per + 2047) / 2048 * 2048);
}

struct NormList {
    const void *grad[kNormTensors];
    long long n[kNormTensors];
    float scale[kNormTensors];
    int first[kNormTensors];  // the tensor's first chunk within this launch
    unsigned char dtype[kNormTensors];
    int count;
    int chunk;
};

struct UpdateList {
    void *param[kUpdateTensors], *grad[kUpdateTensors];
    float *exp_avg[kUpdateTensors], *exp_avg_sq[kUpdateTensors];
    long long n[kUpdateTensors];
    float scale[kUpdateTensors];
    int first[kUpdateTensors];
    unsigned char zero_grad[kUpdateTensors], packets[kUpdateTensors];  // packets: all four pointers are on 16 bytes
    int count;
    int chunk;
};

// The tensor that a chunk lies in: the last one that starts at or before it
__device__ __forceinline__ int tensor_of(const int *first, int count, int chunk) {
    int low = 0, high = count;
    while (high - low > 1) {
        const int mid = (low + high) >> 1;
        if (first[mid] <= chunk) low = mid;
        else high = mid;
    }
    return low;
}

// The square of an element is exact to float32 only within 2^-63 .. 2^63: a packet whose largest element is outside of 2^-50 .. 2^50 is
// summed in float64 (elements that are 2^13 below the largest lose nothing that its square could show).
template <typename T, int N>
__device__ __forceinline__ double packet_squares(const T (&v)[N]) {
    float sum = 0.f, most = 0.f;
#pragma unroll
    for (int k = 0; k < N; ++k) {
        const float x = to_float<T>(v[k]);
        sum = fmaf(x, x, sum);
        most = fmaxf(most, fabsf(x));
    }
    if constexpr (sizeof(T) != 2 || !std::is_same<T, __half>::value) {
        if (most > 0x1p50f || (most < 0x1p-50f && most > 0.f)) {
            double wide = 0.0;
#pragma unroll
            for (int k = 0; k < N; ++k) {
                const double x = static_cast<double>(to_float<T>(v[k]));
                wide += x * x;
            }
            return wide;
        }
    }
    return static_cast<double>(sum);
}

template <typename T>
__device__ __forceinline__ double chunk_squares(const T *__restrict__ g, int n) {
    constexpr int N = kPacket<T>, kAhead = 2;
    const int off = static_cast<int>(reinterpret_cast<uintptr_t>(g) & 15) / static_cast<int>(sizeof(T));
    const int head = min(n, off ? N - off : 0), packets = (n - head) / N, tail = head + packets * N;
    const Packet16<T> *body = reinterpret_cast<const Packet16<T> *>(g + head);
    double sum = 0.0;
    for (int i = threadIdx.x; i < packets; i += kAhead * kClipThreads) {
        Packet16<T> p[kAhead];
#pragma unroll
        for (int a = 0; a < kAhead; ++a)
            if (i + a * kClipThreads < packets) p[a] = body[i + a * kClipThreads];
#pragma unroll
        for (int a = 0; a < kAhead; ++a)
            if (i + a * kClipThreads < packets) sum += packet_squares<T, N>(p[a].v);
    }
    const int lone = head + (n - tail);  // before the first packet and behind the last one: fewer than 2 N
    for (int i = threadIdx.x; i < lone; i += kClipThreads) {
        const T one[1] = {g[i < head ? i : tail + i - head]};
        sum += packet_squares<T, 1>(one);
    }
    return sum;
}

__device__ __forceinline__ double block_sum(double v, double *warps) {
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(~0u, v, off);
    if ((threadIdx.x & 31) == 0) warps[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0.0;
    for (int w = 0; w < static_cast<int>(blockDim.x) / 32; ++w) v += warps[w];
    return v;
}

// Bound by memory: 100 M bfloat16 gradients 35.7 us (5.6 TB/s), float32 61.1 (6.5).  Two packets a thread ahead and eight CTAs on an SM; with four packets and
// four CTAs 37.9 and 63.9, with eight and three 39.8 and 67.2.
__global__ void __launch_bounds__(kClipThreads, 8) grad_squares_kernel(const __grid_constant__ NormList t, double *__restrict__ partial) {
    __shared__ double warps[kClipThreads / 32];
    after_previous();
    const int k = tensor_of(t.first, t.count, blockIdx.x);
    const long long from = static_cast<long long>(static_cast<int>(blockIdx.x) - t.first[k]) * t.chunk;
    const int n = static_cast<int>(min(static_cast<long long>(t.chunk), t.n[k] - from));
    double sum;
    if (t.dtype[k] == TH_F32) sum = chunk_squares(static_cast<const float *>(t.grad[k]) + from, n);
    else if (t.dtype[k] == TH_F16) sum = chunk_squares(static_cast<const __half *>(t.grad[k]) + from, n);
    else sum = chunk_squares(static_cast<const __nv_bfloat16 *>(t.grad[k]) + from, n);
    sum = block_sum(sum, warps);
    if (threadIdx.x == 0) partial[blockIdx.x] = sum * t.scale[k] * t.scale[k];
}

__global__ void __launch_bounds__(1024) norm_factor_kernel(const double *__restrict__ partial, int count, float max_norm, float *__restrict__ pair) {
    __shared__ double warps[32];
    after_previous();
    double sum = 0.0;
    for (int i = threadIdx.x; i < count; i += 1024) sum += partial[i];
    sum = block_sum(sum, warps);
    if (threadIdx.x == 0) {
        const float norm = static_cast<float>(sqrt(sum)), factor = max_norm / (norm + 1e-6f);
        pair[0] = norm;
        pair[1] = factor >= 1.f ? 1.f : factor;  // a NaN stays one
    }
}

template <typename T>
__device__ __forceinline__ void chunk_scale(T *__restrict__ g, int n, float factor) {
    constexpr int N = kPacket<T>;
    const int off = static_cast<int>(reinterpret_cast<uintptr_t>(g) & 15) / static_cast<int>(sizeof(T));
    const int head = min(n, off ? N - off : 0), packets = (n - head) / N, tail = head + packets * N;
    Packet16<T> *body = reinterpret_cast<Packet16<T> *>(g + head);
#pragma unroll 4
    for (int i = threadIdx.x; i < packets; i += kClipThreads) {
        Packet16<T> p = body[i];
#pragma unroll
        for (int k = 0; k < N; ++k) p.v[k] = from_float<T>(to_float<T>(p.v[k]) * factor);
        body[i] = p;
    }
    for (int i = threadIdx.x; i < head + (n - tail); i += kClipThreads) {
        T &at = g[i < head ? i : tail + i - head];
        at = from_float<T>(to_float<T>(at) * factor);
    }
}

__global__ void __launch_bounds__(kClipThreads) scale_tensors_kernel(const __grid_constant__ NormList t, const float *__restrict__ pair) {
    after_previous();
    const float factor = pair[1];
    if (factor == 1.f) return;
    const int k = tensor_of(t.first, t.count, blockIdx.x);
    const long long from = static_cast<long long>(static_cast<int>(blockIdx.x) - t.first[k]) * t.chunk;
    const int n = static_cast<int>(min(static_cast<long long>(t.chunk), t.n[k] - from));
    void *g = const_cast<void *>(t.grad[k]);
    if (t.dtype[k] == TH_F32) chunk_scale(static_cast<float *>(g) + from, n, factor);
    else if (t.dtype[k] == TH_F16) chunk_scale(static_cast<__half *>(g) + from, n, factor);
    else chunk_scale(static_cast<__nv_bfloat16 *>(g) + from, n, factor);
}

// Adam's update (adam.cuh) with the pair's factor in the gradient's scale.  Bound by memory: 60 M bfloat16 parameters with float32 moments 206 us, 1.26 GB at
// 6.1 TB/s.  The tensors' list lets one launch take 256 of them, a chunk a CTA (th_adam_steps walks 16 with the whole grid).
template <typename T>
__global__ void __launch_bounds__(kClipThreads) adam_clipped_kernel(const __grid_constant__ UpdateList t, AdamScalars a, const float *__restrict__ pair,
                                                                    int *__restrict__ skipped_total) {
    constexpr int N = kPacket<T>;
    after_previous();
    const int k = tensor_of(t.first, t.count, blockIdx.x);
    const long long from = static_cast<long long>(static_cast<int>(blockIdx.x) - t.first[k]) * t.chunk;
    const int n = static_cast<int>(min(static_cast<long long>(t.chunk), t.n[k] - from));
    T *param = static_cast<T *>(t.param[k]) + from, *grad = static_cast<T *>(t.grad[k]) + from;
    float *exp_avg = t.exp_avg[k] + from, *exp_avg_sq = t.exp_avg_sq[k] + from;
    // a norm that is not finite: a NaN for every gradient, which adam_one passes over
    a.grad_scale = isfinite(pair[0]) ? t.scale[k] * pair[1] : __int_as_float(0x7fc00000);
    const bool zero = t.zero_grad[k] != 0;
    int skipped = 0;
    const int packets = t.packets[k] ? n / N : 0;
    for (int i = threadIdx.x; i < packets; i += kClipThreads) {
        Packet16<T> p = reinterpret_cast<Packet16<T> *>(param)[i];
        const Packet16<T> g = reinterpret_cast<const Packet16<T> *>(grad)[i];
        Moments<N> m = reinterpret_cast<Moments<N> *>(exp_avg)[i], v = reinterpret_cast<Moments<N> *>(exp_avg_sq)[i];
#pragma unroll
        for (int e = 0; e < N; ++e) p.v[e] = adam_one<T>(p.v[e], g.v[e], m.v[e], v.v[e], a, skipped);
        reinterpret_cast<Packet16<T> *>(param)[i] = p;
        reinterpret_cast<Moments<N> *>(exp_avg)[i] = m;
        reinterpret_cast<Moments<N> *>(exp_avg_sq)[i] = v;
        if (zero) {
            Packet16<T> z;
#pragma unroll
            for (int e = 0; e < N; ++e) z.v[e] = from_float<T>(0.f);
            reinterpret_cast<Packet16<T> *>(grad)[i] = z;
        }
    }
    for (int i = packets * N + threadIdx.x; i < n; i += kClipThreads) {
        param[i] = adam_one<T>(param[i], grad[i], exp_avg[i], exp_avg_sq[i], a, skipped);
        if (zero) grad[i] = from_float<T>(0.f);
    }
    if (skipped_total && skipped) count_skipped(skipped_total, skipped);
}

long long total_elements(int n_tensors, const int64_t *n_elems) {
    long long total = 0;
    for (int k = 0; k < n_tensors; ++k) total += std::max<long long>(0, n_elems[k]);
    return total;
}

int check_list(const char *what, int n_tensors, const void *const *pointers, const int64_t *n_elems, const int *dtypes) {
    if (n_tensors < 0 || (n_tensors > 0 && (!pointers || !n_elems || !dtypes))) return fail(TH_ERR_BAD_ARG, "%s: bad list of %d tensors", what, n_tensors);
    for (int k = 0; k < n_tensors; ++k) {
        if (dtypes[k] != TH_F32 && dtypes[k] != TH_F16 && dtypes[k] != TH_BF16) return fail(TH_ERR_UNSUPPORTED, "%s: unknown dtype code %d", what, dtypes[k]);
        if (n_elems[k] < 0) return fail(TH_ERR_BAD_ARG, "%s: negative element count", what);
        if (n_elems[k] > 0 && !pointers[k]) return fail(TH_ERR_BAD_ARG, "%s: null tensor pointer", what);
        if (int rc = check_elements(what, dtypes[k], {pointers[k]})) return rc;
    }
    return TH_OK;
}

// Launches fn(list, chunks, chunks before) for the tensors in lists of kNormTensors
template <typename Fn>
int for_lists(int n_tensors, const void *const *pointers, const int64_t *n_elems, const int *dtypes, const float *scales, const Fn &fn) {
    const long long chunk = chunk_elements(total_elements(n_tensors, n_elems));
    if (chunk > (1ll << 30)) return fail(TH_ERR_UNSUPPORTED, "tensors of more than 2^41 elements in all");
    NormList t;
    t.chunk = static_cast<int>(chunk);
    t.count = 0;
    int chunks = 0, before = 0;
    for (int k = 0; k <= n_tensors; ++k) {
        if (t.count == kNormTensors || (k == n_tensors && t.count)) {
            if (int rc = fn(t, chunks, before)) return rc;
            before += chunks;
            t.count = chunks = 0;
        }
        if (k == n_tensors || n_elems[k] == 0) continue;
        t.grad[t.count] = pointers[k];
        t.n[t.count] = n_elems[k];
        t.scale[t.count] = scales ? scales[k] : 1.f;
        t.dtype[t.count] = static_cast<unsigned char>(dtypes[k]);
        t.first[t.count++] = chunks;
        chunks += static_cast<int>((n_elems[k] + chunk - 1) / chunk);
    }
    return TH_OK;
}

}  // namespace
}  // namespace th

using namespace th;

extern "C" int64_t th_grad_norm_workspace_bytes(int n_tensors, const int64_t *n_elems) {
    if (n_tensors < 1 || !n_elems) return 0;
    const long long chunk = chunk_elements(total_elements(n_tensors, n_elems));
    int64_t chunks = 0;
    for (int k = 0; k < n_tensors; ++k) chunks += (std::max<int64_t>(0, n_elems[k]) + chunk - 1) / chunk;
    return 8 * chunks;
}

extern "C" int th_grad_norm(int n_tensors, const void *const *grad_dev, const int64_t *n_elems, const int *dtypes, const float *grad_scale, float max_norm,
                            float *norm_factor_dev, void *workspace_dev, int64_t workspace_bytes, void *stream) {
    if (int rc = check_list("th_grad_norm", n_tensors, grad_dev, n_elems, dtypes)) return rc;
    if (!norm_factor_dev) return fail(TH_ERR_BAD_ARG, "th_grad_norm: null pointer");
    if (int rc = check_elements("th_grad_norm", TH_F32, {norm_factor_dev})) return rc;
    const int64_t wanted = th_grad_norm_workspace_bytes(n_tensors, n_elems);
    if (wanted > 0 && (!workspace_dev || workspace_bytes < wanted || !aligned_to(workspace_dev, 8)))
        return fail(TH_ERR_WORKSPACE, "th_grad_norm: scratch missing, too small or off 8 bytes");
    double *partial = static_cast<double *>(workspace_dev);
    cudaStream_t at = static_cast<cudaStream_t>(stream);
    const int rc = for_lists(n_tensors, grad_dev, n_elems, dtypes, grad_scale, [&](const NormList &t, int chunks, int before) {
        return launch_chained("grad_squares_kernel launch", grad_squares_kernel, chunks, kClipThreads, 0, at, 1, t, partial + before);
    });
    if (rc) return rc;
    return launch_chained("norm_factor_kernel launch", norm_factor_kernel, 1, 1024, 0, at, 1, partial, static_cast<int>(wanted / 8), max_norm, norm_factor_dev);
}

extern "C" int th_scale_tensors(int n_tensors, void *const *tensor_dev, const int64_t *n_elems, const int *dtypes, const float *norm_factor_dev, void *stream) {
    if (int rc = check_list("th_scale_tensors", n_tensors, tensor_dev, n_elems, dtypes)) return rc;
    if (!norm_factor_dev) return fail(TH_ERR_BAD_ARG, "th_scale_tensors: null pointer");
    if (int rc = check_elements("th_scale_tensors", TH_F32, {norm_factor_dev})) return rc;
    cudaStream_t at = static_cast<cudaStream_t>(stream);
    return for_lists(n_tensors, tensor_dev, n_elems, dtypes, nullptr, [&](const NormList &t, int chunks, int) {
        return launch_chained("scale_tensors_kernel launch", scale_tensors_kernel, chunks, kClipThreads, 0, at, 1, t, norm_factor_dev);
    });
}

extern "C" int th_adam_clipped(int n_tensors, void *const *param_dev, void *const *grad_dev, float *const *exp_avg_dev, float *const *exp_avg_sq_dev,
                               const int64_t *n_elems, const float *grad_scale, const int *zero_grad, const float *norm_factor_dev, float lr, float beta1,
                               float beta2, float eps, int step, int dtype, int *skipped_dev, void *stream) {
    if (n_tensors < 0 || (n_tensors > 0 && (!param_dev || !grad_dev || !exp_avg_dev || !exp_avg_sq_dev || !n_elems || !grad_scale || !zero_grad)))
        return fail(TH_ERR_BAD_ARG, "th_adam_clipped: bad list of %d tensors", n_tensors);
    if (step < 1) return fail(TH_ERR_BAD_ARG, "step counts from 1");
    if (dtype != TH_F32 && dtype != TH_F16 && dtype != TH_BF16) return fail(TH_ERR_UNSUPPORTED, "th_adam_clipped: unknown dtype code %d", dtype);
    if (!norm_factor_dev) return fail(TH_ERR_BAD_ARG, "th_adam_clipped: null pointer");
    if (int rc = check_elements("th_adam_clipped", TH_F32, {norm_factor_dev, skipped_dev})) return rc;
    for (int k = 0; k < n_tensors; ++k) {
        if (n_elems[k] < 0) return fail(TH_ERR_BAD_ARG, "th_adam_clipped: negative element count");
        if (n_elems[k] == 0) continue;
        if (!param_dev[k] || !grad_dev[k] || !exp_avg_dev[k] || !exp_avg_sq_dev[k]) return fail(TH_ERR_BAD_ARG, "th_adam_clipped: null tensor pointer");
        if (int rc = check_elements("th_adam_clipped", dtype, {param_dev[k], grad_dev[k]})) return rc;
        if (int rc = check_elements("th_adam_clipped", TH_F32, {exp_avg_dev[k], exp_avg_sq_dev[k]})) return rc;
    }
    const long long chunk = chunk_elements(total_elements(n_tensors, n_elems));
    if (chunk > (1ll << 30)) return fail(TH_ERR_UNSUPPORTED, "tensors of more than 2^41 elements in all");
    AdamScalars a{lr, beta1, beta2, eps, 0.f, 0.f, 1.f, 0};
    a.bias1 = static_cast<float>(1.0 - pow(static_cast<double>(beta1), step));
    a.bias2_sqrt = static_cast<float>(sqrt(1.0 - pow(static_cast<double>(beta2), step)));
    cudaStream_t at = static_cast<cudaStream_t>(stream);
    UpdateList t;
    t.chunk = static_cast<int>(chunk);
    t.count = 0;
    int chunks = 0;
    for (int k = 0; k <= n_tensors; ++k) {
        if (t.count == kUpdateTensors || (k == n_tensors && t.count)) {
            const auto launch = [&](auto kernel) {
                return launch_chained("adam_clipped_kernel launch", kernel, chunks, kClipThreads, 0, at, 1, t, a, norm_factor_dev, skipped_dev);
            };
            const int rc = dtype == TH_F32   ? launch(adam_clipped_kernel<float>)
                           : dtype == TH_F16 ? launch(adam_clipped_kernel<__half>)
                                             : launch(adam_clipped_kernel<__nv_bfloat16>);
            if (rc) return rc;
            t.count = chunks = 0;
        }
        if (k == n_tensors || n_elems[k] == 0) continue;
        t.param[t.count] = param_dev[k];
        t.grad[t.count] = grad_dev[k];
        t.exp_avg[t.count] = exp_avg_dev[k];
        t.exp_avg_sq[t.count] = exp_avg_sq_dev[k];
        t.n[t.count] = n_elems[k];
        t.scale[t.count] = grad_scale[k];
        t.zero_grad[t.count] = zero_grad[k] != 0;
        t.packets[t.count] = aligned_to(param_dev[k], 16) && aligned_to(grad_dev[k], 16) && aligned_to(exp_avg_dev[k], 16) && aligned_to(exp_avg_sq_dev[k], 16);
        t.first[t.count++] = chunks;
        chunks += static_cast<int>((n_elems[k] + chunk - 1) / chunk);
    }
    return TH_OK;
}
