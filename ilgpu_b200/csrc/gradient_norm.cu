// The norm of all gradients, over any number of views of any lengths and types, and clipping by it.
//
//   norm = sqrt(sum over all views and elements of x^2)
//   y    = x * min(1, max_norm / norm)
//
// The views of a launch are listed in its parameters; a block takes a stretch of the chunks that they are cut into.
#include <math.h>
#include <type_traits>

#include "elements.cuh"

namespace b200alg {

constexpr int kNormThreads = 256;
constexpr int kChunk = 8192;       // elements
constexpr int kNormBlocksPerSm = 4;
constexpr int kMaxBlocks = 148 * kNormBlocksPerSm;  // partial sums of a launch
constexpr int kMostViews = 1024;   // of a launch: 30 KB of parameters

struct ViewTable {
    const void *in[kMostViews];
    void *out[kMostViews];
    long long length[kMostViews];
    unsigned int chunk[kMostViews + 1];  // first chunk of a view
    unsigned char in_type[kMostViews], out_type[kMostViews];
    int views;
};
static_assert(sizeof(ViewTable) <= 31 << 10, "fits a kernel's parameters");

// Views from `first` on that one launch takes; returns how many.
static int64_t fill_table(ViewTable &t, const void *const *in, void *const *out, const int64_t *lengths, const int *in_types, const int *out_types,
                          int64_t first, int64_t views) {
    int64_t i = first;
    unsigned int chunks = 0;
    t.views = 0;
    for (; i < views && t.views < kMostViews; ++i) {
        const int64_t need = ceil_div(lengths[i], kChunk);
        if (!need) continue;
        const int v = t.views++;
        t.in[v] = in[i];
        t.out[v] = out ? out[i] : (void *)in[i];
        t.length[v] = lengths[i];
        t.chunk[v] = chunks;
        t.in_type[v] = (unsigned char)in_types[i];
        t.out_type[v] = (unsigned char)(out_types ? out_types[i] : in_types[i]);
        chunks += (unsigned int)need;
    }
    t.chunk[t.views] = chunks;
    return i - first;
}

// The view that chunk c belongs to.
__device__ __forceinline__ int view_of_chunk(const ViewTable &t, unsigned int c) {
    int lo = 0, hi = t.views - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (t.chunk[mid] <= c) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// A block's stretch of the chunks.
__device__ __forceinline__ void stretch(unsigned int chunks, unsigned int &begin, unsigned int &end) {
    begin = (unsigned int)((unsigned long long)chunks * blockIdx.x / gridDim.x);
    end = (unsigned int)((unsigned long long)chunks * (blockIdx.x + 1) / gridDim.x);
}

// Squares of G elements in 32 bits; where they overflow or vanish there, in 64.
template <typename T, int G, int N> __device__ __forceinline__ double squares(const Group<T, G> (&v)[N]) {
    float s = 0.0f;
    unsigned int any = 0u;
#pragma unroll
    for (int u = 0; u < N; ++u) {
#pragma unroll
        for (int k = 0; k < G; ++k) s = fmaf(v[u].get(k), v[u].get(k), s);
        if constexpr (!std::is_same<T, __half>::value) {
#pragma unroll
            for (int k = 0; k < Group<T, G>::kWords; ++k) any |= v[u].w[k];
        }
    }
    if constexpr (!std::is_same<T, __half>::value) {  // (the squares of 16-bit floats of five exponent bits are all normal)
        constexpr unsigned int kMagnitude = sizeof(T) == 4 ? 0x7FFFFFFFu : 0x7FFF7FFFu;
        // Squares below 2^-126 lose bits, each at most 2^-126; N * G of them are nothing beside 2^-80.
        if (!(s >= 0x1p-80f && s <= FLT_MAX) && (any & kMagnitude)) {
            double d = 0.0;
#pragma unroll
            for (int u = 0; u < N; ++u)
#pragma unroll
                for (int k = 0; k < G; ++k) d = fma((double)v[u].get(k), (double)v[u].get(k), d);
            return d;
        }
    }
    return (double)s;
}

// Sum of the squares of a chunk, this thread's part.
template <typename T> __device__ __forceinline__ double chunk_squares(const T *__restrict__ p, int64_t n) {
    constexpr int G = 16 / sizeof(T);
    constexpr int N = kChunk / (kNormThreads * G);
    double sum = 0.0;
    int64_t head = (int64_t)(((16u - (unsigned)((uintptr_t)p & 15u)) & 15u) / sizeof(T));
    if (head > n) head = n;
    const int64_t groups = (n - head) / G;
    Group<T, G> v[N];
#pragma unroll
    for (int u = 0; u < N; ++u) {
        const int64_t g = threadIdx.x + u * kNormThreads;
        if (g < groups) v[u].load(p + head + g * G);
        else v[u].clear();
    }
    sum = squares<T, G, N>(v);
    const int64_t tail = head + groups * G;
    const int64_t at = (int64_t)threadIdx.x < head ? (int64_t)threadIdx.x : tail + threadIdx.x - head;  // fewer than 32 elements
    if (at < n && (int64_t)threadIdx.x < head + n - tail) {
        Group<T, 1> one[1];
        one[0].load(p + at);
        sum += squares<T, 1, 1>(one);
    }
    return sum;
}

// Sum over the block, in its first thread.
__device__ __forceinline__ double block_sum(double v) {
    __shared__ double part[kNormThreads / 32];
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) v += __shfl_down_sync(0xffffffffu, v, d);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    if (threadIdx.x == 0) {
        v = part[0];
        for (int i = 1; i < kNormThreads / 32; ++i) v += part[i];
    }
    __syncthreads();
    return v;
}

__global__ void __launch_bounds__(kNormThreads) norm_partial_kernel(const __grid_constant__ ViewTable t, double *partial) {
    grid_dependency_release();
    grid_dependency_wait();
    unsigned int c, end;
    stretch(t.chunk[t.views], c, end);
    double sum = 0.0;
    if (c < end) {
        int v = view_of_chunk(t, c);
        for (; c < end; ++c) {
            while (c >= t.chunk[v + 1]) ++v;
            const int64_t first = (int64_t)(c - t.chunk[v]) * kChunk;
            const int64_t n = t.length[v] - first < kChunk ? t.length[v] - first : kChunk;
            switch (t.in_type[v]) {
            case B200ALG_F32: sum += chunk_squares((const float *)t.in[v] + first, n); break;
            case B200ALG_F16: sum += chunk_squares((const __half *)t.in[v] + first, n); break;
            case B200ALG_BF16: sum += chunk_squares((const __nv_bfloat16 *)t.in[v] + first, n); break;
            }
        }
    }
    sum = block_sum(sum);
    if (threadIdx.x == 0) partial[blockIdx.x] = sum;
}

// The partial sums are added up in a fixed order.
__global__ void __launch_bounds__(kNormThreads) norm_finish_kernel(const double *partial, int64_t count, float *norm) {
    grid_dependency_release();
    grid_dependency_wait();
    double sum = 0.0;
    for (int64_t i = threadIdx.x; i < count; i += kNormThreads) sum += partial[i];
    sum = block_sum(sum);
    if (threadIdx.x == 0) *norm = (float)sqrt(sum);
}

template <typename TIn, typename TOut>
__device__ __forceinline__ void scale_chunk(const TIn *in, TOut *out, int64_t n, float factor) {
    constexpr int G = 16 / sizeof(TIn);
    // groups where both sides can be moved whole: from the input's first boundary on
    int64_t head = (int64_t)(((16u - (unsigned)((uintptr_t)in & 15u)) & 15u) / sizeof(TIn));
    constexpr unsigned int kBoundary = G * sizeof(TOut) < 16 ? G * sizeof(TOut) : 16;
    if (head > n || (uintptr_t)(out + head) % kBoundary) head = n;
    const int64_t groups = (n - head) / G, tail = head + groups * G;
    for (int64_t g = threadIdx.x; g < groups; g += kNormThreads) {
        Group<TIn, G> v;
        v.load(in + head + g * G);
        float x[G];
#pragma unroll
        for (int k = 0; k < G; ++k) x[k] = v.get(k) * factor;
        Group<TOut, G> y;
        y.set(x);
        y.store(out + head + g * G);
    }
    for (int64_t i = threadIdx.x; i < head; i += kNormThreads) out[i] = from_float<TOut>(to_float(in[i]) * factor);
    for (int64_t i = tail + threadIdx.x; i < n; i += kNormThreads) out[i] = from_float<TOut>(to_float(in[i]) * factor);
}

template <typename TIn>
__device__ __forceinline__ void scale_chunk_to(const TIn *in, void *out, int out_type, int64_t first, int64_t n, float factor) {
    switch (out_type) {
    case B200ALG_F32: scale_chunk(in + first, (float *)out + first, n, factor); break;
    case B200ALG_F16: scale_chunk(in + first, (__half *)out + first, n, factor); break;
    case B200ALG_BF16: scale_chunk(in + first, (__nv_bfloat16 *)out + first, n, factor); break;
    }
}

__global__ void __launch_bounds__(kNormThreads) scale_kernel(const __grid_constant__ ViewTable t, const float *norm, double max_norm) {
    grid_dependency_release();
    grid_dependency_wait();
    const float whole = *norm;
    // a norm that is not finite leaves the values as they are: it says so itself
    const float factor = whole <= FLT_MAX && (double)whole > max_norm ? (float)(max_norm / (double)whole) : 1.0f;
    unsigned int begin, c;
    stretch(t.chunk[t.views], begin, c);
    if (c <= begin) return;
    int v = view_of_chunk(t, c - 1);
    // backwards: what the norm's kernel has read last may still be in the cache
    while (c-- > begin) {
        while (c < t.chunk[v]) --v;
        if (factor == 1.0f && t.in[v] == t.out[v]) continue;
        const int64_t first = (int64_t)(c - t.chunk[v]) * kChunk;
        const int64_t n = t.length[v] - first < kChunk ? t.length[v] - first : kChunk;
        switch (t.in_type[v]) {
        case B200ALG_F32: scale_chunk_to((const float *)t.in[v], t.out[v], t.out_type[v], first, n, factor); break;
        case B200ALG_F16: scale_chunk_to((const __half *)t.in[v], t.out[v], t.out_type[v], first, n, factor); break;
        case B200ALG_BF16: scale_chunk_to((const __nv_bfloat16 *)t.in[v], t.out[v], t.out_type[v], first, n, factor); break;
        }
    }
}

static int blocks_of(const ViewTable &t) {
    const int64_t most = kMaxBlocks < (int64_t)sm_count() * kNormBlocksPerSm ? kMaxBlocks : (int64_t)sm_count() * kNormBlocksPerSm;
    const int64_t chunks = t.chunk[t.views];
    return (int)(chunks < most ? chunks : most);
}

// launch_dependent() without its copies of the parameters.
static cudaError_t launch_with_table(const void *kernel, int blocks, cudaStream_t s, void **arguments) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(blocks);
    cfg.blockDim = dim3(kNormThreads);
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelExC(&cfg, kernel, arguments);
}

static int check_views(const void *const *views, void *const *outputs, const int64_t *lengths, const int *types, const int *out_types, int64_t count) {
    if (count < 0 || (count && (!views || !lengths || !types))) return B200ALG_INVALID_ARGUMENT;
    if (count > INT32_MAX) return B200ALG_TOO_LARGE;
    int64_t elements = 0;
    for (int64_t i = 0; i < count; ++i) {
        const int bytes = element_bytes(types[i]), out_bytes = out_types ? element_bytes(out_types[i]) : bytes;
        if (!bytes || !out_bytes) return B200ALG_UNSUPPORTED;
        if (lengths[i] < 0) return B200ALG_INVALID_ARGUMENT;
        if (lengths[i] > kMaxElements - elements) return B200ALG_TOO_LARGE;  // of all together: 31 bits count their chunks
        elements += lengths[i];
        if (lengths[i] == 0) continue;
        if (!views[i] || (outputs && !outputs[i])) return B200ALG_INVALID_ARGUMENT;
        if ((uintptr_t)views[i] % bytes || (outputs && (uintptr_t)outputs[i] % out_bytes)) return B200ALG_MISALIGNED;
        // in place only with the type that is there
        if ((outputs ? outputs[i] == views[i] : out_types != nullptr) && out_types && out_types[i] != types[i]) return B200ALG_INVALID_ARGUMENT;
    }
    return B200ALG_OK;
}

static int64_t norm_temp_bytes(int64_t count) {
    return sizeof(TempHeader) + round_up((ceil_div(count, kMostViews) + 1) * kMaxBlocks * 8, 256);  // every launch but the last takes kMostViews views
}

static int run_norm(cudaStream_t s, const void *const *views, const int64_t *lengths, const int *types, int64_t count, float *norm, void *temp) {
    double *partial = (double *)((char *)temp + sizeof(TempHeader));
    int64_t sums = 0;
    ViewTable t;
    for (int64_t first = 0; first < count;) {
        first += fill_table(t, views, nullptr, lengths, types, nullptr, first, count);
        if (!t.views) break;
        const int blocks = blocks_of(t);
        double *to = partial + sums;
        void *arguments[] = {&t, &to};
        B200ALG_CUDA_TRY(launch_with_table((const void *)norm_partial_kernel, blocks, s, arguments));
        sums += blocks;
    }
    B200ALG_CUDA_TRY(launch_dependent(norm_finish_kernel, dim3(1), dim3(kNormThreads), 0, s, (const double *)partial, sums, norm));
    return B200ALG_OK;
}

static int run_scale(cudaStream_t s, const void *const *views, void *const *outputs, const int64_t *lengths, const int *types, const int *out_types,
                     int64_t count, const float *norm, double max_norm) {
    ViewTable t;
    for (int64_t first = 0; first < count;) {
        first += fill_table(t, views, outputs, lengths, types, out_types, first, count);
        if (!t.views) break;
        void *arguments[] = {&t, &norm, &max_norm};
        B200ALG_CUDA_TRY(launch_with_table((const void *)scale_kernel, blocks_of(t), s, arguments));
    }
    return B200ALG_OK;
}

}  // namespace b200alg

using namespace b200alg;

extern "C" int b200alg_gradient_norm_temp_bytes(int64_t count, int64_t *out_bytes) {
    if (!out_bytes || count < 0) return B200ALG_INVALID_ARGUMENT;
    if (count > INT32_MAX) return B200ALG_TOO_LARGE;
    *out_bytes = norm_temp_bytes(count);
    return B200ALG_OK;
}

extern "C" int b200alg_gradient_norm(void *stream, const void *const *views, const int64_t *lengths, const int *dtypes, int64_t count, float *norm,
                                     void *temp, int64_t temp_bytes) {
    const int rc = check_views(views, nullptr, lengths, dtypes, nullptr, count);
    if (rc != B200ALG_OK) return rc;
    if (!norm || !temp) return B200ALG_INVALID_ARGUMENT;
    if ((uintptr_t)norm % 4 || (uintptr_t)temp % 256) return B200ALG_MISALIGNED;
    if (temp_bytes < norm_temp_bytes(count)) return B200ALG_TEMP_TOO_SMALL;
    return run_norm((cudaStream_t)stream, views, lengths, dtypes, count, norm, temp);
}

extern "C" int b200alg_gradient_scale(void *stream, const void *const *views, void *const *outputs, const int64_t *lengths, const int *dtypes,
                                      const int *out_dtypes, int64_t count, const float *norm, double max_norm) {
    const int rc = check_views(views, outputs, lengths, dtypes, out_dtypes, count);
    if (rc != B200ALG_OK) return rc;
    if (!norm || !(max_norm >= 0.0)) return B200ALG_INVALID_ARGUMENT;
    if ((uintptr_t)norm % 4) return B200ALG_MISALIGNED;
    return run_scale((cudaStream_t)stream, views, outputs, lengths, dtypes, out_dtypes, count, norm, max_norm);
}

extern "C" int b200alg_gradient_clip(void *stream, const void *const *views, void *const *outputs, const int64_t *lengths, const int *dtypes,
                                     const int *out_dtypes, int64_t count, double max_norm, float *norm, void *temp, int64_t temp_bytes) {
    int rc = check_views(views, outputs, lengths, dtypes, out_dtypes, count);
    if (rc != B200ALG_OK) return rc;
    if (!norm || !temp || !(max_norm >= 0.0)) return B200ALG_INVALID_ARGUMENT;
    if ((uintptr_t)norm % 4 || (uintptr_t)temp % 256) return B200ALG_MISALIGNED;
    if (temp_bytes < norm_temp_bytes(count)) return B200ALG_TEMP_TOO_SMALL;
    rc = run_norm((cudaStream_t)stream, views, lengths, dtypes, count, norm, temp);
    if (rc != B200ALG_OK) return rc;
    return run_scale((cudaStream_t)stream, views, outputs, lengths, dtypes, out_dtypes, count, norm, max_norm);
}
