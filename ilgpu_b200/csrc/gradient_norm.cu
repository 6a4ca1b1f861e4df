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
constexpr int kGroupBytes = 16;
constexpr int kAheadGroups = 4;                                          // of a thread in a chunk
constexpr int kChunkGroups = kNormThreads * kAheadGroups;                // 16 KB
constexpr int kNormBlocksPerSm = 4;
constexpr int kMaxBlocks = 148 * kNormBlocksPerSm;  // partial sums of a launch
constexpr int kMostViews = 1024;                    // of a launch: 30 KB of parameters
constexpr int kMostSpan = 8;                        // chunks that a block takes one behind the other

struct ViewTable {
    const void *in[kMostViews];
    void *out[kMostViews];
    long long length[kMostViews];
    unsigned int chunk[kMostViews + 1];  // first chunk of a view
    unsigned char in_type[kMostViews], out_type[kMostViews];
    int views;
    int span;
};
static_assert(sizeof(ViewTable) <= 31 << 10, "fits a kernel's parameters");

// 16-byte groups of a view, from the boundary at or in front of its first element on.
__host__ __device__ __forceinline__ int64_t groups_of(const void *p, int64_t length, int bytes) {
    return ((int64_t)((uintptr_t)p & (kGroupBytes - 1)) + length * bytes + kGroupBytes - 1) / kGroupBytes;
}

// Views from `first` on that one launch takes; returns how many.
static int64_t fill_table(ViewTable &t, const void *const *in, void *const *out, const int64_t *lengths, const int *in_types, const int *out_types,
                          int64_t first, int64_t views) {
    int64_t i = first;
    unsigned int chunks = 0;
    t.views = 0;
    for (; i < views && t.views < kMostViews; ++i) {
        if (!lengths[i]) continue;
        const int v = t.views++;
        t.in[v] = in[i];
        t.out[v] = out ? out[i] : (void *)in[i];
        t.length[v] = lengths[i];
        t.chunk[v] = chunks;
        t.in_type[v] = (unsigned char)in_types[i];
        t.out_type[v] = (unsigned char)(out_types ? out_types[i] : in_types[i]);
        chunks += (unsigned int)ceil_div(groups_of(in[i], lengths[i], element_bytes(in_types[i])), kChunkGroups);
    }
    t.chunk[t.views] = chunks;
    const int64_t each = chunks / ((int64_t)kMaxBlocks * 4);
    t.span = (int)(each < 1 ? 1 : each > kMostSpan ? kMostSpan : each);
    return i - first;
}

// The chunks of a block: spans of a few one behind the other, taken in turn by all blocks, so that all of them read the
// same part of memory at a time (a stretch of its own for each block: 5.4 TB/s instead of XX).  LAST_FIRST: from the end on.
template <bool LAST_FIRST> struct Chunks {
    const ViewTable &t;
    unsigned int span, chunk, left;  // left: chunks of the span behind this one
    int view;
    __device__ __forceinline__ Chunks(const ViewTable &table) : t(table), span(blockIdx.x) {}
    __device__ __forceinline__ unsigned int spans() const { return (t.chunk[t.views] + t.span - 1) / t.span; }
    __device__ __forceinline__ bool enter() {
        if (span >= spans()) return false;
        const unsigned int at = LAST_FIRST ? spans() - 1 - span : span, begin = at * t.span, behind = begin + t.span;
        const unsigned int end = behind < t.chunk[t.views] ? behind : t.chunk[t.views];
        left = end - begin - 1;
        chunk = LAST_FIRST ? end - 1 : begin;
        int lo = 0, hi = t.views - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (t.chunk[mid] <= chunk) lo = mid;
            else hi = mid - 1;
        }
        view = lo;
        return true;
    }
    __device__ __forceinline__ bool next() {
        if (!left) {
            span += gridDim.x;
            return enter();
        }
        --left;
        if (LAST_FIRST) {
            --chunk;
            while (chunk < t.chunk[view]) --view;
        } else {
            ++chunk;
            while (chunk >= t.chunk[view + 1]) ++view;
        }
        return true;
    }
};

// A thread's part of a chunk: kAheadGroups groups, zero where the view has none.
struct Part {
    uint4 w[kAheadGroups];
    int type, view;
    int64_t group;  // of the view, the thread's first
};

template <typename T> __device__ __forceinline__ uint4 edge_group(const T *in, int64_t first, int64_t length) {
    Group<T, kGroupBytes / (int)sizeof(T)> g;
    g.clear();
#pragma unroll
    for (int k = 0; k < kGroupBytes / (int)sizeof(T); ++k) {
        if (first + k < 0 || first + k >= length) continue;
        if constexpr (sizeof(T) == 4) g.w[k] = reinterpret_cast<const unsigned int *>(in)[first + k];
        else g.w[k / 2] |= (unsigned int)reinterpret_cast<const unsigned short *>(in)[first + k] << (k % 2 * 16);
    }
    return make_uint4(g.w[0], g.w[1], g.w[2], g.w[3]);
}

// Loads this thread's part of the chunk; LAST: the data is not needed again.
template <typename Where> __device__ __forceinline__ void load_part(Part &part, const ViewTable &t, const Where &at) {
    const int v = at.view;
    part.view = v;
    part.type = t.in_type[v];
    const int shift = part.type == B200ALG_F32 ? 2 : 1;  // of an element's size
    const int before = (int)((uintptr_t)t.in[v] & (kGroupBytes - 1));  // bytes of the first group in front of the view
    const char *base = (const char *)t.in[v] - before;
    const int64_t bytes = (t.length[v] << shift) + before;
    part.group = (int64_t)(at.chunk - t.chunk[v]) * kChunkGroups + threadIdx.x;
    const int64_t whole = bytes / kGroupBytes;  // groups in front of this one are full, but for the first where `before`
#pragma unroll
    for (int u = 0; u < kAheadGroups; ++u) {
        const int64_t g = part.group + u * kNormThreads;
        if (g < whole && (g || !before)) {
            part.w[u] = __ldcs(reinterpret_cast<const uint4 *>(base) + g);
        } else if (g * kGroupBytes < bytes) {
            const int64_t first = (g * kGroupBytes - before) >> shift;
            part.w[u] = shift == 2 ? edge_group((const float *)t.in[v], first, t.length[v]) : edge_group((const __half *)t.in[v], first, t.length[v]);
        } else {
            part.w[u] = make_uint4(0u, 0u, 0u, 0u);
        }
    }
}

// Squares of a part in 32 bits; where they overflow or vanish there, in 64.
template <typename T> __device__ __forceinline__ double squares(const Part &part) {
    constexpr int G = kGroupBytes / (int)sizeof(T);
    float s = 0.0f;
    unsigned int any = 0u;
    auto group = [&](int u) {
        Group<T, G> g;
        g.w[0] = part.w[u].x, g.w[1] = part.w[u].y, g.w[2] = part.w[u].z, g.w[3] = part.w[u].w;
        return g;
    };
#pragma unroll
    for (int u = 0; u < kAheadGroups; ++u) {
        const Group<T, G> g = group(u);
        float sum = 0.0f;
#pragma unroll
        for (int k = 0; k < G; ++k) sum = fmaf(g.get(k), g.get(k), sum);
        s += sum;
        any |= g.w[0] | g.w[1] | g.w[2] | g.w[3];
    }
    if constexpr (!std::is_same<T, __half>::value) {  // (the squares of 16-bit floats of five exponent bits are all normal)
        constexpr unsigned int kMagnitude = sizeof(T) == 4 ? 0x7FFFFFFFu : 0x7FFF7FFFu;
        // Squares below 2^-126 lose bits, each at most 2^-126; 32 of them are nothing beside 2^-80.
        if (!(s >= 0x1p-80f && s <= FLT_MAX) && (any & kMagnitude)) {
            double d = 0.0;
#pragma unroll
            for (int u = 0; u < kAheadGroups; ++u) {
                const Group<T, G> g = group(u);
#pragma unroll
                for (int k = 0; k < G; ++k) d = ::fma((double)g.get(k), (double)g.get(k), d);
            }
            return d;
        }
    }
    return (double)s;
}

// Sum over the block, in every thread.
__device__ __forceinline__ double block_sum(double v) {
    __shared__ double part[kNormThreads / 32];
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    v = part[0];
#pragma unroll
    for (int i = 1; i < kNormThreads / 32; ++i) v += part[i];
    return v;
}

// The norm from the sums of all blocks, added up in a fixed order.
__device__ __forceinline__ float norm_of(const double *partial, int count) {
    double sum = 0.0;
    for (int i = threadIdx.x; i < count; i += kNormThreads) sum += partial[i];
    return (float)sqrt(block_sum(sum));
}

__global__ void __launch_bounds__(kNormThreads) norm_partial_kernel(const __grid_constant__ ViewTable t, double *partial) {
    grid_dependency_release();
    Chunks<false> at(t);
    bool more = at.enter();
    grid_dependency_wait();
    double sum = 0.0;
    Part next;
    if (more) load_part(next, t, at);
    while (more) {  // the next chunk is under way while this one is added up
        const Part part = next;
        more = at.next();
        if (more) load_part(next, t, at);
        switch (part.type) {
        case B200ALG_F32: sum += squares<float>(part); break;
        case B200ALG_F16: sum += squares<__half>(part); break;
        default: sum += squares<__nv_bfloat16>(part);
        }
    }
    sum = block_sum(sum);
    if (threadIdx.x == 0) partial[blockIdx.x] = sum;
}

__global__ void __launch_bounds__(kNormThreads) norm_finish_kernel(const double *partial, int count, float *norm) {
    grid_dependency_release();
    grid_dependency_wait();
    const float whole = norm_of(partial, count);
    if (threadIdx.x == 0) *norm = whole;
}

template <typename TIn, typename TOut> __device__ __forceinline__ void scale_part(const Part &part, const ViewTable &t, float factor) {
    constexpr int G = kGroupBytes / (int)sizeof(TIn);
    constexpr unsigned int kBoundary = G * sizeof(TOut) < 16 ? G * sizeof(TOut) : 16;
    const int64_t length = t.length[part.view];
    const int before = (int)((uintptr_t)t.in[part.view] & (kGroupBytes - 1)) / (int)sizeof(TIn);
#pragma unroll
    for (int u = 0; u < kAheadGroups; ++u) {
        const int64_t first = (part.group + u * kNormThreads) * G - before;  // the group's first element
        if (first >= length) continue;
        TOut *to = (TOut *)t.out[part.view] + first;
        Group<TIn, G> g;
        g.w[0] = part.w[u].x, g.w[1] = part.w[u].y, g.w[2] = part.w[u].z, g.w[3] = part.w[u].w;
        float x[G];
#pragma unroll
        for (int k = 0; k < G; ++k) x[k] = g.get(k) * factor;
        if (first >= 0 && first + G <= length && (uintptr_t)to % kBoundary == 0) {
            Group<TOut, G> y;
            y.set(x);
            y.store(to);
        } else {
#pragma unroll
            for (int k = 0; k < G; ++k)
                if (first + k >= 0 && first + k < length) to[k] = from_float<TOut>(x[k]);
        }
    }
}

template <typename TIn> __device__ __forceinline__ void scale_part_from(const Part &part, const ViewTable &t, float factor) {
    switch (t.out_type[part.view]) {
    case B200ALG_F32: scale_part<TIn, float>(part, t, factor); break;
    case B200ALG_F16: scale_part<TIn, __half>(part, t, factor); break;
    default: scale_part<TIn, __nv_bfloat16>(part, t, factor);
    }
}

// partial == NULL: by the norm that is there; else the norm comes from the blocks' sums, and the first block stores it.
// (Every block adds them up itself, so that no launch stands between the two passes.)
__global__ void __launch_bounds__(kNormThreads) scale_kernel(const __grid_constant__ ViewTable t, const double *partial, int count, float *norm, double max_norm) {
    grid_dependency_release();
    Chunks<true> at(t);  // backwards: what the norm's pass has read last may still be in the cache
    bool more = at.enter();
    grid_dependency_wait();
    Part next;
    if (more) load_part(next, t, at);
    float whole;
    if (partial) {
        whole = norm_of(partial, count);
        if (blockIdx.x == 0 && threadIdx.x == 0) *norm = whole;
    } else {
        whole = *norm;
    }
    // a norm that is not finite leaves the values as they are: it says so itself
    const float factor = whole <= FLT_MAX && (double)whole > max_norm ? (float)(max_norm / (double)whole) : 1.0f;
    while (more) {
        const Part part = next;
        more = at.next();
        if (more) load_part(next, t, at);
        if (factor == 1.0f && t.in[part.view] == t.out[part.view]) continue;
        switch (part.type) {
        case B200ALG_F32: scale_part_from<float>(part, t, factor); break;
        case B200ALG_F16: scale_part_from<__half>(part, t, factor); break;
        default: scale_part_from<__nv_bfloat16>(part, t, factor);
        }
    }
}

static int blocks_of(const ViewTable &t) {
    const int64_t most = kMaxBlocks < (int64_t)sm_count() * kNormBlocksPerSm ? kMaxBlocks : (int64_t)sm_count() * kNormBlocksPerSm;
    const int64_t spans = ceil_div(t.chunk[t.views], t.span);
    return (int)(spans < most ? spans : most);
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

// The sums of squares of all launches' blocks; *sums: how many there are.
static int run_partial(cudaStream_t s, const void *const *views, const int64_t *lengths, const int *types, int64_t count, void *temp, int *sums) {
    double *partial = (double *)((char *)temp + sizeof(TempHeader));
    *sums = 0;
    ViewTable t;
    for (int64_t first = 0; first < count;) {
        first += fill_table(t, views, nullptr, lengths, types, nullptr, first, count);
        if (!t.views) break;
        const int blocks = blocks_of(t);
        double *to = partial + *sums;
        void *arguments[] = {&t, &to};
        B200ALG_CUDA_TRY(launch_with_table((const void *)norm_partial_kernel, blocks, s, arguments));
        *sums += blocks;
    }
    return B200ALG_OK;
}

static int run_finish(cudaStream_t s, int sums, float *norm, void *temp) {
    B200ALG_CUDA_TRY(launch_dependent(norm_finish_kernel, dim3(1), dim3(kNormThreads), 0, s, (const double *)((char *)temp + sizeof(TempHeader)), sums, norm));
    return B200ALG_OK;
}

// By the norm that is there (partial == NULL), or by that of `sums` partial sums, which the first launch stores.
static int run_scale(cudaStream_t s, const void *const *views, void *const *outputs, const int64_t *lengths, const int *types, const int *out_types,
                     int64_t count, const double *partial, int sums, float *norm, double max_norm) {
    ViewTable t;
    for (int64_t first = 0; first < count;) {
        first += fill_table(t, views, outputs, lengths, types, out_types, first, count);
        if (!t.views) break;
        void *arguments[] = {&t, &partial, &sums, &norm, &max_norm};
        B200ALG_CUDA_TRY(launch_with_table((const void *)scale_kernel, blocks_of(t), s, arguments));
        partial = nullptr;  // the norm is there now
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
    int sums = 0;
    const int status = run_partial((cudaStream_t)stream, views, lengths, dtypes, count, temp, &sums);
    return status != B200ALG_OK ? status : run_finish((cudaStream_t)stream, sums, norm, temp);
}

extern "C" int b200alg_gradient_scale(void *stream, const void *const *views, void *const *outputs, const int64_t *lengths, const int *dtypes,
                                      const int *out_dtypes, int64_t count, const float *norm, double max_norm) {
    const int rc = check_views(views, outputs, lengths, dtypes, out_dtypes, count);
    if (rc != B200ALG_OK) return rc;
    if (!norm || !(max_norm >= 0.0)) return B200ALG_INVALID_ARGUMENT;
    if ((uintptr_t)norm % 4) return B200ALG_MISALIGNED;
    return run_scale((cudaStream_t)stream, views, outputs, lengths, dtypes, out_dtypes, count, nullptr, 0, (float *)norm, max_norm);
}

extern "C" int b200alg_gradient_clip(void *stream, const void *const *views, void *const *outputs, const int64_t *lengths, const int *dtypes,
                                     const int *out_dtypes, int64_t count, double max_norm, float *norm, void *temp, int64_t temp_bytes) {
    int rc = check_views(views, outputs, lengths, dtypes, out_dtypes, count);
    if (rc != B200ALG_OK) return rc;
    if (!norm || !temp || !(max_norm >= 0.0)) return B200ALG_INVALID_ARGUMENT;
    if ((uintptr_t)norm % 4 || (uintptr_t)temp % 256) return B200ALG_MISALIGNED;
    if (temp_bytes < norm_temp_bytes(count)) return B200ALG_TEMP_TOO_SMALL;
    int sums = 0;
    rc = run_partial((cudaStream_t)stream, views, lengths, dtypes, count, temp, &sums);
    if (rc != B200ALG_OK) return rc;
    if (!sums) return run_finish((cudaStream_t)stream, sums, norm, temp);  // nothing to clip
    return run_scale((cudaStream_t)stream, views, outputs, lengths, dtypes, out_dtypes, count, (const double *)((char *)temp + sizeof(TempHeader)), sums,
                     norm, max_norm);
}
