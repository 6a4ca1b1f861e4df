// The norm of all gradients, over any number of views of any lengths and types, and clipping by it.
//
//   norm = sqrt(sum over all views and elements of x^2)
//   y    = x * min(1, max_norm / norm)
//
// The views of a launch are listed in its parameters, which costs no upload; all blocks take chunks of them in turn.  Memory
// is the bound: the norm of 10^9 floats takes 604 us (6.6 TB/s); clipping 60 million bf16 in 219 views takes 62.0, for which
// they are read twice (120 MB do not stay on the chip) and written once.
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

// of a launch with a shorter list, whose parameters (2 and 7 KB) cost the host less time: 1 us a launch with 64 views
constexpr int kFewViews = 64, kSomeViews = 256;

template <int MOST> struct ViewTable {
    const void *in[MOST];
    void *out[MOST];
    long long length[MOST];
    unsigned int chunk[MOST + 1];  // first chunk of a view
    unsigned char in_type[MOST], out_type[MOST];
    int views;
    int span;
    int in_place;  // whether all of them are
};
static_assert(sizeof(ViewTable<kMostViews>) <= 31 << 10, "fits a kernel's parameters");

// 16-byte groups of a view, from the boundary at or in front of its first element on.
__host__ __device__ __forceinline__ int64_t groups_of(const void *p, int64_t length, int bytes) {
    return ((int64_t)((uintptr_t)p & (kGroupBytes - 1)) + length * bytes + kGroupBytes - 1) / kGroupBytes;
}

// Views from `first` on that one launch takes; returns how many.
template <int MOST>
static int64_t fill_table(ViewTable<MOST> &t, const void *const *in, void *const *out, const int64_t *lengths, const int *in_types, const int *out_types,
                          int64_t first, int64_t views) {
    int64_t i = first;
    unsigned int chunks = 0;
    t.views = 0;
    t.in_place = 1;
    for (; i < views && t.views < MOST; ++i) {
        if (!lengths[i]) continue;
        const int v = t.views++;
        t.in[v] = in[i];
        t.out[v] = out ? out[i] : (void *)in[i];
        if (t.out[v] != t.in[v]) t.in_place = 0;
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

// The chunks of a block: spans of a few one behind the other, taken in turn by all blocks, so that all of
// them read the same part of memory at a time (with a stretch of its own for each block 10^9 floats took 743 us instead of
// 605).  LAST_FIRST: the same ones from the end on.
template <bool LAST_FIRST, typename Table> struct Chunks {
    const Table &t;
    unsigned int chunk, left;  // left: chunks of the span that are still to come
    int view;
    int64_t span, step, spans;
    __device__ __forceinline__ Chunks(const Table &table) : t(table) {
        spans = (t.chunk[t.views] + t.span - 1) / t.span;
        span = blockIdx.x;
        step = gridDim.x;
        if (LAST_FIRST) {
            span = span < spans ? span + (spans - 1 - span) / step * step : -1;
            step = -step;
        }
    }
    __device__ __forceinline__ bool enter() {
        if (span < 0 || span >= spans) return false;
        const unsigned int begin = (unsigned int)span * t.span, behind = begin + t.span;
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
            span += step;
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

// Loads this thread's part of the chunk; KEEP: the data is wanted again.
template <bool KEEP, typename Table, typename Where>
__device__ __forceinline__ void load_part(Part &part, const Table &t, const Where &at) {
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
            part.w[u] = KEEP ? reinterpret_cast<const uint4 *>(base)[g] : __ldcs(reinterpret_cast<const uint4 *>(base) + g);
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

// The squares of the block's chunks, this thread's part of them.
template <bool KEEP, typename Table> __device__ __forceinline__ double sum_squares(const Table &t) {
    Chunks<false, Table> at(t);
    bool more = at.enter();
    grid_dependency_wait();
    double sum = 0.0;
    Part next;
    if (more) load_part<KEEP>(next, t, at);
    while (more) {  // the next chunk is under way while this one is added up
        const Part part = next;
        more = at.next();
        if (more) load_part<KEEP>(next, t, at);
        switch (part.type) {
        case B200ALG_F32: sum += squares<float>(part); break;
        case B200ALG_F16: sum += squares<__half>(part); break;
        default: sum += squares<__nv_bfloat16>(part);
        }
    }
    return sum;
}

template <int MOST, bool KEEP> __global__ void __launch_bounds__(kNormThreads) norm_partial_kernel(const __grid_constant__ ViewTable<MOST> t, double *partial) {
    grid_dependency_release();
    const double sum = block_sum(sum_squares<KEEP>(t));
    if (threadIdx.x == 0) partial[blockIdx.x] = sum;
}

// The norm, and the status word of the temp that the partial sums lie in: no wait of these kernels can run out.
__device__ __forceinline__ void store_norm(float *norm, float whole, double *partial) {
    *norm = whole;
    (reinterpret_cast<TempHeader *>(partial) - 1)->wait_limit_hit = 0u;
}

__global__ void __launch_bounds__(kNormThreads) norm_finish_kernel(double *partial, int count, float *norm) {
    grid_dependency_release();
    grid_dependency_wait();
    const float whole = norm_of(partial, count);
    if (threadIdx.x == 0) store_norm(norm, whole, partial);
}

// What the values are multiplied by, one behind the other.  A norm that is not finite leaves them as they are: it says so
// itself.
struct Factor {
    float first, second;  // the second is 1 unless the factor as a whole is below float's normal numbers and would lose bits
    __device__ __forceinline__ Factor(float norm, double max_norm) {
        const double whole = norm <= FLT_MAX && (double)norm > max_norm ? max_norm / (double)norm : 1.0;
        second = whole < (double)FLT_MIN ? FLT_MIN : 1.0f;
        first = (float)(whole / (double)second);
    }
    __device__ __forceinline__ bool none() const { return first == 1.0f && second == 1.0f; }
};

template <typename TIn, typename TOut, typename Table> __device__ __forceinline__ void scale_part(const Part &part, const Table &t, const Factor &factor) {
    constexpr int G = kGroupBytes / (int)sizeof(TIn);
    constexpr unsigned int kBoundary = G * sizeof(TOut);
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
        for (int k = 0; k < G; ++k) x[k] = g.get(k) * factor.first;
        if (factor.second != 1.0f) {
#pragma unroll
            for (int k = 0; k < G; ++k) x[k] *= factor.second;
        }
        if (first >= 0 && first + G <= length && (uintptr_t)to % kBoundary == 0) {
            Group<TOut, G> y;
            y.set(x);
            y.store_streaming(to);
        } else {
#pragma unroll
            for (int k = 0; k < G; ++k)
                if (first + k >= 0 && first + k < length) to[k] = from_float<TOut>(x[k]);
        }
    }
}

template <typename TIn, typename Table> __device__ __forceinline__ void scale_part_from(const Part &part, const Table &t, const Factor &factor) {
    switch (t.out_type[part.view]) {
    case B200ALG_F32: scale_part<TIn, float>(part, t, factor); break;
    case B200ALG_F16: scale_part<TIn, __half>(part, t, factor); break;
    default: scale_part<TIn, __nv_bfloat16>(part, t, factor);
    }
}

// Backwards, and each block what it has read for the norm: what was read last may still be in the cache.
// partial == NULL: by the norm that is there; else the norm comes from the blocks' sums, and the first block stores it.
// (Every block adds them up itself, so that no launch stands between the two passes.)
template <int MOST>
__global__ void __launch_bounds__(kNormThreads) scale_kernel(const __grid_constant__ ViewTable<MOST> t, double *partial, int count, float *norm, double max_norm) {
    grid_dependency_release();
    Chunks<true, ViewTable<MOST>> at(t);
    bool more = at.enter();
    grid_dependency_wait();
    Part next;
    if (more) load_part<false>(next, t, at);  // (one chunk in vain where nothing is to be done)
    float whole;
    if (partial) {
        whole = norm_of(partial, count);
        if (blockIdx.x == 0 && threadIdx.x == 0) store_norm(norm, whole, partial);
    } else {
        whole = *norm;
    }
    const Factor factor(whole, max_norm);
    if (factor.none() && t.in_place) return;
    auto changes = [&](int view) { return !factor.none() || t.in[view] != t.out[view]; };  // else it is neither read nor written
    while (more) {
        const Part part = next;
        more = at.next();
        if (more && changes(at.view)) load_part<false>(next, t, at);
        else next.view = at.view;
        if (!changes(part.view)) continue;
        switch (part.type) {
        case B200ALG_F32: scale_part_from<float>(part, t, factor); break;
        case B200ALG_F16: scale_part_from<__half>(part, t, factor); break;
        default: scale_part_from<__nv_bfloat16>(part, t, factor);
        }
    }
}

template <int MOST> static int blocks_of(const ViewTable<MOST> &t) {
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

// A call's lists.
struct ViewLists {
    const void *const *in;
    void *const *out;
    const int64_t *lengths;
    const int *in_types, *out_types;
    int64_t count;
};

// The sums of squares of all launches' blocks; *sums: how many there are.
template <int MOST> static int run_partial(cudaStream_t s, const ViewLists &l, bool keep, double *partial, int *sums) {
    *sums = 0;
    ViewTable<MOST> t;
    for (int64_t first = 0; first < l.count;) {
        first += fill_table(t, l.in, nullptr, l.lengths, l.in_types, nullptr, first, l.count);
        if (!t.views) break;
        const int blocks = blocks_of(t);
        double *to = partial + *sums;
        void *arguments[] = {&t, &to};
        B200ALG_CUDA_TRY(launch_with_table(keep ? (const void *)norm_partial_kernel<MOST, true> : (const void *)norm_partial_kernel<MOST, false>, blocks, s, arguments));
        *sums += blocks;
    }
    return B200ALG_OK;
}

// By the norm that is there (partial == NULL), or by that of `sums` partial sums, which the first launch stores.
template <int MOST> static int run_scale(cudaStream_t s, const ViewLists &l, double *partial, int sums, float *norm, double max_norm) {
    ViewTable<MOST> t;
    for (int64_t first = 0; first < l.count;) {
        first += fill_table(t, l.in, l.out, l.lengths, l.in_types, l.out_types, first, l.count);
        if (!t.views) break;
        void *arguments[] = {&t, &partial, &sums, &norm, &max_norm};
        B200ALG_CUDA_TRY(launch_with_table((const void *)scale_kernel<MOST>, blocks_of(t), s, arguments));
        partial = nullptr;  // the norm is there now
    }
    return B200ALG_OK;
}

// The norm, and with max_norm >= 0 the clipping by it.
template <int MOST> static int run_clip(cudaStream_t s, const ViewLists &l, float *norm, double max_norm, void *temp) {
    double *const partial = (double *)((char *)temp + sizeof(TempHeader));
    int sums = 0;
    if (l.count <= MOST) {  // one table for both passes
        ViewTable<MOST> t;
        fill_table(t, l.in, l.out, l.lengths, l.in_types, l.out_types, 0, l.count);
        if (t.views) {
            sums = blocks_of(t);
            double *to = partial;
            void *arguments[] = {&t, &to};
            B200ALG_CUDA_TRY(launch_with_table(max_norm >= 0.0 ? (const void *)norm_partial_kernel<MOST, true> : (const void *)norm_partial_kernel<MOST, false>,
                                               sums, s, arguments));
            if (max_norm >= 0.0) {
                void *scale_arguments[] = {&t, &to, &sums, &norm, &max_norm};
                B200ALG_CUDA_TRY(launch_with_table((const void *)scale_kernel<MOST>, sums, s, scale_arguments));
                return B200ALG_OK;
            }
        }
    } else {
        int rc = run_partial<MOST>(s, l, max_norm >= 0.0, partial, &sums);
        if (rc == B200ALG_OK && max_norm >= 0.0 && sums) rc = run_scale<MOST>(s, l, partial, sums, norm, max_norm);
        if (rc != B200ALG_OK || (max_norm >= 0.0 && sums)) return rc;
    }
    B200ALG_CUDA_TRY(launch_dependent(norm_finish_kernel, dim3(1), dim3(kNormThreads), 0, s, partial, sums, norm));
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
    const ViewLists l{views, nullptr, lengths, dtypes, nullptr, count};
    if (count <= kFewViews) return run_clip<kFewViews>((cudaStream_t)stream, l, norm, -1.0, temp);
    if (count <= kSomeViews) return run_clip<kSomeViews>((cudaStream_t)stream, l, norm, -1.0, temp);
    return run_clip<kMostViews>((cudaStream_t)stream, l, norm, -1.0, temp);
}

extern "C" int b200alg_gradient_scale(void *stream, const void *const *views, void *const *outputs, const int64_t *lengths, const int *dtypes,
                                      const int *out_dtypes, int64_t count, const float *norm, double max_norm) {
    const int rc = check_views(views, outputs, lengths, dtypes, out_dtypes, count);
    if (rc != B200ALG_OK) return rc;
    if (!norm || !(max_norm >= 0.0)) return B200ALG_INVALID_ARGUMENT;
    if ((uintptr_t)norm % 4) return B200ALG_MISALIGNED;
    const ViewLists l{views, outputs, lengths, dtypes, out_dtypes, count};
    if (count <= kFewViews) return run_scale<kFewViews>((cudaStream_t)stream, l, nullptr, 0, (float *)norm, max_norm);
    if (count <= kSomeViews) return run_scale<kSomeViews>((cudaStream_t)stream, l, nullptr, 0, (float *)norm, max_norm);
    return run_scale<kMostViews>((cudaStream_t)stream, l, nullptr, 0, (float *)norm, max_norm);
}

extern "C" int b200alg_gradient_clip(void *stream, const void *const *views, void *const *outputs, const int64_t *lengths, const int *dtypes,
                                     const int *out_dtypes, int64_t count, double max_norm, float *norm, void *temp, int64_t temp_bytes) {
    const int rc = check_views(views, outputs, lengths, dtypes, out_dtypes, count);
    if (rc != B200ALG_OK) return rc;
    if (!norm || !temp || !(max_norm >= 0.0)) return B200ALG_INVALID_ARGUMENT;
    if ((uintptr_t)norm % 4 || (uintptr_t)temp % 256) return B200ALG_MISALIGNED;
    if (temp_bytes < norm_temp_bytes(count)) return B200ALG_TEMP_TOO_SMALL;
    const ViewLists l{views, outputs, lengths, dtypes, out_dtypes, count};
    if (count <= kFewViews) return run_clip<kFewViews>((cudaStream_t)stream, l, norm, max_norm, temp);
    if (count <= kSomeViews) return run_clip<kSomeViews>((cudaStream_t)stream, l, norm, max_norm, temp);
    return run_clip<kMostViews>((cudaStream_t)stream, l, norm, max_norm, temp);
}
