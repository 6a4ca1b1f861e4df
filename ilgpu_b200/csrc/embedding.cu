// Embedding: rows of a table looked up by token and scaled, and the table's gradient by sorted tokens.
//
//   out[i, :]  = scale * table[token[i], :]
//   grad[v, :] = scale * sum over {i : token[i] = v} of upstream[i, :]
//
// A token outside [0, rows) has no row: zeros are looked up for it and it adds to no gradient.
#include <type_traits>

#include "elements.cuh"

namespace b200alg {

// ---- lookup --------------------------------------------------------------------------------
// Nothing but memory traffic: a thread moves kLookupItems groups, loads ahead of stores.  A group's row and column come
// from one division by the groups of a row, so that rows of any width fill the warps.
constexpr int kLookupThreads = 256, kLookupItems = 4;

template <typename TIn, typename TOut, int G>
__global__ void __launch_bounds__(kLookupThreads)
lookup_kernel(const TIn *__restrict__ table, int64_t rows, int64_t row_stride, IndexView tokens, int64_t first, TOut *__restrict__ out,
              int64_t out_stride, unsigned int total, FastDivide groups, float scale) {
    grid_dependency_release();
    grid_dependency_wait();
    const unsigned int base = blockIdx.x * (kLookupThreads * kLookupItems) + threadIdx.x;
    Group<TIn, G> in[kLookupItems];
    TOut *to[kLookupItems];
#pragma unroll
    for (int u = 0; u < kLookupItems; ++u) {
        const unsigned int q = base + u * kLookupThreads;
        to[u] = nullptr;
        if (q < total) {
            const unsigned int row = groups(q);
            const int64_t column = (int64_t)(q - row * groups.d) * G;
            const int64_t token = tokens[first + row];
            to[u] = out + (first + row) * out_stride + column;
            if (token >= 0 && token < rows) in[u].load(table + token * row_stride + column);
            else in[u].clear();
        }
    }
#pragma unroll
    for (int u = 0; u < kLookupItems; ++u) {
        if (!to[u]) continue;
        float x[G];
#pragma unroll
        for (int k = 0; k < G; ++k) x[k] = in[u].get(k) * scale;
        Group<TOut, G> y;
        y.set(x);
        y.store(to[u]);
    }
}

template <typename TIn, typename TOut, int G>
static int run_lookup(cudaStream_t s, const void *table, int64_t rows, int64_t width, int64_t row_stride, const IndexView &tokens, int64_t n,
                      double scale, void *out, int64_t out_stride) {
    const int64_t groups = width / G;
    const int64_t most = (((int64_t)1 << 31) - kLookupThreads * kLookupItems) / groups;  // rows of a launch, whose groups 31 bits count
    if (most < 1) return B200ALG_TOO_LARGE;
    for (int64_t first = 0; first < n; first += most) {
        const int64_t total = (n - first < most ? n - first : most) * groups;
        B200ALG_CUDA_TRY(launch_dependent(lookup_kernel<TIn, TOut, G>, dim3((unsigned)ceil_div(total, kLookupThreads * kLookupItems)),
                                          dim3(kLookupThreads), 0, s, (const TIn *)table, rows, row_stride, tokens, first, (TOut *)out, out_stride,
                                          (unsigned int)total, FastDivide((unsigned int)groups), (float)scale));
    }
    return B200ALG_OK;
}

// ---- gradient ------------------------------------------------------------------------------
// The tokens are sorted with their positions (the library's stable sort), so that the rows to be added up lie one behind
// the other in the order of their positions; sums do not depend on how the work falls on the GPU.  A tile of sorted
// positions is summed by the threads of a block, each holding one group of columns in registers and walking along the
// tile.  A run of equal tokens inside a tile is written at once; a tile's share of a run that crosses its border goes to
// temp, and gradient_join_kernel adds the shares up in order.  The same launch clears the rows that no token names.
constexpr int kGradientThreads = 256;
constexpr int kAhead = 8;      // rows a thread has in flight
constexpr int kClearRows = 8;  // rows that a warp looks up and clears

struct GradientCall {
    const unsigned int *keys, *positions;  // sorted
    int64_t n, tile, tiles;
    int64_t upstream_stride;
    int64_t rows, width, row_stride;
    float scale;
    int accumulate;
    float *shares;      // [2][tiles][padded width]: of the run that enters a tile, of the run that leaves it
    int64_t share_stride;
    int groups;         // of a row
    int x, y;           // threads of a block along the columns, tiles of a block
    int slabs;          // blocks along the columns
    int64_t sum_blocks;
};

static __global__ void __launch_bounds__(256) gradient_keys_kernel(IndexView tokens, int64_t n, int64_t rows, unsigned int *keys) {
    grid_dependency_release();
    grid_dependency_wait();
    const int64_t step = (int64_t)gridDim.x * blockDim.x;
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += step) {
        const int64_t token = tokens[i];
        keys[i] = token >= 0 && token < rows ? (unsigned int)token : (unsigned int)rows;  // those without a row sort last
    }
}

// First place in keys[0..n) that is not below `key`.
__device__ __forceinline__ int64_t lower_bound(const unsigned int *keys, int64_t n, unsigned int key) {
    int64_t lo = 0, hi = n;
    while (lo < hi) {
        const int64_t mid = (lo + hi) >> 1;
        if (keys[mid] < key) lo = mid + 1;
        else hi = mid;
    }
    return lo;
}

template <typename TOut, int G>
__device__ __forceinline__ void write_row(const GradientCall &c, TOut *out, unsigned int key, int g, const float (&sum)[G]) {
    TOut *p = out + (int64_t)key * c.row_stride + (int64_t)g * G;
    float y[G];
    Group<TOut, G> o;
    if (c.accumulate) {
        o.load(p);
#pragma unroll
        for (int k = 0; k < G; ++k) y[k] = fmaf(sum[k], c.scale, o.get(k));
    } else {
#pragma unroll
        for (int k = 0; k < G; ++k) y[k] = sum[k] * c.scale;
    }
    o.set(y);
    o.store(p);
}
template <int G> __device__ __forceinline__ void write_share(float *p, const float (&sum)[G]) {
    Group<float, G> o;
    o.set(sum);
    o.store(p);
}

template <typename TIn, typename TOut, int G>
__global__ void __launch_bounds__(kGradientThreads) gradient_sum_kernel(GradientCall c, const TIn *__restrict__ upstream, TOut *__restrict__ out) {
    grid_dependency_release();
    grid_dependency_wait();
    const unsigned int rows = (unsigned int)c.rows;
    if (blockIdx.x >= c.sum_blocks) {  // rows that no token names
        const int lane = threadIdx.x & 31;
        const int64_t first = ((blockIdx.x - c.sum_blocks) * (blockDim.x >> 5) + (threadIdx.x >> 5)) * kClearRows;
        bool empty = false;
        if (lane < kClearRows && first + lane < c.rows) {
            const unsigned int row = (unsigned int)(first + lane);
            const int64_t at = lower_bound(c.keys, c.n, row);
            empty = at == c.n || c.keys[at] != row;
        }
        Group<TOut, G> zero;
        zero.clear();
        for (unsigned int todo = __ballot_sync(0xffffffffu, empty); todo; todo &= todo - 1) {
            TOut *p = out + (first + __ffs(todo) - 1) * c.row_stride;
            for (int g = lane; g < c.groups; g += 32) zero.store(p + (int64_t)g * G);
        }
        return;
    }
    const int tx = threadIdx.x % c.x, ty = threadIdx.x / c.x;
    const int64_t t = (int64_t)(blockIdx.x / c.slabs) * c.y + ty;
    const int g = (int)(blockIdx.x % c.slabs) * c.x + tx;
    if (g >= c.groups || t >= c.tiles || ty >= c.y) return;
    const int64_t begin = t * c.tile, end = begin + c.tile < c.n ? begin + c.tile : c.n;
    const unsigned int *keys = c.keys;
    unsigned int current = keys[begin];
    if (current >= rows) return;
    bool entered = begin > 0 && keys[begin - 1] == current;  // whether the current run began in front of the tile
    float sum[G];
#pragma unroll
    for (int k = 0; k < G; ++k) sum[k] = 0.0f;
    float *const enters = c.shares + t * c.share_stride + (int64_t)g * G, *const leaves = enters + c.tiles * c.share_stride;
    for (int64_t i = begin; i < end; i += kAhead) {
        unsigned int key[kAhead];
        Group<TIn, G> in[kAhead];
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            key[j] = i + j < end ? keys[i + j] : rows;
            // (in range unless a wait of the sort ran out, which its status word says)
            const unsigned int position = key[j] < rows ? c.positions[i + j] : 0u;
            if (position >= (unsigned int)c.n) key[j] = rows;
            if (key[j] < rows) in[j].load(upstream + (int64_t)position * c.upstream_stride + (int64_t)g * G);
        }
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            if (key[j] >= rows) continue;
            if (key[j] != current) {
                if (entered) write_share<G>(enters, sum);
                else write_row<TOut, G>(c, out, current, g, sum);
                entered = false;
                current = key[j];
#pragma unroll
                for (int k = 0; k < G; ++k) sum[k] = 0.0f;
            }
#pragma unroll
            for (int k = 0; k < G; ++k) sum[k] += in[j].get(k);
        }
    }
    if (entered) write_share<G>(enters, sum);
    else if (end < c.n && keys[end] == current) write_share<G>(leaves, sum);
    else write_row<TOut, G>(c, out, current, g, sum);
}

// Runs over several tiles: the block of the tile in which a run begins adds its shares up.
template <typename TOut, int G>
__global__ void __launch_bounds__(kGradientThreads) gradient_join_kernel(GradientCall c, TOut *__restrict__ out) {
    grid_dependency_release();
    grid_dependency_wait();
    const int tx = threadIdx.x % c.x, ty = threadIdx.x / c.x;
    const int64_t t = (int64_t)(blockIdx.x / c.slabs) * c.y + ty;
    const int g = (int)(blockIdx.x % c.slabs) * c.x + tx;
    if (g >= c.groups || t >= c.tiles || ty >= c.y) return;
    const int64_t begin = t * c.tile, end = begin + c.tile;
    if (end >= c.n) return;
    const unsigned int key = c.keys[end - 1];
    if (key >= (unsigned int)c.rows || c.keys[end] != key) return;                       // no run leaves the tile
    if (c.keys[begin] == key && begin > 0 && c.keys[begin - 1] == key) return;           // it began in front of it
    const int64_t last = (lower_bound(c.keys + end, c.n - end, key + 1) + end - 1) / c.tile;  // the tile in which it ends
    float sum[G];
    Group<float, G> share;
    const float *enters = c.shares + (int64_t)g * G;
    share.load(enters + (c.tiles + t) * c.share_stride);
#pragma unroll
    for (int k = 0; k < G; ++k) sum[k] = share.get(k);
    for (int64_t i = t + 1; i <= last; ++i) {
        share.load(enters + i * c.share_stride);
#pragma unroll
        for (int k = 0; k < G; ++k) sum[k] += share.get(k);
    }
    write_row<TOut, G>(c, out, key, g, sum);
}

// Sorted positions of a tile: enough tiles for the GPU, and shares of crossing runs that stay a small part of the traffic.
static int64_t gradient_tile(int64_t n) {
    int64_t tile = 128;
    while (tile > 16 && ceil_div(n, tile) < 148) tile /= 2;
    return tile;
}

struct GradientLayout {
    int64_t tile, tiles, share_stride;
    int64_t sort_bytes, off_keys, off_positions, off_shares, total;
};
static int gradient_layout(int64_t rows, int64_t width, int64_t n, GradientLayout &L) {
    if (rows < 0 || width < 0 || n < 0) return B200ALG_INVALID_ARGUMENT;
    if (rows > INT32_MAX || width > INT32_MAX || n > INT32_MAX) return B200ALG_TOO_LARGE;
    L.tile = gradient_tile(n);
    L.tiles = ceil_div(n, L.tile);
    L.share_stride = round_up(width, 8);
    const int rc = b200alg_radix_sort_temp_bytes(B200ALG_U32, n, 4, &L.sort_bytes);  // its part lies first, and with it its status word
    if (rc != B200ALG_OK) return rc;
    L.off_keys = round_up(L.sort_bytes, 256);
    L.off_positions = L.off_keys + round_up(n * 4, 256);
    L.off_shares = L.off_positions + round_up(n * 4, 256);
    L.total = L.off_shares + round_up(2 * L.tiles * L.share_stride * 4, 256);
    return B200ALG_OK;
}

template <typename TIn, typename TOut, int G>
static int run_gradient(cudaStream_t s, GradientCall c, const void *upstream, void *out) {
    c.groups = (int)(c.width / G);
    for (c.x = 32; c.x < kGradientThreads && c.x < c.groups; c.x *= 2) {}
    c.y = kGradientThreads / c.x;
    c.slabs = (int)ceil_div(c.groups, c.x);
    c.sum_blocks = ceil_div(c.tiles, c.y) * c.slabs;
    const int64_t clear_blocks = c.accumulate ? 0 : ceil_div(c.rows, kClearRows * (kGradientThreads / 32));
    if (c.sum_blocks + clear_blocks > INT32_MAX) return B200ALG_TOO_LARGE;
    if (c.sum_blocks + clear_blocks > 0)
        B200ALG_CUDA_TRY(launch_dependent(gradient_sum_kernel<TIn, TOut, G>, dim3((unsigned)(c.sum_blocks + clear_blocks)), dim3(kGradientThreads), 0, s,
                                          c, (const TIn *)upstream, (TOut *)out));
    if (c.tiles > 1)
        B200ALG_CUDA_TRY(launch_dependent(gradient_join_kernel<TOut, G>, dim3((unsigned)c.sum_blocks), dim3(kGradientThreads), 0, s, c, (TOut *)out));
    return B200ALG_OK;
}

}  // namespace b200alg

using namespace b200alg;

extern "C" int b200alg_embedding(void *stream, const void *table, int64_t rows, int64_t width, int64_t row_stride, int dtype, const void *tokens,
                                 int64_t n, int64_t token_stride, int token_dtype, double scale, void *out, int64_t out_stride, int out_dtype) {
    if (rows < 0 || width < 0 || n < 0 || token_stride < 1) return B200ALG_INVALID_ARGUMENT;
    if (!matrix_ok(rows, width, row_stride) || !matrix_ok(n, width, out_stride)) return B200ALG_INVALID_ARGUMENT;
    const int ib = element_bytes(dtype), ob = element_bytes(out_dtype);
    if (!ib || !ob || !index_dtype(token_dtype)) return B200ALG_UNSUPPORTED;
    if (n > INT32_MAX || width > INT32_MAX || rows > INT32_MAX) return B200ALG_TOO_LARGE;
    if (n == 0 || width == 0) return B200ALG_OK;
    if ((!table && rows) || !tokens || !out) return B200ALG_INVALID_ARGUMENT;
    if ((uintptr_t)table % ib || (uintptr_t)out % ob || (uintptr_t)tokens % dtype_bytes(token_dtype)) return B200ALG_MISALIGNED;
    const IndexView view{tokens, token_stride, token_dtype == B200ALG_I64};
    cudaStream_t s = (cudaStream_t)stream;
    auto fits = [&](int group) {
        return groups_aligned(table, row_stride, rows, width, ib, group) && groups_aligned(out, out_stride, n, width, ob, group);
    };
    const int group = fits(8) ? 8 : fits(4) ? 4 : 1;
    return with_element(dtype, [&](auto in) {
        return with_element(out_dtype, [&](auto to) {
            using TIn = decltype(in);
            using TOut = decltype(to);
            if (group == 8) return run_lookup<TIn, TOut, 8>(s, table, rows, width, row_stride, view, n, scale, out, out_stride);
            if (group == 4) return run_lookup<TIn, TOut, 4>(s, table, rows, width, row_stride, view, n, scale, out, out_stride);
            return run_lookup<TIn, TOut, 1>(s, table, rows, width, row_stride, view, n, scale, out, out_stride);
        });
    });
}

extern "C" int b200alg_embedding_gradient_temp_bytes(int64_t rows, int64_t width, int64_t n, int64_t *out_bytes) {
    if (!out_bytes) return B200ALG_INVALID_ARGUMENT;
    GradientLayout L;
    const int rc = gradient_layout(rows, width, n, L);
    if (rc == B200ALG_OK) *out_bytes = L.total;
    return rc;
}

extern "C" int b200alg_embedding_gradient(void *stream, const void *tokens, int64_t n, int64_t token_stride, int token_dtype, const void *upstream,
                                          int64_t upstream_stride, int upstream_dtype, double scale, void *gradient, int64_t rows, int64_t width,
                                          int64_t row_stride, int dtype, int accumulate, void *temp, int64_t temp_bytes) {
    if (rows < 0 || width < 0 || n < 0 || token_stride < 1) return B200ALG_INVALID_ARGUMENT;
    if (!matrix_ok(rows, width, row_stride) || !matrix_ok(n, width, upstream_stride)) return B200ALG_INVALID_ARGUMENT;
    const int ib = element_bytes(upstream_dtype), ob = element_bytes(dtype);
    if (!ib || !ob || !index_dtype(token_dtype)) return B200ALG_UNSUPPORTED;
    GradientLayout L;
    int rc = gradient_layout(rows, width, n, L);
    if (rc != B200ALG_OK) return rc;
    if (rows == 0 || width == 0) return B200ALG_OK;
    if (!gradient || !temp || (n && (!tokens || !upstream))) return B200ALG_INVALID_ARGUMENT;
    if ((uintptr_t)gradient % ob || (uintptr_t)upstream % ib || (uintptr_t)tokens % dtype_bytes(token_dtype) || (uintptr_t)temp % 256)
        return B200ALG_MISALIGNED;
    if (temp_bytes < L.total) return B200ALG_TEMP_TOO_SMALL;
    cudaStream_t s = (cudaStream_t)stream;
    char *t = (char *)temp;
    unsigned int *keys = (unsigned int *)(t + L.off_keys), *positions = (unsigned int *)(t + L.off_positions);
    if (n) {
        const IndexView view{tokens, token_stride, token_dtype == B200ALG_I64};
        const int64_t want = ceil_div(n, 256 * 2), cap = (int64_t)sm_count() * 8;
        B200ALG_CUDA_TRY(launch_dependent(gradient_keys_kernel, dim3((unsigned)(want < cap ? want : cap)), dim3(256), 0, s, view, n, rows, keys));
        rc = b200alg_radix_sort_pairs_sequence(stream, keys, positions, n, B200ALG_U32, B200ALG_U32, B200ALG_SORT_ASCENDING, temp, L.sort_bytes);
        if (rc != B200ALG_OK) return rc;
    }
    GradientCall c{};
    c.keys = keys, c.positions = positions;
    c.n = n, c.tile = L.tile, c.tiles = L.tiles;
    c.upstream_stride = upstream_stride;
    c.rows = rows, c.width = width, c.row_stride = row_stride;
    c.scale = (float)scale, c.accumulate = accumulate != 0;
    c.shares = (float *)(t + L.off_shares), c.share_stride = L.share_stride;
    return with_element(upstream_dtype, [&](auto in) {
        return with_element(dtype, [&](auto to) {
            using TIn = decltype(in);
            using TOut = decltype(to);
            constexpr int G = 16 / sizeof(TIn);
            if (groups_aligned(upstream, upstream_stride, n, width, ib, G) && groups_aligned(gradient, row_stride, rows, width, ob, G))
                return run_gradient<TIn, TOut, G>(s, c, upstream, gradient);
            return run_gradient<TIn, TOut, 1>(s, c, upstream, gradient);
        });
    });
}
