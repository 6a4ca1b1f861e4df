// Embedding: rows of a table looked up by token and scaled, and the table's gradient by sorted tokens.
//
//   out[i, :]  = scale * table[token[i], :]
//   grad[v, :] = scale * sum over {i : token[i] = v} of upstream[i, :]
//
// A token outside [0, rows) has no row: zeros are looked up for it and it adds to no gradient.
#include <type_traits>

#include "elements.cuh"

namespace b200alg {

// Where rows do not lie on boundaries that groups can be moved from and to whole, groups of four or eight columns begin on the
// boundaries of the OUTPUT row (the first and the last one of a row stick out of it), and are put together from the two
// aligned words of the input that hold them.  SHIFTED below.  (One element at a time: 60001 rows of 1357
// bf16 184 us instead of 59.)
constexpr int kMostShifted = 8;
template <typename TIn, typename TOut> constexpr int shifted_group() { return sizeof(TIn) == 2 && sizeof(TOut) == 2 ? 8 : 4; }

// Extent of a matrix that is read: a word that overlaps it may be loaded whole (an aligned word lies in one page).
struct Extent {
    const char *begin, *end;
};
inline Extent extent_of(const void *p, int64_t rows, int64_t width, int64_t row_stride, int bytes) {
    return Extent{(const char *)p, (const char *)p + (rows ? (rows - 1) * row_stride + width : 0) * bytes};
}

template <typename T, int G, bool SHIFTED> struct Columns {  // G columns of a row, as they are loaded
    Group<T, G> w;
    __device__ __forceinline__ void load(const T *p, const Extent &) { w.load(p); }
    __device__ __forceinline__ void clear() { w.clear(); }
    __device__ __forceinline__ Group<T, G> get() const { return w; }
};
template <typename T, int G> struct Columns<T, G, true> {
    static_assert(G == 4 || (G == 8 && sizeof(T) == 2), "two words of 8 or 16 bytes, of which half the elements are chosen");
    Group<T, G> w, behind;
    int shift;  // elements of w in front of the first column
    __device__ __forceinline__ void load(const T *p, const Extent &matrix) {
        constexpr int kBytes = Group<T, G>::kBytes;
        const char *word = (const char *)((uintptr_t)p & ~(uintptr_t)(kBytes - 1));
        shift = (int)(((const char *)p - word) / (int)sizeof(T));
        if (word + kBytes > matrix.begin && word < matrix.end) w.load((const T *)word);
        else w.clear();
        if (shift && word + kBytes < matrix.end) behind.load((const T *)(word + kBytes));
        else behind.clear();
    }
    __device__ __forceinline__ void clear() {
        w.clear();
        behind.clear();
        shift = 0;
    }
    __device__ __forceinline__ Group<T, G> get() const {
        constexpr int W = Group<T, G>::kWords, PER = 4 / (int)sizeof(T);  // elements of a word
        unsigned int t[2 * W];
#pragma unroll
        for (int i = 0; i < W; ++i) t[i] = w.w[i], t[W + i] = behind.w[i];
        const int words = shift / PER;  // by whole words, then by half a word
#pragma unroll
        for (int by = W / 2; by > 0; by >>= 1)
#pragma unroll
            for (int i = 0; i + by < 2 * W; ++i) t[i] = words & by ? t[i + by] : t[i];
        Group<T, G> r;
#pragma unroll
        for (int i = 0; i < W; ++i) r.w[i] = sizeof(T) == 4 ? t[i] : __funnelshift_r(t[i], t[i + 1], shift % PER * 16);
        return r;
    }
};

// First column of a group of the output row.
template <bool SHIFTED, int G, typename T> __device__ __forceinline__ int64_t column_of(const T *row, int64_t g) {
    return SHIFTED ? g * G - (int64_t)((uintptr_t)row / sizeof(T) % G) : g * G;
}
// Writes y to the columns from `column` on that the row has.
template <bool SHIFTED, typename T, int G> __device__ __forceinline__ void put_columns(T *row, int64_t column, int64_t width, const float (&y)[G]) {
    if (!SHIFTED || (column >= 0 && column + G <= width)) {
        Group<T, G> o;
        o.set(y);
        o.store(row + column);
    } else {
#pragma unroll
        for (int k = 0; k < G; ++k)
            if (column + k >= 0 && column + k < width) row[column + k] = from_float<T>(y[k]);
    }
}
// Groups of a row.
inline int64_t groups_in(int64_t width, int group, bool shifted) { return shifted ? (width + 2 * group - 2) / group : width / group; }

// ---- lookup --------------------------------------------------------------------------------
// Nothing but memory traffic: a thread moves kLookupItems groups of up to 32 bytes, loads ahead of stores.  A group's row
// and column come from one division by the groups of a row, so that rows of any width fill the warps.  (65536 rows of
// 4096 bf16 out of 128000: groups of 16 bytes 127 us, of 32 bytes 114.6, four of those 116.)
constexpr int kLookupThreads = 256, kLookupItems = 2;

struct LookupCall {
    int64_t rows, width, row_stride, out_stride;
    Extent extent;      // of the table
    IndexView tokens;
    int64_t first;      // row of the output
    unsigned int total; // groups
    FastDivide groups;  // of a row
    float scale;        // (of a double, rounded once)
};

template <typename TIn, typename TOut, int G, bool SHIFTED>
__global__ void __launch_bounds__(kLookupThreads) lookup_kernel(const LookupCall c, const TIn *__restrict__ table, TOut *__restrict__ out) {
    grid_dependency_release();
    grid_dependency_wait();
    const FastDivide groups = c.groups;
    const unsigned int base = blockIdx.x * (kLookupThreads * kLookupItems) + threadIdx.x;
    Columns<TIn, G, SHIFTED> in[kLookupItems];
    TOut *to[kLookupItems];
    int64_t column[kLookupItems];
    float scale[kLookupItems];
#pragma unroll
    for (int u = 0; u < kLookupItems; ++u) {
        const unsigned int q = base + u * kLookupThreads;
        to[u] = nullptr;
        if (q < c.total) {
            const unsigned int row = groups(q);
            const int64_t token = c.tokens[c.first + row];
            to[u] = out + (c.first + row) * c.out_stride;
            column[u] = column_of<SHIFTED, G>(to[u], q - row * groups.d);
            const bool there = token >= 0 && token < c.rows;
            if (there) in[u].load(table + token * c.row_stride + column[u], c.extent);
            else in[u].clear();
            scale[u] = there ? c.scale : 1.0f;  // (zeros whatever the scale)
        }
    }
#pragma unroll
    for (int u = 0; u < kLookupItems; ++u) {
        if (!to[u]) continue;
        const Group<TIn, G> g = in[u].get();
        float x[G];
#pragma unroll
        for (int k = 0; k < G; ++k) x[k] = g.get(k) * scale[u];
        put_columns<SHIFTED>(to[u], column[u], c.width, x);
    }
}

template <typename TIn, typename TOut, int G, bool SHIFTED>
static int run_lookup(cudaStream_t s, const void *table, int64_t rows, int64_t width, int64_t row_stride, const IndexView &tokens, int64_t n,
                      double scale, void *out, int64_t out_stride) {
    const int64_t groups = groups_in(width, G, SHIFTED);
    const int64_t most = (((int64_t)1 << 31) - kLookupThreads * kLookupItems) / groups;  // rows of a launch, whose groups 31 bits count
    if (most < 1) return B200ALG_TOO_LARGE;
    for (int64_t first = 0; first < n; first += most) {
        const int64_t total = (n - first < most ? n - first : most) * groups;
        const LookupCall c{rows, width, row_stride, out_stride, extent_of(table, rows, width, row_stride, sizeof(TIn)), tokens, first, (unsigned int)total,
                           FastDivide((unsigned int)groups), (float)scale};
        B200ALG_CUDA_TRY(launch_dependent(lookup_kernel<TIn, TOut, G, SHIFTED>, dim3((unsigned)ceil_div(total, kLookupThreads * kLookupItems)),
                                          dim3(kLookupThreads), 0, s, c, (const TIn *)table, (TOut *)out));
    }
    return B200ALG_OK;
}

// ---- gradient ------------------------------------------------------------------------------
// The tokens are sorted with their positions (the library's stable sort), so that the rows to be added up lie one behind
// the other in the order of their positions; sums do not depend on how the work falls on the GPU.  A tile of sorted
// positions is summed by the threads of a block, each holding one group of columns in registers and walking along the
// tile.  A run of equal tokens inside a tile is written at once; a tile's share of a run that crosses its border goes to
// temp, and gradient_join_kernel adds the shares up in order.  Rows that no token names, which are most of a large
// table, are known from a byte each and cleared by other blocks of the last launch, beside the join, which waits more than it
// moves.  (Beside the sums the join stands alone at the end: 75.8 us instead of 70.3 for 16384 tokens.  The sort, too, is
// independent of the clearing, but a launch that passes it by without a wait is not promised to find the bytes written.)
// Memory is the bound: 131072 rows of 4096 bf16 into 128000 rows of float take 506 us, 3.1 GB at 6.2 TB/s; 16384 of 2048
// into 32000 take 70, some 15 of them for keys and sort in front of 330 MB.
constexpr int kGradientThreads = 256;
constexpr int kAhead = 8;      // rows, or shares, that a thread has in flight

struct GradientCall {
    const unsigned int *keys, *positions;  // sorted
    const unsigned char *named;            // a byte per row of the table: whether a token names it
    int64_t n, tile, tiles;
    int64_t upstream_stride;
    Extent extent;      // of upstream
    int64_t rows, width, row_stride;
    float scale;
    int accumulate;
    float *shares;      // [2][tiles][padded width]: of the run that enters a tile, of the run that leaves it
    int64_t share_stride;
    int groups;         // of a row
    int x, y;           // threads of a block along the columns, tiles of a block
    int slabs;          // blocks along the columns
    int64_t sum_blocks;
    int clear_rows;     // rows of a block that clears
    int flat;           // whether it clears them as one stretch: short rows one behind the other
    FastDivide by_width;
    int64_t clear_blocks, join_blocks;
};

__global__ void __launch_bounds__(256) gradient_forget_kernel(uint4 *named, int64_t words) {
    grid_dependency_release();
    grid_dependency_wait();
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < words; i += (int64_t)gridDim.x * 256) named[i] = make_uint4(0u, 0u, 0u, 0u);
}

// (Bytes, for plain stores to them may meet: with a bit per row and atomics 131072 tokens, 8 % of them the same, took
// 11 us.)
__global__ void __launch_bounds__(256) gradient_keys_kernel(IndexView tokens, int64_t n, int64_t rows, unsigned int *keys, unsigned char *named) {
    grid_dependency_release();
    grid_dependency_wait();
    const int64_t step = (int64_t)gridDim.x * blockDim.x;
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += step) {
        const int64_t token = tokens[i];
        const bool there = token >= 0 && token < rows;
        keys[i] = there ? (unsigned int)token : (unsigned int)rows;  // those without a row sort last
        if (named && there) named[token] = 1;
    }
}

// The scaled sum to group g of a row of the table's gradient.
template <bool SHIFTED, typename TOut, int G>
__device__ __forceinline__ void write_row(const GradientCall &c, TOut *out, unsigned int key, int g, const float (&sum)[G]) {
    TOut *row = out + (int64_t)key * c.row_stride;
    const int64_t column = column_of<SHIFTED, G>(row, g);
    float y[G];
    if (!c.accumulate) {
#pragma unroll
        for (int k = 0; k < G; ++k) y[k] = sum[k] * c.scale;
    } else if (!SHIFTED || (column >= 0 && column + G <= c.width)) {
        Group<TOut, G> o;
        o.load(row + column);
#pragma unroll
        for (int k = 0; k < G; ++k) y[k] = fmaf(sum[k], c.scale, o.get(k));
    } else {
#pragma unroll
        for (int k = 0; k < G; ++k) y[k] = column + k >= 0 && column + k < c.width ? fmaf(sum[k], c.scale, to_float(row[column + k])) : 0.0f;
    }
    put_columns<SHIFTED>(row, column, c.width, y);
}
template <int G> __device__ __forceinline__ void write_share(float *p, const float (&sum)[G]) {
    Group<float, G> o;
    o.set(sum);
    o.store(p);
}

// Clears a row, by `threads` threads of which this is one.
template <bool SHIFTED, int G, typename TOut> __device__ __forceinline__ void clear_row(const GradientCall &c, TOut *out, int64_t at, int thread, int threads) {
    float zero[G];
#pragma unroll
    for (int k = 0; k < G; ++k) zero[k] = 0.0f;
    TOut *row = out + at * c.row_stride;
    for (int g = thread; g < c.groups; g += threads) put_columns<SHIFTED>(row, column_of<SHIFTED, G>(row, g), c.width, zero);
}

// Clears those of the `rows` rows from `first` on, one behind the other in memory, that are not named, word by word of 16
// bytes whatever the rows' width; by a block.  (822 tokens into 60092 rows of 115 bf16: 10.6 us, row by row 22.7.)
template <typename TOut, typename Named> __device__ __forceinline__ void clear_flat(const GradientCall &c, TOut *out, int64_t first, int rows, Named named) {
    constexpr int W = 16 / (int)sizeof(TOut);
    TOut *const base = out + first * c.width;
    const int count = rows * (int)c.width, before = (int)((uintptr_t)base / sizeof(TOut) % W), words = (count + before + W - 1) / W;
    for (int w = threadIdx.x; w < words; w += kGradientThreads) {
        const int begin = w * W - before, from = begin < 0 ? 0 : begin, to = begin + W < count ? begin + W : count;
        const int row = (int)c.by_width(from), last = (int)c.by_width(to - 1);
        if (to - from == W && last - row <= 1 && !named(row) && !named(last)) {
            *reinterpret_cast<uint4 *>(base + begin) = make_uint4(0u, 0u, 0u, 0u);
        } else {
            for (int e = from; e < to; ++e)
                if (!named((int)c.by_width(e))) base[e] = from_float<TOut>(0.0f);
        }
    }
}

template <typename TIn, typename TOut, int G, bool SHIFTED>
__global__ void __launch_bounds__(kGradientThreads) gradient_sum_kernel(GradientCall c, const TIn *__restrict__ upstream, TOut *__restrict__ out) {
    grid_dependency_release();
    grid_dependency_wait();
    const unsigned int rows = (unsigned int)c.rows, block = blockIdx.x;
    const int tx = threadIdx.x % c.x, ty = threadIdx.x / c.x;
    const int64_t t = (int64_t)(block / c.slabs) * c.y + ty;
    const int g = (int)(block % c.slabs) * c.x + tx;
    // the keys and positions of the block's tiles, and the keys in front of each tile and behind it
    extern __shared__ unsigned int smem[];
    const int tile = (int)c.tile;
    unsigned int *const key = smem + ty * (2 * tile + 3) + 1, *const position = key + tile + 1;
    int &length = reinterpret_cast<int &>(position[tile]);  // positions of the tile that have a row
    const int64_t begin = t * tile;
    const int most = t >= c.tiles ? 0 : (int)(c.n - begin < tile ? c.n - begin : tile);
    if (tx == 0) length = most;
    __syncthreads();
    for (int i = tx - 1; i <= most && most; i += c.x) {
        const unsigned int k = begin + i >= 0 && begin + i < c.n ? c.keys[begin + i] : rows;
        key[i] = k;
        if (i < 0 || i >= most) continue;
        if (k >= rows) atomicMin(&length, i);
        // (in range unless a wait of the sort ran out, which its status word says)
        const unsigned int at = c.positions[begin + i];
        position[i] = at < (unsigned int)c.n ? at : 0u;
    }
    __syncthreads();
    const int len = length;
    if (g >= c.groups || !len) return;
    auto fetch = [&](Columns<TIn, G, SHIFTED> &to, int i) {  // what the i-th position of the tile has in the columns of its row
        to.load(upstream + (int64_t)position[i] * c.upstream_stride + column_of<SHIFTED, G>(out + (int64_t)key[i] * c.row_stride, g), c.extent);
    };
    Columns<TIn, G, SHIFTED> in[kAhead];  // a row is replaced by the one kAhead behind it as soon as it has been added
#pragma unroll
    for (int j = 0; j < kAhead; ++j)
        if (j < len) fetch(in[j], j);
    unsigned int current = key[0];
    bool entered = key[-1] == current;  // whether the current run began in front of the tile
    float sum[G];
#pragma unroll
    for (int k = 0; k < G; ++k) sum[k] = 0.0f;
    float *const enters = c.shares + t * c.share_stride + (int64_t)g * G, *const leaves = enters + c.tiles * c.share_stride;
    for (int i = 0; i < len; i += kAhead) {
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            if (i + j >= len) break;
            const unsigned int next = key[i + j];
            if (next != current) {
                if (entered) write_share<G>(enters, sum);
                else write_row<SHIFTED>(c, out, current, g, sum);
                entered = false;
                current = next;
#pragma unroll
                for (int k = 0; k < G; ++k) sum[k] = 0.0f;
            }
            const Group<TIn, G> x = in[j].get();
#pragma unroll
            for (int k = 0; k < G; ++k) sum[k] += x.get(k);
            if (i + j + kAhead < len) fetch(in[j], i + j + kAhead);
        }
    }
    if (entered) write_share<G>(enters, sum);
    else if (len == tile && key[tile] == current) write_share<G>(leaves, sum);
    else write_row<SHIFTED>(c, out, current, g, sum);
}

// Runs over several tiles: where one begins, its shares are added up.  A block is made of parts, each wide enough for its
// columns.  They take a tile each; a run of many shares is added up by all of them, and their sums are joined in order.
constexpr int kPartThreads = 64, kLeastPart = 8;  // threads of a part
constexpr int kParts = kGradientThreads / kPartThreads, kMostParts = kGradientThreads / kLeastPart;
static int part_threads(int groups) {
    int x = kLeastPart;
    while (x < kPartThreads && x < groups) x *= 2;
    return x;
}

// Adds the sums of the parts, of x threads each, up, in those of the first one.
template <int G> __device__ __forceinline__ void join_parts(float (&sum)[G], float *part, int x) {
    __syncthreads();
#pragma unroll
    for (int k = 0; k < G; ++k) part[k * kGradientThreads + threadIdx.x] = sum[k];
    __syncthreads();
    if (threadIdx.x >= x) return;
    for (int p = x; p < kGradientThreads; p += x)
#pragma unroll
        for (int k = 0; k < G; ++k) sum[k] += part[k * kGradientThreads + p + threadIdx.x];
}

// Adds the shares of the tiles [from, to) up: of the tile `start` what leaves it, of the others what enters them.
template <int G>
__device__ __forceinline__ void add_shares(float (&sum)[G], const GradientCall &c, int64_t start, int64_t from, int64_t to, int g) {
    const float *enters = c.shares + (int64_t)g * G;
    for (int64_t i = from; i < to; i += kAhead) {
        Group<float, G> share[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int64_t t = i + u < to ? i + u : to - 1;  // (one load behind the other, without a branch between them)
            share[u].load(enters + (t == start ? c.tiles + start : t) * c.share_stride);
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
#pragma unroll
            for (int k = 0; k < G; ++k) sum[k] += i + u < to ? share[u].get(k) : 0.0f;
    }
}

// Clears those of a block's rows that no token names.
template <bool SHIFTED, int G, typename TOut> __device__ __forceinline__ void clear_unnamed(const GradientCall &c, TOut *out, int64_t block) {
    const int64_t first = block * c.clear_rows, behind = first + c.clear_rows < c.rows ? first + c.clear_rows : c.rows;
    if (c.flat) {
        clear_flat(c, out, first, (int)(behind - first), [&](int row) { return c.named[first + row] != 0; });
        return;
    }
    const int lane = threadIdx.x & 31, each = c.clear_rows / (kGradientThreads / 32);  // rows of a warp
    const int64_t begin = first + (threadIdx.x >> 5) * each, end = begin + each < behind ? begin + each : behind;
    for (int64_t some = begin; some < end; some += 32)
        for (unsigned int rows = __ballot_sync(0xffffffffu, some + lane < end && !c.named[some + lane]); rows; rows &= rows - 1)
            clear_row<SHIFTED, G>(c, out, some + __ffs(rows) - 1, lane, 32);
}

template <typename TOut, int G, bool SHIFTED>
__global__ void __launch_bounds__(kGradientThreads) gradient_join_kernel(GradientCall c, TOut *__restrict__ out, int x) {
    __shared__ float part[kGradientThreads * G];
    __shared__ int64_t ends[kMostParts];  // of the runs that all parts add up: the tile behind the last
    __shared__ unsigned int keys[kMostParts];
    grid_dependency_release();
    grid_dependency_wait();
    if (blockIdx.x >= c.join_blocks) {
        clear_unnamed<SHIFTED, G>(c, out, blockIdx.x - c.join_blocks);
        return;
    }
    const int tx = threadIdx.x & (x - 1), ty = threadIdx.x / x, parts = kGradientThreads / x, lane = threadIdx.x & 31;
    const int slabs = (c.groups + x - 1) / x, g = (int)(blockIdx.x % slabs) * x + tx;
    const int64_t first = (int64_t)(blockIdx.x / slabs) * parts;
    {
        const int64_t t = first + ty, begin = t * c.tile, end = begin + c.tile;
        const bool there = end < c.n;
        const unsigned int key = there ? c.keys[end - 1] : (unsigned int)c.rows, next = there ? c.keys[end] : 0u;
        const unsigned int first_key = there ? c.keys[begin] : 0u, before = there && begin ? c.keys[begin - 1] : ~0u;
        // whether a run begins in the tile and leaves it
        const bool starts = there && key < (unsigned int)c.rows && next == key && (first_key != key || before != key);
        // The first tile that does not begin with the run's key.  The lanes of a part ask at equal steps, which grow until
        // one is past it and shrink again from there.
        int64_t behind = t + 1, step = 1;
        const int asked = x < 32 ? x : 32, own = lane & (asked - 1);
        for (bool open = starts; __any_sync(0xffffffffu, open);) {
            const int64_t at = (behind + (own + 1) * step) * c.tile;
            const unsigned int ended = __ballot_sync(0xffffffffu, open && (at >= c.n || c.keys[at] != key)) >> (lane - own) & (~0u >> (32 - asked));
            if (!open) continue;
            if (!ended) {
                behind += asked * step;
                step *= asked;
            } else {
                behind += (__ffs(ended) - 1) * step;
                open = step > 1;
                if (open) step /= asked;
                else ++behind;
            }
        }
        const bool few = behind - t <= kAhead;
        if (starts && few && g < c.groups) {
            float sum[G];
#pragma unroll
            for (int k = 0; k < G; ++k) sum[k] = 0.0f;
            add_shares<G>(sum, c, t, t, behind, g);
            write_row<SHIFTED>(c, out, key, g, sum);
        }
        if (tx == 0) {
            ends[ty] = starts && !few ? behind : -1;
            keys[ty] = key;
        }
    }
    __syncthreads();
    for (int j = 0; j < parts; ++j) {  // (all threads of the block alike)
        const int64_t t = first + j, count = ends[j] - t;
        if (ends[j] < 0) continue;
        float sum[G];
#pragma unroll
        for (int k = 0; k < G; ++k) sum[k] = 0.0f;
        if (g < c.groups) add_shares<G>(sum, c, t, t + count * ty / parts, t + count * (ty + 1) / parts, g);
        join_parts<G>(sum, part, x);
        if (ty == 0 && g < c.groups) write_row<SHIFTED>(c, out, keys[j], g, sum);
    }
}

// ---- gradient of few tokens, in one launch ----
// A block of a position looks all tokens over: if its token stands in front of it, another block has its row; else it
// lists the positions that name the row and adds them up, in y parts that are joined in order.  What clears does so with
// the bits of its own rows, from all tokens as well.  us, this way / by a sort, into 500 rows and into 32000:
//   257 tokens of   64 floats   4.8 / 14.0    6.1 / 15.2        1024 tokens of   64 floats  10.2 / 14.9   11.0 / 17.0
//   512 tokens of 4096 bf16    15.4 / 15.9   78.0 / 86.0         640 tokens of 4096 bf16    19.3 / 16.8   79.1 / 86.5
//   512 tokens of 1357 bf16    13.1 / 16.4   40.2 / 42.5         640 tokens of 1357 bf16    16.7 / 16.8   44.4 / 42.8
constexpr int64_t kFewTokens = 512, kMostFewTokens = 1024;  // the latter where a row is one part of a block

template <typename TIn, typename TOut, int G, bool SHIFTED>
__global__ void __launch_bounds__(kGradientThreads)
gradient_few_kernel(GradientCall c, IndexView tokens, const TIn *__restrict__ upstream, TOut *__restrict__ out, TempHeader *hdr) {
    grid_dependency_release();
    __shared__ unsigned int bits[kMostFewTokens / 32];
    __shared__ unsigned short list[kMostFewTokens];
    __shared__ float part[kGradientThreads * G];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, n = (int)c.n;
    // blocks that clear evenly between those that sum
    const unsigned int block = (unsigned int)((unsigned long long)blockIdx.x * c.sum_blocks / gridDim.x);
    if (block == (unsigned int)((blockIdx.x + 1ull) * c.sum_blocks / gridDim.x)) {
        const int64_t first = (int64_t)(blockIdx.x - block) * c.clear_rows;  // clear_rows: 32 for each warp at most
        if (threadIdx.x < kGradientThreads / 32) bits[threadIdx.x] = 0u;
        __syncthreads();
        grid_dependency_wait();
        if (blockIdx.x == gridDim.x - 1 && threadIdx.x == 0) hdr->wait_limit_hit = 0u;  // no wait can run out
        for (int i = threadIdx.x; i < n; i += kGradientThreads) {
            const int64_t token = tokens[i];
            if (token >= first && token < first + c.clear_rows) atomicOr(bits + ((token - first) >> 5), 1u << ((token - first) & 31));
        }
        __syncthreads();
        if (c.flat) {
            clear_flat(c, out, first, (int)(first + c.clear_rows < c.rows ? c.clear_rows : c.rows - first),
                       [&](int row) { return (bits[row >> 5] >> (row & 31) & 1) != 0; });
            return;
        }
        const bool one_by_one = c.clear_rows < kGradientThreads / 32;  // long rows: all threads take one at a time
        for (int i = one_by_one ? 0 : warp; i < c.clear_rows; i += one_by_one ? 1 : kGradientThreads / 32)
            if (first + i < c.rows && !(bits[i >> 5] >> (i & 31) & 1))
                clear_row<SHIFTED, G>(c, out, first + i, one_by_one ? threadIdx.x : lane, one_by_one ? kGradientThreads : 32);
        return;
    }
    grid_dependency_wait();
    if (blockIdx.x == gridDim.x - 1 && threadIdx.x == 0) hdr->wait_limit_hit = 0u;
    const int i = (int)(block / c.slabs);
    int64_t some[kMostFewTokens / kGradientThreads];  // this thread's share of the tokens, all under way at once
#pragma unroll
    for (int u = 0; u < kMostFewTokens / kGradientThreads; ++u) {
        const int j = u * kGradientThreads + (int)threadIdx.x;
        some[u] = j < n ? tokens[j] : -1;
    }
    const int64_t token = tokens[i];
    if (token < 0 || token >= c.rows) return;
#pragma unroll
    for (int u = 0; u < kMostFewTokens / kGradientThreads; ++u) {
        const unsigned int same = __ballot_sync(0xffffffffu, some[u] == token);
        if (lane == 0) bits[u * (kGradientThreads / 32) + warp] = same;
    }
    __syncthreads();
    const int words = (n + 31) / 32;
    int count = 0;
    bool earlier = false;
    for (int w = 0; w < words; ++w) {  // (all threads alike)
        const unsigned int same = bits[w];
        if (w < i / 32 ? same : w == i / 32 && same << (31 - i % 32) << 1) earlier = true;
        if (w % (kGradientThreads / 32) == warp && same >> lane & 1) list[count + __popc(same & lanemask_lt())] = (unsigned short)(w * 32 + lane);
        count += __popc(same);
    }
    if (earlier) return;
    __syncthreads();
    const int tx = threadIdx.x % kPartThreads, ty = threadIdx.x / kPartThreads;
    constexpr int kFewAhead = SHIFTED ? 4 : 8;  // (shifted columns take twice the registers, which would cost blocks on an SM)
    const int begin = count * ty / kParts, end = count * (ty + 1) / kParts;
    const int64_t row = token * c.row_stride;
    for (int first = (int)(block % c.slabs) * kPartThreads; first < c.groups; first += c.slabs * kPartThreads) {
        const int g = first + tx;
        float sum[G];
#pragma unroll
        for (int k = 0; k < G; ++k) sum[k] = 0.0f;
        const TIn *from = upstream + column_of<SHIFTED, G>(out + row, g);
        for (int r = begin; r < end && g < c.groups; r += kFewAhead) {
            Columns<TIn, G, SHIFTED> in[kFewAhead];
#pragma unroll
            for (int j = 0; j < kFewAhead; ++j)  // (one load behind the other, without a branch between them)
                in[j].load(from + list[r + j < end ? r + j : end - 1] * c.upstream_stride, c.extent);
#pragma unroll
            for (int j = 0; j < kFewAhead; ++j) {
                const Group<TIn, G> x = in[j].get();
#pragma unroll
                for (int k = 0; k < G; ++k) sum[k] += r + j < end ? x.get(k) : 0.0f;
            }
        }
        join_parts<G>(sum, part, kPartThreads);
        if (ty == 0 && g < c.groups) write_row<SHIFTED>(c, out, (unsigned int)token, g, sum);
    }
}

// Floats of a tile's share of a run (a shifted row has a group or two more than its columns).
static int64_t share_floats(int64_t width) { return round_up(width + kMostShifted, 8) + 8; }

// Sorted positions of a tile: enough blocks for the GPU (a narrow row leaves room for many tiles in one), and shares of
// crossing runs that stay a small part of the traffic.
constexpr int64_t kLeastTile = 16, kMostTile = 128;
constexpr int64_t kEnoughTiles = 148 * 3 / 2, kWideShare = 2064;  // tiles of wide rows, from 2048 columns on
static int64_t gradient_tile(int64_t n, int64_t share) {
    int64_t tile = kMostTile;
    while (tile > kLeastTile && ceil_div(n, tile) * (share < kWideShare ? share : kWideShare) < kEnoughTiles * kWideShare) tile /= 2;
    return tile;
}
// Floats that the shares of this many positions, or of fewer of no wider rows, take at most, so that a temp for the
// longest input serves all.  A tile below the longest is half of one that was too long: kEnoughTiles wide shares were
// more than all its shares, and those of its halves are at most twice as many.
static int64_t most_share_floats(int64_t n, int64_t share) {
    const int64_t longest = ceil_div(n, kMostTile) * share, least = ceil_div(n, kLeastTile) * share;
    const int64_t halves = 2 * kEnoughTiles * (share > kWideShare ? share : kWideShare);
    const int64_t shorter = least < halves ? least : halves;
    return longest > shorter ? longest : shorter;
}

struct GradientLayout {
    int64_t tile, tiles, share_stride;
    int64_t sort_bytes, off_keys, off_positions, off_named, named_words, off_shares, total;
};
static int gradient_layout(int64_t rows, int64_t width, int64_t n, GradientLayout &L) {
    if (rows < 0 || width < 0 || n < 0) return B200ALG_INVALID_ARGUMENT;
    if (rows > INT32_MAX || width > INT32_MAX || n > INT32_MAX) return B200ALG_TOO_LARGE;
    L.share_stride = share_floats(width);
    L.tile = gradient_tile(n, L.share_stride);
    L.tiles = ceil_div(n, L.tile);
    const int rc = b200alg_radix_sort_temp_bytes(B200ALG_U32, n, 4, &L.sort_bytes);  // its part lies first, and with it its status word
    if (rc != B200ALG_OK) return rc;
    L.off_keys = round_up(L.sort_bytes, 256);
    L.off_positions = L.off_keys + round_up(n * 4, 256);
    L.off_named = L.off_positions + round_up(n * 4, 256);
    L.named_words = ceil_div(rows, 16);  // of 16 bytes
    L.off_shares = L.off_named + round_up(L.named_words * 16, 256);
    L.total = L.off_shares + round_up(2 * most_share_floats(n, L.share_stride) * 4, 256);
    return B200ALG_OK;
}

// Rows that a block clears: about 32 KB of them (64 and 128 KB: 9.5 and 15.9 instead of 8.5 us for 301 tokens into 10007
// rows of 768 floats), but not fewer than `least`.  From a row for each warp on they are a multiple of that.
static int rows_to_clear(int64_t width, int bytes, int least, int most) {
    constexpr int kWarps = kGradientThreads / 32;
    int64_t rows = (32 << 10) / (width * bytes);
    rows = rows < least ? least : rows > most ? most : rows;
    return (int)(rows < kWarps ? rows : rows / kWarps * kWarps);
}

// The status word of a call that has nothing else to do.
static int clear_status(cudaStream_t s, void *temp) {
    B200ALG_CUDA_TRY(cudaMemsetAsync(&((TempHeader *)temp)->wait_limit_hit, 0, sizeof(unsigned int), s));
    return B200ALG_OK;
}

template <typename TIn, typename TOut, int G, bool SHIFTED>
static int run_gradient(cudaStream_t s, GradientCall c, const IndexView &tokens, const GradientLayout &L, const void *upstream, void *out, void *temp) {
    c.groups = (int)groups_in(c.width, G, SHIFTED);
    c.extent = extent_of(upstream, c.n, c.width, c.upstream_stride, sizeof(TIn));
    char *t = (char *)temp;
    c.flat = (c.row_stride == c.width || c.rows == 1) && c.width * (int64_t)sizeof(TOut) < 1024;  // (rows of 5 KB: 89 us instead of 80)
    c.by_width = FastDivide((unsigned int)c.width);
    if (c.n <= (c.groups <= kPartThreads ? kMostFewTokens : kFewTokens)) {
        // columns of a position that different blocks take: as many as make some thousands of blocks
        const int64_t slabs = ceil_div(c.groups, kPartThreads), most = ceil_div(2048, c.n ? c.n : 1);
        c.slabs = (int)(slabs < most ? slabs : most);
        c.sum_blocks = c.n * c.slabs;
        c.clear_rows = rows_to_clear(c.width, sizeof(TOut), 1, 256);
        c.clear_blocks = c.accumulate ? 0 : ceil_div(c.rows, c.clear_rows);
        const int64_t blocks = c.sum_blocks + c.clear_blocks;
        if (blocks > INT32_MAX) return B200ALG_TOO_LARGE;
        if (!blocks) return clear_status(s, temp);
        B200ALG_CUDA_TRY(launch_dependent(gradient_few_kernel<TIn, TOut, G, SHIFTED>, dim3((unsigned)blocks), dim3(kGradientThreads), 0, s, c, tokens,
                                          (const TIn *)upstream, (TOut *)out, (TempHeader *)temp));
        return B200ALG_OK;
    }
    unsigned int *keys = (unsigned int *)(t + L.off_keys), *positions = (unsigned int *)(t + L.off_positions);
    unsigned char *named = c.accumulate ? nullptr : (unsigned char *)(t + L.off_named);
    c.keys = keys, c.positions = positions, c.named = named;
    c.tile = L.tile, c.tiles = L.tiles;
    c.shares = (float *)(t + L.off_shares), c.share_stride = L.share_stride;
    for (c.x = 8; c.x < kGradientThreads && c.x < c.groups; c.x *= 2) {}
    c.y = kGradientThreads / c.x;
    c.slabs = (int)ceil_div(c.groups, c.x);
    c.sum_blocks = ceil_div(c.tiles, c.y) * c.slabs;
    // (a row for each warp at least: with one row a block 131072 tokens of 4096 took 559 us instead of 528)
    c.clear_rows = rows_to_clear(c.width, sizeof(TOut), kGradientThreads / 32, 1 << 20);
    c.clear_blocks = named ? ceil_div(c.rows, c.clear_rows) : 0;
    const int x = part_threads(c.groups);
    c.join_blocks = ceil_div(c.tiles, kGradientThreads / x) * ceil_div(c.groups, x);
    if (c.sum_blocks > INT32_MAX || c.join_blocks + c.clear_blocks > INT32_MAX) return B200ALG_TOO_LARGE;
    const int64_t cap = (int64_t)sm_count() * 8;
    auto some = [&](int64_t want) { return dim3((unsigned)(want < cap ? want : cap)); };
    if (named)
        B200ALG_CUDA_TRY(launch_dependent(gradient_forget_kernel, some(ceil_div(L.named_words, 256)), dim3(256), 0, s, (uint4 *)named, L.named_words));
    B200ALG_CUDA_TRY(launch_dependent(gradient_keys_kernel, some(ceil_div(c.n, 256 * 2)), dim3(256), 0, s, tokens, c.n, c.rows, keys, named));
    const int rc = b200alg_radix_sort_pairs_sequence(s, keys, positions, c.n, B200ALG_U32, B200ALG_U32, B200ALG_SORT_ASCENDING, temp, L.sort_bytes);
    if (rc != B200ALG_OK) return rc;
    const size_t smem = (size_t)c.y * (2 * c.tile + 3) * 4;  // (33 KB at most)
    B200ALG_CUDA_TRY(launch_dependent(gradient_sum_kernel<TIn, TOut, G, SHIFTED>, dim3((unsigned)c.sum_blocks), dim3(kGradientThreads), smem, s, c,
                                      (const TIn *)upstream, (TOut *)out));
    B200ALG_CUDA_TRY(launch_dependent(gradient_join_kernel<TOut, G, SHIFTED>, dim3((unsigned)(c.join_blocks + c.clear_blocks)), dim3(kGradientThreads), 0, s, c, (TOut *)out, x));
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
    return with_element(dtype, [&](auto in) {
        return with_element(out_dtype, [&](auto to) {
            using TIn = decltype(in);
            using TOut = decltype(to);
            constexpr int G = 32 / (sizeof(TIn) > sizeof(TOut) ? sizeof(TIn) : sizeof(TOut));
            if (fits(G)) return run_lookup<TIn, TOut, G, false>(s, table, rows, width, row_stride, view, n, scale, out, out_stride);
            if constexpr (G == 16)
                if (fits(8)) return run_lookup<TIn, TOut, 8, false>(s, table, rows, width, row_stride, view, n, scale, out, out_stride);
            return run_lookup<TIn, TOut, shifted_group<TIn, TOut>(), true>(s, table, rows, width, row_stride, view, n, scale, out, out_stride);
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
    if (rows == 0 || width == 0) return temp && temp_bytes >= (int64_t)sizeof(TempHeader) ? clear_status((cudaStream_t)stream, temp) : B200ALG_OK;
    if (!gradient || !temp || (n && (!tokens || !upstream))) return B200ALG_INVALID_ARGUMENT;
    if ((uintptr_t)gradient % ob || (uintptr_t)upstream % ib || (uintptr_t)tokens % dtype_bytes(token_dtype) || (uintptr_t)temp % 256)
        return B200ALG_MISALIGNED;
    if (temp_bytes < L.total) return B200ALG_TEMP_TOO_SMALL;
    cudaStream_t s = (cudaStream_t)stream;
    const IndexView view{tokens, token_stride, token_dtype == B200ALG_I64};
    GradientCall c{};
    c.n = n;
    c.upstream_stride = upstream_stride;
    c.rows = rows, c.width = width, c.row_stride = row_stride;
    c.scale = (float)scale, c.accumulate = accumulate != 0;
    return with_element(upstream_dtype, [&](auto in) {
        return with_element(dtype, [&](auto to) {
            using TIn = decltype(in);
            using TOut = decltype(to);
            constexpr int G = 16 / sizeof(TIn);
            if (groups_aligned(upstream, upstream_stride, n, width, ib, G) && groups_aligned(gradient, row_stride, rows, width, ob, G))
                return run_gradient<TIn, TOut, G, false>(s, c, view, L, upstream, gradient, temp);
            return run_gradient<TIn, TOut, shifted_group<TIn, TOut>(), true>(s, c, view, L, upstream, gradient, temp);
        });
    });
}
