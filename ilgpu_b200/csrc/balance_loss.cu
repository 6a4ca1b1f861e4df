// The balance loss of a router with the counts per expert, and its gradient in the logits.
//
//   p_t  = softmax(logits[t, :])                    (a row of nothing but -inf: zeros)
//   c_e  = #{(t, j) : token t counts, experts[t, j] = e}
//   P_e  = 1/T' sum over the tokens that count of p_te       (T' of them)
//   loss = coefficient * E * sum_e c_e / (T' k) * P_e
//
//   d loss / d logits[t, e] = coefficient * E / (T'^2 k) * p_te * (c_e - sum_j c_j p_tj)
//
// The counts are taken as constants, as they have no derivative.
//
// One read of the logits (and one write of the gradient).  262144 tokens of 128 experts in bf16, 68 MB, take 25.7 us: 17.7 for the
// probabilities, whose loads and exponentials 16 warps an SM do not hide altogether, 3.5 for the counts and 4.5 for the launch
// that adds the blocks' shares up.  The gradient of 131072 tokens of 256 experts in float, 255 MB, takes 42.2 (6.0 TB/s).
#include <math.h>
#include <type_traits>

#include <cooperative_groups.h>

#include "elements.cuh"

namespace cg = cooperative_groups;

namespace b200alg {

constexpr int kBalanceThreads = 512;  // (256, and so twice the shares to add up: 28.7 us instead of 25.2 for 262144 tokens and 128 experts in bf16)
constexpr int kBalanceWarps = kBalanceThreads / 32;
constexpr int kMostExperts = 1024;
constexpr int kBalanceCluster = 8;  // blocks that add up in each other's shared memory
constexpr int kMostBalanceBlocks = 148 * 2;  // (with 64 registers a thread or more no third one fits an SM)
// Rows of a launch that a lane adds up.  With the lanes beside it and the block's warps a column's sum is 123 additions in 32
// bits at most; blocks, clusters and launches go on in 64, so that the error does not grow with the tokens.  (Sums that
// go on in 64 within a launch cost registers: 131072 tokens of 256 experts in float 33 us instead of 30.)
constexpr int kLaneRows = 104;
constexpr int kFinishThreads = 1024;
constexpr int kIndexSlots = 2;        // indices of a row that a lane fetches ahead
constexpr int kShareAhead = 8;      // blocks' shares that a thread has in flight

struct BalanceCall {
    int64_t tokens, logits_stride;
    int experts, choices;
    const unsigned char *mask;  // of the tokens that count, NULL: all do
    int groups;                 // of a row
};

__host__ __device__ constexpr int padded_bins(int experts) { return (experts + 4) / 4 * 4; }
constexpr int kGradientWarps = 8;
// Shared memory of balance_kernel: counts, the warps' sums, and where one cluster is all a block's part of what it adds up.
static size_t balance_smem(int64_t experts, int cluster) {
    return (size_t)padded_bins((int)experts) * (1 + kBalanceWarps) * 4 + (cluster ? (size_t)ceil_div(experts, cluster) * 12 : 0);
}

__device__ __forceinline__ float exp2_approximate(float x) {  // 2^x; below 2^-126 zero
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

template <typename T> struct LowestBits;  // -inf, in each part of a word
template <> struct LowestBits<float> { static constexpr unsigned int value = 0xFF800000u; };
template <> struct LowestBits<__half> { static constexpr unsigned int value = 0xFC00FC00u; };
template <> struct LowestBits<__nv_bfloat16> { static constexpr unsigned int value = 0xFF80FF80u; };

// How a row lies in a warp: LANES lanes share it, each with C groups of V elements; group c of lane l holds the columns
// (c * LANES + l) * V on.  A lane has U rows in flight.
template <int V_, int C_, int LANES_, int U_> struct RowShape {
    static constexpr int V = V_, C = C_, LANES = LANES_, U = U_, E = V_ * C_;
    static constexpr int ROWS = 32 / LANES_;  // of a warp at a time
};

// Two floats in one instruction, which is what these kernels are made of.
struct Pair {
    unsigned long long bits;
    __device__ __forceinline__ Pair() {}
    __device__ __forceinline__ Pair(float a, float b) { asm("mov.b64 %0, {%1, %2};" : "=l"(bits) : "f"(a), "f"(b)); }
    __device__ __forceinline__ void apart(float &a, float &b) const { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(bits)); }
};
__device__ __forceinline__ Pair operator+(Pair a, Pair b) {
    Pair r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.bits) : "l"(a.bits), "l"(b.bits));
    return r;
}
__device__ __forceinline__ Pair operator*(Pair a, Pair b) {
    Pair r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.bits) : "l"(a.bits), "l"(b.bits));
    return r;
}
__device__ __forceinline__ Pair fma(Pair a, Pair b, Pair c) {
    Pair r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.bits) : "l"(a.bits), "l"(b.bits), "l"(c.bits));
    return r;
}

template <typename T, typename S> struct RouterRow {
    Group<T, S::V> raw[S::C];

    // -inf in the places that the row does not have, and in all of a row that does not count: their exp is zero.
    __device__ __forceinline__ void load(const T *p, bool there, int groups, int lane_of_row) {
#pragma unroll
        for (int c = 0; c < S::C; ++c) {
#pragma unroll
            for (int i = 0; i < Group<T, S::V>::kWords; ++i) raw[c].w[i] = LowestBits<T>::value;
            const int g = c * S::LANES + lane_of_row;
            if (there && g < groups) raw[c].load(p + g * S::V);
        }
    }
    // The largest value of the row (a NaN is left out here and comes back from the exponentials); all lanes take part.
    __device__ __forceinline__ float top() const {
        float top = -INFINITY;
        if constexpr (sizeof(T) == 2 && S::V > 1) {  // two at a time
            using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
            unsigned int most = LowestBits<T>::value;
#pragma unroll
            for (int c = 0; c < S::C; ++c)
#pragma unroll
                for (int i = 0; i < Group<T, S::V>::kWords; ++i) {
                    const T2 m = __hmax2(*reinterpret_cast<const T2 *>(&most), *reinterpret_cast<const T2 *>(&raw[c].w[i]));
                    most = *reinterpret_cast<const unsigned int *>(&m);
                }
            Group<T, 2> two;
            two.w[0] = most;
            top = fmaxf(two.get(0), two.get(1));
        } else {
#pragma unroll
            for (int c = 0; c < S::C; ++c)
#pragma unroll
                for (int v = 0; v < S::V; ++v) top = fmaxf(top, raw[c].get(v));
        }
#pragma unroll
        for (int d = S::LANES >> 1; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
        return top;
    }
    __device__ __forceinline__ float element(int i) const { return raw[i / S::V].get(i % S::V); }
    // e = exp(x - max x) times a power of two below 2 that is the row's own and leaves with its sum.  x log2(e) less a
    // whole number is one fused operation, rounded once; where the largest value is so large that its product with
    // log2(e) is not near a whole number any more, x - max x is taken first.
    __device__ __forceinline__ void exponentials(Pair (&e)[S::E / 2]) const {
        constexpr float kLog2e = 1.4426950408889634f;
        float most = top();
        if (most == -INFINITY) most = 0.0f;
        if (fabsf(most) <= 0x1p20f) {
            const float whole = -rintf(most * kLog2e);
            const Pair by(kLog2e, kLog2e), from(whole, whole);
#pragma unroll
            for (int i = 0; i < S::E / 2; ++i) {
                float a, b;
                fma(Pair(element(2 * i), element(2 * i + 1)), by, from).apart(a, b);
                e[i] = Pair(exp2_approximate(a), exp2_approximate(b));
            }
        } else {
#pragma unroll
            for (int i = 0; i < S::E / 2; ++i)
                e[i] = Pair(exp2_approximate((element(2 * i) - most) * kLog2e), exp2_approximate((element(2 * i + 1) - most) * kLog2e));
        }
    }
};

template <int LANES> __device__ __forceinline__ float row_sum(float x) {
#pragma unroll
    for (int d = LANES >> 1; d > 0; d >>= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
    return x;
}
__device__ __forceinline__ float sum_of(Pair x) {
    float a, b;
    x.apart(a, b);
    return a + b;
}

// 1 / x of a row's sum: between 1/2 and twice the number of experts, zero where every logit is -inf, NaN where one is.
__device__ __forceinline__ float inverse_of(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return x == 0.0f ? 0.0f : y;
}

// What the blocks found, in temp: sums of p by expert, and counts by expert with the tokens that count behind them.
struct BalanceShares {
    double *sums;          // [blocks][experts]
    unsigned int *counts;  // [blocks][experts + 1]
    int add;               // to those of the launch before
};

struct BalanceResult {
    TempHeader *hdr;
    double factor;  // coefficient * experts / choices
    float *loss;
    int *counts;
    float *probabilities;
};

__device__ __forceinline__ double sum_of_warp(double sum) {
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    return sum;
}

// The results from the sums and counts of all tokens, by the blocks of a cluster that are known to run: `sums` and
// `counts` hold this block's columns [first, last) of the experts; `valid` tokens count.
template <int THREADS>
__device__ void finish_balance(const double *sums, const unsigned int *counts, int first, int last, unsigned int valid, int experts,
                               const BalanceResult &to) {
    __shared__ double share[kBalanceCluster], part[THREADS / 32];
    cg::cluster_group cluster = cg::this_cluster();
    const int blocks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank(), lane = threadIdx.x & 31;
    const double inverse = valid ? 1.0 / valid : 0.0;
    double sum = 0.0;
    for (int e = first + threadIdx.x; e < last; e += THREADS) {
        const double p = sums[e - first] * inverse;
        to.counts[e] = (int)counts[e - first];
        to.probabilities[e] = (float)p;
        sum += counts[e - first] * p;
    }
    sum = sum_of_warp(sum);
    if (lane == 0) part[threadIdx.x >> 5] = sum;
    __syncthreads();
    if (threadIdx.x < 32) {
        sum = sum_of_warp(lane < THREADS / 32 ? part[lane] : 0.0);
        if (lane == 0) *cluster.map_shared_rank(share + rank, 0) = sum;
    }
    cluster.sync();
    if (rank == 0 && threadIdx.x < 32) {
        sum = sum_of_warp(lane < blocks ? share[lane] : 0.0);
        if (lane == 0) {
            *to.loss = (float)(sum * inverse * to.factor);
            to.counts[experts] = (int)valid;
            to.hdr->wait_limit_hit = 0u;  // no wait can run out
        }
    }
}

template <typename T, typename S>
__global__ void __launch_bounds__(kBalanceThreads, S::E <= 16 ? 2 : 1)
balance_kernel(BalanceCall call, const T *__restrict__ logits, IndexView chosen, BalanceShares shares, BalanceResult to, int alone) {
    grid_dependency_release();
    extern __shared__ __align__(16) unsigned char smem[];
    const int experts = call.experts;
    unsigned int *bins = reinterpret_cast<unsigned int *>(smem);                 // [experts + 1]
    float *sums = reinterpret_cast<float *>(bins + padded_bins(experts));        // [warps][experts], then [experts]
    for (int e = threadIdx.x; e <= experts; e += kBalanceThreads) bins[e] = 0u;
    __syncthreads();
    grid_dependency_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int lane_of_row = lane & (S::LANES - 1), row_of_warp = lane / S::LANES;
    const unsigned int tokens = (unsigned int)call.tokens;
    const unsigned int apart = gridDim.x * (kBalanceWarps * S::ROWS);  // rows that the grid takes at a time

    // An index that no expert has is out of range in 32 bits, too.
    auto index_at = [&](int64_t at) -> unsigned int {
        if (!chosen.wide) return reinterpret_cast<const unsigned int *>(chosen.p)[at];
        const uint2 w = reinterpret_cast<const uint2 *>(chosen.p)[at];
        return w.y ? ~0u : w.x;
    };
    unsigned int valid = 0u;
    Pair sum[S::E / 2];
#pragma unroll
    for (int i = 0; i < S::E / 2; ++i) sum[i] = Pair(0.0f, 0.0f);
    // (no row's number passes 32 bits: tokens is at most 2^31 - 1, the grid takes fewer than 2^20 rows at a time)
    // A lane's rows come round in turn: each is loaded again, for the row U steps on, as soon as its values are in use, and
    // whether that row counts is known a round before.
    RouterRow<T, S> r[S::U];
    bool there[S::U], soon[S::U];
    unsigned int index[S::U][kIndexSlots];
    auto counts_in = [&](unsigned int row) { return row < tokens && (!call.mask || call.mask[row]); };
    auto fetch = [&](int u, unsigned int row) {
        r[u].load(logits + row * call.logits_stride, there[u], call.groups, lane_of_row);
#pragma unroll
        for (int k = 0; k < kIndexSlots; ++k) {
            const int j = lane_of_row + k * S::LANES;
            index[u][k] = there[u] && j < call.choices ? index_at(row * chosen.stride + j) : ~0u;
        }
    };
    unsigned int t = (blockIdx.x * kBalanceWarps + warp) * S::ROWS + row_of_warp;
#pragma unroll
    for (int u = 0; u < S::U; ++u) there[u] = counts_in(t + u * apart);
#pragma unroll
    for (int u = 0; u < S::U; ++u) {
        fetch(u, t + u * apart);
        soon[u] = counts_in(t + (u + S::U) * apart);
    }
    for (; t - row_of_warp < tokens; t += apart * S::U) {
#pragma unroll
        for (int u = 0; u < S::U; ++u) {
            const unsigned int row = t + u * apart;
            if (row - row_of_warp >= tokens) break;
            valid += there[u] && lane_of_row == 0;
#pragma unroll
            for (int k = 0; k < kIndexSlots; ++k)
                if (index[u][k] < (unsigned int)experts) atomicAdd(bins + index[u][k], 1u);
            if (there[u])
                for (int j = lane_of_row + kIndexSlots * S::LANES; j < call.choices; j += S::LANES) {
                    const unsigned int e = index_at(row * chosen.stride + j);
                    if (e < (unsigned int)experts) atomicAdd(bins + e, 1u);
                }
            Pair e[S::E / 2];
            r[u].exponentials(e);
            there[u] = soon[u];
            fetch(u, row + apart * S::U);
            soon[u] = counts_in(row + apart * (2 * S::U));
            Pair whole = e[0];
#pragma unroll
            for (int i = 1; i < S::E / 2; ++i) whole = whole + e[i];
            const float inverse = inverse_of(row_sum<S::LANES>(sum_of(whole)));
            const Pair by(inverse, inverse);
#pragma unroll
            for (int i = 0; i < S::E / 2; ++i) sum[i] = fma(e[i], by, sum[i]);
        }
    }
    valid = __reduce_add_sync(0xffffffffu, valid);
    if (lane == 0 && valid) atomicAdd(bins + experts, valid);
    float column[S::E];
#pragma unroll
    for (int i = 0; i < S::E / 2; ++i) sum[i].apart(column[2 * i], column[2 * i + 1]);
#pragma unroll
    for (int i = 0; i < S::E; ++i)
#pragma unroll
        for (int d = S::LANES; d < 32; d <<= 1) column[i] += __shfl_xor_sync(0xffffffffu, column[i], d);
    if (row_of_warp == 0) {
#pragma unroll
        for (int c = 0; c < S::C; ++c) {
            const int g = c * S::LANES + lane_of_row;
            if (g >= call.groups) continue;
#pragma unroll
            for (int v = 0; v < S::V; ++v) sums[warp * experts + g * S::V + v] = column[c * S::V + v];
        }
    }
    __syncthreads();
    for (int e = threadIdx.x; e <= experts; e += kBalanceThreads) {
        if (e < experts) {
            float p = sums[e];
#pragma unroll
            for (int w = 1; w < kBalanceWarps; ++w) p += sums[w * experts + e];
            if (alone) {
                sums[e] = p;  // (this thread's own column)
            } else {
                double *share = shares.sums + (int64_t)blockIdx.x * experts + e;
                *share = shares.add ? *share + p : p;
            }
        }
        if (!alone) {
            unsigned int *share = shares.counts + (int64_t)blockIdx.x * (experts + 1) + e;
            *share = shares.add ? *share + bins[e] : bins[e];
        }
    }
    if (!alone) return;
    // One cluster has all tokens: it adds up by columns and needs no other launch.
    cg::cluster_group cluster = cg::this_cluster();
    const int blocks = (int)cluster.num_blocks(), part = (experts + blocks - 1) / blocks, first = (int)cluster.block_rank() * part;
    const int last = first + part < experts ? first + part : experts;
    double *all_sums = reinterpret_cast<double *>(sums + kBalanceWarps * padded_bins(experts));  // [part]
    unsigned int *all_counts = reinterpret_cast<unsigned int *>(all_sums + part);    // [part]
    __shared__ unsigned int all_valid;
    cluster.sync();
    for (int e = first + threadIdx.x; e < last; e += kBalanceThreads) {
        double p = 0.0;
        unsigned int n = 0u;
        for (int b = 0; b < blocks; ++b) {
            p += cluster.map_shared_rank(sums, b)[e];
            n += cluster.map_shared_rank(bins, b)[e];
        }
        all_sums[e - first] = p;
        all_counts[e - first] = n;
    }
    if (warp == kBalanceWarps - 1) {
        const unsigned int n = __reduce_add_sync(0xffffffffu, lane < blocks ? cluster.map_shared_rank(bins, lane)[experts] : 0u);
        if (lane == 0) all_valid = n;
    }
    cluster.sync();  // (nobody leaves while its shared memory is read)
    finish_balance<kBalanceThreads>(all_sums, all_counts, first, last, all_valid, experts, to);
}

// The shares of all blocks, by a cluster whose blocks take a part of the columns each.  (The threads of one block would
// add up a few hundred shares one behind the other.)
__global__ void __launch_bounds__(kFinishThreads) balance_finish_kernel(BalanceShares shares, int blocks, int experts, BalanceResult to) {
    constexpr int kMostColumns = kMostExperts / kBalanceCluster;
    __shared__ double sums[kMostColumns], part[kFinishThreads];
    __shared__ unsigned int counts[kMostColumns], part_counts[kFinishThreads], valid[kFinishThreads / 32];
    grid_dependency_release();
    const int columns = (experts + kBalanceCluster - 1) / kBalanceCluster, first = (int)blockIdx.x * columns;
    const int last = first + columns < experts ? first + columns : experts;
    // x threads along the columns, y along the shares
    int x = 1;
    while (x < columns) x *= 2;
    const int y = kFinishThreads / x, tx = threadIdx.x & (x - 1), ty = threadIdx.x / x, e = first + tx;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    cg::this_cluster().sync();  // all its blocks run: they write to the first one's shared memory
    grid_dependency_wait();
    const unsigned int some_valid = threadIdx.x < blocks ? shares.counts[threadIdx.x * (experts + 1) + experts] : 0u;
    double p = 0.0;
    unsigned int n = 0u;
    for (int b = ty; e < last && b < blocks; b += y * kShareAhead) {
        double some[kShareAhead];
        unsigned int count[kShareAhead];
#pragma unroll
        for (int u = 0; u < kShareAhead; ++u) {
            const unsigned int at = b + u * y;  // (fewer than 2^20 values in all)
            some[u] = at < blocks ? shares.sums[at * experts + e] : 0.0;
            count[u] = at < blocks ? shares.counts[at * (experts + 1) + e] : 0u;
        }
#pragma unroll
        for (int u = 0; u < kShareAhead; ++u) {
            p += some[u];
            n += count[u];
        }
    }
    part[threadIdx.x] = p;
    part_counts[threadIdx.x] = n;
    n = __reduce_add_sync(0xffffffffu, some_valid);
    if (lane == 0) valid[warp] = n;
    __syncthreads();
    for (int c = warp; c < columns; c += kFinishThreads / 32) {  // a warp adds up a column
        p = 0.0;
        n = 0u;
        for (int i = lane; i < y; i += 32) {
            p += part[i * x + c];
            n += part_counts[i * x + c];
        }
        p = sum_of_warp(p);
        n = __reduce_add_sync(0xffffffffu, n);
        if (lane == 0) {
            sums[c] = p;
            counts[c] = n;
        }
    }
    const unsigned int all_valid = __reduce_add_sync(0xffffffffu, valid[lane]);
    __syncthreads();
    finish_balance<kFinishThreads>(sums, counts, first, last, all_valid, experts, to);
}

template <typename T, typename S>
__global__ void __launch_bounds__(kGradientWarps * 32)
balance_gradient_kernel(BalanceCall call, const T *__restrict__ logits, const int *counts, const float *loss_gradient, double coefficient,
                        T *gradient, int64_t gradient_stride, int accumulate) {
    grid_dependency_release();
    grid_dependency_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int lane_of_row = lane & (S::LANES - 1), row_of_warp = lane / S::LANES;
    const unsigned int rows = (unsigned int)call.tokens, apart = gridDim.x * (kGradientWarps * S::ROWS);
    // Counts from the smallest one on: what all experts share takes no part in c - dot, and left in it would round it.
    // Where all are chosen as often the gradient is zero.
    int number[S::E], least = INT32_MAX;
#pragma unroll
    for (int i = 0; i < S::E; ++i) {
        const int g = i / S::V * S::LANES + lane_of_row;
        number[i] = g < call.groups ? counts[g * S::V + i % S::V] : INT32_MAX;  // of the lane's i-th element
        least = min(least, number[i]);
    }
    least = __reduce_min_sync(0xFFFFFFFFu, least);
    auto often_of = [&](int i) { return i / S::V * S::LANES + lane_of_row < call.groups ? (float)((unsigned int)number[i] - (unsigned int)least) : 0.0f; };
    Pair often[S::E / 2];
#pragma unroll
    for (int i = 0; i < S::E / 2; ++i) often[i] = Pair(often_of(2 * i), often_of(2 * i + 1));
    const double tokens = counts[call.experts];
    const float factor = tokens > 0.0 ? (float)((double)*loss_gradient * coefficient * call.experts / call.choices / (tokens * tokens)) : 0.0f;
    for (unsigned int t = (blockIdx.x * kGradientWarps + warp) * S::ROWS; t < rows; t += apart * S::U) {
        RouterRow<T, S> r[S::U];
        bool there[S::U];
#pragma unroll
        for (int u = 0; u < S::U; ++u) {
            const unsigned int row = t + u * apart + row_of_warp;
            there[u] = row < rows && (!call.mask || call.mask[row]);
            r[u].load(logits + row * call.logits_stride, there[u], call.groups, lane_of_row);
        }
#pragma unroll
        for (int u = 0; u < S::U; ++u) {
            const unsigned int row = t + u * apart + row_of_warp;
            Pair e[S::E / 2];
            r[u].exponentials(e);
            Pair whole = e[0], dots = e[0] * often[0];
#pragma unroll
            for (int i = 1; i < S::E / 2; ++i) {
                whole = whole + e[i];
                dots = fma(e[i], often[i], dots);
            }
            const float inverse = inverse_of(row_sum<S::LANES>(sum_of(whole)));
            const float dot = row_sum<S::LANES>(sum_of(dots)) * inverse;
            if (row >= rows || (!there[u] && accumulate)) continue;
            const Pair by(factor * inverse, factor * inverse), less(-dot, -dot);
            float y[S::E];
#pragma unroll
            for (int i = 0; i < S::E / 2; ++i) (e[i] * (often[i] + less) * by).apart(y[2 * i], y[2 * i + 1]);
            T *p = gradient + row * gradient_stride;
#pragma unroll
            for (int c = 0; c < S::C; ++c) {
                const int g = c * S::LANES + lane_of_row;
                if (g >= call.groups) continue;
                float z[S::V];
                Group<T, S::V> o;
#pragma unroll
                for (int v = 0; v < S::V; ++v) z[v] = there[u] ? y[c * S::V + v] : 0.0f;
                if (accumulate) {
                    o.load(p + g * S::V);
#pragma unroll
                    for (int v = 0; v < S::V; ++v) z[v] += o.get(v);
                }
                o.set(z);
                o.store(p + g * S::V);
            }
        }
    }
}

// Elements of a group that a router's rows can be moved in: 16 bytes, or four, two or one element.
static int router_group(int64_t experts, int bytes, const void *logits, int64_t logits_stride, const void *gradient, int64_t gradient_stride, int64_t tokens) {
    auto fits = [&](int group) {
        return groups_aligned(logits, logits_stride, tokens, experts, bytes, group) && groups_aligned(gradient, gradient_stride, tokens, experts, bytes, group);
    };
    const int most = 16 / bytes;
    return fits(most) ? most : fits(4) ? 4 : fits(2) ? 2 : 1;
}

// Calls `call` with the element type and the shape of a row.  A lane holds 16 or 32 elements of a row where the row is
// that long, so that few lanes share a row and few shuffles go into its maximum and its sum.
template <int V, typename T, typename Call> static int with_shape(int experts, Call call) {
    const int groups = experts / V;
    if constexpr (V >= 4) {
        if (groups <= 2) return call(T{}, RowShape<V, 1, 2, 4>{});
        if (groups <= 8) return call(T{}, RowShape<V, 2, 4, 2>{});
        if (groups <= 16) return call(T{}, RowShape<V, 4, 4, 1>{});
        if (groups <= 32) return call(T{}, RowShape<V, 4, 8, 1>{});
        if (groups <= 64) return call(T{}, RowShape<V, 4, 16, 1>{});
        if constexpr (V == 4) {
            if (groups <= 128) return call(T{}, RowShape<V, 4, 32, 1>{});
            return call(T{}, RowShape<V, 8, 32, 1>{});
        } else {
            return call(T{}, RowShape<V, 4, 32, 1>{});
        }
    } else {
        constexpr int C = 8;
        if constexpr (V == 2)  // (two lanes a row would read 16 bytes of it at a time)
            if (groups <= 2 * C) return call(T{}, RowShape<V, 4, 4, 2>{});
        if constexpr (V == 1)
            if (groups <= 2 * C) return call(T{}, RowShape<V, C, 2, 2>{});
        if (groups <= 4 * C) return call(T{}, RowShape<V, C, 4, 2 / V>{});
        if (groups <= 8 * C) return call(T{}, RowShape<V, C, 8, 2 / V>{});
        if constexpr (V == 1)
            if (groups <= 12 * C) return call(T{}, RowShape<V, 12, 8, 1>{});
        if (groups <= 16 * C) return call(T{}, RowShape<V, C, 16, 2 / V>{});
        if (groups <= 32 * C) return call(T{}, RowShape<V, C, 32, 2 / V>{});
        return call(T{}, RowShape<V, 32 / V, 32, 1>{});
    }
}
template <typename Call> static int with_row(int dtype, int experts, int group, Call call) {
    return with_element(dtype, [&](auto element) {
        using T = decltype(element);
        if (group == 1) return with_shape<1, T>(experts, call);
        if (group == 2) return with_shape<2, T>(experts, call);
        if constexpr (sizeof(T) == 2)
            if (group == 8) return with_shape<8, T>(experts, call);
        return with_shape<4, T>(experts, call);
    });
}

template <typename S> static BalanceCall balance_call(int64_t tokens, int64_t logits_stride, int64_t experts, int64_t choices, const void *mask) {
    return BalanceCall{tokens, logits_stride, (int)experts, (int)choices, (const unsigned char *)mask, (int)experts / S::V};
}

// Blocks of a call: one for a few rows, then a cluster of them, and from where one is slower than two launches (0) as
// many as there is work for.  In bf16 64 experts, us, cluster / two launches: 128 tokens 5.7 / 7.3, 2048 6.9 / 8.5, 2437
// 7.7 / 8.4; rows that do not lie on boundaries take longer: of 99 experts in float 330 tokens 5.3 / 7.4, 1323 7.9 / 7.5.
static int balance_cluster(int64_t tokens, int64_t experts, bool long_groups) {
    const int64_t cells = tokens * experts;
    return cells <= 4096 ? 1 : cells <= (long_groups ? 1 << 17 : 1 << 15) ? kBalanceCluster : 0;
}

// Resident blocks of a kernel on the whole GPU (asked once per context; `cache` is the kernel's own).
template <typename KernelT> static int resident_blocks(KernelT kernel, int threads, size_t smem, ContextCache<int> &cache, int *blocks) {
    int per_sm = 0;
    if (!cache.find(&per_sm)) {
        if (smem > 48 << 10) B200ALG_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
        B200ALG_CUDA_TRY(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, threads, smem));
        if (per_sm < 1) per_sm = 1;
        cache.store(per_sm);
    }
    *blocks = sm_count() * per_sm;
    return B200ALG_OK;
}

static int check_router(int64_t tokens, int64_t experts, int64_t choices, int64_t logits_stride, int dtype) {
    if (tokens < 0 || experts < 1 || choices < 1 || !matrix_ok(tokens, experts, logits_stride)) return B200ALG_INVALID_ARGUMENT;
    if (!element_bytes(dtype)) return B200ALG_UNSUPPORTED;
    if (experts > kMostExperts || choices > kMostExperts) return B200ALG_UNSUPPORTED;
    if (tokens > INT32_MAX / choices) return B200ALG_TOO_LARGE;  // the counts are 32-bit integers
    return B200ALG_OK;
}

static int64_t balance_temp_bytes(int64_t experts, int64_t tokens) {
    const int64_t blocks = balance_cluster(tokens, experts, false) ? 0 : kMostBalanceBlocks;
    return sizeof(TempHeader) + round_up(blocks * experts * 8, 256) + round_up(blocks * (experts + 1) * 4, 256);
}

}  // namespace b200alg

using namespace b200alg;

extern "C" int b200alg_balance_loss_temp_bytes(int64_t experts, int64_t tokens, int64_t *out_bytes) {
    if (!out_bytes || experts < 1 || tokens < 0) return B200ALG_INVALID_ARGUMENT;
    if (experts > kMostExperts) return B200ALG_UNSUPPORTED;
    if (tokens > INT32_MAX) return B200ALG_TOO_LARGE;
    *out_bytes = balance_temp_bytes(experts, tokens);
    return B200ALG_OK;
}

extern "C" int b200alg_balance_loss(void *stream, const void *logits, int64_t tokens, int64_t experts, int64_t logits_stride, int dtype,
                                    const void *chosen, int64_t choices, int64_t chosen_stride, int chosen_dtype, const void *mask,
                                    double coefficient, float *loss, int32_t *counts, float *probabilities, void *temp, int64_t temp_bytes) {
    int rc = check_router(tokens, experts, choices, logits_stride, dtype);
    if (rc != B200ALG_OK) return rc;
    if (!index_dtype(chosen_dtype)) return B200ALG_UNSUPPORTED;
    if (!matrix_ok(tokens, choices, chosen_stride) || !isfinite(coefficient)) return B200ALG_INVALID_ARGUMENT;
    if (!loss || !counts || !probabilities || !temp || (tokens && (!logits || !chosen))) return B200ALG_INVALID_ARGUMENT;
    const int bytes = element_bytes(dtype);
    if ((uintptr_t)logits % bytes || (uintptr_t)chosen % dtype_bytes(chosen_dtype) || (uintptr_t)loss % 4 || (uintptr_t)counts % 4 ||
        (uintptr_t)probabilities % 4 || (uintptr_t)temp % 256)
        return B200ALG_MISALIGNED;
    if (temp_bytes < balance_temp_bytes(experts, tokens)) return B200ALG_TEMP_TOO_SMALL;
    cudaStream_t s = (cudaStream_t)stream;
    int blocks = 0;
    BalanceShares shares;
    shares.sums = (double *)((char *)temp + sizeof(TempHeader));
    shares.counts = (unsigned int *)((char *)temp + sizeof(TempHeader) + round_up(kMostBalanceBlocks * experts * 8, 256));
    shares.add = 0;
    const BalanceResult to{(TempHeader *)temp, coefficient * experts / choices, loss, counts, probabilities};
    const int group = router_group(experts, bytes, logits, logits_stride, logits, logits_stride, tokens);
    const int cluster = balance_cluster(tokens, experts, group >= 4);
    const size_t smem = balance_smem(experts, cluster);
    rc = with_row(dtype, (int)experts, group, [&](auto element, auto shape) -> int {
        using T = decltype(element);
        using S = decltype(shape);
        auto kernel = balance_kernel<T, S>;
        static ContextCache<int> cache;
        const int status = resident_blocks(kernel, kBalanceThreads, balance_smem(kMostExperts, 1), cache, &blocks);
        if (status != B200ALG_OK) return status;
        int64_t most = tokens;  // of a launch
        if (cluster) {
            blocks = cluster;
        } else {
            const int64_t want = ceil_div(tokens, kBalanceWarps * S::ROWS * S::U);
            if (blocks > kMostBalanceBlocks) blocks = kMostBalanceBlocks;
            if (blocks > want) blocks = (int)want;
            const int64_t rows = (int64_t)blocks * kBalanceWarps * S::ROWS;  // that the grid takes at a time
            const int64_t rounds = ceil_div(tokens, rows);
            most = ceil_div(rounds, ceil_div(rounds, kLaneRows)) * rows;  // as many rounds in each launch
        }
        const int index_bytes = dtype_bytes(chosen_dtype);
        int64_t first = 0;
        do {
            const int64_t some = tokens - first < most ? tokens - first : most;
            B200ALG_CUDA_TRY(launch_dependent_cluster(
                kernel, dim3(blocks), dim3(kBalanceThreads), smem, s, cluster ? cluster : 1,
                balance_call<S>(some, logits_stride, experts, choices, mask ? (const char *)mask + first : nullptr), (const T *)logits + first * logits_stride,
                IndexView{(const char *)chosen + first * chosen_stride * index_bytes, chosen_stride, chosen_dtype == B200ALG_I64}, shares, to, cluster != 0));
            shares.add = 1;
            first += most;
        } while (first < tokens);
        return B200ALG_OK;
    });
    if (rc != B200ALG_OK || cluster) return rc;
    B200ALG_CUDA_TRY(launch_dependent_cluster(balance_finish_kernel, dim3(kBalanceCluster), dim3(kFinishThreads), 0, s, kBalanceCluster, shares, blocks,
                                              (int)experts, to));
    return B200ALG_OK;
}

extern "C" int b200alg_balance_loss_gradient(void *stream, const void *logits, int64_t tokens, int64_t experts, int64_t logits_stride, int dtype,
                                             const void *mask, const int32_t *counts, int64_t choices, double coefficient,
                                             const float *loss_gradient, void *gradient, int64_t gradient_stride, int accumulate) {
    const int rc = check_router(tokens, experts, choices, logits_stride, dtype);
    if (rc != B200ALG_OK) return rc;
    if (!matrix_ok(tokens, experts, gradient_stride) || !isfinite(coefficient)) return B200ALG_INVALID_ARGUMENT;
    if (tokens == 0) return B200ALG_OK;
    if (!logits || !counts || !loss_gradient || !gradient) return B200ALG_INVALID_ARGUMENT;
    const int bytes = element_bytes(dtype);
    if ((uintptr_t)logits % bytes || (uintptr_t)gradient % bytes || (uintptr_t)counts % 4 || (uintptr_t)loss_gradient % 4) return B200ALG_MISALIGNED;
    cudaStream_t s = (cudaStream_t)stream;
    const int group = router_group(experts, bytes, logits, logits_stride, gradient, gradient_stride, tokens);
    return with_row(dtype, (int)experts, group, [&](auto element, auto shape) -> int {
        using T = decltype(element);
        using S = decltype(shape);
        auto kernel = balance_gradient_kernel<T, S>;
        int blocks = 0;
        static ContextCache<int> cache;
        const int status = resident_blocks(kernel, kGradientWarps * 32, 0, cache, &blocks);
        if (status != B200ALG_OK) return status;
        const int64_t want = ceil_div(tokens, kGradientWarps * S::ROWS * S::U);
        B200ALG_CUDA_TRY(launch_dependent(kernel, dim3((unsigned)(want < blocks ? want : blocks)), dim3(kGradientWarps * 32), 0, s,
                                          balance_call<S>(tokens, logits_stride, experts, choices, mask), (const T *)logits, counts, loss_gradient,
                                          coefficient, (T *)gradient, gradient_stride, accumulate != 0));
        return B200ALG_OK;
    });
}
