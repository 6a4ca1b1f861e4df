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
#include <math.h>
#include <type_traits>

#include "elements.cuh"

namespace b200alg {

constexpr int kBalanceThreads = 256;
constexpr int kBalanceWarps = kBalanceThreads / 32;
constexpr int kMostExperts = 1024;
constexpr int kBalanceBlocksPerSm = 4;
constexpr int kMostBalanceBlocks = 148 * kBalanceBlocksPerSm;

struct BalanceCall {
    int64_t tokens, logits_stride;
    int experts, choices;
    const unsigned char *mask;  // of the tokens that count, NULL: all do
    int lanes;                  // of a row: a power of two
    int groups;                 // of a row
};

__host__ __device__ constexpr int padded_bins(int experts) { return (experts + 4) / 4 * 4; }

__device__ __forceinline__ float exp2_approximate(float x) {  // 2^x; below 2^-126 zero
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// A row's logits in the registers of `lanes` lanes: group c of lane l holds the columns (c * lanes + l) * V on.
template <typename T, int V, int C> struct RouterRow {
    Group<T, V> raw[C];

    __device__ __forceinline__ void load(const T *p, const BalanceCall &call, int lane_of_row) {
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int g = c * call.lanes + lane_of_row;
            if (g < call.groups) raw[c].load(p + (int64_t)g * V);
        }
    }
    // e = exp(x - max x), zero in places that the row does not have; all lanes take part.
    __device__ __forceinline__ void exponentials(float (&e)[C * V], const BalanceCall &call, int lane_of_row, bool there) const {
        float top = -INFINITY;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const bool in = there && c * call.lanes + lane_of_row < call.groups;
#pragma unroll
            for (int v = 0; v < V; ++v) {
                e[c * V + v] = in ? raw[c].get(v) : -INFINITY;
                top = fmaxf(top, e[c * V + v]);  // (a NaN is left out here and comes back below)
            }
        }
        for (int d = call.lanes >> 1; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
        if (top == -INFINITY) top = 0.0f;
#pragma unroll
        for (int i = 0; i < C * V; ++i) e[i] = exp2_approximate((e[i] - top) * 1.4426950408889634f);
    }
};

__device__ __forceinline__ float row_sum(float x, int lanes) {
    for (int d = lanes >> 1; d > 0; d >>= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
    return x;
}

// What a block found, in temp: sums of p by expert, counts by expert, tokens that count.
struct BalanceShares {
    float *sums;      // [blocks][experts]
    unsigned int *counts;  // [blocks][experts + 1]
};

// The shares of all blocks as the call's results, by one block.
__device__ void finish_balance(const BalanceShares &shares, int blocks, int experts, int choices, double coefficient, float *loss, int *counts,
                               float *probabilities) {
    __shared__ unsigned int valid;
    __shared__ double part[kBalanceWarps];
    __syncthreads();
    if (threadIdx.x < 32) {
        unsigned int n = 0u;
        for (int b = threadIdx.x; b < blocks; b += 32) n += __ldcg(shares.counts + (int64_t)b * (experts + 1) + experts);
        n = __reduce_add_sync(0xffffffffu, n);
        if (threadIdx.x == 0) valid = n;
    }
    __syncthreads();
    const double inverse = valid ? 1.0 / valid : 0.0;
    double sum = 0.0;
    for (int e = threadIdx.x; e < experts; e += kBalanceThreads) {
        double p = 0.0;
        unsigned int n = 0u;
        for (int b = 0; b < blocks; ++b) {
            p += __ldcg(shares.sums + (int64_t)b * experts + e);
            n += __ldcg(shares.counts + (int64_t)b * (experts + 1) + e);
        }
        p *= inverse;
        counts[e] = (int)n;
        probabilities[e] = (float)p;
        sum += n * inverse / choices * p;
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) sum += __shfl_down_sync(0xffffffffu, sum, d);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < kBalanceWarps; ++w) sum += part[w];
        *loss = (float)(coefficient * experts * sum);
        counts[experts] = (int)valid;
    }
}

template <typename T, int V, int C>
__global__ void __launch_bounds__(kBalanceThreads)
balance_kernel(BalanceCall call, const T *__restrict__ logits, IndexView chosen, FastDivide by_choices, BalanceShares shares, double coefficient,
               float *loss, int *counts, float *probabilities) {
    grid_dependency_release();
    extern __shared__ unsigned char smem[];
    unsigned int *bins = reinterpret_cast<unsigned int *>(smem);                  // [experts + 1]
    float *sums = reinterpret_cast<float *>(bins + padded_bins(call.experts));  // [warps][experts]
    for (int e = threadIdx.x; e <= call.experts; e += kBalanceThreads) bins[e] = 0u;
    __syncthreads();
    grid_dependency_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t begin = call.tokens * blockIdx.x / gridDim.x, end = call.tokens * (blockIdx.x + 1) / gridDim.x;

    // counts
    unsigned int valid = 0u;
    for (int64_t t = begin + threadIdx.x; t < end; t += kBalanceThreads) valid += call.mask ? call.mask[t] != 0 : 1u;
    valid = __reduce_add_sync(0xffffffffu, valid);
    if (lane == 0) atomicAdd(bins + call.experts, valid);
    const unsigned int ids = (unsigned int)((end - begin) * call.choices);
    for (unsigned int i = threadIdx.x; i < ids; i += kBalanceThreads) {
        const unsigned int t = by_choices(i), j = i - t * call.choices;
        if (call.mask && !call.mask[begin + t]) continue;
        const int64_t e = chosen.wide ? reinterpret_cast<const long long *>(chosen.p)[(begin + t) * chosen.stride + j]
                                      : reinterpret_cast<const int *>(chosen.p)[(begin + t) * chosen.stride + j];
        if (e >= 0 && e < call.experts) atomicAdd(bins + e, 1u);
    }

    // sums of probabilities
    const int rows = 32 / call.lanes;  // of a warp at a time
    const int lane_of_row = lane & (call.lanes - 1), row_of_warp = lane / call.lanes;
    float sum[C * V];
#pragma unroll
    for (int i = 0; i < C * V; ++i) sum[i] = 0.0f;
    for (int64_t t = begin + warp * rows; t < end; t += kBalanceWarps * rows) {
        const int64_t row = t + row_of_warp;
        const bool there = row < end && (!call.mask || call.mask[row]);
        RouterRow<T, V, C> r;
        if (there) r.load(logits + row * call.logits_stride, call, lane_of_row);
        float e[C * V], whole = 0.0f;
        r.exponentials(e, call, lane_of_row, there);
#pragma unroll
        for (int i = 0; i < C * V; ++i) whole += e[i];
        whole = row_sum(whole, call.lanes);
        const float inverse = whole == 0.0f ? 0.0f : 1.0f / whole;
#pragma unroll
        for (int i = 0; i < C * V; ++i) sum[i] = fmaf(e[i], inverse, sum[i]);
    }
#pragma unroll
    for (int i = 0; i < C * V; ++i)
        for (int d = call.lanes; d < 32; d <<= 1) sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], d);
    if (row_of_warp == 0) {
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int g = c * call.lanes + lane_of_row;
            if (g >= call.groups) continue;
#pragma unroll
            for (int v = 0; v < V; ++v) sums[warp * call.experts + g * V + v] = sum[c * V + v];
        }
    }
    __syncthreads();
    for (int e = threadIdx.x; e < call.experts; e += kBalanceThreads) {
        float p = 0.0f;
#pragma unroll
        for (int w = 0; w < kBalanceWarps; ++w) p += sums[w * call.experts + e];
        shares.sums[(int64_t)blockIdx.x * call.experts + e] = p;
    }
    for (int e = threadIdx.x; e <= call.experts; e += kBalanceThreads) shares.counts[(int64_t)blockIdx.x * (call.experts + 1) + e] = bins[e];
    if (gridDim.x == 1) finish_balance(shares, 1, call.experts, call.choices, coefficient, loss, counts, probabilities);
}

__global__ void __launch_bounds__(kBalanceThreads) balance_finish_kernel(BalanceShares shares, int blocks, int experts, int choices, double coefficient,
                                                                          float *loss, int *counts, float *probabilities) {
    grid_dependency_release();
    grid_dependency_wait();
    finish_balance(shares, blocks, experts, choices, coefficient, loss, counts, probabilities);
}

template <typename T, int V, int C>
__global__ void __launch_bounds__(kBalanceThreads)
balance_gradient_kernel(BalanceCall call, const T *__restrict__ logits, const int *counts, const float *loss_gradient, double coefficient,
                        T *gradient, int64_t gradient_stride, int accumulate) {
    grid_dependency_release();
    grid_dependency_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int rows = 32 / call.lanes;
    const int lane_of_row = lane & (call.lanes - 1), row_of_warp = lane / call.lanes;
    float often[C * V];
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const int g = c * call.lanes + lane_of_row;
#pragma unroll
        for (int v = 0; v < V; ++v) often[c * V + v] = g < call.groups ? (float)counts[g * V + v] : 0.0f;
    }
    const double tokens = counts[call.experts];
    const float factor = tokens > 0.0 ? (float)((double)*loss_gradient * coefficient * call.experts / call.choices / (tokens * tokens)) : 0.0f;
    const int64_t step = (int64_t)gridDim.x * kBalanceWarps * rows;
    for (int64_t t = ((int64_t)blockIdx.x * kBalanceWarps + warp) * rows; t < call.tokens; t += step) {
        const int64_t row = t + row_of_warp;
        const bool there = row < call.tokens && (!call.mask || call.mask[row]);
        RouterRow<T, V, C> r;
        if (there) r.load(logits + row * call.logits_stride, call, lane_of_row);
        float e[C * V], whole = 0.0f, dot = 0.0f;
        r.exponentials(e, call, lane_of_row, there);
#pragma unroll
        for (int i = 0; i < C * V; ++i) {
            whole += e[i];
            dot = fmaf(e[i], often[i], dot);
        }
        whole = row_sum(whole, call.lanes);
        dot = row_sum(dot, call.lanes);
        const float inverse = whole == 0.0f ? 0.0f : 1.0f / whole;
        dot *= inverse;
        if (row >= call.tokens || (!there && accumulate)) continue;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int g = c * call.lanes + lane_of_row;
            if (g >= call.groups) continue;
            T *p = gradient + row * gradient_stride + (int64_t)g * V;
            float y[V];
            Group<T, V> o;
#pragma unroll
            for (int v = 0; v < V; ++v) y[v] = there ? factor * (e[c * V + v] * inverse) * (often[c * V + v] - dot) : 0.0f;
            if (accumulate) {
                o.load(p);
#pragma unroll
                for (int v = 0; v < V; ++v) y[v] += o.get(v);
            }
            o.set(y);
            o.store(p);
        }
    }
}

// Calls `call` with the element type, the elements of a group and the groups of a lane that fit the logits.
template <typename Call> static int with_row(int dtype, int experts, bool whole_groups, Call call) {
    return with_element(dtype, [&](auto element) {
        using T = decltype(element);
        constexpr int V = 16 / sizeof(T);
        const int lane_groups = (int)ceil_div(whole_groups ? experts / V : experts, 32);
        if (whole_groups) {
            if (lane_groups <= 1) return call(element, std::integral_constant<int, V>{}, std::integral_constant<int, 1>{});
            if (lane_groups <= 2) return call(element, std::integral_constant<int, V>{}, std::integral_constant<int, 2>{});
            if constexpr (V == 8) {
                return call(element, std::integral_constant<int, V>{}, std::integral_constant<int, 4>{});
            } else {
                if (lane_groups <= 4) return call(element, std::integral_constant<int, V>{}, std::integral_constant<int, 4>{});
                return call(element, std::integral_constant<int, V>{}, std::integral_constant<int, 8>{});
            }
        }
        if (lane_groups <= 2) return call(element, std::integral_constant<int, 1>{}, std::integral_constant<int, 2>{});
        if (lane_groups <= 8) return call(element, std::integral_constant<int, 1>{}, std::integral_constant<int, 8>{});
        return call(element, std::integral_constant<int, 1>{}, std::integral_constant<int, 32>{});
    });
}

static BalanceCall balance_call(int64_t tokens, int64_t logits_stride, int64_t experts, int64_t choices, const void *mask, int group) {
    BalanceCall c{tokens, logits_stride, (int)experts, (int)choices, (const unsigned char *)mask, 1, (int)experts / group};
    while (c.lanes < 32 && c.lanes < c.groups) c.lanes *= 2;
    return c;
}

// Blocks that a call's tokens fill: every warp has a few rows.
static int64_t balance_blocks(int64_t tokens, int64_t most) {
    const int64_t want = ceil_div(tokens, kBalanceWarps * 8);
    return want < 1 ? 1 : want < most ? want : most;
}

static int check_router(int64_t tokens, int64_t experts, int64_t choices, int64_t logits_stride, int dtype) {
    if (tokens < 0 || experts < 1 || choices < 1 || !matrix_ok(tokens, experts, logits_stride)) return B200ALG_INVALID_ARGUMENT;
    if (!element_bytes(dtype)) return B200ALG_UNSUPPORTED;
    if (experts > kMostExperts || choices > kMostExperts) return B200ALG_UNSUPPORTED;
    if (tokens > INT32_MAX / choices) return B200ALG_TOO_LARGE;  // the counts are 32-bit integers
    return B200ALG_OK;
}

static int64_t balance_temp_bytes(int64_t experts, int64_t tokens) {
    const int64_t blocks = balance_blocks(tokens, kMostBalanceBlocks);
    return sizeof(TempHeader) + round_up(blocks * experts * 4, 256) + round_up(blocks * (experts + 1) * 4, 256);
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
    const int64_t resident = (int64_t)sm_count() * kBalanceBlocksPerSm;
    const int blocks = (int)balance_blocks(tokens, resident < kMostBalanceBlocks ? resident : kMostBalanceBlocks);
    BalanceShares shares;
    shares.sums = (float *)((char *)temp + sizeof(TempHeader));
    shares.counts = (unsigned int *)((char *)temp + sizeof(TempHeader) + round_up((int64_t)blocks * experts * 4, 256));
    const bool whole = groups_aligned(logits, logits_stride, tokens, experts, bytes, 16 / bytes);
    const size_t smem = (size_t)(padded_bins((int)experts) + kBalanceWarps * experts) * 4;
    rc = with_row(dtype, (int)experts, whole, [&](auto element, auto v, auto c) -> int {
        using T = decltype(element);
        const BalanceCall call = balance_call(tokens, logits_stride, experts, choices, mask, v.value);
        B200ALG_CUDA_TRY(launch_dependent(balance_kernel<T, v.value, c.value>, dim3(blocks), dim3(kBalanceThreads), smem, s, call, (const T *)logits,
                                          IndexView{chosen, chosen_stride, chosen_dtype == B200ALG_I64}, FastDivide((unsigned int)choices), shares,
                                          coefficient, loss, counts, probabilities));
        return B200ALG_OK;
    });
    if (rc != B200ALG_OK || blocks == 1) return rc;
    B200ALG_CUDA_TRY(launch_dependent(balance_finish_kernel, dim3(1), dim3(kBalanceThreads), 0, s, shares, blocks, (int)experts, (int)choices,
                                      coefficient, loss, counts, probabilities));
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
    const bool whole = groups_aligned(logits, logits_stride, tokens, experts, bytes, 16 / bytes) &&
                       groups_aligned(gradient, gradient_stride, tokens, experts, bytes, 16 / bytes);
    return with_row(dtype, (int)experts, whole, [&](auto element, auto v, auto c) -> int {
        using T = decltype(element);
        const BalanceCall call = balance_call(tokens, logits_stride, experts, choices, mask, v.value);
        const int64_t want = ceil_div(tokens, (32 / call.lanes) * kBalanceWarps), most = (int64_t)sm_count() * 8;
        B200ALG_CUDA_TRY(launch_dependent(balance_gradient_kernel<T, v.value, c.value>, dim3((unsigned)(want < most ? want : most)),
                                          dim3(kBalanceThreads), 0, s, call, (const T *)logits, counts, loss_gradient, coefficient, (T *)gradient,
                                          gradient_stride, accumulate != 0));
        return B200ALG_OK;
    });
}
