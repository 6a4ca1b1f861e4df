// Elements of the operators of a training step: F32, F16 and BF16, read and written in groups and computed in 32 bits.
#pragma once

#include "common.cuh"
#include "fast_divide.cuh"

#include <cuda_bf16.h>

namespace b200alg {

// Size of an element type of these operators, 0 for any other type.
inline int element_bytes(int dt) {
    switch (dt) {
    case B200ALG_F16: case B200ALG_BF16: return 2;
    case B200ALG_F32: return 4;
    }
    return 0;
}

// Whether groups of `group` elements of a matrix lie on boundaries that they can be moved from and to whole.
inline bool groups_aligned(const void *p, int64_t row_stride, int64_t rows, int64_t width, int bytes, int group) {
    const int64_t boundary = group * bytes;
    return width % group == 0 && (uintptr_t)p % boundary == 0 && (rows <= 1 || row_stride * bytes % boundary == 0);
}

// Whether a matrix of `rows` rows `row_stride` elements apart is one: rows that do not overlap, and whose last
// element an index of 64 bits reaches.
inline bool matrix_ok(int64_t rows, int64_t width, int64_t row_stride) {
    return rows <= 1 || (row_stride >= width && row_stride <= ((int64_t)1 << 60) / rows);
}

inline bool index_dtype(int dt) { return dt == B200ALG_I32 || dt == B200ALG_I64; }

#ifdef __CUDACC__

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T> __device__ __forceinline__ T from_float(float x);
template <> __device__ __forceinline__ float from_float<float>(float x) { return x; }
template <> __device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// G consecutive elements as the words that they are moved in.
template <typename T, int G> struct Group {
    static constexpr int kBytes = G * (int)sizeof(T);
    static constexpr int kWords = kBytes < 4 ? 1 : kBytes / 4;
    unsigned int w[kWords];

    // 32 bytes go in one instruction: as two of 16 each would touch half of what it covers (clearing rows by such stores
    // ran at 4.3 TB/s instead of 7.2).
    __device__ __forceinline__ void load(const T *p) {
        static_assert(kBytes <= 32, "one instruction");
        if constexpr (kBytes == 32) {
            asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                         : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7]) : "l"(p));
        } else if constexpr (kBytes == 16) {
            const uint4 v = *reinterpret_cast<const uint4 *>(p);
            w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
        } else if constexpr (kBytes == 8) {
            const uint2 v = *reinterpret_cast<const uint2 *>(p);
            w[0] = v.x, w[1] = v.y;
        } else if constexpr (kBytes == 4) {
            w[0] = *reinterpret_cast<const unsigned int *>(p);
        } else {
            w[0] = *reinterpret_cast<const unsigned short *>(p);
        }
    }
    __device__ __forceinline__ void store(T *p) const {
        if constexpr (kBytes == 32) {
            asm volatile("st.global.v8.b32 [%8], {%0, %1, %2, %3, %4, %5, %6, %7};" ::"r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]),
                         "r"(w[6]), "r"(w[7]), "l"(p)
                         : "memory");
        } else if constexpr (kBytes == 16) {
            *reinterpret_cast<uint4 *>(p) = make_uint4(w[0], w[1], w[2], w[3]);
        } else if constexpr (kBytes == 8) {
            *reinterpret_cast<uint2 *>(p) = make_uint2(w[0], w[1]);
        } else if constexpr (kBytes == 4) {
            *reinterpret_cast<unsigned int *>(p) = w[0];
        } else {
            *reinterpret_cast<unsigned short *>(p) = (unsigned short)w[0];
        }
    }
    // For what is not read again soon.
    __device__ __forceinline__ void store_streaming(T *p) const {
        if constexpr (kBytes == 32) {
            asm volatile("st.global.cs.v8.b32 [%8], {%0, %1, %2, %3, %4, %5, %6, %7};" ::"r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]),
                         "r"(w[6]), "r"(w[7]), "l"(p)
                         : "memory");
        } else if constexpr (kBytes == 16) {
            __stcs(reinterpret_cast<uint4 *>(p), make_uint4(w[0], w[1], w[2], w[3]));
        } else if constexpr (kBytes == 8) {
            __stcs(reinterpret_cast<uint2 *>(p), make_uint2(w[0], w[1]));
        } else {
            store(p);
        }
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < kWords; ++i) w[i] = 0u;
    }
    __device__ __forceinline__ float get(int i) const {  // i is known when this is compiled
        if constexpr (sizeof(T) == 4) {
            return __uint_as_float(w[i]);
        } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {  // the upper half of a float
            return __uint_as_float(i % 2 ? w[i / 2] & 0xFFFF0000u : w[i / 2] << 16);
        } else {
            return __half2float(__ushort_as_half((unsigned short)(i % 2 ? w[i / 2] >> 16 : w[i / 2])));
        }
    }
    // Rounded to the nearest, once.
    __device__ __forceinline__ void set(const float (&x)[G]) {
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < G; ++i) w[i] = __float_as_uint(x[i]);
        } else if constexpr (G == 1) {
            const T t = from_float<T>(x[0]);
            w[0] = *reinterpret_cast<const unsigned short *>(&t);
        } else {
#pragma unroll
            for (int i = 0; i < G / 2; ++i) {
                if constexpr (std::is_same<T, __nv_bfloat16>::value) {
                    const __nv_bfloat162 t = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
                    w[i] = *reinterpret_cast<const unsigned int *>(&t);
                } else {
                    const __half2 t = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
                    w[i] = *reinterpret_cast<const unsigned int *>(&t);
                }
            }
        }
    }
};

// Calls `call` with a value of the element type that `dt` stands for (one of the three).
template <typename Call> inline int with_element(int dt, Call call) {
    switch (dt) {
    case B200ALG_F16: return call(__half{});
    case B200ALG_BF16: return call(__nv_bfloat16{});
    case B200ALG_F32: return call(float{});
    }
    return B200ALG_UNSUPPORTED;
}

// Indices of 32 or 64 bits.
struct IndexView {
    const void *p;
    int64_t stride;
    int wide;
    __device__ __forceinline__ int64_t operator[](int64_t i) const {
        return wide ? (int64_t) reinterpret_cast<const long long *>(p)[i * stride] : (int64_t) reinterpret_cast<const int *>(p)[i * stride];
    }
};

#endif  // __CUDACC__

}  // namespace b200alg
