// sequence_device.hpp -- loads and stores of a few neighbouring elements of a
// row, at any alignment, for the sequence operators' kernels.
#pragma once

#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

namespace vkfx {

template <typename T, int N>
using Some = T __attribute__((ext_vector_type(N)));
// The same in memory, at any alignment of its elements.
template <typename T, int N>
struct Packed {
    typedef T type __attribute__((ext_vector_type(N), aligned(sizeof(T))));
};

template <typename T>
constexpr int kVector = 16 / (int)sizeof(T);

// Elements c .. c + N - 1 of a row of `width`, zeros past its end.
template <typename T, int N>
__device__ __forceinline__ Some<T, N> load_some(const T* row, int c, int width) {
    Some<T, N> r;
    if (c + N <= width) {
        r = *(const typename Packed<T, N>::type*)(row + c);
    } else {
#pragma unroll
        for (int e = 0; e < N; ++e) r[e] = c + e < width ? row[c + e] : (T)0.f;
    }
    return r;
}

template <typename T, int N>
__device__ __forceinline__ void store_some(T* row, int c, int width, const Some<T, N>& r) {
    if (c + N <= width) {
        *(typename Packed<T, N>::type*)(row + c) = r;
        return;
    }
#pragma unroll
    for (int e = 0; e < N; ++e)
        if (c + e < width) row[c + e] = r[e];
}

}  // namespace vkfx
