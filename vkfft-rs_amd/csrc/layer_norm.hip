// layer_norm.hip -- layer norm of rows and its gradients.
//
// Both passes are bound by memory: a row of any width that fits the registers
// of a block is read once. Vectors of 16 bytes go to consecutive lanes; a row
// belongs to 8 .. 64 lanes of a wave, so that short rows fill it, or to a whole
// block. The variance is the mean of squared distances from the mean, both from
// registers, so a mean far from zero costs no digits. Rows may start at any
// alignment of their elements.
//
// Backward, with n = (x - mean) rstd and g = dy weight:
//   dx = rstd (g - mean(g) - n mean(g n)),  dweight = sum dy n,  dbias = sum dy
// over the rows. The lane that holds a column in one row holds it in the
// block's every row, so the sums over rows stay in registers; each block then
// writes one row of sums and a second launch adds those in their order.
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

#include <algorithm>

#include "sequence.hpp"
#include "vkfx.h"

namespace vkfx {

namespace {

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

// Makes the compiler take `r` for new: where it is used again it is converted
// once more, rather than kept in 32 bits from the first time.
template <typename T, int N>
__device__ __forceinline__ void again(Some<T, N>& r) {
    typedef unsigned words __attribute__((ext_vector_type(sizeof(r) / 4)));
    words w = __builtin_bit_cast(words, r);
    asm volatile("" : "+v"(w));
    r = __builtin_bit_cast(Some<T, N>, w);
}

// Sum over the LPR threads of a row, the same on each. Rows wider than a wave
// meet in `lds`, of which every call takes the other half: one barrier each.
template <int LPR, int N>
__device__ __forceinline__ void row_sum(float (&v)[N], float* lds, int& half) {
#pragma unroll
    for (int o = 1; o < (LPR < 64 ? LPR : 64); o <<= 1)
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] += __shfl_xor(v[i], o);
    if constexpr (LPR > 64) {
        constexpr int waves = LPR / 64;
        const int wave = threadIdx.x >> 6, all = blockDim.x >> 6;
        float* at = lds + half * all * N;
        half ^= 1;
        if ((threadIdx.x & 63) == 0)
#pragma unroll
            for (int i = 0; i < N; ++i) at[wave * N + i] = v[i];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; ++i) {
            v[i] = 0.f;
#pragma unroll
            for (int w = 0; w < waves; ++w) v[i] += at[(wave / waves * waves + w) * N + i];
        }
    }
}

// LPR threads a row, NV vectors each, NT threads a block.
template <typename T, typename W, int LPR, int NV, int NT>
__global__ __launch_bounds__(NT) void k_norm_forward(const NormArgs a) {
    constexpr int V = kVector<T>, R = NT / LPR;
    __shared__ float lds[2 * (NT / 64)];
    int half = 0;
    const int lane = threadIdx.x % LPR, group = threadIdx.x / LPR;
    Some<W, V> w[NV], b[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int c = (j * LPR + lane) * V;
#pragma unroll
        for (int e = 0; e < V; ++e) w[j][e] = (W)1.f, b[j][e] = (W)0.f;
        if (a.weight) w[j] = load_some<W, V>((const W*)a.weight, c, a.width);
        if (a.bias) b[j] = load_some<W, V>((const W*)a.bias, c, a.width);
    }
    Some<T, V> next[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) next[j] = (T)0.f;
    const auto fetch = [&](long long r) {
        if (r < a.rows)
#pragma unroll
            for (int j = 0; j < NV; ++j)
                next[j] = load_some<T, V>((const T*)a.x + r * a.x_stride, (j * LPR + lane) * V, a.width);
    };
    const float over = 1.f / (float)a.width;
    const long long stride = (long long)gridDim.x * R;
    constexpr bool kAhead = NT < 1024 || NV == 1;  // the next row on its way, where the registers hold it
    if constexpr (kAhead) fetch((long long)blockIdx.x * R + group);
    for (long long r0 = (long long)blockIdx.x * R; r0 < a.rows; r0 += stride) {
        const long long r = r0 + group;
        const bool live = r < a.rows;  // where not, the group still meets the block's barriers
        if constexpr (!kAhead) fetch(r);
        Some<T, V> x[NV];
#pragma unroll
        for (int j = 0; j < NV; ++j) x[j] = next[j];
        if constexpr (kAhead) fetch(r + stride);
        float s[1] = {0.f};
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int e = 0; e < V; ++e) s[0] += (float)x[j][e];
        row_sum<LPR>(s, lds, half);
        const float mean = s[0] * over;
        s[0] = 0.f;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int left = a.width - (j * LPR + lane) * V;
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float d = e < left ? (float)x[j][e] - mean : 0.f;
                s[0] = fmaf(d, d, s[0]);
            }
        }
        row_sum<LPR>(s, lds, half);
        const float rstd = 1.f / sqrtf(fmaf(s[0], over, a.epsilon));
        if (!live) continue;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            Some<T, V> y;
#pragma unroll
            for (int e = 0; e < V; ++e) y[e] = (T)fmaf(((float)x[j][e] - mean) * rstd, (float)w[j][e], (float)b[j][e]);
            store_some<T, V>((T*)a.y + r * a.y_stride, (j * LPR + lane) * V, a.width, y);
        }
        if (a.stats_out && lane == 0) {
            a.stats_out[2 * r] = mean;
            a.stats_out[2 * r + 1] = rstd;
        }
    }
}

// Floats in which half of a block's row groups hand the other half their sums,
// both kinds at a time where that stays within 48 KB.
template <typename T, int LPR, int NV, int NT>
constexpr int kHalf = NT > LPR ? NV * LPR * kVector<T> * (LPR < 64 ? NT / 64 : NT / LPR) / 2 : 0;
template <typename T, int LPR, int NV, int NT>
constexpr bool kSumsBoth = kHalf<T, LPR, NV, NT> * 8 <= 48 * 1024;
template <typename T, int LPR, int NV, int NT>
constexpr int kSums = kHalf<T, LPR, NV, NT> * (kSumsBoth<T, LPR, NV, NT> ? 2 : 1);

// SUMS: with the gradients of weight and bias. ADD: the blocks' sums are added
// to those that an earlier launch left in the workspace (as an argument of the
// kernel it costs calls of 10 us 0.3).
template <typename T, typename W, int LPR, int NV, int NT, bool SUMS, bool ADD>
__global__ __launch_bounds__(NT) void k_norm_backward(const NormArgs a) {
    constexpr int V = kVector<T>, R = NT / LPR;
    constexpr bool kAhead = NT < 1024 || NV == 1;  // the next row on its way, where the registers hold it
    extern __shared__ float sums[];  // kSums floats
    __shared__ float lds[4 * (NT / 64)];
    int half = 0;
    const int lane = threadIdx.x % LPR, group = threadIdx.x / LPR;
    Some<W, V> w[NV];
    float dw[NV][V], db[NV][V];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
#pragma unroll
        for (int e = 0; e < V; ++e) w[j][e] = (W)1.f, dw[j][e] = db[j][e] = 0.f;
        if (kAhead && a.weight) w[j] = load_some<W, V>((const W*)a.weight, (j * LPR + lane) * V, a.width);
    }
    // the weights, from registers or, where the sums take those, from the cache
    const auto weight = [&](int j) {
        if constexpr (kAhead) return w[j];
        if (a.weight) return load_some<W, V>((const W*)a.weight, (j * LPR + lane) * V, a.width);
        return Some<W, V>((W)1.f);
    };
    Some<T, V> nx[NV], ng[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) nx[j] = ng[j] = (T)0.f;
    float nmean = 0.f, nrstd = 0.f;
    const auto fetch = [&](long long r) {
        if (r >= a.rows) return;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            nx[j] = load_some<T, V>((const T*)a.x + r * a.x_stride, (j * LPR + lane) * V, a.width);
            ng[j] = load_some<T, V>((const T*)a.dy + r * a.dy_stride, (j * LPR + lane) * V, a.width);
        }
        nmean = a.stats_in[2 * r];
        nrstd = a.stats_in[2 * r + 1];
    };
    const float over = 1.f / (float)a.width;
    const long long stride = (long long)gridDim.x * R;
    if constexpr (kAhead) fetch((long long)blockIdx.x * R + group);
    for (long long r0 = (long long)blockIdx.x * R; r0 < a.rows; r0 += stride) {
        const long long r = r0 + group;
        const bool live = r < a.rows;
        if constexpr (!kAhead) fetch(r);
        Some<T, V> x[NV], dy[NV];
#pragma unroll
        for (int j = 0; j < NV; ++j) x[j] = nx[j], dy[j] = ng[j];
        const float mean = nmean, rstd = nrstd;
        if constexpr (kAhead) fetch(r + stride);
        float s[2] = {0.f, 0.f};
        if (live)
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const Some<W, V> wj = weight(j);
#pragma unroll
                for (int e = 0; e < V; ++e) {  // past the row's end dy is zero
                    const float n = ((float)x[j][e] - mean) * rstd, d = (float)dy[j][e], g = d * (float)wj[e];
                    if constexpr (SUMS) {
                        dw[j][e] = fmaf(d, n, dw[j][e]);
                        db[j][e] += d;
                    }
                    s[0] += g;
                    s[1] = fmaf(g, n, s[1]);
                }
            }
        if (!a.y) continue;
        row_sum<LPR>(s, lds, half);
        if (!live) continue;
        const float m1 = s[0] * over, m2 = s[1] * over;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            Some<T, V> dx;
            if constexpr (!SUMS) again<T, V>(x[j]), again<T, V>(dy[j]);
            const Some<W, V> wj = weight(j);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float n = ((float)x[j][e] - mean) * rstd, g = (float)dy[j][e] * (float)wj[e];
                dx[e] = (T)((g - m1 - n * m2) * rstd);
            }
            store_some<T, V>((T*)a.y + r * a.y_stride, (j * LPR + lane) * V, a.width, dx);
        }
    }
    if (!SUMS || (!a.dweight && !a.dbias)) return;
    // the block's rows side by side: lanes of a wave, then its waves one after the other
    if constexpr (LPR < 64)
#pragma unroll
        for (int o = LPR; o < 64; o <<= 1)
#pragma unroll
            for (int j = 0; j < NV; ++j)
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    dw[j][e] += __shfl_xor(dw[j][e], o);
                    db[j][e] += __shfl_xor(db[j][e], o);
                }
    if constexpr (R > 1) {
        // by halves: the upper ones hand their sums to the lower ones
        constexpr int parts = LPR < 64 ? NT / 64 : R;
        const int part = LPR < 64 ? (int)(threadIdx.x >> 6) : group;
        const bool mine = LPR >= 64 || (threadIdx.x & 63) < LPR;
        const auto at = [&](int p, int j, int e) { return ((p * V + e) * NV + j) * LPR + lane; };
#pragma unroll
        for (int h = parts / 2; h; h >>= 1) {
            constexpr int D = parts / 2 * LPR * NV * V;
#pragma unroll
            for (int both = kSumsBoth<T, LPR, NV, NT> ? 1 : 2, i = 0; i < both; ++i) {
                const bool w = both == 1 || i == 0, b = both == 1 || i == 1;
                const int second = both == 1 ? D : 0;
                if (part >= h && part < 2 * h && mine)
#pragma unroll
                    for (int j = 0; j < NV; ++j)
#pragma unroll
                        for (int e = 0; e < V; ++e) {
                            if (w) sums[at(part - h, j, e)] = dw[j][e];
                            if (b) sums[at(part - h, j, e) + second] = db[j][e];
                        }
                __syncthreads();
                if (part < h && mine)
#pragma unroll
                    for (int j = 0; j < NV; ++j)
#pragma unroll
                        for (int e = 0; e < V; ++e) {
                            if (w) dw[j][e] += sums[at(part, j, e)];
                            if (b) db[j][e] += sums[at(part, j, e) + second];
                        }
                __syncthreads();
            }
        }
        if (part || !mine) return;
    }
    // one block: its sums are the gradients
    const bool last = a.parts == 1;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int c = (j * LPR + lane) * V;
        if (last) {
            Some<W, V> p, q;
#pragma unroll
            for (int e = 0; e < V; ++e) p[e] = (W)dw[j][e], q[e] = (W)db[j][e];
            if (a.dweight) store_some<W, V>((W*)a.dweight, c, a.width, p);
            if (a.dbias) store_some<W, V>((W*)a.dbias, c, a.width, q);
        } else {
            float *const w_at = a.partial + (long long)blockIdx.x * 2 * a.width, *const b_at = w_at + a.width;
            Some<float, V> p, q;
#pragma unroll
            for (int e = 0; e < V; ++e) p[e] = dw[j][e], q[e] = db[j][e];
            if constexpr (ADD) p += load_some<float, V>(w_at, c, a.width), q += load_some<float, V>(b_at, c, a.width);
            store_some<float, V>(w_at, c, a.width, p);
            store_some<float, V>(b_at, c, a.width, q);
        }
    }
}

// Adds the blocks' sums: 64 columns a block, its 16 waves each an equal share
// of the blocks in their order. blockIdx.y: weight or bias; blockIdx.z: columns
// past what a launch's threads along x can count.
template <typename W>
__global__ __launch_bounds__(1024) void k_norm_backward_sum(const NormArgs a, int parts) {
    __shared__ float lds[16][64];
    W* const to = (W*)(blockIdx.y ? a.dbias : a.dweight);
    if (!to) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const long long c = ((long long)blockIdx.z * gridDim.x + blockIdx.x) * 64 + lane;
    const int first = (int)((long long)parts * wave / 16), end = (int)((long long)parts * (wave + 1) / 16);
    float s = 0.f;
    if (c < a.width) {
        const float* p = a.partial + (long long)blockIdx.y * a.width + c;
#pragma unroll 8
        for (int i = first; i < end; ++i) s += p[(long long)i * 2 * a.width];
    }
    lds[wave][lane] = s;
    __syncthreads();
    if (wave || c >= a.width) return;
    s = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) s += lds[i][lane];
    to[c] = (W)s;
}

// ---- rows too wide for a block's registers: read once for each sum. A thread's
// own sums are long (a row of 2^20 elements gives it 1024 terms, which are added
// one by one), so they are in 64 bits: equal elements would round to one side
// each time.

template <typename T, typename W>
__global__ __launch_bounds__(1024) void k_norm_forward_wide(const NormArgs a) {
    __shared__ float lds[2 * 16];
    int half = 0;
    for (long long r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const T* x = (const T*)a.x + r * a.x_stride;
        T* y = (T*)a.y + r * a.y_stride;
        double sum = 0.0;
        for (int i = threadIdx.x; i < a.width; i += 1024) sum += (double)(float)x[i];
        float s[1] = {(float)sum};
        row_sum<1024>(s, lds, half);
        const float mean = s[0] / (float)a.width;
        sum = 0.0;
        for (int i = threadIdx.x; i < a.width; i += 1024) {
            const float d = (float)x[i] - mean;
            sum += (double)(d * d);
        }
        s[0] = (float)sum;
        row_sum<1024>(s, lds, half);
        const float rstd = 1.0f / sqrtf(s[0] / (float)a.width + a.epsilon);
        for (int i = threadIdx.x; i < a.width; i += 1024) {
            const float w = a.weight ? (float)((const W*)a.weight)[i] : 1.f;
            const float b = a.bias ? (float)((const W*)a.bias)[i] : 0.f;
            y[i] = (T)fmaf(((float)x[i] - mean) * rstd, w, b);
        }
        if (a.stats_out && threadIdx.x == 0) {
            a.stats_out[2 * r] = mean;
            a.stats_out[2 * r + 1] = rstd;
        }
    }
}

template <typename T, typename W>
__global__ __launch_bounds__(1024) void k_norm_backward_wide(const NormArgs a) {
    __shared__ float lds[4 * 16];
    int half = 0;
    for (long long r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const T* x = (const T*)a.x + r * a.x_stride;
        const T* dy = (const T*)a.dy + r * a.dy_stride;
        T* dx = (T*)a.y + r * a.y_stride;
        const float mean = a.stats_in[2 * r], rstd = a.stats_in[2 * r + 1];
        double sum = 0.0, product = 0.0;
        for (int i = threadIdx.x; i < a.width; i += 1024) {
            const float g = (float)dy[i] * (a.weight ? (float)((const W*)a.weight)[i] : 1.f);
            sum += (double)g;
            product += (double)(g * (((float)x[i] - mean) * rstd));
        }
        float s[2] = {(float)sum, (float)product};
        row_sum<1024>(s, lds, half);
        const float m1 = s[0] / (float)a.width, m2 = s[1] / (float)a.width;
        for (int i = threadIdx.x; i < a.width; i += 1024) {
            const float g = (float)dy[i] * (a.weight ? (float)((const W*)a.weight)[i] : 1.f);
            dx[i] = (T)((g - m1 - ((float)x[i] - mean) * rstd * m2) * rstd);
        }
    }
}

// Sums over every gridDim.y-th row, a thread four columns, in 64 bits: there may
// be many rows.
template <typename T>
__global__ __launch_bounds__(256) void k_norm_backward_wide_rows(const NormArgs a) {
    const int c = (blockIdx.x * 256 + threadIdx.x) * 4;
    if (c >= a.width) return;
    double w[4] = {}, b[4] = {};
    for (long long r = blockIdx.y; r < a.rows; r += gridDim.y) {
        const Some<T, 4> dy = load_some<T, 4>((const T*)a.dy + r * a.dy_stride, c, a.width);
        const Some<T, 4> x = load_some<T, 4>((const T*)a.x + r * a.x_stride, c, a.width);
        const float mean = a.stats_in[2 * r], rstd = a.stats_in[2 * r + 1];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            w[e] += (double)((float)dy[e] * (((float)x[e] - mean) * rstd));
            b[e] += (double)(float)dy[e];
        }
    }
    Some<float, 4> dw, db;
#pragma unroll
    for (int e = 0; e < 4; ++e) dw[e] = (float)w[e], db[e] = (float)b[e];
    store_some<float, 4>(a.partial + (long long)blockIdx.y * 2 * a.width, c, a.width, dw);
    store_some<float, 4>(a.partial + ((long long)blockIdx.y * 2 + 1) * a.width, c, a.width, db);
}

template <typename W>
void launch_sum(const NormArgs& a, int parts, hipStream_t s) {
    const unsigned blocks = (unsigned)((a.width + 63) / 64), x = std::min(blocks, 1u << 21);
    hipLaunchKernelGGL((k_norm_backward_sum<W>), dim3(x, 2, (blocks + x - 1) / x), dim3(1024), 0, s, a, parts);
}

// Whether a row's sums over the rows stay in a block's registers.
bool sums_in_registers(int element, int width) {
    return element == VKFX_ELEMENT_F32 ? width <= 4096 * kVector<float> : width <= 2048 * kVector<_Float16>;
}

// Rows of sums that the rows of a wider one are split over: 64, and fewer where
// the columns alone fill the GPU (gradients of 64 rows of 2^20 f32: 1336 us with the
// 4 that this gives, 1542 with 64).
int wide_parts(int width) { return std::max(1, std::min(64, (1 << 22) / width)); }

template <typename T, typename W, int LPR, int NV, int NT>
int forward_with(const NormArgs& a, hipStream_t s) {
    constexpr int R = NT / LPR;
    // blocks that fill the CUs; further rows in their loop, which reads a row ahead
    const long long blocks = std::min((a.rows + R - 1) / R, (long long)a.cus * (2048 / NT));
    hipLaunchKernelGGL((k_norm_forward<T, W, LPR, NV, NT>), dim3((unsigned)blocks), dim3(NT), 0, s, a);
    return (int)hipGetLastError();
}

// Equal numbers round to one side wherever they are added one by one: 512 are off by up to 7.6e-6 of their sum, 64
// by 1e-6.
constexpr int kTurns = 64;

template <typename T, typename W, int LPR, int NV, int NT, bool SUMS = true>
int backward_with(const NormArgs& a, hipStream_t s) {
    constexpr int R = NT / LPR;
    // one block a CU: every block costs a row of sums to write and to add
    const auto blocks_of = [&](long long rows) { return std::min((rows + R - 1) / R, (long long)a.cus); };
    constexpr size_t lds = sizeof(float) * kSums<T, LPR, NV, NT>;
    const bool sums = SUMS && (a.dweight || a.dbias);
    NormArgs b = a;
    b.parts = (int)blocks_of(a.rows);
    // A launch's groups add at most kTurns rows one after the other, then the next launch adds to the same rows of sums
    const long long most = sums ? (long long)a.cus * R * kTurns : a.rows;
    for (long long first = 0; first < a.rows; first += most) {
        b.rows = std::min(a.rows - first, most);
        const auto kernel = first ? k_norm_backward<T, W, LPR, NV, NT, SUMS, SUMS> : k_norm_backward<T, W, LPR, NV, NT, SUMS, false>;
        hipLaunchKernelGGL(kernel, dim3((unsigned)blocks_of(b.rows)), dim3(NT), lds, s, b);
        b.x = (const T*)b.x + most * a.x_stride;
        b.dy = (const T*)b.dy + most * a.dy_stride;
        b.y = b.y ? (T*)b.y + most * a.y_stride : nullptr;
        b.stats_in += 2 * most;
    }
    if (sums && b.parts > 1) launch_sum<W>(a, b.parts, s);
    return (int)hipGetLastError();
}

// By vectors in a row: lanes of a wave as long as a lane's vectors fit its
// registers well, then a block.
template <typename T, typename W>
int forward_as(const NormArgs& a, hipStream_t s) {
    const int n = (a.width + kVector<T> - 1) / kVector<T>;
    if (n <= 8) return forward_with<T, W, 8, 1, 256>(a, s);
    if (n <= 16) return forward_with<T, W, 16, 1, 256>(a, s);
    if (n <= 32) return forward_with<T, W, 32, 1, 256>(a, s);
    if (n <= 64) return forward_with<T, W, 64, 1, 256>(a, s);
    if (n <= 128) return forward_with<T, W, 128, 1, 256>(a, s);
    if (n <= 256) return forward_with<T, W, 256, 1, 256>(a, s);
    if (n <= 512) return forward_with<T, W, 512, 1, 512>(a, s);
    if (n <= 1024) return forward_with<T, W, 512, 2, 512>(a, s);
    if (n <= 2048) return forward_with<T, W, 512, 4, 512>(a, s);
    if (n <= 4096) return forward_with<T, W, 1024, 4, 1024>(a, s);
    hipLaunchKernelGGL((k_norm_forward_wide<T, W>), dim3((unsigned)std::min(a.rows, (long long)a.cus * 2)), dim3(1024), 0, s, a);
    return (int)hipGetLastError();
}

template <typename T, typename W>
int backward_as(const NormArgs& a, hipStream_t s) {
    if (!a.rows) {
        if (a.dweight || a.dbias) launch_sum<W>(a, 0, s);
        return (int)hipGetLastError();
    }
    const int n = (a.width + kVector<T> - 1) / kVector<T>;
    if (n <= 8) return backward_with<T, W, 8, 1, 1024>(a, s);
    if (n <= 16) return backward_with<T, W, 16, 1, 1024>(a, s);
    if (n <= 32) return backward_with<T, W, 32, 1, 1024>(a, s);
    if (n <= 64) return backward_with<T, W, 64, 1, 1024>(a, s);
    if (n <= 128) return backward_with<T, W, 64, 2, 512>(a, s);
    if (n <= 256) return backward_with<T, W, 256, 1, 1024>(a, s);
    if (n <= 512) return backward_with<T, W, 512, 1, 1024>(a, s);
    if (n <= 1024) return backward_with<T, W, 256, 4, 512>(a, s);
    if (n <= 2048) return backward_with<T, W, 512, 4, 512>(a, s);
    if constexpr (sizeof(T) == 4)
        if (sums_in_registers(a.element, a.width)) return backward_with<T, W, 1024, 4, 1024>(a, s);
    // dx may overwrite dy: the sums over the rows go first
    if (a.dweight || a.dbias) {
        const int parts = (int)std::min(a.rows, (long long)wide_parts(a.width));
        hipLaunchKernelGGL((k_norm_backward_wide_rows<T>), dim3((unsigned)((a.width + 1023) / 1024), parts), dim3(256), 0, s, a);
        launch_sum<W>(a, parts, s);
    }
    if (!a.y) return (int)hipGetLastError();
    if constexpr (sizeof(T) < 4)
        if (n <= 4096) return backward_with<T, W, 1024, 4, 1024, false>(a, s);
    hipLaunchKernelGGL((k_norm_backward_wide<T, W>), dim3((unsigned)std::min(a.rows, (long long)a.cus * 2)), dim3(1024), 0, s, a);
    return (int)hipGetLastError();
}

template <typename T>
int pick(const NormArgs& a, hipStream_t s, bool forward) {
    if (a.weight_element == VKFX_ELEMENT_F32) return forward ? forward_as<T, float>(a, s) : backward_as<T, float>(a, s);
    return forward ? forward_as<T, T>(a, s) : backward_as<T, T>(a, s);
}

int pick_element(const NormArgs& a, hipStream_t s, bool forward) {
    if (a.element == VKFX_ELEMENT_F32) return pick<float>(a, s, forward);
    if (a.element == VKFX_ELEMENT_F16) return pick<_Float16>(a, s, forward);
    return pick<__bf16>(a, s, forward);
}

}  // namespace

int launch_norm_forward(const NormArgs& a, hipStream_t s) { return pick_element(a, s, true); }
int launch_norm_backward(const NormArgs& a, hipStream_t s) { return pick_element(a, s, false); }
size_t norm_workspace_bytes(int element, int width, int cus) {
    return (size_t)(sums_in_registers(element, width) ? cus : wide_parts(width)) * 2 * (size_t)width * sizeof(float);
}

}  // namespace vkfx
