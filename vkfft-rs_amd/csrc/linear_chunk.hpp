// linear_chunk.hpp -- linear attention over many tokens, chunk by chunk on the
// matrix cores. Instantiated per element type in linear_f32/f16/bf16.hip.
//
// For a chunk of C tokens and the state X before it (sequence.hpp has the
// scan's definition; g the head's decay, n <= C the tokens that are left):
//   P[i][j] = scale_update g^(i-j) (A[i] . B[j])           for j <= i, else 0
//   out[i]  = scale_in ( g^(i+1-lead) A[i] X + sum_j P[i][j] C[j] )
//   X      <- g^n X + scale_update sum_j g^(n-1-j+lead) B[j] C[j]^T
// four products of small matrices, all on mfma 16x16x32 bf16 with f32 sums.
//
// Operands of more than 8 bits are sums of bf16 parts: an f16 value is two
// parts exactly, an f32 value three, and so are P, X and the weighted C:
// P and X take two parts where the output has 16 bits (2^-17 of a term is lost,
// the output itself keeps 2^-9 or 2^-12) and three for f32; the state's own
// update takes three always, since the state is an f32 result. Products of
// parts that lie below the kept bits are left out.
//
// Four waves share the chunk's A, B, C and P in LDS. Each wave owns 16 NT of
// the block's 64 NT columns of C, X and out, so that X stays in its
// accumulators from the first token to the last. The layout of accumulators
// (lane: one column, four rows) is that of an operand (lane: one row or column,
// eight along the summed axis) when that axis is taken in the order 0-3, 16-19
// of lane group 0, 4-7, 20-23 of group 1, ...: X enters A X without moving, and
// A and B are read from LDS in that order. out is formed transposed, so that a
// lane holds four neighbours of one token. Operands summed over tokens (C in
// P C, B and C in the update) come from LDS by transposing reads.
#pragma once

#include <hip/hip_runtime.h>

#include "sequence.hpp"

namespace vkfx {

typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x8 __attribute__((ext_vector_type(8)));

struct ChunkArgs {
    ScanArgs scan[3];
    int scans;
    int slices;     // blocks side by side over dv
    int segments;   // parts of the tokens, each `segment` long (a multiple of the chunk)
    long long segment;
    float* slots;   // segments > 1: [scan][batch][head][segment][dk][dv] states before each segment
    const float* powers;
};

template <typename T>
struct Parts;  // bf16 parts of an input, and of P and X
template <>
struct Parts<__bf16> {
    static constexpr int in = 1, mid = 2;
};
template <>
struct Parts<_Float16> {
    static constexpr int in = 2, mid = 2;
};
template <>
struct Parts<float> {
    static constexpr int in = 3, mid = 3;
};

__device__ __forceinline__ f32x4 mma(bf16x8 a, bf16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// Sum of the products of parts whose orders add up to less than `orders`.
template <int N, int M>
__device__ __forceinline__ f32x4 mma_parts(const bf16x8 (&a)[N], const bf16x8 (&b)[M], f32x4 c, int orders) {
#pragma unroll
    for (int o = N + M - 2; o >= 0; --o)  // small ones first
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int j = 0; j < M; ++j)
                if (i + j == o && o < orders) c = mma(a[i], b[j], c);
    return c;
}

template <int N>
__device__ __forceinline__ void split8(const float (&x)[8], bf16x8 (&p)[N]) {
    float r[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) r[e] = x[e];
#pragma unroll
    for (int i = 0; i < N; ++i) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            p[i][e] = (__bf16)r[e];
            if (i + 1 < N) r[e] -= (float)p[i][e];
        }
    }
}

// Eight neighbours of a row at any alignment of its elements.
template <typename T>
struct __attribute__((packed, aligned(sizeof(T)))) Eight {
    T v[8];
};

// One thread's share of a chunk of rows [C][D] on its way to LDS: vectors of
// eight elements, read ahead while the chunk before is worked on.
template <typename T, int C, int D>
struct Staged {
    static constexpr int kVectors = C * D / 8;
    static constexpr int kEach = (kVectors + 255) / 256;
    Eight<T> r[kEach];

    // rows: tokens first .. first + n - 1 (in scan order), zeros from there on
    __device__ __forceinline__ void load(const T* base, long long token, long long first, int n, int step, int col0, int dim) {
#pragma unroll
        for (int u = 0; u < kEach; ++u) {
            const int v = (int)threadIdx.x + 256 * u;
            const int row = v / (D / 8), c = col0 + v % (D / 8) * 8;
            if ((kVectors % 256 == 0 || v < kVectors) && row < n && c + 8 <= dim) {
                r[u] = *(const Eight<T>*)(base + (first + (long long)step * row) * token + c);
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) r[u].v[e] = (T)0.f;
                if ((kVectors % 256 == 0 || v < kVectors) && row < n && c < dim) {
                    const T* p = base + (first + (long long)step * row) * token + c;
#pragma unroll
                    for (int e = 0; e < 7; ++e)
                        if (c + e < dim) r[u].v[e] = p[e];
                }
            }
        }
    }

    // to lds[part][C][pitch]
    __device__ __forceinline__ void store(__bf16* lds, int pitch) const {
#pragma unroll
        for (int u = 0; u < kEach; ++u) {
            const int v = (int)threadIdx.x + 256 * u;
            if (kVectors % 256 != 0 && v >= kVectors) continue;
            __bf16* to = lds + v / (D / 8) * pitch + v % (D / 8) * 8;
            if constexpr (Parts<T>::in == 1) {
                bf16x8 p;
#pragma unroll
                for (int e = 0; e < 8; ++e) p[e] = r[u].v[e];
                *(bf16x8*)to = p;
            } else {
                float x[8];
                bf16x8 p[Parts<T>::in];
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = (float)r[u].v[e];
                split8(x, p);
#pragma unroll
                for (int i = 0; i < Parts<T>::in; ++i) *(bf16x8*)(to + i * C * pitch) = p[i];
            }
        }
    }
};

// Row `row` of a matrix in LDS as an operand: elements k0 + (0-3, 16-19) + 4 g.
__device__ __forceinline__ bf16x8 row_operand(const __bf16* m, int pitch, int row, int k0, int g) {
    const bf16x4 a = *(const bf16x4*)(m + row * pitch + k0 + 4 * g);
    const bf16x4 b = *(const bf16x4*)(m + row * pitch + k0 + 16 + 4 * g);
    return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
}

// Column c0 + lane % 16 of a matrix in LDS as an operand over the rows
// r0 + 8 g .. + 7: two transposing reads of 4 rows x 16 columns a lane group.
__device__ __forceinline__ bf16x8 column_operand(const __bf16* m, int pitch, int r0, int c0, int lane) {
    typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
    const __bf16* p = m + (r0 + 8 * (lane >> 4) + ((lane & 15) >> 2)) * pitch + c0 + 4 * (lane & 3);
    const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)p);
    const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p + 4 * pitch));
    return __builtin_bit_cast(bf16x8, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
}

template <typename T, int DK, int NT, int C>
struct ChunkShape {
    static constexpr int kIn = Parts<T>::in, kMid = Parts<T>::mid;
    static constexpr int kCols = 64 * NT;
    // 16 bytes more a row: a quarter wave's 8-byte reads down the rows meet different banks
    static constexpr int kPitchK = DK + 8, kPitchV = kCols + 8, kPitchP = C + 8;
    static constexpr size_t kA = 0, kB = kA + (size_t)kIn * C * kPitchK, kC = kB + (size_t)kIn * C * kPitchK,
                            kP = kC + (size_t)kIn * C * kPitchV, kEnd = kP + (size_t)kMid * C * kPitchP;
    static constexpr size_t kLds = kEnd * 2 + kDecayPowers * 4 + 16;
};

template <typename T, int DK, int NT, int C, bool STATE_ONLY>
__global__ __launch_bounds__(256, 2) void k_chunk(const ChunkArgs args) {
    using S = ChunkShape<T, DK, NT, C>;
    constexpr int IN = S::kIn, MID = S::kMid, TI = C / 16;
    extern __shared__ __align__(16) char lds[];
    __bf16* const la = (__bf16*)lds + S::kA;
    __bf16* const lb = (__bf16*)lds + S::kB;
    __bf16* const lc = (__bf16*)lds + S::kC;
    __bf16* const lp = (__bf16*)lds + S::kP;
    float* const pw = (float*)((__bf16*)lds + S::kEnd);

    // block -> (scan, sequence, head, segment, slice), slices side by side
    long long id = blockIdx.x;
    const int slice = (int)(id % args.slices);
    id /= args.slices;
    const int seg = (int)(id % args.segments);
    id /= args.segments;
    const int h = (int)(id % args.scan[0].heads);
    id /= args.scan[0].heads;
    const int b = (int)(id % args.scan[0].batch);
    const int z = (int)(id / args.scan[0].batch);
    const ScanArgs& s = args.scan[z];

    long long n = s.tokens;
    if (s.lengths) {
        const long long l = s.lengths[b];
        n = l < 0 ? 0 : l < n ? l : n;
    }
    const long long begin = seg * args.segment;
    const long long end = begin + args.segment < s.tokens ? begin + args.segment : s.tokens;
    // a state before the next segment is needed only where that one has tokens
    if (STATE_ONLY && begin + args.segment >= n) return;

    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int g = lane >> 4, l16 = lane & 15;
    const int col0 = slice * S::kCols, wcol = wave * 16 * NT;
    const int lead = s.reverse;
    if (tid < kDecayPowers) pw[tid] = args.powers[(long long)h * kDecayPowers + tid];
    if (!STATE_ONLY)  // tiles of P right of the diagonal that a product of 32 tokens meets
        for (int i = tid; i < MID * C * S::kPitchP; i += 256) lp[i] = (__bf16)0.f;

    const T* const A = (const T*)s.a.p + b * s.a.batch + (h / s.a.group) * s.a.head;
    const T* const B = (const T*)s.b.p + b * s.b.batch + (h / s.b.group) * s.b.head;
    const T* const Cc = (const T*)s.c.p + b * s.c.batch + (h / s.c.group) * s.c.head;
    const int step = s.reverse ? -1 : 1;
    const auto token_of = [&](long long i) { return s.reverse ? n - 1 - i : i; };

    // the state: rows 16 a + 4 g + r, columns col0 + wcol + 16 t + l16
    f32x4 X[DK / 16][NT];
    const long long head_state = ((long long)b * s.heads + h) * s.dk * s.dv;
    float* const slot = args.slots + ((((long long)z * s.batch + b) * s.heads + h) * args.segments + seg) * s.dk * s.dv;
    {
        const float* from = STATE_ONLY ? nullptr : args.segments > 1 ? slot : s.state_in ? s.state_in + head_state : nullptr;
        const bool native = args.segments > 1;
        const int sr = native ? s.dv : s.state_row, sc = native ? 1 : s.state_col;
#pragma unroll
        for (int a = 0; a < DK / 16; ++a)
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int row = 16 * a + 4 * g + r, col = col0 + wcol + 16 * t + l16;
                    X[a][t][r] = from && row < s.dk && col < s.dv ? from[(long long)row * sr + (long long)col * sc] : 0.f;
                }
    }

    Staged<T, C, DK> sa, sb;
    Staged<T, C, S::kCols> sc;
    const auto fetch = [&](long long at) {
        const int left = (int)(n - at < C ? (n - at > 0 ? n - at : 0) : C);
        const long long first = token_of(at);
        if (!STATE_ONLY) sa.load(A, s.a.token, first, left, step, 0, s.dk);
        sb.load(B, s.b.token, first, left, step, 0, s.dk);
        sc.load(Cc, s.c.token, first, left, step, col0, s.dv);
    };

    long long at = begin;
    if (at < n) fetch(at);
    for (; at < end && at < n; at += C) {
        const int left = (int)(n - at < C ? n - at : C);
        __syncthreads();  // the chunk before has been read
        if (!STATE_ONLY) sa.store(la, S::kPitchK);
        sb.store(lb, S::kPitchK);
        sc.store(lc, S::kPitchV);
        __syncthreads();
        if (at + C < end && at + C < n) fetch(at + C);

        f32x4 o[TI][NT];
        if constexpr (!STATE_ONLY) {
            // P, transposed: rows j, columns i; the tiles on and left of the diagonal dealt to the waves
            int tile = 0;
#pragma unroll
            for (int I = 0; I < TI; ++I)
#pragma unroll
                for (int J = 0; J <= I; ++J, ++tile) {
                    if ((tile & 3) != wave) continue;
                    f32x4 p = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int k = 0; k < DK / 32; ++k) {
                        bf16x8 bj[IN], ai[IN];
#pragma unroll
                        for (int i = 0; i < IN; ++i) {
                            bj[i] = row_operand(lb + i * C * S::kPitchK, S::kPitchK, 16 * J + l16, 32 * k, g);
                            ai[i] = row_operand(la + i * C * S::kPitchK, S::kPitchK, 16 * I + l16, 32 * k, g);
                        }
                        p = mma_parts(bj, ai, p, IN == 3 ? 3 : 2);
                    }
                    const int i = 16 * I + l16, j0 = 16 * J + 4 * g;
                    bf16x4 q[MID];
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int d = i - (j0 + r);
                        float x = d < 0 ? 0.f : p[r] * (pw[d < 0 ? 0 : d] * s.scale_update);
#pragma unroll
                        for (int m = 0; m < MID; ++m) {
                            q[m][r] = (__bf16)x;
                            x -= (float)q[m][r];
                        }
                    }
#pragma unroll
                    for (int m = 0; m < MID; ++m) *(bf16x4*)(lp + (m * C + i) * S::kPitchP + j0) = q[m];
                }

            // out = A X, transposed
#pragma unroll
            for (int I = 0; I < TI; ++I)
#pragma unroll
                for (int t = 0; t < NT; ++t) o[I][t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int k = 0; k < DK / 32; ++k) {
                bf16x8 x[NT][MID];
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    float v[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[e] = X[2 * k + e / 4][t][e % 4];
                    split8(v, x[t]);
                }
#pragma unroll
                for (int I = 0; I < TI; ++I) {
                    bf16x8 ai[IN];
#pragma unroll
                    for (int i = 0; i < IN; ++i)
                        ai[i] = row_operand(la + i * C * S::kPitchK, S::kPitchK, 16 * I + l16, 32 * k, g);
#pragma unroll
                    for (int t = 0; t < NT; ++t) o[I][t] = mma_parts(x[t], ai, o[I][t], MID);
                }
            }
#pragma unroll
            for (int I = 0; I < TI; ++I) {
                const float w = pw[16 * I + l16 + 1 - lead];
#pragma unroll
                for (int t = 0; t < NT; ++t) o[I][t] *= w;
            }
            __syncthreads();  // P is written
        }

        const float whole = pw[left];
#pragma unroll
        for (int a = 0; a < DK / 16; ++a)
#pragma unroll
            for (int t = 0; t < NT; ++t) X[a][t] *= whole;
#pragma unroll
        for (int k = 0; k < C / 32; ++k) {
            bf16x8 cv[NT][IN], cw[NT][3];
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int i = 0; i < IN; ++i)
                    cv[t][i] = column_operand(lc + i * C * S::kPitchV, S::kPitchV, 32 * k, wcol + 16 * t, lane);
            if constexpr (!STATE_ONLY) {
#pragma unroll
                for (int I = 2 * k; I < TI; ++I) {
                    bf16x8 p[MID];
#pragma unroll
                    for (int m = 0; m < MID; ++m)
                        p[m] = *(const bf16x8*)(lp + (m * C + 16 * I + l16) * S::kPitchP + 32 * k + 8 * g);
#pragma unroll
                    for (int t = 0; t < NT; ++t) o[I][t] = mma_parts(cv[t], p, o[I][t], MID);
                }
            }
            float w[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int d = left - 1 - (32 * k + 8 * g + e) + lead;
                w[e] = pw[d < 0 ? 0 : d] * s.scale_update;
            }
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                float v[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    v[e] = 0.f;
#pragma unroll
                    for (int i = IN - 1; i >= 0; --i) v[e] += (float)cv[t][i][e];
                    v[e] *= w[e];
                }
                split8(v, cw[t]);
            }
#pragma unroll
            for (int a = 0; a < DK / 16; ++a) {
                bf16x8 bt[IN];
#pragma unroll
                for (int i = 0; i < IN; ++i) bt[i] = column_operand(lb + i * C * S::kPitchK, S::kPitchK, 32 * k, 16 * a, lane);
#pragma unroll
                for (int t = 0; t < NT; ++t) X[a][t] = mma_parts(bt, cw[t], X[a][t], 3);
            }
        }

        if constexpr (!STATE_ONLY) {
#pragma unroll
            for (int I = 0; I < TI; ++I) {
                const int i = 16 * I + l16;
                if (i >= left) continue;
                const long long row = b * s.out_batch + token_of(at + i) * s.out_token + h * s.out_head;
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    const int c = col0 + wcol + 16 * t + 4 * g;
                    const f32x4 y = o[I][t] * s.scale_in;
                    if (s.out_f32) {
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            if (c + r < s.dv) ((float*)s.out)[row + c + r] = y[r];
                    } else if (c + 4 <= s.dv) {
                        struct __attribute__((packed, aligned(sizeof(T)))) Four {
                            T v[4];
                        } f;
#pragma unroll
                        for (int r = 0; r < 4; ++r) f.v[r] = (T)y[r];
                        *(Four*)((T*)s.out + row + c) = f;
                    } else {
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            if (c + r < s.dv) ((T*)s.out)[row + c + r] = (T)y[r];
                    }
                }
            }
        }
    }

    if constexpr (STATE_ONLY) {
        // what this segment adds goes to the next one's slot
        float* const to = slot + (long long)s.dk * s.dv;
#pragma unroll
        for (int a = 0; a < DK / 16; ++a)
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int row = 16 * a + 4 * g + r, col = col0 + wcol + 16 * t + l16;
                    if (row < s.dk && col < s.dv) to[(long long)row * s.dv + col] = X[a][t][r];
                }
        return;
    }
    // rows past the sequence's length
    for (long long i = (begin > n ? begin : n) + wave; i < end; i += 4) {
        const long long row = b * s.out_batch + i * s.out_token + h * s.out_head;
        for (int c = col0 + lane; c < s.dv && c < col0 + S::kCols; c += 64) {
            if (s.out_f32) ((float*)s.out)[row + c] = 0.f;
            else ((T*)s.out)[row + c] = (T)0.f;
        }
    }
    if (s.state_out && seg == (n > 0 ? (n - 1) / args.segment : 0)) {
#pragma unroll
        for (int a = 0; a < DK / 16; ++a)
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int row = 16 * a + 4 * g + r, col = col0 + wcol + 16 * t + l16;
                    if (row < s.dk && col < s.dv)
                        s.state_out[head_state + (long long)row * s.state_row + (long long)col * s.state_col] = X[a][t][r];
                }
    }
}

// Joins the segments: slot 0 = state_in, slot k+1 = g^segment slot k + what
// segment k added (which the slot holds).
__global__ void k_chunk_join(const ChunkArgs args);

struct ChunkKernel {
    int dk, cols, chunk;  // padded key width, columns of a block, tokens of a chunk
    size_t lds;
    const void* run;
    const void* state_only;
};
// The element's kernel for a scan of dk x dv.
const ChunkKernel* chunk_kernel_f32(int dk, int dv);
const ChunkKernel* chunk_kernel_f16(int dk, int dv);
const ChunkKernel* chunk_kernel_bf16(int dk, int dv);

template <typename T, int DK, int NT, int C>
ChunkKernel chunk_kernel_of() {
    return ChunkKernel{DK, 64 * NT, C, ChunkShape<T, DK, NT, C>::kLds, (const void*)k_chunk<T, DK, NT, C, false>,
                       (const void*)k_chunk<T, DK, NT, C, true>};
}

// Key widths are padded to one of six. Blocks take 128 columns where there are
// more than 64 and the state of 128 rows or fewer still fits the registers.
template <typename T, int C>
const ChunkKernel* pick_chunk_kernel(int dk, int dv) {
    static const ChunkKernel narrow[6] = {chunk_kernel_of<T, 32, 1, C>(),  chunk_kernel_of<T, 64, 1, C>(),
                                          chunk_kernel_of<T, 96, 1, C>(),  chunk_kernel_of<T, 128, 1, C>(),
                                          chunk_kernel_of<T, 192, 1, C>(), chunk_kernel_of<T, 256, 1, C>()};
    static const ChunkKernel wide[4] = {chunk_kernel_of<T, 32, 2, C>(), chunk_kernel_of<T, 64, 2, C>(),
                                        chunk_kernel_of<T, 96, 2, C>(), chunk_kernel_of<T, 128, 2, C>()};
    const int i = dk <= 32 ? 0 : dk <= 64 ? 1 : dk <= 96 ? 2 : dk <= 128 ? 3 : dk <= 192 ? 4 : 5;
    return dv > 64 && i < 4 ? &wide[i] : &narrow[i];
}

}  // namespace vkfx
