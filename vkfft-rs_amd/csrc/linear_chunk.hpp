// linear_chunk.hpp -- linear attention over many tokens, chunk by chunk on the
// matrix cores. Instantiated per element type in linear_f32/f16/bf16.hip.
//
// For a chunk of C tokens and the state X before it (sequence.hpp has the
// scan's definition; g the head's decay, n <= C the tokens that are left):
//   P[i][j] = scale_in scale_update g^(i-j) (A[i] . B[j])           for j <= i, else 0
//   out[i]  = scale_in g^(i+1-lead) A[i] X + sum_j P[i][j] C[j]
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
// A block's waves share the chunk's A, B, C and P in LDS. Each owns 16 NT
// columns of C, X and out, so that X stays in its accumulators from the first
// token to the last. The layout of accumulators
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

// The decay of n tokens, by squaring, from a head's table.
__device__ __forceinline__ double decay_of(const float* powers, long long n) {
    double power = 1.0, square = (double)powers[kDecayHigh] + (double)powers[kDecayLow];
    for (long long i = n; i; i >>= 1, square *= square)
        if (i & 1) power *= square;
    return power;
}

// A number that is the same in every lane, held in scalar registers.
__device__ __forceinline__ double same_in_all(double x) {
    typedef int two __attribute__((ext_vector_type(2)));
    const two w = __builtin_bit_cast(two, x);
    return __builtin_bit_cast(double, two{__builtin_amdgcn_readfirstlane(w[0]), __builtin_amdgcn_readfirstlane(w[1])});
}

// Tokens of a chunk: what one product sums over. With 64 the state is split
// half as often, but o, the weights and what is read ahead take the registers of
// a second wave (bf16, 8 x 2048 tokens, 16 heads of 128: 157 us, with 32 90).
constexpr int kChunk = 32;

struct ChunkArgs {
    ScanArgs scan[3];
    int scans;
    long long blocks;  // of the launch: more than 2^32 threads take a second dimension of the grid
    int slices;     // blocks side by side over dv
    int segments;   // parts of the tokens, each `segment` long (a multiple of the chunk)
    long long segment;
    // segments > 1: each scan's [batch][head][segment][dk][dv], the state before each segment; until k_chunk_join ran,
    // from the third on what the segment before it adds. The first is state_in itself, or with in_place (another
    // block's state_out may then overwrite that) its copy. A scan whose state another one forms reads that transposed.
    float* slots[3];
    int slot_row[3], slot_col[3];
    int in_place;
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

// c[u] += sum of the products of a[u]'s and b[u]'s parts whose orders add up to
// less than `orders`, small ones first. One product of every u before the next:
// a product that adds to the one before it would wait for that.
template <int U, int N, int M>
__device__ __forceinline__ void mma_parts(const bf16x8 (&a)[U][N], const bf16x8 (&b)[U][M], f32x4 (&c)[U], int orders) {
#pragma unroll
    for (int o = N + M - 2; o >= 0; --o)
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int j = 0; j < M; ++j)
                if (i + j == o && o < orders)
#pragma unroll
                    for (int u = 0; u < U; ++u) c[u] = mma(a[u][i], b[u][j], c[u]);
}
// The same with one first operand for all.
template <int U, int N, int M>
__device__ __forceinline__ void mma_parts(const bf16x8 (&a)[N], const bf16x8 (&b)[U][M], f32x4* c, int orders) {
#pragma unroll
    for (int o = N + M - 2; o >= 0; --o)
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int j = 0; j < M; ++j)
                if (i + j == o && o < orders)
#pragma unroll
                    for (int u = 0; u < U; ++u) c[u] = mma(a[i], b[u][j], c[u]);
}
// And with one second operand for all.
template <int U, int N, int M>
__device__ __forceinline__ void mma_parts(const bf16x8 (&a)[U][N], const bf16x8 (&b)[M], f32x4* c, int orders) {
#pragma unroll
    for (int o = N + M - 2; o >= 0; --o)
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int j = 0; j < M; ++j)
                if (i + j == o && o < orders)
#pragma unroll
                    for (int u = 0; u < U; ++u) c[u] = mma(a[u][i], b[j], c[u]);
}

// x as a sum of N bf16 parts, each the rounding of what the ones before leave.
// SUMMED: elements that meet in one sum. There v_dot2_f32_bf16 takes a part off
// in one instruction, x - 1 p[0] - 0 p[1], exactly; elsewhere an infinite
// neighbour must not make that a NaN.
template <bool SUMMED, int N, int E, typename V>
__device__ __forceinline__ void split(const float (&x)[E], V (&p)[N]) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    typedef unsigned u32s __attribute__((ext_vector_type(E / 2)));
    // in registers: as an immediate the instruction takes (-1, 0) for another value
    unsigned first, second;
    asm("s_mov_b32 %0, 0xbf80" : "=s"(first));
    asm("s_mov_b32 %0, 0xbf800000" : "=s"(second));
    u32s q[N];
#pragma unroll
    for (int e = 0; e < E / 2; ++e) {
        float a = x[2 * e], b = x[2 * e + 1];
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const bf16x2 both = __builtin_convertvector(f32x2{a, b}, bf16x2);
            q[i][e] = __builtin_bit_cast(unsigned, both);
            if (i + 1 == N) continue;
            if constexpr (SUMMED) {
                a = __builtin_amdgcn_fdot2_f32_bf16(both, __builtin_bit_cast(bf16x2, first), a, false);
                b = __builtin_amdgcn_fdot2_f32_bf16(both, __builtin_bit_cast(bf16x2, second), b, false);
            } else {
                a -= __builtin_bit_cast(float, q[i][e] << 16);
                b -= __builtin_bit_cast(float, q[i][e] & 0xffff0000u);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < N; ++i) p[i] = __builtin_bit_cast(V, q[i]);
}

template <typename T>
using Eight = T __attribute__((ext_vector_type(8)));
// The same in memory, at any alignment of its elements.
template <typename T>
struct PackedEight {
    typedef T type __attribute__((ext_vector_type(8), aligned(sizeof(T))));
};

// Zero, or a NaN where x or its rounding to bf16 is infinite or a NaN. In units
// of 2^120 bf16's largest number is 255, what rounds past it begins at 255.5, and
// kPast leads that, but not 255, past the end of 32 bits at 256.
constexpr float kPast = 1.003f;
__device__ __forceinline__ float times_zero(float x) { return x * kPast * 0.f; }
// s, or a NaN where an element is such a one.
__device__ __forceinline__ float times_zero(const Eight<float>& x, float s) {
#pragma unroll
    for (int e = 0; e < 8; ++e) s = fmaf(x[e] * kPast, 0.f, s);
    return s;
}
__device__ __forceinline__ float times_zero(const Eight<_Float16>& x, float s) {
    typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int e = 0; e < 8; e += 2) s = __builtin_amdgcn_fdot2(f16x2{x[e], x[e + 1]}, f16x2{0, 0}, s, false);
    return s;
}
__device__ __forceinline__ float times_zero(const Eight<__bf16>& x, float s) {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int e = 0; e < 8; e += 2)
        s = __builtin_amdgcn_fdot2_f32_bf16(bf16x2{x[e], x[e + 1]}, bf16x2{(__bf16)0.f, (__bf16)0.f}, s, false);
    return s;
}

// One thread's share of a chunk of rows [C][D] on its way to LDS: vectors of
// eight elements at one column of every kRows-th row, read ahead while the
// chunk before is worked on. The reads take no branch, which would make the
// compiler wait for them on the spot: rows past the last one read that again,
// threads without a column read the first, and what does not belong is left
// out on the way to LDS.
template <typename T, int C, int D, int THREADS>
struct Staged {
    static constexpr int kLanes = D / 8 <= 4 ? 4 : D / 8 <= 8 ? 8 : D / 8 <= 16 ? 16 : 32;  // threads along a row
    static constexpr int kRows = THREADS / kLanes, kEach = kRows < C ? C / kRows : 1;
    Eight<T> r[kEach];
    const char* next;  // the row of the next chunk's first token, at the block's first column
    long long token;   // bytes from a token to the next in the order of the scan
    unsigned step;     // the same, of the lower address to the higher
    int row, col, at;  // this thread's first row and column, and the column where its vectors start
    int width;         // columns that the block has
    bool slow;         // rows of fewer than eight elements or 2^24 bytes apart: read when they are needed
    bool plain;        // no vector starts early

    __device__ __forceinline__ void init(const ScanSide& s, int b, int h, int col0, int dim, long long first, int reverse) {
        const long long apart = s.token * (long long)sizeof(T);
        next = (const char*)((const T*)s.p + b * s.batch + (h / s.group) * s.head + col0) + first * apart;
        token = reverse ? -apart : apart;
        row = (int)threadIdx.x / kLanes;
        col = (int)threadIdx.x % kLanes * 8;
        width = dim - col0 < D ? dim - col0 : D;
        slow = width < 8 || apart >= 1 << 24;
        step = slow ? 0u : (unsigned)apart;
        plain = !slow && width % 8 == 0;
        // the vector over the last column starts early, on what its neighbour reads too
        at = col >= width || slow ? 0 : col + 8 > width ? width - 8 : col;  // slow: of what is read for nothing
    }

    // Asks for the next chunk's `left` rows.
    __device__ __forceinline__ void load(int left, int reverse, const void* elsewhere) {
        const char* p = slow ? (const char*)elsewhere : reverse ? next - (unsigned)(left - 1) * step : next;
#pragma unroll
        for (int u = 0; u < kEach; ++u) {
            int i = row + u * kRows;
            i = i < left ? i : left - 1;
            i = reverse ? left - 1 - i : i;
            const unsigned offset = __umul24((unsigned)i, step) + (unsigned)at * (unsigned)sizeof(T);
            r[u] = *(const typename PackedEight<T>::type*)(p + offset);
        }
    }

    // Waits for what was read ahead.
    __device__ __forceinline__ void arrive() {
#pragma unroll
        for (int u = 0; u < kEach; ++u) asm volatile("" : "+v"(r[u]));
    }

    // Infinities and NaN of the chunk that was asked for become zeros, and *bad tells of them.
    __device__ __forceinline__ void make_finite(unsigned* bad) {
        float none = 0.f;
#pragma unroll
        for (int u = 0; u < kEach; ++u) none = times_zero(r[u], none);
        if (none == 0.f) return;
        *bad = 1;
#pragma unroll
        for (int u = 0; u < kEach; ++u)
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (times_zero((float)r[u][e]) != 0.f) r[u][e] = (T)0.f;
    }

    // The chunk that was asked for to lds[part][C][pitch], rows from `left` on as zeros; then on to the next.
    __device__ __forceinline__ void store(__bf16* lds, int pitch, int left, unsigned* bad = nullptr) {
        if (plain && left == C) {
            if (col < width && row < C)
#pragma unroll
                for (int u = 0; u < kEach; ++u) put(lds + (row + u * kRows) * pitch + col, pitch, r[u], true);
        } else if (!slow) {
            if (col < width && row < C)
#pragma unroll
                for (int u = 0; u < kEach; ++u) {
                    const Eight<T> zero = (T)0.f;
                    put(lds + (row + u * kRows) * pitch + at, pitch, row + u * kRows < left ? r[u] : zero, at == col);
                }
        } else {
#pragma unroll 1
            for (int j = (int)threadIdx.x; j < C * D; j += THREADS) {
                const int i = j / D, c = j % D;
                float f = i < left && c < width ? (float)((const T*)(next + i * token))[c] : 0.f;
                if (bad && times_zero(f) != 0.f) *bad = 1, f = 0.f;
#pragma unroll
                for (int k = 0; k < Parts<T>::in; ++k) {
                    const __bf16 v = (__bf16)f;
                    lds[(k * C + i) * pitch + c] = v;
                    f -= (float)v;
                }
            }
        }
        next += C * token;
    }

    // Eight elements' parts; aligned: as vectors.
    static __device__ __forceinline__ void put(__bf16* to, int pitch, const Eight<T>& x, bool aligned) {
        bf16x8 p[Parts<T>::in];
        if constexpr (Parts<T>::in == 1) {
            p[0] = x;
        } else {
            float f[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = (float)x[e];
            split<false>(f, p);
        }
#pragma unroll
        for (int i = 0; i < Parts<T>::in; ++i) {
            if (aligned) {
                *(bf16x8*)(to + i * C * pitch) = p[i];
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) to[i * C * pitch + e] = p[i][e];
            }
        }
    }
};

// A row of a matrix in LDS as an operand: elements k0 + (0-3, 16-19) + 4 g.
__device__ __forceinline__ bf16x8 row_operand(const __bf16* row, int k0, int g) {
    const bf16x4 a = *(const bf16x4*)(row + k0 + 4 * g);
    const bf16x4 b = *(const bf16x4*)(row + k0 + 16 + 4 * g);
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

// Four neighbours, as many as there is room for.
template <typename T>
__device__ __forceinline__ void store_four(T* to, f32x4 y, int room) {
    typedef T four __attribute__((ext_vector_type(4), aligned(sizeof(T))));
    if (room >= 4) {
        *(four*)to = four{(T)y[0], (T)y[1], (T)y[2], (T)y[3]};
    } else {
#pragma unroll
        for (int r = 0; r < 3; ++r)
            if (r < room) to[r] = (T)y[r];
    }
}

template <typename T, int DK, int WAVES, int NT, int C, bool STATE_ONLY>
struct ChunkShape {
    static constexpr int kIn = Parts<T>::in, kMid = Parts<T>::mid;
    static constexpr int kThreads = 64 * WAVES, kCols = 16 * NT * WAVES;
    // 16 bytes more a row: a quarter wave's 8-byte reads down the rows meet different banks
    static constexpr int kPitchK = DK + 8, kPitchV = kCols + 8, kPitchP = C + 8;
    // A, B and C, twice where a CU's LDS then still holds a second block or there is none anyway: the next chunk is
    // written while other waves read this one
    static constexpr size_t kA = 0, kB = STATE_ONLY ? 0 : (size_t)kIn * C * kPitchK, kC = kB + (size_t)kIn * C * kPitchK,
                            kOne = kC + (size_t)kIn * C * kPitchV, kScores = STATE_ONLY ? 0 : (size_t)kMid * C * kPitchP, kRest = kScores * 2 + kDecayPowers * 4 + 16;
    static constexpr size_t kCu = 160 * 1024;
    static constexpr bool kTwice = 2 * (4 * kOne + kRest) <= kCu || (2 * (2 * kOne + kRest) > kCu && 4 * kOne + kRest <= kCu);
    static constexpr size_t kP = kTwice ? 2 * kOne : kOne, kEnd = kP + kScores;
    static constexpr size_t kLds = kEnd * 2 + kDecayPowers * 4 + 16;
    // waves that share a SIMD's registers: two, or the one that the LDS leaves
    static constexpr int kShare = (int)(kCu / kLds) * WAVES >= 8 ? 2 : 1;
};

template <typename T, int DK, int WAVES, int NT, int C, bool STATE_ONLY>
__global__ __launch_bounds__(64 * WAVES, (ChunkShape<T, DK, WAVES, NT, C, STATE_ONLY>::kShare)) void k_chunk(const ChunkArgs args) {
    using S = ChunkShape<T, DK, WAVES, NT, C, STATE_ONLY>;
    constexpr int IN = S::kIn, MID = S::kMid, TI = C / 16, THREADS = S::kThreads;
    extern __shared__ __align__(16) char lds[];
    __bf16* la = (__bf16*)lds + S::kA;
    __bf16* lb = (__bf16*)lds + S::kB;
    __bf16* lc = (__bf16*)lds + S::kC;
    int other = S::kTwice ? (int)S::kOne : 0;  // from this chunk's buffer to the next one's
    __bf16* const lp = (__bf16*)lds + S::kP;
    float* const pw = (float*)((__bf16*)lds + S::kEnd);
    unsigned* const bad = (unsigned*)(pw + kDecayPowers);  // of this chunk and of the next, in turn

    // block -> (scan, sequence, head, segment, slice), slices side by side
    long long id = blockIdx.x + (long long)blockIdx.y * gridDim.x;
    if (id >= args.blocks) return;
    const int slice = (int)(id % args.slices);
    id /= args.slices;
    const int seg = (int)(id % args.segments);
    id /= args.segments;
    const int h = (int)(id % args.scan[0].heads);
    id /= args.scan[0].heads;
    const int b = (int)(id % args.scan[0].batch);
    const int z = (int)(id / args.scan[0].batch);
    const ScanArgs& s = args.scan[z];

    const int tokens = (int)s.tokens, segment = (int)args.segment;
    int n = tokens;
    if (s.lengths) n = s.lengths[b] < 0 ? 0 : s.lengths[b] < n ? s.lengths[b] : n;
    const int begin = seg * segment, end = tokens - begin > segment ? begin + segment : tokens;
    const int stop = end < n ? end : n;  // of what the scan reads
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int g = lane >> 4, l16 = lane & 15;
    const int col0 = slice * S::kCols, wcol = wave * 16 * NT;
    const int lead = s.reverse;
    if (tid < 2) bad[tid] = 0;
    if (tid < kDecayPowers) pw[tid] = args.powers[(long long)h * kDecayPowers + tid];
    // columns past the tensors', and tiles of P right of the diagonal that a product of 32 tokens meets
    for (int i = tid; i < (int)(S::kEnd / 8); i += THREADS) ((bf16x8*)lds)[i] = (__bf16)0.f;

    // the state: rows 16 a + 4 g + r, columns col0 + wcol + 16 t + l16
    f32x4 X[NT][DK / 16];
    const int col = col0 + wcol + l16;
    const long long head_state = ((long long)b * s.heads + h) * s.dk * s.dv;
    float* const slot = args.slots[z] + (((long long)b * s.heads + h) * args.segments + seg) * s.dk * s.dv;
    // All of a state's elements are asked for before the first is waited for: rows and columns past the last
    // read the last one, and are left out by what they meet - zeros in A, B and C - and where X is written.
    const auto read_state = [&](const float* from, int row_step, int col_step) {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const int c = col + 16 * t < s.dv ? col + 16 * t : s.dv - 1;
#pragma unroll
            for (int a = 0; a < DK / 16; ++a)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int row = 16 * a + 4 * g + r < s.dk ? 16 * a + 4 * g + r : s.dk - 1;
                    X[t][a][r] = from[row * row_step + c * col_step];
                }
        }
    };
    const auto write_state = [&](float* to, int row_step, int col_step) {
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int a = 0; a < DK / 16; ++a)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int row = 16 * a + 4 * g + r, c = col + 16 * t;
                    if (row < s.dk && c < s.dv) to[row * row_step + c * col_step] = X[t][a][r];
                }
    };
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int a = 0; a < DK / 16; ++a) X[t][a] = f32x4{0.f, 0.f, 0.f, 0.f};
    // The state is factor X. In 64 bits: in 32 the decay of a chunk, rounded once, would round every chunk's state to the
    // same side (after 512 chunks a state would be off by 1.4e-5 at a decay of 0.999997).
    double factor = 1.0;
    const int state_size = s.dk * s.dv;
    if constexpr (STATE_ONLY) {
        if (seg == 0 && s.state_in) read_state(s.state_in + head_state, s.state_row, s.state_col);
        if (seg == 0 && args.in_place) write_state(slot, args.slot_row[z], args.slot_col[z]);
        // a state before the next segment is needed only where that one has tokens
        if (n - begin <= segment) return;
    } else if (seg == 0 && !args.in_place) {
        if (s.state_in) read_state(s.state_in + head_state, s.state_row, s.state_col);
    } else if (begin < n || seg == 0) {
        read_state(slot, args.slot_row[z], args.slot_col[z]);
    }

    const int reverse = s.reverse;
    const long long first = reverse ? (long long)n - 1 - begin : begin;
    const float scale_update = s.scale_update, scale_in = s.scale_in;
    Staged<T, C, DK, THREADS> sa, sb;
    Staged<T, C, S::kCols, THREADS> sc;
    if (!STATE_ONLY) sa.init(s.a, b, h, 0, s.dk, first, reverse);
    sb.init(s.b, b, h, 0, s.dk, first, reverse);
    sc.init(s.c, b, h, col0, s.dv, first, reverse);
    const auto fetch = [&](int left) {
        if (!STATE_ONLY) sa.load(left, reverse, args.powers);
        sb.load(left, reverse, args.powers);
        sc.load(left, reverse, args.powers);
    };
    // on every way to the loop's next turn, or the compiler waits where that asks for more
    const auto arrive = [&]() {
        if (!STATE_ONLY) sa.arrive();
        sb.arrive();
        sc.arrive();
    };
    const auto stage = [&](int left, unsigned* marks) {
        // rows of C that are not finite would reach the tokens before them through their zeros in P
        if (!STATE_ONLY) sc.make_finite(marks);
        if (!STATE_ONLY) sa.store(la, S::kPitchK, left);
        sb.store(lb, S::kPitchK, left);
        sc.store(lc, S::kPitchV, left, STATE_ONLY ? nullptr : marks);
    };

    // where this lane's token of a chunk's first 16 goes, from its first column on
    const int out_col = col0 + wcol + 4 * g, room = s.dv - out_col, out_f32 = s.out_f32;
    const long long out_step = (reverse ? -s.out_token : s.out_token) * (out_f32 ? 4ll : (long long)sizeof(T));
    char* out = (char*)s.out + (b * s.out_batch + h * s.out_head + first * s.out_token + out_col) * (out_f32 ? 4ll : (long long)sizeof(T)) +
                l16 * out_step;

    // Weights, the same for every whole chunk. P: the tiles on and left of the diagonal, dealt to the waves; a wave
    // without a tile of its own in the last turn does the last one once more.
    constexpr int tiles = TI * (TI + 1) / 2, each = (tiles + WAVES - 1) / WAVES;
    int pi[each], pj[each];
    float pweight[each][4], oweight[TI], uweight[C / 32][8];
    __syncthreads();  // pw, and the clearing
    if constexpr (!STATE_ONLY) {
#pragma unroll
        for (int u = 0; u < each; ++u) {
            const int tile = wave + u * WAVES < tiles ? wave + u * WAVES : tiles - 1;
            const int I = tile < 1 ? 0 : tile < 3 ? 1 : tile < 6 ? 2 : 3;
            pi[u] = 16 * I, pj[u] = 16 * (tile - I * (I + 1) / 2);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int d = pi[u] + l16 - (pj[u] + 4 * g + r);
                pweight[u][r] = d < 0 ? 0.f : pw[d] * scale_update * scale_in;
            }
        }
#pragma unroll
        for (int I = 0; I < TI; ++I) oweight[I] = pw[16 * I + l16 + 1 - lead] * scale_in;
    }
    const auto update_weights = [&](int left) {
#pragma unroll
        for (int k = 0; k < C / 32; ++k)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int d = left - 1 - (32 * k + 8 * g + e) + lead;
                uweight[k][e] = pw[d < 0 ? 0 : d] * scale_update;
            }
    };
    update_weights(C);
    const double whole = same_in_all(decay_of(pw, C));

    // the state is here before the loop begins: a wait for it inside would be one for the chunk that is read ahead
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int a = 0; a < DK / 16; ++a) asm volatile("" : "+v"(X[t][a]));
    if (begin < stop) fetch(stop - begin < C ? stop - begin : C);
    arrive();
    if (begin < stop) stage(stop - begin < C ? stop - begin : C, bad);
    int turn = 0;
#pragma unroll 1
    for (int at = begin; at < stop; at += C) {
        const int left = stop - at < C ? stop - at : C;
        const int more = stop - at - left < C ? stop - at - left : C;  // tokens of the next chunk
        __syncthreads();
        if (more) fetch(more);
        if (left < C) update_weights(left);
        const unsigned* const marks = bad + turn;
        turn ^= 1;
        if (!STATE_ONLY && tid == 0) bad[turn] = 0;  // nobody marks the next chunk before P's barrier

        // The state decays by its factor, which runs from 2^7 down to 1: X is never larger than the state, which may come
        // near the largest number, and at most 2^7 times smaller, where the parts of small numbers vanish. X itself decays
        // in every second chunk at most, or in each one where a chunk leaves so little that this saves nothing.
        const float before = (float)factor;
        factor = same_in_all(factor * (left < C ? (double)pw[left] : whole));
        const bool fast = whole < 0x1p-7, decays = factor < 1.0;
        const float shrink = (float)factor * (fast ? 1.f : 0x1p-7f);
        if (decays) factor = fast ? 1.0 : 0x1p7;
        const float added = 1.f / (float)factor;

        f32x4 o[NT][TI];
        if constexpr (!STATE_ONLY) {
            // P, transposed: rows j, columns i
            f32x4 p[each];
#pragma unroll
            for (int u = 0; u < each; ++u) p[u] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int k = 0; k < DK / 32; ++k) {
                bf16x8 bj[each][IN], ai[each][IN];
#pragma unroll
                for (int u = 0; u < each; ++u)
#pragma unroll
                    for (int i = 0; i < IN; ++i) {
                        bj[u][i] = row_operand(lb + (i * C + pj[u] + l16) * S::kPitchK, 32 * k, g);
                        ai[u][i] = row_operand(la + (i * C + pi[u] + l16) * S::kPitchK, 32 * k, g);
                    }
                mma_parts(bj, ai, p, IN == 3 ? 3 : 2);
            }
#pragma unroll
            for (int u = 0; u < each; ++u) {
                bf16x4 q[MID];
                float x[4];
#pragma unroll
                for (int r = 0; r < 4; ++r)  // not by a product: what is masked may be infinite
                    x[r] = pi[u] + l16 < pj[u] + 4 * g + r ? 0.f : p[u][r] * pweight[u][r];
                split<true>(x, q);
#pragma unroll
                for (int m = 0; m < MID; ++m) *(bf16x4*)(lp + (m * C + pi[u] + l16) * S::kPitchP + pj[u] + 4 * g) = q[m];
            }

            // out = A X, transposed
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int I = 0; I < TI; ++I) o[t][I] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int k = 0; k < DK / 32; ++k) {
                bf16x8 ai[TI][IN];
#pragma unroll
                for (int I = 0; I < TI; ++I)
#pragma unroll
                    for (int i = 0; i < IN; ++i)
                        ai[I][i] = row_operand(la + (i * C + 16 * I + l16) * S::kPitchK, 32 * k, g);
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    bf16x8 x[MID];
                    float v[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[e] = X[t][2 * k + e / 4][e % 4];
                    split<true>(v, x);
                    mma_parts(x, ai, o[t], MID);
                }
            }
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int I = 0; I < TI; ++I) {
                    o[t][I] *= oweight[I] * before;
                    // Here, and not after the branch below: the compiler counts the wait for a matrix product's result
                    // along one way to a place that two lead to, which may be the longer one.
                    asm volatile("" : "+v"(o[t][I]));
                }
            __syncthreads();  // P is written
        }

        if (decays) {
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int a = 0; a < DK / 16; ++a) X[t][a] *= shrink;
        }
#pragma unroll
        for (int k = 0; k < C / 32; ++k) {
            bf16x8 cv[NT][IN], cw[NT][3];
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int i = 0; i < IN; ++i)
                    cv[t][i] = column_operand(lc + i * C * S::kPitchV, S::kPitchV, 32 * k, wcol + 16 * t, lane);
            if constexpr (!STATE_ONLY) {
                // tiles of 16 tokens from 32 k on, two at a time
#pragma unroll
                for (int I = 2 * k; I < TI; I += 2) {
                    bf16x8 p[2][MID];
#pragma unroll
                    for (int u = 0; u < 2; ++u)
#pragma unroll
                        for (int m = 0; m < MID; ++m)
                            p[u][m] = *(const bf16x8*)(lp + (m * C + 16 * (I + u) + l16) * S::kPitchP + 32 * k + 8 * g);
#pragma unroll
                    for (int t = 0; t < NT; ++t) mma_parts(cv[t], p, o[t] + I, MID);
                }
            }
            float w[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) w[e] = uweight[k][e] * added;
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                float v[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    v[e] = (float)cv[t][IN - 1][e];
#pragma unroll
                    for (int i = IN - 2; i >= 0; --i) v[e] += (float)cv[t][i][e];
                    v[e] *= w[e];
                }
                split<true>(v, cw[t]);
            }
#pragma unroll
            for (int a = 0; a < DK / 16; a += 2) {
                bf16x8 bt[2][IN];
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int i = 0; i < IN; ++i)
                        bt[u][i] = column_operand(lb + i * C * S::kPitchK, S::kPitchK, 32 * k, 16 * (a + u), lane);
#pragma unroll
                for (int t = 0; t < NT; ++t) mma_parts(bt, cw[t], X[t] + a, 3);
            }
        }

        if constexpr (!STATE_ONLY) {
            if (*marks) {  // what was left out of C, where it belongs
#pragma unroll 1
                for (int j = 0; j < left; ++j) {
                    const T* const row = (const T*)s.c.p + b * s.c.batch + (h / s.c.group) * s.c.head +
                                         (reverse ? (long long)n - 1 - at - j : (long long)at + j) * s.c.token;
                    const float weight = pw[left - 1 - j + lead] * scale_update * added;
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            const float c = room > 16 * t + r ? (float)row[out_col + 16 * t + r] : 0.f;
                            if (times_zero(c) == 0.f) continue;
#pragma unroll
                            for (int I = 0; I < TI; ++I) {
                                float p = 0.f;
#pragma unroll
                                for (int m = MID - 1; m >= 0; --m) p += (float)lp[(m * C + 16 * I + l16) * S::kPitchP + j];
                                if (16 * I + l16 >= j) o[t][I][r] = fmaf(p, c, o[t][I][r]);
                            }
                        }
                        const float c = col + 16 * t < s.dv ? (float)row[col + 16 * t] : 0.f;
                        if (times_zero(c) == 0.f) continue;
#pragma unroll
                        for (int a = 0; a < DK / 16; ++a)
#pragma unroll
                            for (int r = 0; r < 4; ++r) {
                                float k = 0.f;
#pragma unroll
                                for (int i = IN - 1; i >= 0; --i) k += (float)lb[(i * C + j) * S::kPitchK + 16 * a + 4 * g + r];
                                X[t][a][r] = fmaf(k, weight * c, X[t][a][r]);
                            }
                    }
                }
            }
        }
        if (!S::kTwice) __syncthreads();  // the chunk has been read
        arrive();
        la += other, lb += other, lc += other;
        other = -other;
        // before this chunk's stores: loads and stores are waited for in their order
        if (more) stage(more, bad + turn);
        if constexpr (!STATE_ONLY) {
#pragma unroll
            for (int I = 0; I < TI; ++I) {
                if (16 * I + l16 >= left) continue;
                char* const to = out + 16 * I * out_step;
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    const f32x4 y = o[t][I];
                    if (out_f32) store_four((float*)to + 16 * t, y, room - 16 * t);
                    else store_four((T*)to + 16 * t, y, room - 16 * t);
                }
            }
            out += C * out_step;
        }
    }

#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int a = 0; a < DK / 16; ++a) X[t][a] *= (float)factor;
    if constexpr (STATE_ONLY) {
        write_state(slot + state_size, args.slot_row[z], args.slot_col[z]);  // to the next segment's place
        return;
    }
    // rows past the sequence's length
    for (int i = (begin > n ? begin : n) + wave; i < end; i += WAVES) {
        const long long row = b * s.out_batch + (long long)i * s.out_token + h * s.out_head;
        for (int c = col0 + lane; c < s.dv && c < col0 + S::kCols; c += 64) {
            if (s.out_f32) ((float*)s.out)[row + c] = 0.f;
            else ((T*)s.out)[row + c] = (T)0.f;
        }
    }
    if (s.state_out && seg == (n > 0 ? (n - 1) / segment : 0)) write_state(s.state_out + head_state, s.state_row, s.state_col);
}

struct ChunkKernel {
    int cols, threads;  // of a block
    size_t lds, state_lds;
    const void* run;
    const void* state_only;
};
// The element's kernel for a scan of dk x dv, on its own or of a gradient's three.
const ChunkKernel* chunk_kernel_f32(int dk, int dv, bool gradient);
const ChunkKernel* chunk_kernel_f16(int dk, int dv, bool gradient);
const ChunkKernel* chunk_kernel_bf16(int dk, int dv, bool gradient);

template <typename T, int DK, int WAVES, int NT, int C>
ChunkKernel chunk_kernel_of() {
    using S = ChunkShape<T, DK, WAVES, NT, C, false>;
    return ChunkKernel{S::kCols,
                       S::kThreads,
                       S::kLds,
                       ChunkShape<T, DK, WAVES, NT, C, true>::kLds,
                       (const void*)k_chunk<T, DK, WAVES, NT, C, false>,
                       (const void*)k_chunk<T, DK, WAVES, NT, C, true>};
}

// Key widths are padded to one of six. Up to 64 values a block has their 64
// columns, above that 128, so that what it reads of A and B serves more of them
// (bf16, 8 x 2048 tokens, 16 heads of 128 x 128: 127 us, with 64 columns 141;
// 64 x 128: 91 and 97), except where keys are wider than 128 and the CU holds
// two blocks of 64 columns but one of 128 (8 heads of 256 x 256, bf16 201 us and
// 213; where the LDS has no room for the second, f16 gradients 600 and 462).
//
// A wave has 32 columns where that leaves enough waves: what it reads of A, B
// and P then serves two products (bf16, 64 x 128: 95 us, with 16 columns 112;
// 96 x 96: 105 and 128). Not where it leaves two waves a block and these have
// much to do between them: operands of two or three parts, 96 keys or the scans
// of a gradient (16 heads of 64 x 64, with 16 columns and with 32: f16 86 us and
// 119, f32 109 and 188, bf16 gradients 133 and 153; 96 x 64 bf16 79 and 114), nor
// where a state of more than 128 rows, for f32 96, takes the registers. Two parts
// and 32 keys run as fast either way (73 and 76); bf16 forward is slower with 16
// columns where the sequence is long (1 x 65536, 64 x 64: 182 and 170).
template <typename T>
const ChunkKernel* pick_chunk_kernel(int dk, int dv, bool gradient) {
    constexpr int C = kChunk;
    constexpr int parts = Parts<T>::in;
    constexpr int wide192 = 2 * ChunkShape<T, 192, 4, 1, C, false>::kLds <= ChunkShape<T, 192, 4, 1, C, false>::kCu ? 4 : 8;
    constexpr int wide256 = 2 * ChunkShape<T, 256, 4, 1, C, false>::kLds <= ChunkShape<T, 256, 4, 1, C, false>::kCu ? 4 : 8;
    constexpr int few32 = parts == 3 ? 4 : 2, few64 = parts > 1 ? 4 : 2, many128 = parts == 3 ? 8 : 4;
    static const ChunkKernel kernels[6][2] = {
        {chunk_kernel_of<T, 32, few32, 4 / few32, C>(), chunk_kernel_of<T, 32, 4, 2, C>()},
        {chunk_kernel_of<T, 64, few64, 4 / few64, C>(), chunk_kernel_of<T, 64, 4, 2, C>()},
        {chunk_kernel_of<T, 96, 4, 1, C>(), chunk_kernel_of<T, 96, 4, 2, C>()},
        {chunk_kernel_of<T, 128, 4, 1, C>(), chunk_kernel_of<T, 128, many128, 8 / many128, C>()},
        {chunk_kernel_of<T, 192, 4, 1, C>(), chunk_kernel_of<T, 192, wide192, 1, C>()},
        {chunk_kernel_of<T, 256, 4, 1, C>(), chunk_kernel_of<T, 256, wide256, 1, C>()}};
    static const ChunkKernel gradient64 = chunk_kernel_of<T, 64, 4, 1, C>();
    if (gradient && dk > 32 && dk <= 64 && dv <= 64) return &gradient64;
    return &kernels[dk <= 32 ? 0 : dk <= 64 ? 1 : dk <= 96 ? 2 : dk <= 128 ? 3 : dk <= 192 ? 4 : 5][dv > 64];
}

}  // namespace vkfx
