// recurrence.hip -- the gated recurrence h[t] = a[t] h[t-1] + m[t] x[t] of every
// channel, and its gradients.
//
// With D the gradient of the state after a token and E = a D that of the state
// before it,
//   D[t] = dy[t] + E[t+1],  dx = m D,  da = D (h[t-1] - (m = 1 - a ? x : 0))
// and dgate = da a (1 - a) or da a.
//
// Bound by memory, where the sequence is long enough to be read side by side. A
// lane has 4 bytes of channels, a wave 16 tokens of them in its registers: it
// forms what they make of any state before them (state -> A state + H), a
// block's waves, one behind the other in time, fold these in LDS, and each goes
// over its tokens once more from the state that it now knows. The next 16 times
// as many tokens are on their way meanwhile. Where channels are too few to fill
// the machine, a sequence is cut into segments whose (A, H) an earlier launch
// forms.
//
// A decay near 1 is kept as what it is short of 1: rounded to 24 bits itself, a
// memory of n tokens would be off by n 2^-25 of its length. So is A.
#include <algorithm>
#include <type_traits>

#include "sequence.hpp"
#include "sequence_device.hpp"
#include "vkfx.h"

namespace vkfx {

namespace {

constexpr int U = kSpan;  // tokens of a wave

// exp(g), off by 2^-22 of it, for -87 <= g <= 0: the product with log2(e) keeps
// its rounding.
__device__ __forceinline__ float exp_near(float g) {
    constexpr float log2e = 1.44269502f, rest = 1.92596299e-8f;
    const float t = g * log2e, low = fmaf(g, rest, fmaf(g, log2e, -t));
    const float e = __builtin_amdgcn_exp2f(t);
    return fmaf(e, low * 0.693147181f, e);
}
// exp(g) - 1 for -ln 2 < g <= 0: its series, the next term below 2^-26 of it.
__device__ __forceinline__ float exp_less_1(float g) {
    float p = 1.f / 3628800;
    p = fmaf(p, g, 1.f / 362880);
    p = fmaf(p, g, 1.f / 40320);
    p = fmaf(p, g, 1.f / 5040);
    p = fmaf(p, g, 1.f / 720);
    p = fmaf(p, g, 1.f / 120);
    p = fmaf(p, g, 1.f / 24);
    p = fmaf(p, g, 1.f / 6);
    p = fmaf(p, g, 0.5f);
    return fmaf(g * p, g, g);
}

// A gate: s is the smaller of a and 1 - a, negative (-0 too) where that is 1 - a;
// w is 1 - a. NEAR: no |g| is past 87, from where on the hardware's exponential
// gives 0; there it is the square of its root.
struct Gate {
    float s, w;
};
constexpr float kNear = 87.f;
template <bool NEAR>
__device__ __forceinline__ float exp_of(float g) {
    if (NEAR || !(g < -kNear)) return exp_near(g);
    const float root = exp_near(fmaxf(0.5f * g, -kNear));
    return root * root;
}
template <bool SIGMOID, bool NEAR>
__device__ __forceinline__ Gate gate_of(float g) {
    if constexpr (SIGMOID) {
        const float e = exp_of<NEAR>(-fabsf(g));
        const float large = __builtin_amdgcn_rcpf(1.f + e), small = e * large;
        return g > 0.f ? Gate{-small, small} : Gate{small, large};
    } else {
        g = g > 0.f ? 0.f : g;  // a NaN stays one
        const float less = exp_less_1(g), e = exp_of<NEAR>(g);
        return g > -0.6931472f ? Gate{__int_as_float(__float_as_int(less) | (int)0x80000000), -less} : Gate{e, 1.f - e};
    }
}
// v where a >= 1/2, else 0.
__device__ __forceinline__ float if_slow(float s, float v) { return __int_as_float((__float_as_int(s) >> 31) & __float_as_int(v)); }
__device__ __forceinline__ float decayed(float s, float v) { return fmaf(s, v, if_slow(s, v)); }  // a v
__device__ __forceinline__ float short_of(float s) { return __float_as_int(s) < 0 ? -s : 1.f - s; }  // 1 - a

// What some tokens make of the state before them: a v + h, a by its smaller side
// like a gate.
struct Join {
    float s, h;
    __device__ __forceinline__ float operator()(float v) const { return decayed(s, v) + h; }
};

__device__ __forceinline__ int clamped(const int* lengths, int b, long long tokens) {
    const long long n = lengths ? lengths[b] : tokens;
    return __builtin_amdgcn_readfirstlane((int)(n < 0 ? 0 : n < tokens ? n : tokens));
}

// The next row. Kept from the compiler, which would hold every row's place in
// scalar registers, and these, past 100 of them, in lanes of vector registers.
template <typename T>
__device__ __forceinline__ T* behind(T* row, long long stride) {
    row += stride;
    asm volatile("" : "+s"(row));
    return row;
}

// A lane's place among the channels: CH of them, or none. Lanes without any read
// the block's first.
template <typename T, int CH>
struct Lane {
    typedef T Vec __attribute__((ext_vector_type(CH)));
    // A token's channels as they lie in memory: as elements, the compiler would
    // take them apart, and wait for them, where they arrive.
    typedef std::conditional_t<sizeof(Vec) == 4, unsigned, unsigned short> Raw;
    long long first;  // the block's first channel
    int at;           // the lane's
    bool have;

    __device__ __forceinline__ explicit Lane(long long channels) {
        first = (long long)blockIdx.x * (64 * CH);
        have = first + (threadIdx.x & 63) * CH < channels;
        at = have ? (threadIdx.x & 63) * CH : 0;
    }
    // Tokens t .. t + m - 1 of sequence b, the last one again behind them.
    __device__ __forceinline__ void fetch(unsigned (&r)[U], const RecurrenceSide& s, long long b, long long t, int m) const {
        if (m <= 0) return;
        const T* row = (const T*)s.p + b * s.batch + t * s.token + first;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            r[u] = *(const Raw*)(row + at);
            row += u + 1 < m ? s.token : 0;
        }
    }
    __device__ __forceinline__ static float value(unsigned r, int c) { return (float)__builtin_bit_cast(Vec, (Raw)r)[c]; }
    __device__ __forceinline__ void store(T* row, const float (&y)[CH]) const {
        Vec r;
#pragma unroll
        for (int c = 0; c < CH; ++c) r[c] = (T)y[c];
        *(Vec*)(row + at) = r;
    }
    // Zeros in rows t .. of a tensor.
    __device__ __forceinline__ void clear(const RecurrenceSide& s, long long b, long long t, int rows) const {
        T* row = (T*)s.p + b * s.batch + t * s.token + first;
        const float zero[CH] = {};
        for (int u = 0; have && u < rows; ++u, row += s.token) store(row, zero);
    }
    __device__ __forceinline__ void load_state(float (&h)[CH], const float* row) const {
#pragma unroll
        for (int c = 0; c < CH; ++c) h[c] = row ? row[first + at + c] : 0.f;
    }
    __device__ __forceinline__ void store_state(float* row, const float (&h)[CH]) const {
#pragma unroll
        for (int c = 0; c < CH; ++c)
            if (have) row[first + at + c] = h[c];
    }
};

// Goes over the wave's gates: f(u, c, gate) for each. WHOLE: all U tokens, none
// past kNear; otherwise tokens from m on leave every state as it is.
template <typename T, int CH, bool SIGMOID, typename F>
__device__ __forceinline__ void each_gate(const unsigned (&g)[U], int m, F f) {
    float most = 0.f;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
        for (int c = 0; c < CH; ++c) most = fmaxf(most, fabsf(Lane<T, CH>::value(g[u], c)));
    if (__builtin_expect(m == U && !__any(most > kNear), 1)) {
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int c = 0; c < CH; ++c) f(u, c, gate_of<SIGMOID, true>(Lane<T, CH>::value(g[u], c)));
    } else {
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int c = 0; c < CH; ++c) f(u, c, u < m ? gate_of<SIGMOID, false>(Lane<T, CH>::value(g[u], c)) : Gate{-0.f, 0.f});
    }
}

// The product of decays: a, and low = 1 - a.
struct Product {
    float a = 1.f, low = 0.f;
    __device__ __forceinline__ void by(float s, float w) {
        a = decayed(s, a);
        low = decayed(s, low) + w;
    }
    // The smaller of both, as a gate has it.
    __device__ __forceinline__ float smaller() const { return low < 0.5f ? -low : a; }
};

// A block's waves' Joins one after the other (BACK: from the last on): h, the
// state before the tile, becomes that before the wave, and v that behind the
// tile. all: the whole segment's decay, where it is wanted.
template <int CH, int W, bool BACK, bool ALL>
__device__ __forceinline__ void fold(float (&h)[CH], float (&v)[CH], Product (&all)[CH], const Join (&at)[W][64][CH]) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int c = 0; c < CH; ++c) v[c] = h[c];
#pragma unroll
    for (int i = 0; i < W; ++i) {
        const int w = BACK ? W - 1 - i : i;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const Join k = at[w][lane][c];
            h[c] = w == wave ? v[c] : h[c];
            v[c] = k(v[c]);
            if constexpr (ALL) all[c].by(k.s, short_of(k.s));
        }
    }
}

// Segment z of a call: tokens z length .. + length.
struct Cut {
    int length, segments;
};
// Place of a segment's Joins in the workspace: [2][batch][segment][channel].
__device__ __forceinline__ float* join_at(const RecurrenceArgs& a, const Cut& cut, int part, int b, int z) {
    return a.work + (((long long)part * a.batch + b) * cut.segments + z) * a.channels;
}

// The state that reaches segment z from those before it (BACK: behind it).
template <typename T, int CH, bool BACK>
__device__ __forceinline__ void arrive(float (&h)[CH], const Lane<T, CH>& lane, const RecurrenceArgs& a, const Cut& cut, int b, int z, int n) {
    lane.load_state(h, a.state_in ? a.state_in + (long long)b * a.channels : nullptr);
    const int live = (n + cut.length - 1) / cut.length;  // segments with tokens
    for (int i = BACK ? live - 1 : 0; BACK ? i > z : i < z && i < live; i += BACK ? -1 : 1) {
        float s[CH], v[CH];
        lane.load_state(s, join_at(a, cut, 0, b, i));
        lane.load_state(v, join_at(a, cut, 1, b, i));
#pragma unroll
        for (int c = 0; c < CH; ++c) h[c] = Join{s[c], v[c]}(h[c]);
    }
}

// W waves a block, one behind the other in time. JOIN: the segment's Joins alone,
// nothing else written.
template <typename T, int CH, bool SIGMOID, bool COMPLEMENT, int W, bool JOIN>
__global__ __launch_bounds__(64 * W) void k_recurrence(const RecurrenceArgs a, const Cut cut) {
    __shared__ Join lds[2][W][64][CH];
    const Lane<T, CH> lane(a.channels);
    const int b = blockIdx.y, z = blockIdx.z;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n = clamped(a.lengths, b, a.tokens);
    const int begin = z * cut.length, end = (int)std::min(a.tokens, (long long)begin + cut.length), live = std::min(n, end);
    const long long spans = (a.tokens + U - 1) / U;
    float h[CH] = {};  // the state before the tile
    Product all[CH];
    if constexpr (!JOIN) arrive<T, CH, false>(h, lane, a, cut, b, z, n);
    unsigned x[U] = {}, g[U] = {};
    const auto fetch = [&](int t) {
        lane.fetch(x, a.x, b, t, live - t);
        lane.fetch(g, a.gate, b, t, live - t);
    };
    fetch(begin + wave * U);
    int t0 = begin;
    for (int half = 0; t0 < live; t0 += W * U, half ^= 1) {
        const int t = t0 + wave * U, m = std::min(live - t, U);
        // what the wave's tokens make of a state: p a + l
        float s[U][CH], in[U][CH], l[CH] = {}, after[CH];
        Product p[CH];
        each_gate<T, CH, SIGMOID>(g, m, [&](int u, int c, Gate q) {
            s[u][c] = q.s;
            in[u][c] = COMPLEMENT ? q.w * lane.value(x[u], c) : u < m ? lane.value(x[u], c) : 0.f;
            if constexpr (W > 1 || JOIN) {
                p[c].by(q.s, q.w);
                l[c] = decayed(q.s, l[c]) + in[u][c];
            }
        });
        fetch(t + W * U);
        if constexpr (W > 1 || JOIN) {
#pragma unroll
            for (int c = 0; c < CH; ++c) lds[half][threadIdx.x >> 6][threadIdx.x & 63][c] = Join{p[c].smaller(), l[c]};
            __syncthreads();
            fold<CH, W, false, JOIN>(h, after, all, lds[half]);
        }
        if constexpr (!JOIN) {
            if (a.saved && t < end) lane.store_state(a.saved + ((long long)b * spans + t / U) * a.channels, h);
            T* row = (T*)a.y.p + b * a.y.batch + t * a.y.token + lane.first;
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int c = 0; c < CH; ++c) in[u][c] = h[c] = decayed(s[u][c], h[c]) + in[u][c];
            if (m == U) {
                if (lane.have)
#pragma unroll
                    for (int u = 0; u < U; ++u, row = behind(row, a.y.token)) lane.store(row, in[u]);
            } else {
                if (lane.have)
#pragma unroll
                    for (int u = 0; u < U; ++u, row = behind(row, a.y.token))
                        if (u < m) lane.store(row, in[u]);
                lane.clear(a.y, b, t + std::max(m, 0), std::min(end - t, U) - std::max(m, 0));
            }
        }
        if constexpr (W > 1 || JOIN)
#pragma unroll
            for (int c = 0; c < CH; ++c) h[c] = after[c];
    }
    if constexpr (JOIN) {
        if (wave) return;
        float decay[CH];
#pragma unroll
        for (int c = 0; c < CH; ++c) decay[c] = all[c].smaller();
        lane.store_state(join_at(a, cut, 0, b, z), decay);
        lane.store_state(join_at(a, cut, 1, b, z), h);
    } else {
        for (int t = t0 + wave * U; t < end; t += W * U) {  // past the sequence
            if (a.saved) lane.store_state(a.saved + ((long long)b * spans + t / U) * a.channels, h);
            lane.clear(a.y, b, t, std::min(end - t, U));
        }
        if (!wave && z == cut.segments - 1 && a.state_out) lane.store_state(a.state_out + (long long)b * a.channels, h);
    }
}

// The same backwards: h is the gradient that arrives from the tokens behind.
template <typename T, int CH, bool SIGMOID, bool COMPLEMENT, int W, bool JOIN>
__global__ __launch_bounds__(64 * W) void k_recurrence_back(const RecurrenceArgs a, const Cut cut) {
    __shared__ Join lds[2][W][64][CH];
    const Lane<T, CH> lane(a.channels);
    const int b = blockIdx.y, z = blockIdx.z;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n = clamped(a.lengths, b, a.tokens);
    const int begin = z * cut.length, end = (int)std::min(a.tokens, (long long)begin + cut.length), live = std::min(n, end);
    const long long spans = (a.tokens + U - 1) / U;
    float h[CH] = {};
    Product all[CH];
    if constexpr (!JOIN) arrive<T, CH, true>(h, lane, a, cut, b, z, n);
    unsigned x[U] = {}, g[U] = {}, dy[U] = {};
    const auto fetch = [&](int t) {
        if constexpr (!JOIN) lane.fetch(x, a.x, b, t, live - t);
        lane.fetch(g, a.gate, b, t, live - t);
        lane.fetch(dy, a.dy, b, t, live - t);
    };
    const int tiles = (std::max(0, live - begin) + W * U - 1) / (W * U);
    if (tiles) fetch(begin + (tiles - 1) * (W * U) + wave * U);
    for (int i = tiles - 1, half = 0; i >= 0; --i, half ^= 1) {
        const int t = begin + i * (W * U) + wave * U, m = std::min(live - t, U);
        float s[U][CH], p[U][CH], v[CH], l[CH] = {}, after[CH];  // v: the state before each token
        Product q[CH];
        unsigned d[U];
        if constexpr (!JOIN) lane.load_state(v, m > 0 ? a.saved + ((long long)b * spans + t / U) * a.channels : nullptr);
        each_gate<T, CH, SIGMOID>(g, m, [&](int u, int c, Gate k) {
            s[u][c] = k.s;
            if constexpr (W > 1 || JOIN) q[c].by(k.s, k.w);
            if constexpr (!JOIN) {
                const float xv = lane.value(x[u], c);
                p[u][c] = COMPLEMENT ? v[c] - xv : v[c];
                if (!SIGMOID && lane.value(g[u], c) > 0.f) p[u][c] = 0.f;
                v[c] = decayed(k.s, v[c]) + (COMPLEMENT ? k.w * xv : xv);
            }
        });
#pragma unroll
        for (int u = 0; u < U; ++u) d[u] = dy[u];
        if (m < U)
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (u >= m) d[u] = 0;
        if (i > 0) fetch(t - W * U);
        if constexpr (W > 1 || JOIN) {
#pragma unroll
            for (int u = U - 1; u >= 0; --u)
#pragma unroll
                for (int c = 0; c < CH; ++c) l[c] = decayed(s[u][c], l[c] + lane.value(d[u], c));
#pragma unroll
            for (int c = 0; c < CH; ++c) lds[half][threadIdx.x >> 6][threadIdx.x & 63][c] = Join{q[c].smaller(), l[c]};
            __syncthreads();
            fold<CH, W, true, JOIN>(h, after, all, lds[half]);
        }
        if constexpr (!JOIN) {
            T* dx = (T*)a.y.p + b * a.y.batch + (t + U - 1) * a.y.token + lane.first;
            T* dg = (T*)a.dgate.p + b * a.dgate.batch + (t + U - 1) * a.dgate.token + lane.first;
            const auto gradients = [&](int u, float (&to_x)[CH], float (&to_g)[CH]) {
#pragma unroll
                for (int c = 0; c < CH; ++c) {
                    const float k = s[u][c], D = lane.value(d[u], c) + h[c];
                    to_x[c] = COMPLEMENT ? short_of(k) * D : D;
                    to_g[c] = p[u][c] * D * (SIGMOID ? fabsf(k) * (1.f - fabsf(k)) : decayed(k, 1.f));
                    h[c] = decayed(k, D);
                }
            };
            float to_x[CH], to_g[CH];
            if (m == U) {
                if (lane.have)
#pragma unroll
                    for (int u = U - 1; u >= 0; --u, dx = behind(dx, -a.y.token), dg = behind(dg, -a.dgate.token)) {
                        gradients(u, to_x, to_g);
                        lane.store(dx, to_x);
                        lane.store(dg, to_g);
                    }
            } else if (lane.have) {
#pragma unroll
                for (int u = U - 1; u >= 0; --u, dx = behind(dx, -a.y.token), dg = behind(dg, -a.dgate.token))
                    if (u < m) {
                        gradients(u, to_x, to_g);
                        lane.store(dx, to_x);
                        lane.store(dg, to_g);
                    }
            }
        }
        if constexpr (W > 1 || JOIN)
#pragma unroll
            for (int c = 0; c < CH; ++c) h[c] = after[c];
    }
    if constexpr (JOIN) {
        if (wave) return;
        float decay[CH];
#pragma unroll
        for (int c = 0; c < CH; ++c) decay[c] = all[c].smaller();
        lane.store_state(join_at(a, cut, 0, b, z), decay);
        lane.store_state(join_at(a, cut, 1, b, z), h);
    } else {
        for (int t = std::max(begin, live) + wave * U; t < end; t += W * U) {  // past the sequence
            lane.clear(a.y, b, t, std::min(end - t, U));
            lane.clear(a.dgate, b, t, std::min(end - t, U));
        }
        if (!wave && !z && a.state_out) lane.store_state(a.state_out + (long long)b * a.channels, h);
    }
}

// Blocks a CU that segments may make.
constexpr int kCutBlocks = 2;

template <typename T, int CH, bool SIGMOID, bool COMPLEMENT, int W>
int launch_as(const RecurrenceArgs& a, hipStream_t s, bool back) {
    const long long columns = (a.channels + 64 * CH - 1) / (64 * CH);
    const dim3 block(64 * W);
    Cut cut{(int)std::max(a.tokens, 1ll), 1};
    if constexpr (W >= 8) {
        const long long tile = W * U, most = (long long)a.cus * kCutBlocks / (columns * a.batch);
        const long long segments = std::min(most, a.tokens / (2 * tile));
        if (segments > 1) {
            cut.length = (int)((a.tokens + segments * tile - 1) / (segments * tile) * tile);
            cut.segments = (int)((a.tokens + cut.length - 1) / cut.length);
        }
        if (cut.segments > 1) {
            const auto kernel = back ? k_recurrence_back<T, CH, SIGMOID, COMPLEMENT, W, true> : k_recurrence<T, CH, SIGMOID, COMPLEMENT, W, true>;
            hipLaunchKernelGGL(kernel, dim3((unsigned)columns, (unsigned)a.batch, (unsigned)cut.segments), block, 0, s, a, cut);
        }
    }
    const auto kernel = back ? k_recurrence_back<T, CH, SIGMOID, COMPLEMENT, W, false> : k_recurrence<T, CH, SIGMOID, COMPLEMENT, W, false>;
    hipLaunchKernelGGL(kernel, dim3((unsigned)columns, (unsigned)a.batch, (unsigned)cut.segments), block, 0, s, a, cut);
    return (int)hipGetLastError();
}

template <typename T, int CH, bool SIGMOID, bool COMPLEMENT>
int launch_waves(const RecurrenceArgs& a, hipStream_t s, bool back) {
    if (a.tokens <= U) return launch_as<T, CH, SIGMOID, COMPLEMENT, 1>(a, s, back);
    if (a.tokens <= 4 * U) return launch_as<T, CH, SIGMOID, COMPLEMENT, 4>(a, s, back);
    return launch_as<T, CH, SIGMOID, COMPLEMENT, 8>(a, s, back);
}

template <typename T, int CH>
int launch_gate(const RecurrenceArgs& a, hipStream_t s, bool back) {
    if (a.gate_kind == VKFX_GATE_SIGMOID) return a.complement ? launch_waves<T, CH, true, true>(a, s, back) : launch_waves<T, CH, true, false>(a, s, back);
    return a.complement ? launch_waves<T, CH, false, true>(a, s, back) : launch_waves<T, CH, false, false>(a, s, back);
}

// Two 16-bit channels a lane where every pair of them is a word.
template <typename T>
int launch_channels(const RecurrenceArgs& a, hipStream_t s, bool back) {
    uintptr_t all = (uintptr_t)a.channels * 2;
    for (const RecurrenceSide* x : {&a.x, &a.gate, &a.dy, &a.y, &a.dgate}) all |= (uintptr_t)x->p | (uintptr_t)(x->batch * 2) | (uintptr_t)(x->token * 2);
    return all % 4 ? launch_gate<T, 1>(a, s, back) : launch_gate<T, 2>(a, s, back);
}

int launch_element(const RecurrenceArgs& a, hipStream_t s, bool back) {
    if (a.element == VKFX_ELEMENT_F32) return launch_gate<float, 1>(a, s, back);
    if (a.element == VKFX_ELEMENT_F16) return launch_channels<_Float16>(a, s, back);
    return launch_channels<__bf16>(a, s, back);
}

}  // namespace

int launch_recurrence_forward(const RecurrenceArgs& a, hipStream_t s) { return launch_element(a, s, false); }
int launch_recurrence_backward(const RecurrenceArgs& a, hipStream_t s) { return launch_element(a, s, true); }
// segments times columns is at most kCutBlocks a CU, of up to 128 channels each
size_t recurrence_workspace_bytes(int, long long, int cus) { return (size_t)cus * kCutBlocks * 128 * 2 * sizeof(float); }

}  // namespace vkfx
