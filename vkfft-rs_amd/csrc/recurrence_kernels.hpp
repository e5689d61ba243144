// recurrence_kernels.hpp -- the gated recurrence h[t] = a[t] h[t-1] + m[t] x[t] of every
// channel, and its gradients.
//
// With D the gradient of the state after a token and E = a D that of the state
// before it,
//   D[t] = dy[t] + E[t+1],  dx = m D,  da = D (h[t-1] - (m = 1 - a ? x : 0))
// and dgate = da a (1 - a) or da a.
//
// A lane has 4 bytes of channels, a wave 16 tokens of them in its registers: it
// forms what they make of any state before them (state -> A state + H), a
// block's waves, one behind the other in time, fold these in LDS, and each goes
// over its tokens once more from the state that it now knows. So everything is
// read once. Where sequences and channels fill the machine, a block goes along
// its sequence with the next tokens on their way; where they do not, a sequence
// is a chain of blocks that hand (A, H) on through memory.
//
// A decay near 1 is kept as what it is short of 1: rounded to 24 bits itself, a
// memory of n tokens would be off by n 2^-25 of its length. So is A.
#pragma once

#include <algorithm>
#include <type_traits>

#include "sequence.hpp"
#include "sequence_device.hpp"
#include "vkfx.h"

// Products and sums join where it is written: a result does not depend on which of
// two ways through a kernel its neighbours' values made its wave take.
#pragma clang fp contract(off)

namespace vkfx {

namespace {

constexpr int U = kSpan;  // tokens of a wave
constexpr float kNear = 87.f;

// exp(g), off by 2^-22 of it, for -87 <= g <= 0: 2^t with what t's rounding left.
__device__ __forceinline__ float exp_near(float g) {
    const float t = g * 1.44269504f, e = __builtin_amdgcn_exp2f(t);
    return fmaf(e, fmaf(t, -0.693147181f, g), e);
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

// Several of them in their order.
struct Joins {
    Product p;
    float h = 0.f;
    __device__ __forceinline__ void add(const Join& j) {
        p.by(j.s, short_of(j.s));
        h = j(h);
    }
    __device__ __forceinline__ Join join() const { return Join{p.smaller(), h}; }
};

__device__ __forceinline__ int clamped(const int* lengths, int b, long long tokens) {
    const long long n = lengths ? lengths[b] : tokens;
    return __builtin_amdgcn_readfirstlane((int)(n < 0 ? 0 : n < tokens ? n : tokens));
}

// A count of its own for the compiler, which would form what follows from it
// once for all places, and keep that in scalar registers.
__device__ __forceinline__ int apart(int m) {
    asm volatile("" : "+s"(m));
    return m;
}
// Pointers that are to global memory, which the compiler does not see behind asm.
template <typename T>
using Global = __attribute__((address_space(1))) T*;
// The next row. Kept from the compiler, which would hold every row's place in
// scalar registers, and these, past 100 of them, in lanes of vector registers.
template <typename T>
__device__ __forceinline__ Global<T> behind(Global<T> row, long long stride) {
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

    __device__ __forceinline__ Lane(unsigned column, long long channels) {
        first = (long long)column * (64 * CH);
        have = first + (threadIdx.x & 63) * CH < channels;
        at = have ? (threadIdx.x & 63) * CH : 0;
    }
    // Tokens t .. t + m - 1 of sequence b. FEW: those alone, where a call may be of one
    // token; otherwise the last one again behind them (without branches: both passes of
    // 4 x 4096 tokens of 2048 channels 149 us, 157 with).
    template <bool FEW>
    __device__ __forceinline__ void fetch(unsigned (&r)[U], const RecurrenceSide& s, long long b, long long t, int m) const {
        Global<const T> row = (Global<const T>)((const T*)s.p + b * s.batch + t * s.token + first);
        if (m >= U) {
#pragma unroll
            for (int u = 0; u < U; ++u, row = behind<const T>(row, s.token)) r[u] = *(Global<const Raw>)(row + at);
        } else if (m > 0) {
            m = apart(m);
#pragma unroll
            for (int u = 0; u < U; ++u, row = behind<const T>(row, FEW || u < m ? s.token : 0))
                if (!FEW || u < m) r[u] = *(Global<const Raw>)(row + at);
        }
    }
    __device__ __forceinline__ static float value(unsigned r, int c) { return (float)__builtin_bit_cast(Vec, (Raw)r)[c]; }
    // Whether an element is past kNear; of 16 bits by its bits, two at a time.
    __device__ __forceinline__ static bool far(const unsigned (&r)[U]) {
        if constexpr (sizeof(T) == 4) {
            float most = 0.f;
#pragma unroll
            for (int u = 0; u < U; ++u) most = fmaxf(most, fabsf(value(r[u], 0)));
            return most > kNear;
        } else {
            typedef unsigned short Pair __attribute__((ext_vector_type(2)));
            Pair most = {0, 0};
#pragma unroll
            for (int u = 0; u < U; ++u) most = __builtin_elementwise_max(most, __builtin_bit_cast(Pair, r[u] & 0x7fff7fffu));
            constexpr unsigned short limit = __builtin_bit_cast(unsigned short, (T)kNear);
            return most[0] > limit || most[1] > limit;
        }
    }
    __device__ __forceinline__ void store(Global<T> row, const float (&y)[CH]) const {
        Vec r;
#pragma unroll
        for (int c = 0; c < CH; ++c) r[c] = (T)y[c];
        *(Global<Vec>)(row + at) = r;
    }
    // Zeros in rows t .. of a tensor.
    __device__ __forceinline__ void clear(const RecurrenceSide& s, long long b, long long t, int rows) const {
        Global<T> row = (Global<T>)((T*)s.p + b * s.batch + t * s.token + first);
        const float zero[CH] = {};
        for (int u = 0; have && u < rows; ++u, row += s.token) store(row, zero);
    }
    __device__ __forceinline__ void load_state(float (&h)[CH], const float* row) const {
#pragma unroll
        for (int c = 0; c < CH; ++c) h[c] = row ? ((Global<const float>)row)[first + at + c] : 0.f;
    }
    __device__ __forceinline__ void store_state(float* row, const float (&h)[CH]) const {
#pragma unroll
        for (int c = 0; c < CH; ++c)
            if (have) ((Global<float>)row)[first + at + c] = h[c];
    }
};

// Goes over the wave's gates: f(u, c, gate, m) for each, m: how many tokens there
// are, a constant where there are all (and no gate is past kNear). Tokens from m on
// leave every state as it is.
template <typename T, int CH, bool SIGMOID, typename F>
__device__ __forceinline__ void each_gate(const unsigned (&g)[U], int m, F f) {
    if (__builtin_expect(m == U && !__any(Lane<T, CH>::far(g)), 1)) {
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int c = 0; c < CH; ++c) f(u, c, gate_of<SIGMOID, true>(Lane<T, CH>::value(g[u], c)), U);
    } else {
        m = apart(m);
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int c = 0; c < CH; ++c) f(u, c, u < m ? gate_of<SIGMOID, false>(Lane<T, CH>::value(g[u], c)) : Gate{-0.f, 0.f}, m);
    }
}

// Which tokens a launch runs, and the states before and behind them (BACK: the
// gradients behind and before them).
struct Range {
    int from, to;
    const float* in;  // null: zeros
    float* out;       // null: not wanted
};

// One block's tile: W waves of U tokens, the first at t0, those before `live` in
// the sequence. Each wave's part of its work:
//   fetch     the tokens on their way
//   prepare   gates; what the wave makes of a state (with JOIN), in `join`
//   finish    outputs, from h, the state before the wave's tokens
template <typename T, int CH, bool SIGMOID, bool COMPLEMENT, bool JOIN>
struct Forward {
    static constexpr bool BACK = false;
    const RecurrenceArgs& a;
    const Lane<T, CH>& lane;
    const int b;
    unsigned x[U] = {}, g[U] = {};
    float s[U][CH], in[U][CH];
    Join join[CH];

    __device__ __forceinline__ Forward(const RecurrenceArgs& a, const Lane<T, CH>& lane, int b) : a(a), lane(lane), b(b) {}
    __device__ __forceinline__ void fetch(int t, int live) {
        lane.template fetch<!JOIN>(x, a.x, b, t, live - t);
        lane.template fetch<!JOIN>(g, a.gate, b, t, live - t);
    }
    __device__ __forceinline__ void prepare(int m) {
        float l[CH] = {};
        Product p[CH];
        each_gate<T, CH, SIGMOID>(g, m, [&](int u, int c, Gate q, int m) {
            s[u][c] = q.s;
            in[u][c] = u < m ? COMPLEMENT ? q.w * lane.value(x[u], c) : lane.value(x[u], c) : 0.f;
            if constexpr (JOIN) {
                p[c].by(q.s, q.w);
                l[c] = decayed(q.s, l[c]) + in[u][c];
            }
        });
#pragma unroll
        for (int c = 0; c < CH; ++c) join[c] = Join{p[c].smaller(), l[c]};
    }
    __device__ __forceinline__ void finish(int t, int m, float (&h)[CH]) {
        if (m <= 0) return;
        const long long spans = (a.tokens + U - 1) / U;
        if (a.saved) lane.store_state(a.saved + ((long long)b * spans + t / U) * a.channels, h);
        Global<T> row = (Global<T>)((T*)a.y.p + b * a.y.batch + t * a.y.token + lane.first);
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int c = 0; c < CH; ++c) in[u][c] = h[c] = decayed(s[u][c], h[c]) + in[u][c];
        if (!lane.have) return;
        if (m == U) {
#pragma unroll
            for (int u = 0; u < U; ++u, row = behind<T>(row, a.y.token)) lane.store(row, in[u]);
        } else {
            m = apart(m);
#pragma unroll
            for (int u = 0; u < U; ++u, row = behind<T>(row, a.y.token))
                if (u < m) lane.store(row, in[u]);
        }
    }
    __device__ __forceinline__ void clear(int t, int rows) const { lane.clear(a.y, b, t, rows); }
};

template <typename T, int CH, bool SIGMOID, bool COMPLEMENT, bool JOIN>
struct Backward {
    static constexpr bool BACK = true;
    const RecurrenceArgs& a;
    const Lane<T, CH>& lane;
    const int b;
    unsigned x[U] = {}, g[U] = {}, dy[U] = {};
    float first[CH];  // the state before the first token
    float s[U][CH], p[U][CH];
    unsigned d[U];
    Join join[CH];

    __device__ __forceinline__ Backward(const RecurrenceArgs& a, const Lane<T, CH>& lane, int b) : a(a), lane(lane), b(b) {}
    __device__ __forceinline__ void fetch(int t, int live) {
        lane.template fetch<!JOIN>(x, a.x, b, t, live - t);
        lane.template fetch<!JOIN>(g, a.gate, b, t, live - t);
        lane.template fetch<!JOIN>(dy, a.dy, b, t, live - t);
        const long long spans = (a.tokens + U - 1) / U;
        lane.load_state(first, t < live ? a.saved + ((long long)b * spans + t / U) * a.channels : nullptr);
    }
    __device__ __forceinline__ void prepare(int m) {
        float v[CH], l[CH] = {};  // v: the state before each token
        Product q[CH];
#pragma unroll
        for (int c = 0; c < CH; ++c) v[c] = first[c];
        each_gate<T, CH, SIGMOID>(g, m, [&](int u, int c, Gate k, int m) {
            s[u][c] = k.s;
            if constexpr (JOIN) q[c].by(k.s, k.w);
            const float xv = u < m ? lane.value(x[u], c) : 0.f;
            p[u][c] = COMPLEMENT ? v[c] - xv : v[c];
            if (!SIGMOID && lane.value(g[u], c) > 0.f) p[u][c] = 0.f;
            v[c] = decayed(k.s, v[c]) + (COMPLEMENT ? k.w * xv : xv);
        });
#pragma unroll
        for (int u = 0; u < U; ++u) d[u] = dy[u];
        if (m < U) {
            m = apart(m);
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (u >= m) d[u] = 0;
        }
        if constexpr (JOIN) {
#pragma unroll
            for (int u = U - 1; u >= 0; --u)
#pragma unroll
                for (int c = 0; c < CH; ++c) l[c] = decayed(s[u][c], l[c] + lane.value(d[u], c));
        }
#pragma unroll
        for (int c = 0; c < CH; ++c) join[c] = Join{q[c].smaller(), l[c]};
    }
    __device__ __forceinline__ void finish(int t, int m, float (&h)[CH]) {
        if (m <= 0) return;
        Global<T> dx = (Global<T>)((T*)a.y.p + b * a.y.batch + (t + U - 1) * a.y.token + lane.first);
        Global<T> dg = (Global<T>)((T*)a.dgate.p + b * a.dgate.batch + (t + U - 1) * a.dgate.token + lane.first);
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
                for (int u = U - 1; u >= 0; --u, dx = behind<T>(dx, -a.y.token), dg = behind<T>(dg, -a.dgate.token)) {
                    gradients(u, to_x, to_g);
                    lane.store(dx, to_x);
                    lane.store(dg, to_g);
                }
        } else if (lane.have) {
            m = apart(m);
#pragma unroll
            for (int u = U - 1; u >= 0; --u, dx = behind<T>(dx, -a.y.token), dg = behind<T>(dg, -a.dgate.token))
                if (u < m) {
                    gradients(u, to_x, to_g);
                    lane.store(dx, to_x);
                    lane.store(dg, to_g);
                }
        }
    }
    __device__ __forceinline__ void clear(int t, int rows) const {
        lane.clear(a.y, b, t, rows);
        lane.clear(a.dgate, b, t, rows);
    }
};

// A block's waves' Joins one after the other (BACK: from the last on): h, the
// state before the tile, becomes that before the wave, and v that behind the tile.
template <int CH, int W, bool BACK>
__device__ __forceinline__ void fold(float (&h)[CH], float (&v)[CH], const Join (&at)[W][64][CH]) {
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
        }
    }
}

template <int CH>
__device__ __forceinline__ void arrived(float (&h)[CH]) {
#pragma unroll
    for (int c = 0; c < CH; ++c) asm volatile("" : "+v"(h[c]));
}

// ---- a block along its sequence: blockIdx.x 64 CH channels, blockIdx.y the
// sequence; W waves, one behind the other in time.

template <typename T, int CH, int W, typename Pass>
__device__ __forceinline__ void along(const RecurrenceArgs& a, const Range& r) {
    __shared__ Join lds[2][W][64][CH];
    const Lane<T, CH> lane(blockIdx.x, a.channels);
    const int b = blockIdx.y, l = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int live = std::max(r.from, std::min(clamped(a.lengths, b, a.tokens), r.to)), tiles = (live - r.from + W * U - 1) / (W * U);
    Pass pass(a, lane, b);
    float h[CH];  // the state before the tile
    lane.load_state(h, r.in ? r.in + (long long)b * a.channels : nullptr);
    const auto first = [&](int i) { return r.from + (Pass::BACK ? tiles - 1 - i : i) * (W * U) + wave * U; };
    if (tiles) pass.fetch(first(0), live);
    if constexpr (W > 1) arrived(h);  // r.out may be r.in: all waves have read it before one writes
    for (int i = 0; i < tiles; ++i) {
        const int t = first(i), m = std::min(live - t, U);
        pass.prepare(m);
        if (i + 1 < tiles) pass.fetch(first(i + 1), live);
        if constexpr (W > 1) {
            float after[CH];
#pragma unroll
            for (int c = 0; c < CH; ++c) lds[i & 1][threadIdx.x >> 6][l][c] = pass.join[c];
            __syncthreads();
            fold<CH, W, Pass::BACK>(h, after, lds[i & 1]);
            pass.finish(t, m, h);
#pragma unroll
            for (int c = 0; c < CH; ++c) h[c] = after[c];
        } else {
            pass.finish(t, m, h);
        }
    }
    for (int t = live + wave * U; t < r.to; t += W * U) pass.clear(t, std::min(r.to - t, U));  // past the sequence
    if (!wave && r.out) lane.store_state(r.out + (long long)b * a.channels, h);
}

// ---- a chain of blocks along a sequence, each with one tile. A block hands the
// Join of its tile on, and the last block of a group the state behind it, as the
// first block does with the state that the sequence starts from (which it alone
// reads: the last may write its successor over it). A block joins the Joins of its
// group's blocks before it, always in this order, and applies that to the state
// before its group. So from a state to the next it takes one exchange and one
// application.
//
// A lane has one channel here, so that three blocks fit a CU (their phases, loads,
// gates, the exchange, outputs, are alike; two channels and two blocks: 1 x 65536
// tokens of 1024 channels 131 us, 112 with one).
//
// Every word is handed on by itself, 64 bits at once: 0 until it is there, and
// never 0 then. A chain's blocks take their places in the order in which they
// start, by a counter. So a block waits for such only as have started, and hands
// its Join on before it waits: every wait ends, whatever else runs. Each chain
// counts by itself, in a line of its own: one counter for all gives a place in 23
// ns, 8192 of them in 188 us.

constexpr int kLeastGroup = 4, kMostGroup = 32, kChainWaves = 8;
constexpr int kChainTokens = kChainWaves * U;
// Times that a wait asks again before it gives up, some seconds: nothing that
// this file launches needs it, a workspace that two calls share at once may.
constexpr int kPatience = 1 << 20;

struct Chain {
    unsigned* counters;
    uint64_t *joins, *states;  // [place][batch][channel]; before a group, [group][batch][channel]
    int columns, places, group;  // blocks of a group, a power of 2
};

__device__ __forceinline__ void hand_on(uint64_t* to, uint64_t word) { __hip_atomic_store(to, word, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
// N CH words at from, from + stride, ...: the first `count` times CH. All are asked
// for at once.
template <int N, int CH>
__device__ __forceinline__ void wait_for(uint64_t (&w)[N][CH], const uint64_t* from, long long stride, int count) {
    for (int tries = 0;; ++tries) {
        bool there = true;
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int c = 0; c < CH; ++c)
                w[i][c] = __hip_atomic_load(from + (i < count ? i : 0) * stride + c, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int c = 0; c < CH; ++c) there = there && w[i][c];
        if (__all(there)) return;
        if (tries == kPatience) break;
        __builtin_amdgcn_s_sleep(1);
    }
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int c = 0; c < CH; ++c) w[i][c] = ~0ull;  // NaN
}
constexpr unsigned kNever = 0x7fffffffu;  // bits that no gate of a Join has
__device__ __forceinline__ uint64_t word_of(const Join& j) {
    const unsigned s = j.s == j.s ? __float_as_uint(j.s) : 0x7fc00000u;
    return (uint64_t)__float_as_uint(j.h) << 32 | (s ^ kNever);
}
__device__ __forceinline__ Join join_of(uint64_t w) { return Join{__uint_as_float((unsigned)w ^ kNever), __uint_as_float((unsigned)(w >> 32))}; }
__device__ __forceinline__ uint64_t word_of(float v) { return (uint64_t)__float_as_uint(v) << 32 | 1; }
__device__ __forceinline__ float state_of(uint64_t w) { return __uint_as_float((unsigned)(w >> 32)); }

__global__ __launch_bounds__(256) void k_chain_clear(uint64_t* words, long long count, unsigned* counters, int chains) {
    typedef uint64_t Two __attribute__((ext_vector_type(2)));
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    if (2 * i + 1 < count) ((Two*)words)[i] = Two{0, 0};
    else if (2 * i < count) words[2 * i] = 0;
    if (i < chains) counters[i * kChainLine] = 0;
}

template <typename T, typename Pass>
__device__ __forceinline__ void chained(const RecurrenceArgs& a, const Range& r, const Chain& chain) {
    constexpr int W = kChainWaves, CH = 1;
    __shared__ Join own[W][64][CH], before[W - 1][64][CH];
    __shared__ float start[64][CH];
    __shared__ unsigned ticket;
    // neighbours in the order of launch are of different chains, those of one chain on different XCDs
    const unsigned chains = (unsigned)(chain.columns * a.batch), mine = (blockIdx.x + blockIdx.x / chains) % chains;
    if (!threadIdx.x) ticket = __hip_atomic_fetch_add(chain.counters + mine * kChainLine, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    const int order = (int)__builtin_amdgcn_readfirstlane(ticket);
    const int b = (int)(mine / (unsigned)chain.columns), l = threadIdx.x & 63;
    const Lane<T, CH> lane(mine - (unsigned)(b * chain.columns), a.channels);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int live = std::max(r.from, std::min(clamped(a.lengths, b, a.tokens), r.to)), tiles = (live - r.from + W * U - 1) / (W * U);
    const int tile = Pass::BACK ? chain.places - 1 - order : order;
    const int place = Pass::BACK ? tiles - 1 - tile : tile;  // in the sequence's chain
    const int t = r.from + tile * (W * U) + wave * U, m = std::min(live - t, U);
    Pass pass(a, lane, b);
    const long long channel = lane.first + lane.at, width = (long long)a.batch * a.channels, at = (long long)b * a.channels + channel;
    // a place there is not: only where another call counts in the same workspace
    if (tile < tiles && order < chain.places) {
        pass.fetch(t, live);
        pass.prepare(m);
#pragma unroll
        for (int c = 0; c < CH; ++c) own[threadIdx.x >> 6][l][c] = pass.join[c];
        __syncthreads();
        const int group = place / chain.group, count = place % chain.group;
        const bool last = place + 1 == tiles;
        constexpr int N = (kMostGroup + W - 3) / (W - 1);  // of kMostGroup - 1 Joins, a wave's
        float h[CH];
        Join all[CH];
        if (!wave) {
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                Joins k;
#pragma unroll
                for (int i = 0; i < W; ++i) k.add(own[Pass::BACK ? W - 1 - i : i][l][c]);
                all[c] = k.join();
                if (lane.have && count < chain.group - 1 && !last) hand_on(chain.joins + place * width + at + c, word_of(all[c]));
            }
            if (!place) {
                lane.load_state(h, r.in ? r.in + (long long)b * a.channels : nullptr);
#pragma unroll
                for (int c = 0; c < CH; ++c)
                    if (lane.have && !last) hand_on(chain.states + at + c, word_of(h[c]));
            }
        } else {
            const int first = (wave - 1) * N, some = std::min(count - first, N);
            if (some > 0) {
                uint64_t w[N][CH];
                wait_for(w, chain.joins + ((long long)group * chain.group + first) * width + at, width, some);
#pragma unroll
                for (int c = 0; c < CH; ++c) {
                    Joins k;
#pragma unroll
                    for (int i = 0; i < N; ++i)
                        if (i < some) k.add(join_of(w[i][c]));
                    before[wave - 1][l][c] = k.join();
                }
            }
        }
        __syncthreads();
        if (!wave) {
            const int parts = (count + N - 1) / N;
            Join to[CH], behind[CH];  // from the state before the group to that before the tile, and behind it
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                Joins k;
#pragma unroll
                for (int i = 0; i < W - 1; ++i)
                    if (i < parts) k.add(before[i][l][c]);
                to[c] = k.join();
                k.add(all[c]);
                behind[c] = k.join();
            }
            if (place) {
                uint64_t w[1][CH];
                wait_for(w, chain.states + group * width + at, 0, 1);
#pragma unroll
                for (int c = 0; c < CH; ++c) h[c] = state_of(w[0][c]);
            }
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                if (lane.have && count == chain.group - 1 && !last) hand_on(chain.states + (group + 1) * width + at + c, word_of(behind[c](h[c])));
                start[l][c] = count ? to[c](h[c]) : h[c];
            }
        }
        __syncthreads();
        float after[CH];
#pragma unroll
        for (int c = 0; c < CH; ++c) h[c] = start[l][c];
        fold<CH, W, Pass::BACK>(h, after, own);
        pass.finish(t, m, h);
        if (!wave && place + 1 == tiles && r.out) lane.store_state(r.out + (long long)b * a.channels, after);
    } else if (!wave && !tiles && !order && r.out && r.out != r.in) {  // no tokens: the state goes on as it is
        float h[CH];
        lane.load_state(h, r.in ? r.in + (long long)b * a.channels : nullptr);
        lane.store_state(r.out + (long long)b * a.channels, h);
    }
    const int past = std::max(live, t);
    if (past < r.to && past < t + U) pass.clear(past, std::min(r.to, t + U) - past);
}

// Forward with 128 registers, so that two blocks fit a CU (64 x 100 tokens of 4096
// channels 39 us, 54 with 130 registers).
template <typename T, int CH, bool SIGMOID, bool COMPLEMENT, int W, bool BACK>
__global__ __launch_bounds__(64 * W, W == 8 && !BACK ? 4 : 1) void k_recurrence(const RecurrenceArgs a, const Range r) {
    along<T, CH, W, std::conditional_t<BACK, Backward<T, CH, SIGMOID, COMPLEMENT, (W > 1)>, Forward<T, CH, SIGMOID, COMPLEMENT, (W > 1)>>>(a, r);
}
template <typename T, bool SIGMOID, bool COMPLEMENT, bool BACK>
__global__ __launch_bounds__(64 * kChainWaves) void k_recurrence_chain(const RecurrenceArgs a, const Range r, const Chain chain) {
    chained<T, std::conditional_t<BACK, Backward<T, 1, SIGMOID, COMPLEMENT, true>, Forward<T, 1, SIGMOID, COMPLEMENT, true>>>(a, r, chain);
}

// Whether a call is for chains: blocks that go along their sequences would leave
// a quarter of the CUs' time unused (320 blocks for 256 CUs, 5 x 2048 tokens of 8192
// channels: 134 us, 125 in chains; 256 blocks 93 and 106).
bool for_chains(const RecurrenceArgs& a, long long blocks) {
    if (a.tokens <= kChainTokens) return false;
    const long long rounds = (blocks + a.cus - 1) / a.cus;
    return blocks * 4 < rounds * a.cus * 3;
}

// The workspace (recurrence_workspace_bytes): the chains' counters, their states
// between launches, the words of a launch.
struct Workspace {
    unsigned* counters;
    float* states;
    uint64_t* words;
};
Workspace workspace_of(const RecurrenceArgs& a) {
    float* states = a.work + most_chained(a.cus) / 64 * kChainLine;
    return Workspace{(unsigned*)a.work, states, (uint64_t*)(states + most_chained(a.cus))};
}

template <typename T, bool SIGMOID, bool COMPLEMENT, bool BACK>
int launch_chains(const RecurrenceArgs& a, hipStream_t s) {
    const Workspace w = workspace_of(a);
    const long long width = a.channels * a.batch, columns = (a.channels + 63) / 64, chains = columns * a.batch;
    // groups of about as many blocks as a chain has side by side
    int group = kMostGroup;
    while (group > kLeastGroup && group * chains > a.cus * 2) group /= 2;
    // places of one launch: their words, and those of their groups
    const long long most = (words_of(a.cus) / width - 1) * group / (group + 1), places = (a.tokens + kChainTokens - 1) / kChainTokens;
    const long long launches = (places + most - 1) / most, each = (places + launches - 1) / launches;
    for (long long i = 0; i < launches; ++i) {
        const long long first = (BACK ? launches - 1 - i : i) * each, last = std::min(first + each, places);
        const Range r{(int)(first * kChainTokens), (int)std::min(last * kChainTokens, a.tokens), i ? w.states : a.state_in,
                      i + 1 < launches ? w.states : a.state_out};
        const Chain chain{w.counters, w.words, w.words + (last - first) * width, (int)columns, (int)(last - first), group};
        const long long words = ((last - first) + (last - first + group - 1) / group) * width;
        hipLaunchKernelGGL(k_chain_clear, dim3((unsigned)((std::max((words + 1) / 2, chains) + 255) / 256)), dim3(256), 0, s, w.words, words, w.counters,
                           (int)chains);
        const auto kernel = k_recurrence_chain<T, SIGMOID, COMPLEMENT, BACK>;
        hipLaunchKernelGGL(kernel, dim3((unsigned)(chains * (last - first))), dim3(64 * kChainWaves), 0, s, a, r, chain);
    }
    return (int)hipGetLastError();
}

template <typename T, int CH, bool SIGMOID, bool COMPLEMENT, bool BACK>
int launch_as(const RecurrenceArgs& a, hipStream_t s) {
    const long long columns = (a.channels + 64 * CH - 1) / (64 * CH);
    if (for_chains(a, columns * a.batch)) return launch_chains<T, SIGMOID, COMPLEMENT, BACK>(a, s);
    const Range r{0, (int)a.tokens, a.state_in, a.state_out};
    const dim3 grid((unsigned)columns, (unsigned)a.batch);
    if (a.tokens <= U) hipLaunchKernelGGL((k_recurrence<T, CH, SIGMOID, COMPLEMENT, 1, BACK>), grid, dim3(64), 0, s, a, r);
    else if (a.tokens <= 4 * U) hipLaunchKernelGGL((k_recurrence<T, CH, SIGMOID, COMPLEMENT, 4, BACK>), grid, dim3(256), 0, s, a, r);
    else hipLaunchKernelGGL((k_recurrence<T, CH, SIGMOID, COMPLEMENT, 8, BACK>), grid, dim3(512), 0, s, a, r);
    return (int)hipGetLastError();
}

template <typename T, int CH, bool BACK>
int launch_gate(const RecurrenceArgs& a, hipStream_t s) {
    if (a.gate_kind == VKFX_GATE_SIGMOID) return a.complement ? launch_as<T, CH, true, true, BACK>(a, s) : launch_as<T, CH, true, false, BACK>(a, s);
    return a.complement ? launch_as<T, CH, false, true, BACK>(a, s) : launch_as<T, CH, false, false, BACK>(a, s);
}

// Two 16-bit channels a lane where every pair of them is a word.
template <typename T>
int launch_channels(const RecurrenceArgs& a, hipStream_t s, bool back) {
    if constexpr (sizeof(T) == 2) {
        uintptr_t all = (uintptr_t)a.channels * 2;
        for (const RecurrenceSide* x : {&a.x, &a.gate, &a.dy, &a.y, &a.dgate}) all |= (uintptr_t)x->p | (uintptr_t)(x->batch * 2) | (uintptr_t)(x->token * 2);
        if (all % 4 == 0) return back ? launch_gate<T, 2, true>(a, s) : launch_gate<T, 2, false>(a, s);
    }
    return back ? launch_gate<T, 1, true>(a, s) : launch_gate<T, 1, false>(a, s);
}

}  // namespace

}  // namespace vkfx
