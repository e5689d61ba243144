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
template <typename T>
constexpr int kChannels = 4 / (int)sizeof(T);  // of a lane

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

// The smaller of a and 1 - a; negative (-0 too) where that is 1 - a. NEAR: no
// |g| is past 87, from where on the hardware's exponential gives 0.
template <bool SIGMOID, bool NEAR>
__device__ __forceinline__ float gate_of(float g) {
    if constexpr (SIGMOID) {
        const float e = NEAR ? exp_near(-fabsf(g)) : expf(-fabsf(g));
        const float small = e * __builtin_amdgcn_rcpf(1.f + e);
        return g > 0.f ? -small : small;
    } else {
        g = g > 0.f ? 0.f : g;  // a NaN stays one
        if (NEAR) return g > -0.6931472f ? __int_as_float(__float_as_int(exp_less_1(g)) | (int)0x80000000) : exp_near(g);
        return g > -0.6931472f ? g == 0.f ? -0.f : expm1f(g) : expf(g);
    }
}
// v where a >= 1/2, else 0.
__device__ __forceinline__ float if_slow(float s, float v) { return __int_as_float((__float_as_int(s) >> 31) & __float_as_int(v)); }
__device__ __forceinline__ float decayed(float s, float v) { return fmaf(s, v, if_slow(s, v)); }  // a v
__device__ __forceinline__ float short_of(float s) { return __float_as_int(s) < 0 ? -s : 1.f - s; }  // 1 - a

// What some tokens make of the state before them: a v + h, short = 1 - a.
struct Join {
    float a, low, h;  // low: 1 - a
    __device__ __forceinline__ float operator()(float v) const { return (low < 0.5f ? fmaf(-low, v, v) : a * v) + h; }
};

__device__ __forceinline__ int clamped(const int* lengths, int b, long long tokens) {
    const long long n = lengths ? lengths[b] : tokens;
    return (int)(n < 0 ? 0 : n < tokens ? n : tokens);
}

// A wave's place: channels first .. + have of the lane, tokens of the wave.
template <typename T>
struct Lane {
    static constexpr int CH = kChannels<T>;
    typedef Some<T, CH> Vec;
    long long first;  // the block's first channel
    int at, have;     // the lane's, and how many it has

    __device__ __forceinline__ explicit Lane(long long channels) {
        first = (long long)blockIdx.x * (64 * CH);
        at = (threadIdx.x & 63) * CH;
        const long long left = channels - first - at;
        have = left < 0 ? 0 : left < CH ? (int)left : CH;
    }
    // rows[0 .. m) of a tensor
    template <bool FULL>
    __device__ __forceinline__ void fetch(Vec (&r)[U], const RecurrenceSide& s, long long b, long long t, int m) const {
        const T* row = (const T*)s.p + b * s.batch + t * s.token + first;
        if (have == CH) {
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (FULL || u < m) r[u] = *(const typename Packed<T, CH>::type*)(row + u * s.token + at);
        } else if (have) {
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (FULL || u < m) r[u][0] = row[u * s.token + at];
        }
    }
    __device__ __forceinline__ void fetch(Vec (&r)[U], const RecurrenceSide& s, long long b, long long t, int m) const {
        if (m == U) fetch<true>(r, s, b, t, U);
        else if (m > 0) fetch<false>(r, s, b, t, m);
    }
    __device__ __forceinline__ void store(T* row, const float (&y)[CH]) const {
        Vec r;
#pragma unroll
        for (int c = 0; c < CH; ++c) r[c] = (T)y[c];
        if (have == CH) *(typename Packed<T, CH>::type*)(row + at) = r;
        else if (have) row[at] = r[0];
    }
    __device__ __forceinline__ void load_state(float (&h)[CH], const float* row) const {
#pragma unroll
        for (int c = 0; c < CH; ++c) h[c] = c < have && row ? row[first + at + c] : 0.f;
    }
    __device__ __forceinline__ void store_state(float* row, const float (&h)[CH]) const {
        if (have == CH) {
            Some<float, CH> r;
#pragma unroll
            for (int c = 0; c < CH; ++c) r[c] = h[c];
            *(typename Packed<float, CH>::type*)(row + first + at) = r;
        } else if (have) {
            row[first + at] = h[0];
        }
    }
};

// Gates of a wave's first m tokens.
template <typename T, bool SIGMOID>
__device__ __forceinline__ void gates(float (&s)[U][kChannels<T>], const Some<T, kChannels<T>> (&g)[U]) {
    float most = 0.f;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
        for (int c = 0; c < kChannels<T>; ++c) most = fmaxf(most, fabsf((float)g[u][c]));
    if (__builtin_expect(__any(most > 87.f), 0)) {
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int c = 0; c < kChannels<T>; ++c) {
                const float v = (float)g[u][c];  // a gate's bits do not depend on its neighbours
                s[u][c] = fabsf(v) <= 87.f ? gate_of<SIGMOID, true>(v) : gate_of<SIGMOID, false>(v);
            }
    } else {
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int c = 0; c < kChannels<T>; ++c) s[u][c] = gate_of<SIGMOID, true>((float)g[u][c]);
    }
}

// Calls f(u) for the wave's tokens u = 0 .. m - 1, or the other way round.
template <bool BACK, typename F>
__device__ __forceinline__ void each(int m, F f) {
    if (m == U) {
#pragma unroll
        for (int u = 0; u < U; ++u) f(BACK ? U - 1 - u : u);
    } else {
#pragma unroll
        for (int u = 0; u < U; ++u)
            if ((BACK ? U - 1 - u : u) < m) f(BACK ? U - 1 - u : u);
    }
}

// What the wave's tokens make of a state: in(u, c) is what token u adds to it
// behind its decay (forward) or in front of it (BACK).
template <typename T, bool BACK, typename F>
__device__ __forceinline__ void local(Join (&j)[kChannels<T>], const float (&s)[U][kChannels<T>], int m, F in) {
#pragma unroll
    for (int c = 0; c < kChannels<T>; ++c) j[c] = Join{1.f, 0.f, 0.f};
    each<BACK>(m, [&](int u) {
#pragma unroll
        for (int c = 0; c < kChannels<T>; ++c) {
            j[c].a = decayed(s[u][c], j[c].a);
            j[c].low = decayed(s[u][c], j[c].low) + short_of(s[u][c]);
            j[c].h = BACK ? decayed(s[u][c], j[c].h + in(u, c)) : decayed(s[u][c], j[c].h) + in(u, c);
        }
    });
}

// Segment z of a call: tokens z length .. + length.
struct Cut {
    int length, segments;
};
// Place of a segment's Join of a channel in the workspace: [3][batch][segment][channel].
__device__ __forceinline__ float* join_at(const RecurrenceArgs& a, const Cut& cut, int part, int b, int z) {
    return a.work + (((long long)part * a.batch + b) * cut.segments + z) * a.channels;
}

// W waves a block, one behind the other in time. JOIN: the segment's Join alone,
// nothing else written.
template <typename T, bool SIGMOID, bool COMPLEMENT, int W, bool JOIN>
__global__ __launch_bounds__(64 * W) void k_recurrence(const RecurrenceArgs a, const Cut cut) {
    constexpr int CH = kChannels<T>;
    __shared__ Join lds[W > 1 ? 2 : 1][W][CH][64];
    const Lane<T> lane(a.channels);
    const int b = blockIdx.y, z = blockIdx.z, l = threadIdx.x & 63;
    const int wave = W > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : 0;
    const int n = clamped(a.lengths, b, a.tokens);
    const int begin = z * cut.length, end = (int)std::min(a.tokens, (long long)begin + cut.length), live = std::min(n, end);
    float h[CH];  // the state before the block's tokens
    Join all[CH];
    if constexpr (JOIN) {
#pragma unroll
        for (int c = 0; c < CH; ++c) all[c] = Join{1.f, 0.f, 0.f}, h[c] = 0.f;
    } else {
        lane.load_state(h, a.state_in ? a.state_in + (long long)b * a.channels : nullptr);
        for (int i = 0; i < z && i * cut.length < n; ++i) {
            float v[3][CH];
#pragma unroll
            for (int p = 0; p < 3; ++p) lane.load_state(v[p], join_at(a, cut, p, b, i));
#pragma unroll
            for (int c = 0; c < CH; ++c) h[c] = Join{v[0][c], v[1][c], v[2][c]}(h[c]);
        }
    }
    const long long spans = (a.tokens + U - 1) / U;
    typename Lane<T>::Vec x[U], g[U];
#pragma unroll
    for (int u = 0; u < U; ++u) x[u] = g[u] = (T)0.f;
    const auto tokens_of = [&](int t) { return std::max(0, std::min(live - t, U)); };
    const int stop = JOIN ? live : end;
    {
        const int t = begin + wave * U, m = tokens_of(t);
        lane.fetch(x, a.x, b, t, m);
        lane.fetch(g, a.gate, b, t, m);
    }
    for (int t0 = begin, half = 0; t0 < stop; t0 += W * U, half ^= 1) {
        const int t = t0 + wave * U, m = tokens_of(t);
        float s[U][CH], in[U][CH];
        gates<T, SIGMOID>(s, g);
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int c = 0; c < CH; ++c) in[u][c] = COMPLEMENT ? short_of(s[u][c]) * (float)x[u][c] : (float)x[u][c];
        if (t0 + W * U < stop) {
            const int next = t + W * U, k = tokens_of(next);
            lane.fetch(x, a.x, b, next, k);
            lane.fetch(g, a.gate, b, next, k);
        }
        if constexpr (W > 1 || JOIN) {
            Join j[CH];
            local<T, false>(j, s, m, [&](int u, int c) { return in[u][c]; });
            if constexpr (W > 1) {
#pragma unroll
                for (int c = 0; c < CH; ++c) lds[half][wave][c][l] = j[c];
                __syncthreads();
            }
            const int waves = W > 1 ? std::min(W, (live - t0 + U - 1) / U) : 1;  // that have tokens
            float v[CH];
#pragma unroll
            for (int c = 0; c < CH; ++c) v[c] = h[c];
            for (int i = 0; i < waves; ++i)
#pragma unroll
                for (int c = 0; c < CH; ++c) {
                    const Join k = W > 1 ? lds[half][i][c][l] : j[c];
                    if (i == wave) h[c] = v[c];
                    v[c] = k(v[c]);
                    if constexpr (JOIN) {
                        all[c].low = Join{k.a, k.low, k.low}(all[c].low);
                        all[c].a *= k.a;
                    }
                }
            if constexpr (JOIN) {
#pragma unroll
                for (int c = 0; c < CH; ++c) h[c] = v[c];
                continue;
            }
            if (wave >= waves)
#pragma unroll
                for (int c = 0; c < CH; ++c) h[c] = v[c];
            if (a.saved && t < end) lane.store_state(a.saved + ((long long)b * spans + t / U) * a.channels, h);
            T* row = (T*)a.y.p + b * a.y.batch + t * a.y.token + lane.first;
            each<false>(m, [&](int u) {
#pragma unroll
                for (int c = 0; c < CH; ++c) h[c] = decayed(s[u][c], h[c]) + in[u][c];
                lane.store(row + u * a.y.token, h);
            });
            const float zero[CH] = {};
            for (int u = m; u < U && t + u < end; ++u) lane.store(row + u * a.y.token, zero);
#pragma unroll
            for (int c = 0; c < CH; ++c) h[c] = v[c];
        } else {
            if (a.saved) lane.store_state(a.saved + ((long long)b * spans + t / U) * a.channels, h);
            T* row = (T*)a.y.p + b * a.y.batch + t * a.y.token + lane.first;
            each<false>(m, [&](int u) {
#pragma unroll
                for (int c = 0; c < CH; ++c) h[c] = decayed(s[u][c], h[c]) + in[u][c];
                lane.store(row + u * a.y.token, h);
            });
            const float zero[CH] = {};
            for (int u = m; u < U && t + u < end; ++u) lane.store(row + u * a.y.token, zero);
        }
    }
    if (wave) return;
    if constexpr (JOIN) {
        float v[CH];
#pragma unroll
        for (int c = 0; c < CH; ++c) v[c] = all[c].a;
        lane.store_state(join_at(a, cut, 0, b, z), v);
#pragma unroll
        for (int c = 0; c < CH; ++c) v[c] = all[c].low;
        lane.store_state(join_at(a, cut, 1, b, z), v);
        lane.store_state(join_at(a, cut, 2, b, z), h);
    } else if (z == cut.segments - 1 && a.state_out) {
        lane.store_state(a.state_out + (long long)b * a.channels, h);
    }
}

// The same backwards: h is the gradient that arrives from the tokens behind.
template <typename T, bool SIGMOID, bool COMPLEMENT, int W, bool JOIN>
__global__ __launch_bounds__(64 * W) void k_recurrence_back(const RecurrenceArgs a, const Cut cut) {
    constexpr int CH = kChannels<T>;
    __shared__ Join lds[W > 1 ? 2 : 1][W][CH][64];
    const Lane<T> lane(a.channels);
    const int b = blockIdx.y, z = blockIdx.z, l = threadIdx.x & 63;
    const int wave = W > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : 0;
    const int n = clamped(a.lengths, b, a.tokens);
    const int begin = z * cut.length, end = (int)std::min(a.tokens, (long long)begin + cut.length), live = std::min(n, end);
    float h[CH];
    Join all[CH];
    if constexpr (JOIN) {
#pragma unroll
        for (int c = 0; c < CH; ++c) all[c] = Join{1.f, 0.f, 0.f}, h[c] = 0.f;
    } else {
        lane.load_state(h, a.state_in ? a.state_in + (long long)b * a.channels : nullptr);
        for (int i = std::min(cut.segments, (n + cut.length - 1) / cut.length) - 1; i > z; --i) {
            float v[3][CH];
#pragma unroll
            for (int p = 0; p < 3; ++p) lane.load_state(v[p], join_at(a, cut, p, b, i));
#pragma unroll
            for (int c = 0; c < CH; ++c) h[c] = Join{v[0][c], v[1][c], v[2][c]}(h[c]);
        }
    }
    const long long spans = (a.tokens + U - 1) / U;
    typename Lane<T>::Vec x[U], g[U], dy[U];
#pragma unroll
    for (int u = 0; u < U; ++u) x[u] = g[u] = dy[u] = (T)0.f;
    const auto tokens_of = [&](int t) { return std::max(0, std::min(live - t, U)); };
    const auto fetch = [&](int t) {
        const int m = tokens_of(t);
        if constexpr (!JOIN) lane.fetch(x, a.x, b, t, m);
        lane.fetch(g, a.gate, b, t, m);
        lane.fetch(dy, a.dy, b, t, m);
    };
    const int stop = JOIN ? live : end, tiles = (std::max(0, stop - begin) + W * U - 1) / (W * U);
    if (tiles) fetch(begin + (tiles - 1) * (W * U) + wave * U);
    for (int i = tiles - 1, half = 0; i >= 0; --i, half ^= 1) {
        const int t0 = begin + i * (W * U), t = t0 + wave * U, m = tokens_of(t);
        float s[U][CH], p[U][CH], d[U][CH];
        gates<T, SIGMOID>(s, g);
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int c = 0; c < CH; ++c) d[u][c] = (float)dy[u][c];
        if constexpr (!JOIN) {
            float v[CH];  // the state before each token
            lane.load_state(v, m ? a.saved + ((long long)b * spans + t / U) * a.channels : nullptr);
            each<false>(m, [&](int u) {
#pragma unroll
                for (int c = 0; c < CH; ++c) {
                    const float xv = (float)x[u][c];
                    p[u][c] = COMPLEMENT ? v[c] - xv : v[c];
                    if (!SIGMOID && (float)g[u][c] > 0.f) p[u][c] = 0.f;
                    v[c] = decayed(s[u][c], v[c]) + (COMPLEMENT ? short_of(s[u][c]) * xv : xv);
                }
            });
        }
        if (i > 0) fetch(t - W * U);
        float v[CH];
        if constexpr (W > 1 || JOIN) {
            Join j[CH];
            local<T, true>(j, s, m, [&](int u, int c) { return d[u][c]; });
            if constexpr (W > 1) {
#pragma unroll
                for (int c = 0; c < CH; ++c) lds[half][wave][c][l] = j[c];
                __syncthreads();
            }
            const int waves = W > 1 ? std::min(W, (live - t0 + U - 1) / U) : 1;
#pragma unroll
            for (int c = 0; c < CH; ++c) v[c] = h[c];
            for (int k = waves - 1; k >= 0; --k)
#pragma unroll
                for (int c = 0; c < CH; ++c) {
                    const Join q = W > 1 ? lds[half][k][c][l] : j[c];
                    if (k == wave) h[c] = v[c];
                    v[c] = q(v[c]);
                    if constexpr (JOIN) {
                        all[c].low = Join{q.a, q.low, q.low}(all[c].low);
                        all[c].a *= q.a;
                    }
                }
        }
        if constexpr (!JOIN) {
            T* dx = (T*)a.y.p + b * a.y.batch + t * a.y.token + lane.first;
            T* dg = (T*)a.dgate.p + b * a.dgate.batch + t * a.dgate.token + lane.first;
            each<true>(m, [&](int u) {
                float to_x[CH], to_g[CH];
#pragma unroll
                for (int c = 0; c < CH; ++c) {
                    const float q = s[u][c], w = short_of(q), D = d[u][c] + h[c];
                    to_x[c] = COMPLEMENT ? w * D : D;
                    const float slope = SIGMOID ? fabsf(q) * (1.f - fabsf(q)) : decayed(q, 1.f);
                    to_g[c] = D * p[u][c] * slope;
                    h[c] = decayed(q, D);
                }
                lane.store(dx + u * a.y.token, to_x);
                lane.store(dg + u * a.dgate.token, to_g);
            });
            const float zero[CH] = {};
            for (int u = m; u < U && t + u < end; ++u) {
                lane.store(dx + u * a.y.token, zero);
                lane.store(dg + u * a.dgate.token, zero);
            }
        }
        if constexpr (W > 1 || JOIN)
#pragma unroll
            for (int c = 0; c < CH; ++c) h[c] = v[c];
    }
    if (wave) return;
    if constexpr (JOIN) {
        float v[CH];
#pragma unroll
        for (int c = 0; c < CH; ++c) v[c] = all[c].a;
        lane.store_state(join_at(a, cut, 0, b, z), v);
#pragma unroll
        for (int c = 0; c < CH; ++c) v[c] = all[c].low;
        lane.store_state(join_at(a, cut, 1, b, z), v);
        lane.store_state(join_at(a, cut, 2, b, z), h);
    } else if (!z && a.state_out) {
        lane.store_state(a.state_out + (long long)b * a.channels, h);
    }
}

constexpr int kCutBlocks = 4;  // a CU, that segments may make

template <typename T, bool SIGMOID, bool COMPLEMENT, int W>
int launch_as(const RecurrenceArgs& a, hipStream_t s, bool back) {
    const long long columns = (a.channels + 64 * kChannels<T> - 1) / (64 * kChannels<T>);
    const dim3 block(64 * W);
    Cut cut{(int)std::max(a.tokens, 1ll), 1};
    if constexpr (W >= 8) {
        const long long tile = W * U, most = (long long)a.cus * (16 / W) / (columns * a.batch);
        const long long segments = std::min(most, a.tokens / (2 * tile));
        if (segments > 1) {
            cut.length = (int)((a.tokens + segments * tile - 1) / (segments * tile) * tile);
            cut.segments = (int)((a.tokens + cut.length - 1) / cut.length);
        }
        if (cut.segments > 1) {
            const auto kernel = back ? k_recurrence_back<T, SIGMOID, COMPLEMENT, W, true> : k_recurrence<T, SIGMOID, COMPLEMENT, W, true>;
            hipLaunchKernelGGL(kernel, dim3((unsigned)columns, (unsigned)a.batch, (unsigned)cut.segments), block, 0, s, a, cut);
        }
    }
    const auto kernel = back ? k_recurrence_back<T, SIGMOID, COMPLEMENT, W, false> : k_recurrence<T, SIGMOID, COMPLEMENT, W, false>;
    hipLaunchKernelGGL(kernel, dim3((unsigned)columns, (unsigned)a.batch, (unsigned)cut.segments), block, 0, s, a, cut);
    return (int)hipGetLastError();
}

template <typename T, bool SIGMOID, bool COMPLEMENT>
int launch_waves(const RecurrenceArgs& a, hipStream_t s, bool back) {
    if (a.tokens <= U) return launch_as<T, SIGMOID, COMPLEMENT, 1>(a, s, back);
    if (a.tokens <= 4 * U) return launch_as<T, SIGMOID, COMPLEMENT, 4>(a, s, back);
    return launch_as<T, SIGMOID, COMPLEMENT, 8>(a, s, back);
}

template <typename T>
int launch_gate(const RecurrenceArgs& a, hipStream_t s, bool back) {
    if (a.gate_kind == VKFX_GATE_SIGMOID) return a.complement ? launch_waves<T, true, true>(a, s, back) : launch_waves<T, true, false>(a, s, back);
    return a.complement ? launch_waves<T, false, true>(a, s, back) : launch_waves<T, false, false>(a, s, back);
}

int launch_element(const RecurrenceArgs& a, hipStream_t s, bool back) {
    if (a.element == VKFX_ELEMENT_F32) return launch_gate<float>(a, s, back);
    if (a.element == VKFX_ELEMENT_F16) return launch_gate<_Float16>(a, s, back);
    return launch_gate<__bf16>(a, s, back);
}

}  // namespace

int launch_recurrence_forward(const RecurrenceArgs& a, hipStream_t s) { return launch_element(a, s, false); }
int launch_recurrence_backward(const RecurrenceArgs& a, hipStream_t s) { return launch_element(a, s, true); }
// segments times columns is at most kCutBlocks a CU, of up to 128 channels each
size_t recurrence_workspace_bytes(int, long long, int cus) { return (size_t)cus * kCutBlocks * 128 * 3 * sizeof(float); }

}  // namespace vkfx
