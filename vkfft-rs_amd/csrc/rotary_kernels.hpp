// rotary_kernels.hpp -- heads turned by their positions, with a norm of each in front
// where it is wanted, and the gradients of both.
//
// A pair (u1, u2) at position p turns by p f: (u1 c - u2 s, u1 s + u2 c); its
// gradient turns back, by -p f. f is kept as 64 bits of a turn, so p f is one
// product that wraps where an angle does, and its first bits are its quadrant:
// no position is too far. With the norm, n = x rstd, u = n weight:
//   du = the gradient turned back, g = du weight
//   dx = rstd (g - n mean(g n)),  dweight = sum du n
// over tokens and heads.
//
// Bound by memory: every row is read once, in vectors of 16 bytes. A row belongs
// to 4 .. 32 lanes of a wave, each of which holds both elements of its pairs. A
// lane forms its pairs' cosines and sines once for up to 4 heads of a token,
// whose loads are on their way meanwhile.
#pragma once

#include <algorithm>

#include "sequence.hpp"
#include "sequence_device.hpp"
#include "vkfx.h"

namespace vkfx {

namespace {

// Cosine and sine of 2^-64 `phase` turns: the nearest quarter turn, then the series of
// what is left (to pi/4: the next terms are 2^-28.5 of the sine, 2^-32.5 of the cosine).
// With two roundings of t, one of its product with 2 pi and those of the series the
// sine is off by up to 2^-21.6 of itself (2^-21.9 seen), the cosine by 2^-21.9 (2^-22.7);
// angles under 2^-32 turns by 2^-54. (t rounded once, and what r's rounding leaves in
// the sine, make both 2^-22.5 and calls 1 to 3% longer.)
__device__ __forceinline__ void turn(uint64_t phase, float& c, float& s) {
    const unsigned quarter = ((unsigned)(phase >> 61) + 1) >> 1;
    const long long left = (long long)(phase - ((uint64_t)quarter << 62));
    const float t = fmaf((float)(unsigned)left, 0x1p-64f, (float)(int)(left >> 32) * 0x1p-32f);
    const float r = t * 6.283185307179586f, q = r * r;
    const float sn = r * fmaf(q, fmaf(q, fmaf(q, fmaf(q, 1.f / 362880, -1.f / 5040), 1.f / 120), -1.f / 6), 1.f);
    const float cs = fmaf(q, fmaf(q, fmaf(q, fmaf(q, fmaf(q, -1.f / 3628800, 1.f / 40320), -1.f / 720), 1.f / 24), -0.5f), 1.f);
    c = quarter & 1 ? sn : cs;
    s = quarter & 1 ? cs : sn;
    if ((quarter + 1) & 2) c = -c;
    if (quarter & 2) s = -s;
}

// Sum over the G lanes of a row, the same on each.
template <int G>
__device__ __forceinline__ float row_sum(float v) {
#pragma unroll
    for (int o = 1; o < G; o <<= 1) v += __shfl_xor(v, o);
    return v;
}

// A lane's share of a row: two vectors of V elements that hold its V pairs
// between them, and with TAILS two more of what does not turn.
//   HALF: elements l V .. of the first half and of the second, then the tail's
//   else: elements l V .. and (G + l) V .., pairs of neighbours
// A last vector that passes the end of its part begins earlier instead, so that the
// part ends with it: what it shares with the vector before is computed twice, to the
// same bits, and counts once in sums over the row (16 and 4 heads of 90 bf16, 8 x 2048
// tokens: 36 us, 51 with the last elements one by one). A part that is shorter than a
// vector, or of odd length where neighbours pair, has them one by one.
template <typename T, int G, int TAILS, bool HALF>
struct Share {
    static constexpr int V = kVector<T>, N = 2 + TAILS;
    typedef Some<T, V> Vectors[N];
    int at[N], end[N], skip[N], half;
    bool overlap;  // any lane has elements of another's

    // Vector j of lane l, and the end of what it is a part of.
    __device__ __forceinline__ static int place(const RotaryArgs& a, int j, int l) {
        if constexpr (!HALF) return (j * G + l) * V;
        return j < 2 ? j * (a.turned / 2) + l * V : a.turned + ((j - 2) * G + l) * V;
    }
    __device__ __forceinline__ static int limit(const RotaryArgs& a, int j) {
        return HALF && j < 2 ? (j + 1) * (a.turned / 2) : a.dim;
    }
    // How many elements of vector j of lane l are of the vector before.
    __device__ __forceinline__ static int shared(const RotaryArgs& a, int j, int l) {
        const int from = place(a, j, l), end = limit(a, j), past = from + V - end;
        return past > 0 && past < V && end - place(a, j, 0) >= V && (HALF || end % 2 == 0) ? past : 0;
    }
    __device__ __forceinline__ Share(const RotaryArgs& a, int l) {
        half = a.turned / 2;
        overlap = (HALF ? half : a.dim) % V || (a.dim - a.turned) % V;
#pragma unroll
        for (int j = 0; j < N; ++j) skip[j] = shared(a, j, l), at[j] = place(a, j, l) - skip[j], end[j] = limit(a, j);
    }
    __device__ __forceinline__ void load(Vectors& x, const T* row) const {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            x[j] = (T)0.f;
            if (at[j] + V <= end[j]) x[j] = *(const typename Packed<T, V>::type*)(row + at[j]);
            else if (at[j] < end[j]) x[j] = load_some<T, V>(row, at[j], end[j]);
        }
    }
    // v = term(j, e, v) over the row's elements, each once, added over its lanes.
    template <typename F>
    __device__ __forceinline__ float sum(F term) const {
        float v = 0.f;
        if (!overlap) {
#pragma unroll
            for (int j = 0; j < N; ++j)
#pragma unroll
                for (int e = 0; e < V; ++e) v = term(j, e, v);
        } else {
#pragma unroll
            for (int j = 0; j < N; ++j)
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const float with = term(j, e, v);
                    if (e >= skip[j]) v = with;
                }
        }
        return row_sum<G>(v);
    }
    __device__ __forceinline__ void store(const float (&y)[N][V], T* row) const {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            Some<T, V> r;
#pragma unroll
            for (int e = 0; e < V; ++e) r[e] = (T)y[j][e];
            if (at[j] + V <= end[j]) *(typename Packed<T, V>::type*)(row + at[j]) = r;
            else if (at[j] < end[j]) store_some<T, V>(row, at[j], end[j], r);
        }
    }
    // The norm's weights; 1 without.
    __device__ __forceinline__ void weights(float (&w)[N][V], const void* p, bool f32) const {
#pragma unroll
        for (int j = 0; j < N; ++j)
#pragma unroll
            for (int e = 0; e < V; ++e) w[j][e] = 1.f;
        if (!p) return;
#pragma unroll
        for (int j = 0; j < N; ++j) {
            if (f32) {
                const Some<float, V> v = load_some<float, V>((const float*)p, at[j], end[j]);
#pragma unroll
                for (int e = 0; e < V; ++e) w[j][e] = v[e];
            } else {
                const Some<T, V> v = load_some<T, V>((const T*)p, at[j], end[j]);
#pragma unroll
                for (int e = 0; e < V; ++e) w[j][e] = (float)v[e];
            }
        }
    }
    // The lane's pair e, of the row's.
    __device__ __forceinline__ int pair(int e) const { return HALF ? at[0] + e : at[e / (V / 2)] / 2 + e % (V / 2); }
    // Cosines and sines of the lane's pairs at position p, amplitude included.
    __device__ __forceinline__ void turns(float (&c)[V], float (&s)[V], const RotaryArgs& a, long long p, float sign) const {
#pragma unroll
        for (int e = 0; e < V; ++e) {
            c[e] = 1.f;
            s[e] = 0.f;
            if (pair(e) >= half) continue;
            turn((uint64_t)p * a.turns[pair(e)], c[e], s[e]);
            c[e] *= a.amplitude;
            s[e] *= sign;
        }
    }
    // Pairs of neighbours that do not turn stay what they are: with a cosine of 1 and a
    // sine of 0, an infinity would make its neighbour a NaN, and -0 become 0. (Selected
    // for rows that turn whole, too: 16 and 4 heads of 128 bf16, 8 x 2048 tokens, 39.0 us,
    // 38.3 without, 41.7 with a branch for them.)
    __device__ __forceinline__ void turn_by(float (&y)[N][V], const float (&c)[V], const float (&s)[V]) const {
#pragma unroll
        for (int e = 0; e < V; ++e) {
            float& u = HALF ? y[0][e] : y[e / (V / 2)][e % (V / 2) * 2];
            float& v = HALF ? y[1][e] : y[e / (V / 2)][e % (V / 2) * 2 + 1];
            const float first = fmaf(u, c[e], -v * s[e]), second = fmaf(u, s[e], v * c[e]);
            const bool turns = HALF || pair(e) < half;
            u = turns ? first : u;
            v = turns ? second : v;
        }
    }
};

// 1 / sqrt(mean of squares + epsilon) of a row; where that passes 32 bits, from 2^-68
// of the row and 2^-136 of epsilon.
template <typename S, int N, int V>
__device__ __forceinline__ float deviation(const S& share, const float (&x)[N][V], float over, float epsilon) {
    const float square = share.sum([&](int j, int e, float v) { return fmaf(x[j][e], x[j][e], v); });
    const float mean = fmaf(square, over, epsilon);
    if (mean != INFINITY) return 1.f / sqrtf(mean);
    const float small = share.sum([&](int j, int e, float v) {
        const float part = x[j][e] * 0x1p-68f;
        return fmaf(part, part, v);
    });
    return 0x1p-68f / sqrtf(fmaf(small, over, epsilon * 0x1p-68f * 0x1p-68f));
}

// Which token and which heads of it a group of lanes takes: heads phase, phase +
// phases, ... up to HB of them.
struct Place {
    long long b, t, position;
    int phase;
    bool live;  // before the sequence's length
    __device__ __forceinline__ Place(const RotaryArgs& a, long long i, long long count, int phases) {
        const unsigned token = count >> 32 ? (unsigned)(i / phases) : (unsigned)i / (unsigned)phases;
        phase = (int)(i - (long long)token * phases);
        const unsigned row = token / (unsigned)a.tokens;
        b = row;
        t = token - row * (unsigned)a.tokens;
        live = !a.lengths || t < a.lengths[b];
        position = a.positions ? a.positions[b * a.tokens + t] : a.starts ? a.starts[b] + t : t;
    }
};

template <typename T>
__device__ __forceinline__ T* row_of(const RotarySide& s, const Place& p, int head) {
    return (T*)s.p + p.b * s.batch + p.t * s.token + head * s.head;
}

// Turns rows, by `sign` times their angle, behind the norm where NORM. The first
// `split` blocks take rows[0].
template <typename T, int G, int TAILS, int HB, bool HALF, bool NORM>
__global__ __launch_bounds__(256) void k_turn(const RotaryArgs a, unsigned split, float sign) {
    typedef Share<T, G, TAILS, HALF> S;
    constexpr int V = S::V, N = S::N;
    const bool second = blockIdx.x >= split;
    const RotaryRows& h = a.rows[second];
    const int phases = (h.heads + HB - 1) / HB;
    const long long count = a.all * phases, stride = (long long)(second ? gridDim.x - split : split) * (256 / G);
    const S share(a, threadIdx.x % G);
    float w[N][V];
    if constexpr (NORM) share.weights(w, h.weight, a.weight_element == VKFX_ELEMENT_F32);
    for (long long i = (long long)(blockIdx.x - (second ? split : 0)) * (256 / G) + threadIdx.x / G; i < count; i += stride) {
        const Place p(a, i, count, phases);
        typename S::Vectors x[HB];
        if (p.live)
#pragma unroll
            for (int k = 0; k < HB; ++k)
                if (p.phase + k * phases < h.heads) share.load(x[k], row_of<const T>(h.x, p, p.phase + k * phases));
        float c[V], s[V];
        share.turns(c, s, a, p.position, sign * a.amplitude);
#pragma unroll
        for (int k = 0; k < HB; ++k) {
            const int head = p.phase + k * phases;
            if (head >= h.heads) break;
            float y[N][V] = {};
            if (p.live) {
#pragma unroll
                for (int j = 0; j < N; ++j)
#pragma unroll
                    for (int e = 0; e < V; ++e) y[j][e] = (float)x[k][j][e];
                if constexpr (NORM) {
                    const float rstd = deviation(share, y, 1.f / (float)a.dim, a.epsilon);
#pragma unroll
                    for (int j = 0; j < N; ++j)
#pragma unroll
                        for (int e = 0; e < V; ++e) y[j][e] = y[j][e] * rstd * w[j][e];  // rstd w may leave 32 bits
                }
                share.turn_by(y, c, s);
            }
            share.store(y, row_of<T>(h.out, p, head));
        }
    }
}

// Gradients behind the norm. A lane's sums of du n are of kTurns turns in 32 bits
// (equal numbers would round to one side each time), then in 64, in LDS; the
// block's go to the workspace, row blockIdx.x.
constexpr int kTurns = 8;

// Blocks of the backward pass, whose sums each are a row of the workspace: as many
// as fit at once (4 x 4096 tokens of 16 and 4 heads of 128 bf16: 68 us with 3 a CU,
// 85 with 4).
template <typename T, int TAILS>
constexpr int kBackBlocks = TAILS ? 2 : sizeof(T) == 4 ? 4 : 3;

template <typename T, int G, int TAILS, int HB, bool HALF>
__global__ __launch_bounds__(256, (kBackBlocks<T, TAILS>)) void k_norm_turn_back(const RotaryArgs a, unsigned split) {
    typedef Share<T, G, TAILS, HALF> S;
    constexpr int V = S::V, N = S::N;
    __shared__ double sums[N * V][256];  // a thread's own
    const bool second = blockIdx.x >= split;
    const RotaryRows& h = a.rows[second];
    const int phases = (h.heads + HB - 1) / HB;
    const long long count = a.all * phases, stride = (long long)(second ? gridDim.x - split : split) * (256 / G);
    const S share(a, threadIdx.x % G);
    const float over = 1.f / (float)a.dim;
    float w[N][V], part[N][V];
    share.weights(w, h.weight, a.weight_element == VKFX_ELEMENT_F32);
#pragma unroll
    for (int j = 0; j < N; ++j)
#pragma unroll
        for (int e = 0; e < V; ++e) part[j][e] = 0.f, sums[j * V + e][threadIdx.x] = 0.0;
    const auto flush = [&]() {
#pragma unroll
        for (int j = 0; j < N; ++j)
#pragma unroll
            for (int e = 0; e < V; ++e) {
                sums[j * V + e][threadIdx.x] += (double)part[j][e];
                part[j][e] = 0.f;
            }
    };
    int turns = 0;
    for (long long i = (long long)(blockIdx.x - (second ? split : 0)) * (256 / G) + threadIdx.x / G; i < count; i += stride) {
        const Place p(a, i, count, phases);
        typename S::Vectors x[HB], dy[HB];
        if (p.live)
#pragma unroll
            for (int k = 0; k < HB; ++k)
                if (p.phase + k * phases < h.heads) {
                    share.load(dy[k], row_of<const T>(h.x, p, p.phase + k * phases));
                    share.load(x[k], row_of<const T>(h.in, p, p.phase + k * phases));
                }
        float c[V], s[V];
        share.turns(c, s, a, p.position, -a.amplitude);
#pragma unroll
        for (int k = 0; k < HB; ++k) {
            const int head = p.phase + k * phases;
            if (head >= h.heads) break;
            float g[N][V] = {};
            if (p.live) {
                float n[N][V];
#pragma unroll
                for (int j = 0; j < N; ++j)
#pragma unroll
                    for (int e = 0; e < V; ++e) g[j][e] = (float)dy[k][j][e], n[j][e] = (float)x[k][j][e];
                const float rstd = deviation(share, n, over, a.epsilon);
                share.turn_by(g, c, s);
#pragma unroll
                for (int j = 0; j < N; ++j)
#pragma unroll
                    for (int e = 0; e < V; ++e) {
                        n[j][e] *= rstd;
                        part[j][e] = fmaf(g[j][e], n[j][e], part[j][e]);
                        g[j][e] *= w[j][e];
                    }
                const float dot = over * share.sum([&](int j, int e, float v) { return fmaf(g[j][e], n[j][e], v); });
#pragma unroll
                for (int j = 0; j < N; ++j)
#pragma unroll
                    for (int e = 0; e < V; ++e) g[j][e] = fmaf(-n[j][e], dot, g[j][e]) * rstd;
            }
            share.store(g, row_of<T>(h.out, p, head));
        }
        if (++turns % kTurns == 0) flush();
    }
    if (!h.dweight) return;
    flush();
    // the wave's groups, then the block's waves
#pragma unroll
    for (int k = 0; k < N * V; ++k) {
        double v = sums[k][threadIdx.x];
#pragma unroll
        for (int o = G; o < 64; o <<= 1) v += __shfl_xor(v, o);
        sums[k][threadIdx.x] = v;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < N * V * G; i += 256) {
        const int k = i / G, l = i % G, skip = S::shared(a, k / V, l), at = S::place(a, k / V, l) - skip + k % V;
        if (k % V >= skip && at < S::limit(a, k / V))
            a.partial[(long long)blockIdx.x * a.dim + at] = (float)((sums[k][l] + sums[k][64 + l]) + (sums[k][128 + l] + sums[k][192 + l]));
    }
}

// Adds the blocks' sums: 16 elements a block, 64 threads for each of them, which
// take the blocks in turn. blockIdx.y: q's weight, k's.
template <typename W>
__global__ __launch_bounds__(1024) void k_norm_weights(const RotaryArgs a, int split, int blocks) {
    __shared__ double lds[64][16];
    W* const to = (W*)a.rows[blockIdx.y].dweight;
    if (!to) return;
    const int lane = threadIdx.x % 16, slice = threadIdx.x / 16, e = blockIdx.x * 16 + lane;
    const int end = blockIdx.y ? blocks : split;
    double sum = 0.0;
    if (e < a.dim)
#pragma unroll 8
        for (int i = (blockIdx.y ? split : 0) + slice; i < end; i += 64) sum += (double)a.partial[(long long)i * a.dim + e];
    lds[slice][lane] = sum;
#pragma unroll
    for (int n = 8; n; n /= 8) {  // 64 slices to 8, then to one
        __syncthreads();
        if (slice < n) {
            sum = 0.0;
#pragma unroll
            for (int i = 0; i < 8; ++i) sum += lds[slice * (64 / n) + i * (8 / n)][lane];
        }
        __syncthreads();
        if (slice < n) lds[slice * (64 / n)][lane] = sum;
    }
    if (!slice && e < a.dim) to[e] = (W)(float)sum;
}

// Groups of `lanes` that a tensor's rows fill, in blocks.
inline long long blocks_of(const RotaryArgs& a, const RotaryRows& r, int lanes, int heads) {
    const int groups = 256 / lanes;
    return (a.all * ((r.heads + heads - 1) / heads) + groups - 1) / groups;
}

template <typename T, int G, int TAILS, int HB, bool HALF>
int launch_turn(const RotaryArgs& a, hipStream_t s, bool back) {
    const auto blocks = [&](int i) { return (unsigned)std::min(blocks_of(a, a.rows[i], G, HB), 1ll << 22); };
    const unsigned first = blocks(0), all = first + blocks(1);
    if (!all) return (int)hipSuccess;
    const auto kernel = a.norm ? k_turn<T, G, TAILS, HB, HALF, true> : k_turn<T, G, TAILS, HB, HALF, false>;
    hipLaunchKernelGGL(kernel, dim3(all), dim3(256), 0, s, a, first, back ? -1.f : 1.f);
    return (int)hipGetLastError();
}

template <typename T, int G, int TAILS, int HB, bool HALF>
int launch_norm_back(const RotaryArgs& a, hipStream_t s) {
    long long blocks[2] = {blocks_of(a, a.rows[0], G, HB), blocks_of(a, a.rows[1], G, HB)};
    const long long most = (long long)a.cus * kBackBlocks<T, TAILS>, all = blocks[0] + blocks[1];
    if (all > most) {  // in the proportion of their rows, each at least one
        const long long n = blocks[0] ? std::max(1ll, (long long)((double)blocks[0] / (double)all * (double)most)) : 0;
        blocks[0] = blocks[1] ? std::min(n, most - 1) : most;
        blocks[1] = most - blocks[0];
    }
    if (all)
        hipLaunchKernelGGL((k_norm_turn_back<T, G, TAILS, HB, HALF>), dim3((unsigned)(blocks[0] + blocks[1])), dim3(256), 0, s, a, (unsigned)blocks[0]);
    if (a.rows[0].dweight || a.rows[1].dweight) {
        const auto kernel = a.weight_element == VKFX_ELEMENT_F32 ? k_norm_weights<float> : k_norm_weights<T>;
        hipLaunchKernelGGL(kernel, dim3((a.dim + 15) / 16, 2), dim3(1024), 0, s, a, (int)blocks[0], (int)(blocks[0] + blocks[1]));
    }
    return (int)hipGetLastError();
}

// One head a group of lanes while there are few rows, where latency counts; several,
// as far as there are so many, from 8 waves a CU on.
template <typename T, int G, int TAILS, bool HALF>
int launch_heads(const RotaryArgs& a, hipStream_t s, bool back) {
    const long long waves = a.all * ((a.rows[0].heads + a.rows[1].heads + 3) / 4) * G / 64;
    const int heads = waves < (long long)a.cus * 8 ? 1 : std::max(a.rows[0].heads, a.rows[1].heads);
    if (a.norm && back) {
        // two with tails are more than a lane's registers hold
        if constexpr (!(TAILS && sizeof(T) == 2))
            if (heads > 1) return launch_norm_back<T, G, TAILS, 2, HALF>(a, s);
        return launch_norm_back<T, G, TAILS, 1, HALF>(a, s);
    }
    if (heads < 2) return launch_turn<T, G, TAILS, 1, HALF>(a, s, back);
    return heads < 3 ? launch_turn<T, G, TAILS, 2, HALF>(a, s, back) : launch_turn<T, G, TAILS, 4, HALF>(a, s, back);
}

template <typename T, int TAILS, bool HALF>
int launch_lanes(const RotaryArgs& a, hipStream_t s, bool back) {
    constexpr int V = kVector<T>;
    const int pairs = HALF ? (a.turned / 2 + V - 1) / V : (a.dim + 2 * V - 1) / (2 * V);
    const int lanes = std::max(pairs, TAILS ? (a.dim - a.turned + 2 * V - 1) / (2 * V) : 0);
    if (lanes <= 4) return launch_heads<T, 4, TAILS, HALF>(a, s, back);
    if (lanes <= 8) return launch_heads<T, 8, TAILS, HALF>(a, s, back);
    if constexpr (sizeof(T) == 4)
        if (lanes > 16) return launch_heads<T, 32, TAILS, HALF>(a, s, back);
    return launch_heads<T, 16, TAILS, HALF>(a, s, back);
}

template <typename T>
int launch_layout(const RotaryArgs& a, hipStream_t s, bool back) {
    if (a.layout == VKFX_ROTARY_INTERLEAVED) return launch_lanes<T, 0, false>(a, s, back);
    return a.turned == a.dim ? launch_lanes<T, 0, true>(a, s, back) : launch_lanes<T, 2, true>(a, s, back);
}

}  // namespace

}  // namespace vkfx
