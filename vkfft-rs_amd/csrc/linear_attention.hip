// linear_attention.hip -- which kernels a linear attention call runs, the join
// of a long sequence's segments and the sum over a shared head's query heads.
#include <algorithm>

#include "kernels.hpp"
#include "linear_chunk.hpp"
#include "vkfx.h"

namespace vkfx {

namespace {

// Joins the segments: place k = g^segment place k-1 + what segment k-1 added.
// A thread takes EACH elements of a state, 256 apart, and reads AHEAD segments
// before it needs the first.
template <int EACH, int AHEAD>
__global__ __launch_bounds__(256) void k_chunk_join(const ChunkArgs args) {
    const int batch = args.scan[0].batch, z = blockIdx.z / batch, b = blockIdx.z % batch, h = blockIdx.y;
    const ScanArgs& s = args.scan[z];
    long long n = s.tokens;
    if (s.lengths) n = s.lengths[b] < 0 ? 0 : s.lengths[b] < n ? s.lengths[b] : n;
    const int last = (int)((n + args.segment - 1) / args.segment);  // segments that have tokens
    if (last < 3) return;
    const int size = s.dk * s.dv, e = blockIdx.x * 256 * EACH + threadIdx.x;
    float* slot = args.slots[z] + ((long long)b * s.heads + h) * args.segments * size + size;
    int at[EACH];
    float x[EACH];
#pragma unroll
    for (int j = 0; j < EACH; ++j) {
        at[j] = e + 256 * j < size ? e + 256 * j : size - 1;
        x[j] = slot[at[j]];
    }
    const float decay = (float)decay_of(args.powers + (long long)h * kDecayPowers, args.segment);
    for (int k = 2; k < last; k += AHEAD) {
        float added[AHEAD][EACH];
#pragma unroll
        for (int u = 0; u < AHEAD; ++u)
#pragma unroll
            for (int j = 0; j < EACH; ++j)
                added[u][j] = slot[(long long)(k + u < last ? u + 1 : last - k) * size + at[j]];
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            if (k + u >= last) break;
            slot += size;
#pragma unroll
            for (int j = 0; j < EACH; ++j) {
                x[j] = fmaf(x[j], decay, added[u][j]);
                if (e + 256 * j < size) slot[at[j]] = x[j];
            }
        }
    }
}

template <int EACH, int AHEAD>
int launch_join(const ChunkArgs& a, hipStream_t s) {
    const ScanArgs& f = a.scan[0];
    const dim3 grid((unsigned)((f.dk * f.dv + 256 * EACH - 1) / (256 * EACH)), (unsigned)f.heads, (unsigned)(f.batch * a.scans));
    hipLaunchKernelGGL((k_chunk_join<EACH, AHEAD>), grid, dim3(256), 0, s, a);
    return (int)hipGetLastError();
}

// Threads side by side over a row of a sum: a power of two, four elements each.
__host__ __device__ inline int group_sum_lanes(int dim) {
    int lanes = 1;
    while (4 * lanes < dim) lanes *= 2;
    return lanes;
}

// blockIdx.y: one of the two tensors. Bound by memory: 4 group + sizeof(T) bytes
// an element. A thread sums four neighbours of one row of (sequence, token,
// shared head), so that a row's place costs its divisions once for them (6 x 1215
// tokens, 8 heads on 2, widths of 64 and 112, f16: 8.5 us, 5.8 TB/s; 13.8 with one
// element a thread).
template <typename T>
__global__ __launch_bounds__(256) void k_group_sum(const GroupSum a, const GroupSum b, long long batch, long long tokens,
                                                   int kv_heads, int group) {
    typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));
    const GroupSum& s = blockIdx.y ? b : a;
    const int dim = s.dim, lanes = group_sum_lanes(dim), c = (int)threadIdx.x % lanes * 4, room = dim - c;
    if (room <= 0) return;
    const long long rows = batch * tokens * kv_heads, step = (long long)gridDim.x * (256 / lanes);
    for (long long row = (long long)blockIdx.x * (256 / lanes) + threadIdx.x / lanes; row < rows; row += step) {
        const float* from = s.from + row * group * dim + c;
        f32x4 sum = {0.f, 0.f, 0.f, 0.f};
        if (room >= 4) {
#pragma unroll 4
            for (int g = 0; g < group; ++g) sum += *(const f32x4_any*)(from + (long long)g * dim);
        } else {
            for (int g = 0; g < group; ++g)
#pragma unroll
                for (int e = 0; e < 3; ++e)
                    if (e < room) sum[e] += from[(long long)g * dim + e];
        }
        long long t, n;
        int h;
        if (rows >> 32) {
            h = (int)(row % kv_heads);
            t = row / kv_heads % tokens, n = row / kv_heads / tokens;
        } else {
            const unsigned r = (unsigned)row, token = r / (unsigned)kv_heads;
            h = (int)(r % (unsigned)kv_heads);
            t = token % (unsigned)tokens, n = token / (unsigned)tokens;
        }
        store_four((T*)s.to.p + n * s.to.batch + t * s.to.token + h * s.to.head + c, sum, room);
    }
}

const ChunkKernel* chunk_kernel(int element, int dk, int dv, bool gradient) {
    return element == VKFX_ELEMENT_F32   ? chunk_kernel_f32(dk, dv, gradient)
           : element == VKFX_ELEMENT_F16 ? chunk_kernel_f16(dk, dv, gradient)
                                         : chunk_kernel_bf16(dk, dv, gradient);
}

// Blocks of a kernel that the GPU holds at a time: two waves on each SIMD, as
// far as the LDS goes. That is what the outputs' kernels have; the states' ones
// would fit three to five by their registers and are counted as two as well.
long long resident(const ChunkKernel* k, size_t lds, int cus) {
    return (long long)cus * std::max(1, std::min(8 / (k->threads / 64), (int)(160 * 1024 / lds)));
}

// Most states that a call keeps between segments: with a block for each there
// are four a CU, which is what a CU holds of blocks of two waves (16 heads of 64
// over 65536 tokens, 64 segments: 165 us; 264 with 32) and twice what it holds of
// blocks of four.
constexpr long long kStates = 1024;

// Blocks along x: their threads have to stay under 2^32 (a launch of more starts the remainder only).
constexpr long long kGridX = 1 << 22;

int launch_with(const void* fn, long long blocks, int threads, size_t lds, ChunkArgs a, hipStream_t s) {
    if (lds > 65536)
        if (int e = raise_lds_limit(fn, lds)) return e;
    a.blocks = blocks;
    void* kargs[1] = {(void*)&a};
    const dim3 grid((unsigned)std::min(blocks, kGridX), (unsigned)((blocks + kGridX - 1) / kGridX));
    const hipError_t e = hipLaunchKernel(fn, grid, dim3((unsigned)threads), kargs, lds, s);
    return e != hipSuccess ? (int)e : (int)hipGetLastError();
}

// Scans of one shape: one launch.
struct Part {
    const ChunkKernel* k;
    ChunkArgs a;
    int members[3], states;  // scans that form a state come first
    long long run, state;    // blocks of a segment
};

// Tokens of a segment. Where whole sequences leave part of the GPU idle, the
// tokens are split; every segment but the last is then read once more for its
// share of the state, at about 0.4 of the cost. The time of k segments is that
// of the rounds of resident blocks, each 1/k of the tokens long at 3 us a chunk,
// and of the states' bytes, written, joined and read at 4 TB/s. (bf16, 4 x 4096
// tokens, 16 heads of 128, backward, 192 blocks: 309 us with the 5 segments that
// this gives, two rounds; 397 with 1, 355 with 2, 337 with 8. 8 x 2048 forward:
// 128 with its 4, 203 with 1, 155 with 2, 169 with 8. 32 x 1024, whole: 165, 232
// with 2.) A segment has two chunks or more (f32, 3 x 1001 tokens, 12 heads of
// 80 x 96: 55 us with the 11 segments that this gives, 81 with 4). The join's
// steps from segment to segment are not counted: one head of 64 over 65536 tokens
// gets 683 segments and takes 95 us, with 256 it would take 65.
//
// Times in this file and in linear_chunk.hpp are of calls on the same inputs one
// after the other, part of which the Infinity Cache keeps; on new inputs the same
// calls take up to 6% longer.
long long split_tokens(const Part* parts, int count, long long states, int size, long long tokens, int cus) {
    const long long most = std::max(1ll, std::min(tokens / (2 * kChunk), kStates / states));
    const double whole = 3.0 * (double)std::max(1ll, tokens / kChunk), state = 16.0 * (double)states * size / 4e6 / whole;
    const auto rounds = [](long long blocks, long long fit) { return (double)((blocks + fit - 1) / fit); };
    long long best = 1;
    double least = 0;
    for (long long k = 1; k <= most; ++k) {
        double time = state * (double)(k - 1);
        for (int i = 0; i < count; ++i) {
            const Part& p = parts[i];
            time += (rounds(p.run * k, resident(p.k, p.k->lds, cus)) +
                     0.4 * rounds(p.state * (k - 1), resident(p.k, p.k->state_lds, cus))) / (double)k;
        }
        if (k == 1 || time < least) best = k, least = time;
    }
    const long long chunks = (tokens + kChunk - 1) / kChunk;
    return std::max(1ll, (chunks + best - 1) / best) * kChunk;
}

int launch_chunks(int element, const ScanArgs* scans, int count, const float* powers, float* work, int cus, hipStream_t st) {
    const ScanArgs& first = scans[0];
    Part parts[3] = {};
    int n = 0, part_of[3], place[3], states = 0;
    for (int i = 0; i < count; ++i) {
        int p = 0;
        while (p < n && (scans[parts[p].members[0]].dk != scans[i].dk || scans[parts[p].members[0]].dv != scans[i].dv)) ++p;
        if (p == n) {
            ++n;
            parts[p].k = chunk_kernel(element, scans[i].dk, scans[i].dv, count > 1);
            parts[p].a.slices = (scans[i].dv + parts[p].k->cols - 1) / parts[p].k->cols;
            parts[p].a.powers = powers;
        }
        part_of[i] = p;
        place[i] = parts[p].a.scans++;
        parts[p].members[place[i]] = i;
        parts[p].a.scan[place[i]] = scans[i];
        const long long blocks = first.batch * (long long)first.heads * parts[p].a.slices;
        parts[p].run += blocks;
        if (scans[i].like < 0) {
            ++parts[p].states;
            ++states;
            parts[p].state += blocks;
        }
    }
    const long long heads = first.batch * (long long)first.heads;
    const long long segment = split_tokens(parts, n, states * heads, first.dk * first.dv, first.tokens, cus);
    const int segments = (int)std::max(1ll, (first.tokens + segment - 1) / segment);
    const long long floats = heads * segments * first.dk * first.dv;
    float* slots[3];
    for (int i = 0; i < count; ++i) {
        const int from = scans[i].like < 0 ? i : scans[i].like;
        ChunkArgs& a = parts[part_of[i]].a;
        a.segments = segments;
        a.segment = segment;
        if (segments == 1) continue;
        if (from == i) {
            slots[i] = work;
            work += floats;
        }
        a.slots[place[i]] = slots[from];
        a.slot_row[place[i]] = from == i ? scans[i].dv : 1;
        a.slot_col[place[i]] = from == i ? 1 : scans[i].dk;
        // a whole sequence's block reads its state before it writes it: only segments need the copy
        if (scans[i].state_in && scans[i].state_in == scans[i].state_out) a.in_place = 1;
    }
    for (int p = 0; p < n && segments > 1; ++p) {
        ChunkArgs a = parts[p].a;
        a.scans = parts[p].states;
        if (!a.scans) continue;
        if (int e = launch_with(parts[p].k->state_only, parts[p].state * segments, parts[p].k->threads, parts[p].k->state_lds, a, st))
            return e;
        // Few segments come with many states and are joined four elements a thread, many segments with few states one
        // element a thread (bf16 prompts: 8 x 2048 tokens of 16 heads of 128, 4 segments, 128 us, 137 the other way;
        // 1 x 16384 of 4 heads of 64, 171 segments, 50 and 77)
        if (segments > 2)
            if (int e = segments <= 8 ? launch_join<4, 4>(a, st) : launch_join<1, 16>(a, st)) return e;
    }
    for (int p = 0; p < n; ++p)
        if (int e = launch_with(parts[p].k->run, parts[p].run * segments, parts[p].k->threads, parts[p].k->lds, parts[p].a, st)) return e;
    return (int)hipSuccess;
}

}  // namespace

size_t scan_work_floats(int dk, int dv, int heads, int states, long long max_batch, long long max_tokens) {
    const long long most = max_tokens / (2 * kChunk);
    return most > 1 ? (size_t)std::min(states * max_batch * heads * most, kStates) * (size_t)(dk * dv) : 0;
}

int launch_scans(int element, const ScanArgs* scans, int count, const float* powers, float* work, int cus, hipStream_t s) {
    // The recurrence itself while a chunk would be mostly empty: for one sequence of 16 heads of 128 x 128 a step of 8
    // tokens takes 10.4 us and a chunk 12.6, of 2 tokens 4.7 and 12.6; 8 sequences 15.4 and 15.1 at 8 tokens, 10.2 and
    // 15.1 at 4. Only large batches turn sooner (64 sequences: 52 and 43 at 8, 35 and 41 at 4).
    if (scans[0].tokens <= kStepTokens) return launch_steps(element, scans, count, powers, cus, s);
    return launch_chunks(element, scans, count, powers, work, cus, s);
}

int launch_group_sum(int element, const GroupSum& a, const GroupSum& b, long long batch, long long tokens, int kv_heads,
                     int group, hipStream_t s) {
    const int rows = 256 / group_sum_lanes(std::max(a.dim, b.dim));  // of a block, the fewer
    const long long blocks = (batch * tokens * kv_heads + rows - 1) / rows;
    const dim3 grid((unsigned)std::min(blocks, 4096ll), 2);
    if (element == VKFX_ELEMENT_F32)
        hipLaunchKernelGGL(k_group_sum<float>, grid, dim3(256), 0, s, a, b, batch, tokens, kv_heads, group);
    else if (element == VKFX_ELEMENT_F16)
        hipLaunchKernelGGL(k_group_sum<_Float16>, grid, dim3(256), 0, s, a, b, batch, tokens, kv_heads, group);
    else
        hipLaunchKernelGGL(k_group_sum<__bf16>, grid, dim3(256), 0, s, a, b, batch, tokens, kv_heads, group);
    return (int)hipGetLastError();
}

}  // namespace vkfx
