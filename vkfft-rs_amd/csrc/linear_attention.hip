// linear_attention.hip -- which kernels a linear attention call runs, the join
// of a long sequence's segments and the sum over a shared head's query heads.
#include <algorithm>

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
    float* slot = args.slots + (((long long)z * batch + b) * s.heads + h) * args.segments * size + size;
    int at[EACH];
    float x[EACH];
#pragma unroll
    for (int j = 0; j < EACH; ++j) {
        at[j] = e + 256 * j < size ? e + 256 * j : size - 1;
        x[j] = slot[at[j]];
    }
    const float decay = whole_segment(args.powers + (long long)h * kDecayPowers, args.segment);
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

// blockIdx.y: one of the two tensors.
template <typename T>
__global__ __launch_bounds__(256) void k_group_sum(const GroupSum a, const GroupSum b, long long batch, long long tokens,
                                                   int kv_heads, int group) {
    const GroupSum& s = blockIdx.y ? b : a;
    const long long total = batch * tokens * kv_heads * s.dim;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long long)gridDim.x * 256) {
        const int c = (int)(i % s.dim);
        const long long row = i / s.dim;  // batch, token, shared head
        const int h = (int)(row % kv_heads);
        const long long t = row / kv_heads % tokens, n = row / kv_heads / tokens;
        const float* from = s.from + row * group * s.dim + c;
        float sum = 0.f;
        for (int g = 0; g < group; ++g) sum += from[(long long)g * s.dim];
        ((T*)s.to.p)[n * s.to.batch + t * s.to.token + h * s.to.head + c] = (T)sum;
    }
}

const ChunkKernel* chunk_kernel(int element, int dk, int dv) {
    return element == VKFX_ELEMENT_F32   ? chunk_kernel_f32(dk, dv)
           : element == VKFX_ELEMENT_F16 ? chunk_kernel_f16(dk, dv)
                                         : chunk_kernel_bf16(dk, dv);
}

// Waves that keep the GPU's 256 CUs busy: two on each SIMD. (Half as many, with
// fewer segments to join: bf16, 8 x 2048 tokens of 16 heads of 128, 114 us
// instead of 88; 1 x 65536 of 16 heads of 64, 188 instead of 112.)
constexpr long long kWaves = 2048;

struct Split {
    int segments;
    long long segment;
};

// Where the waves of whole sequences are fewer than half of kWaves, the tokens
// are split too: every segment but the last is read once more for its share of
// the state. A segment has two chunks or more (f32, 3 x 1001 tokens of 12 heads
// of 80 x 96: 44 us; 49 with four or more).
Split split_tokens(long long waves, long long tokens) {
    long long k = waves * 2 > kWaves ? 1 : kWaves / std::max(1ll, waves);
    k = std::max(1ll, std::min(k, tokens / (2 * kChunk)));
    const long long chunks = (tokens + kChunk - 1) / kChunk;
    Split s;
    s.segment = std::max(1ll, (chunks + k - 1) / k) * kChunk;
    s.segments = (int)std::max(1ll, (tokens + s.segment - 1) / s.segment);
    return s;
}

int launch_with(const void* fn, long long blocks, int threads, size_t lds, const ChunkArgs& a, hipStream_t s) {
    if (lds > 65536) {
        const hipError_t e = hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        if (e != hipSuccess) return (int)e;
    }
    void* kargs[1] = {(void*)&a};
    const hipError_t e = hipLaunchKernel(fn, dim3((unsigned)blocks), dim3((unsigned)threads), kargs, lds, s);
    return e != hipSuccess ? (int)e : (int)hipGetLastError();
}

long long slot_floats(const ScanArgs& s, int count, int segments) {
    return segments > 1 ? (long long)count * s.batch * s.heads * segments * s.dk * s.dv : 0;
}

int launch_chunks(int element, const ScanArgs* scans, int count, const float* powers, float*& work, hipStream_t st) {
    const ScanArgs& first = scans[0];
    const ChunkKernel* k = chunk_kernel(element, first.dk, first.dv);
    ChunkArgs a{};
    for (int i = 0; i < count; ++i) a.scan[i] = scans[i];
    a.scans = count;
    a.slices = (first.dv + k->cols - 1) / k->cols;
    const long long whole = (long long)count * first.batch * first.heads * a.slices;
    const Split sp = split_tokens(whole * (k->threads / 64), first.tokens);
    a.segments = sp.segments;
    a.segment = sp.segment;
    a.powers = powers;
    a.slots = work;
    // a whole sequence's block reads its state before it writes it: only segments need the copy
    for (int i = 0; i < count && a.segments > 1; ++i)
        if (scans[i].state_in && scans[i].state_in == scans[i].state_out) a.in_place = 1;
    if (whole * a.segments > 0x7fffffffll) return (int)hipErrorInvalidConfiguration;
    if (a.segments > 1) {
        work += slot_floats(first, count, a.segments);
        if (int e = launch_with(k->state_only, whole * a.segments, k->threads, k->state_lds, a, st)) return e;
        // few segments come with many states, many segments with few
        if (a.segments > 2)
            if (int e = a.segments <= 8 ? launch_join<4, 4>(a, st) : launch_join<1, 16>(a, st)) return e;
    }
    return launch_with(k->run, whole * a.segments, k->threads, k->lds, a, st);
}

}  // namespace

size_t scan_work_floats(int element, int dk, int dv, int heads, int count, long long max_batch, long long max_tokens) {
    const ChunkKernel* k = chunk_kernel(element, dk, dv);
    const int slices = (dv + k->cols - 1) / k->cols;
    // segments > 1 only below kWaves waves in all, and never over tokens / (2 kChunk) of them
    const long long most = std::max(1ll, max_tokens / (2 * kChunk));
    const long long states = std::min((long long)count * max_batch * heads * most, kWaves / (k->threads / 64) / slices);
    return most > 1 ? (size_t)states * dk * dv : 0;
}

int launch_scans(int element, const ScanArgs* scans, int count, const float* powers, float* work, int cus, hipStream_t s) {
    // the recurrence itself while a chunk would be mostly empty
    if (scans[0].tokens <= kStepTokens) return launch_steps(element, scans, count, powers, cus, s);
    // scans of one shape run side by side
    for (int i = 0; i < count;) {
        int j = i + 1;
        while (j < count && scans[j].dk == scans[i].dk && scans[j].dv == scans[i].dv) ++j;
        if (int e = launch_chunks(element, scans + i, j - i, powers, work, s)) return e;
        i = j;
    }
    return (int)hipSuccess;
}

int launch_group_sum(int element, const GroupSum& a, const GroupSum& b, long long batch, long long tokens, int kv_heads,
                     int group, hipStream_t s) {
    const long long blocks = (batch * tokens * kv_heads * std::max(a.dim, b.dim) + 255) / 256;
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
