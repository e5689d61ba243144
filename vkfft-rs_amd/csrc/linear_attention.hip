// linear_attention.hip -- which kernels a linear attention call runs, the join
// of a long sequence's segments and the sum over a shared head's query heads.
#include <algorithm>

#include "linear_chunk.hpp"
#include "vkfx.h"

namespace vkfx {

__global__ __launch_bounds__(256) void k_chunk_join(const ChunkArgs args) {
    const int z = blockIdx.z;
    const ScanArgs& s = args.scan[z];
    const int b = blockIdx.y / s.heads, h = blockIdx.y % s.heads;
    const int e = blockIdx.x * 256 + threadIdx.x;
    const int size = s.dk * s.dv;
    if (e >= size) return;
    long long n = s.tokens;
    if (s.lengths) {
        const long long l = s.lengths[b];
        n = l < 0 ? 0 : l < n ? l : n;
    }
    // the decay of a whole segment, by squaring
    const float* p = args.powers + (long long)h * kDecayPowers;
    double power = 1.0, square = (double)p[1] + (double)p[kDecayPowers - 1];
    for (long long i = args.segment; i; i >>= 1, square *= square)
        if (i & 1) power *= square;
    const float decay = (float)power;
    const int row = e / s.dv, col = e % s.dv;
    const long long head = (long long)b * s.heads + h;
    float x = s.state_in ? s.state_in[head * size + (long long)row * s.state_row + (long long)col * s.state_col] : 0.f;
    float* slot = args.slots + ((long long)z * s.batch * s.heads + head) * args.segments * size + e;
    // segments before the last that has tokens; eight are read before the first is needed
    const int last = (int)((n + args.segment - 1) / args.segment);
    slot[0] = x;
    for (int k = 1; k < last; k += 8) {
        float added[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) added[u] = k + u < last ? slot[(long long)(k + u) * size] : 0.f;
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            x = fmaf(x, decay, added[u]);
            if (k + u < last) slot[(long long)(k + u) * size] = x;
        }
    }
}

namespace {

template <typename T>
__global__ __launch_bounds__(256) void k_group_sum(const float* __restrict__ from, const ScanSide to, long long batch,
                                                   long long tokens, int kv_heads, int group, int dim) {
    const long long total = batch * tokens * kv_heads * dim;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long long)gridDim.x * 256) {
        const int c = (int)(i % dim);
        const long long row = i / dim;  // batch, token, shared head
        const int h = (int)(row % kv_heads);
        const long long t = row / kv_heads % tokens, b = row / kv_heads / tokens;
        float sum = 0.f;
        for (int g = 0; g < group; ++g) sum += from[(row * group + g) * dim + c];
        ((T*)to.p)[b * to.batch + t * to.token + h * to.head + c] = (T)sum;
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
// are split too: every segment but the last is read once more for its
// share of the state. A segment has four chunks or more.
Split split_tokens(long long waves, long long tokens, int chunk) {
    long long k = waves * 2 > kWaves ? 1 : kWaves / std::max(1ll, waves);
    k = std::max(1ll, std::min(k, tokens / (4 * chunk)));
    const long long chunks = (tokens + chunk - 1) / chunk;
    const long long each = (chunks + k - 1) / k;
    Split s;
    s.segment = std::max(1ll, each) * chunk;
    s.segments = (int)std::max(1ll, (tokens + s.segment - 1) / s.segment);
    return s;
}

int launch_with(const void* fn, long long blocks, const ChunkKernel* k, const ChunkArgs& a, hipStream_t s) {
    const size_t lds = k->lds;
    if (lds > 65536) {
        const hipError_t e = hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        if (e != hipSuccess) return (int)e;
    }
    void* kargs[1] = {(void*)&a};
    const hipError_t e = hipLaunchKernel(fn, dim3((unsigned)blocks), dim3((unsigned)k->threads), kargs, lds, s);
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
    const Split sp = split_tokens(whole * (k->threads / 64), first.tokens, k->chunk);
    a.segments = sp.segments;
    a.segment = sp.segment;
    a.powers = powers;
    a.slots = work;
    if (whole * a.segments > 0x7fffffffll) return (int)hipErrorInvalidConfiguration;
    if (a.segments > 1) {
        work += slot_floats(first, count, a.segments);
        if (int e = launch_with(k->state_only, whole * a.segments, k, a, st)) return e;
        const dim3 grid((unsigned)((first.dk * first.dv + 255) / 256), (unsigned)(first.batch * first.heads), (unsigned)count);
        hipLaunchKernelGGL(k_chunk_join, grid, dim3(256), 0, st, a);
        if (hipError_t e = hipGetLastError()) return (int)e;
    }
    return launch_with(k->run, whole * a.segments, k, a, st);
}

}  // namespace

size_t scan_work_floats(int element, int dk, int dv, int heads, int count, long long max_batch, long long max_tokens) {
    const ChunkKernel* k = chunk_kernel(element, dk, dv);
    const int slices = (dv + k->cols - 1) / k->cols;
    // segments > 1 only below kWaves waves in all, and never over tokens / (4 chunk) of them
    const long long most = std::max(1ll, max_tokens / (4 * k->chunk));
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

int launch_group_sum(int element, const float* from, const ScanSide& to, long long batch, long long tokens, int kv_heads,
                     int group, int dim, hipStream_t s) {
    const long long blocks = (batch * tokens * kv_heads * dim + 255) / 256;
    const dim3 grid((unsigned)(blocks < 4096 ? blocks : 4096));
    if (element == VKFX_ELEMENT_F32)
        hipLaunchKernelGGL(k_group_sum<float>, grid, dim3(256), 0, s, from, to, batch, tokens, kv_heads, group, dim);
    else if (element == VKFX_ELEMENT_F16)
        hipLaunchKernelGGL(k_group_sum<_Float16>, grid, dim3(256), 0, s, from, to, batch, tokens, kv_heads, group, dim);
    else
        hipLaunchKernelGGL(k_group_sum<__bf16>, grid, dim3(256), 0, s, from, to, batch, tokens, kv_heads, group, dim);
    return (int)hipGetLastError();
}

}  // namespace vkfx
