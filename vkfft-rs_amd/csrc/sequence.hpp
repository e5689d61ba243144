// sequence.hpp -- launch interface of the sequence operators' kernels
// (layer_norm.hip, linear_*.hip, rotary_*.hip, recurrence_*.hip), used by
// sequence.cpp, rotary_plan.cpp and recurrence_plan.cpp.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace vkfx {

// ------------------------------------------------------------- layer norm

struct NormArgs {
    const void* x;
    const void* weight;  // null: 1
    const void* bias;    // null: 0
    const float* stats_in;
    const void* dy;
    void* y;  // forward: y; backward: dx
    float* stats_out;
    void* dweight;
    void* dbias;
    float* partial;  // backward: [blocks][2][width] sums of a block's rows, norm_workspace_bytes
    long long rows, x_stride, dy_stride, y_stride;
    int parts;  // backward: rows of sums
    int width;
    int element, weight_element;  // vkfx_element
    float epsilon;
    int cus;
};

int launch_norm_forward(const NormArgs& a, hipStream_t s);
int launch_norm_backward(const NormArgs& a, hipStream_t s);
size_t norm_workspace_bytes(int element, int width, int cus);

// ------------------------------------------------------- linear attention

// One scan over a batch of sequences: with inputs A (rows of `dk`), B (rows of
// `dk`) and C (rows of `dv`), and a state X (dk x dv),
//   out[i] = scale_in ( scale_update sum_{j <= i} g^(i-j) (A[i] . B[j]) C[j]
//                       + g^(i + 1 - lead) A[i] X )
//   X'     = g^n X + scale_update sum_j g^(n - 1 - j + lead) B[j] C[j]^T.
// The forward pass and the gradient of q run it in the order of the tokens
// with lead 0 (A, B, C = q, k, v and dout, v, k), the gradients of v and k
// backwards from each sequence's last token with lead 1 (k, q, dout and v,
// dout, q), where X is the gradient of the state after a token.
struct ScanSide {
    const void* p;
    long long batch, token, head;  // element strides
    int group;                     // head h reads row h / group
};
struct ScanArgs {
    ScanSide a, b, c;
    void* out;  // elements, or floats with out_f32
    long long out_batch, out_token, out_head;
    int out_f32;
    const int* lengths;     // null: tokens
    const float* state_in;  // null: zeros
    float* state_out;       // null: not wanted
    // a state's element (row of dk, column of dv) is at row * state_row + column * state_col
    int state_row, state_col;
    long long tokens;
    int batch, heads, dk, dv;
    int reverse;  // and lead
    float scale_in, scale_update;
    int like;  // -1, or the scan whose state is this one's transpose, which then forms it for both
};

// Powers 0, 1, ... of each head's decay, kDecayPowers floats a head; the last
// two are the decay itself as a sum: its 24 bits towards zero and the rest. The
// rest is never negative, nor zero unless the decay is, so that a state times
// both parts stays infinite where it is.
constexpr int kDecayPowers = 72, kDecayHigh = kDecayPowers - 2, kDecayLow = kDecayPowers - 1;

// Up to kStepTokens tokens one after the other (linear_step.hip).
constexpr int kStepTokens = 8;
int launch_steps(int element, const ScanArgs* scans, int count, const float* powers, int cus, hipStream_t s);

// `count` scans (up to 3) of the same batch, tokens and heads, by the kernels
// that suit the number of tokens (linear_attention.hip). `work` holds
// scan_work_floats, `states`: scans without a `like`.
int launch_scans(int element, const ScanArgs* scans, int count, const float* powers, float* work, int cus, hipStream_t s);
size_t scan_work_floats(int dk, int dv, int heads, int states, long long max_batch, long long max_tokens);

// Sums the floats [batch][token][head][dim] of each shared head's `group`
// query heads, in their order; two tensors at once.
struct GroupSum {
    const float* from;
    ScanSide to;
    int dim;
};
int launch_group_sum(int element, const GroupSum& a, const GroupSum& b, long long batch, long long tokens, int kv_heads,
                     int group, hipStream_t s);

// ----------------------------------------------------------------- rotary

struct RotarySide {
    const void* p;
    long long batch, token, head;  // element strides
};
// Queries or keys. No heads: left out.
struct RotaryRows {
    RotarySide x;   // backward: dy
    RotarySide in;  // backward with the norm: the forward pass's input
    RotarySide out;
    const void* weight;  // null: 1
    void* dweight;       // null: not wanted
    int heads;
};
struct RotaryArgs {
    RotaryRows rows[2];
    const uint64_t* turns;  // [turned / 2] 2^-64 turns a position
    const int *positions, *starts, *lengths;  // null: none
    float* partial;  // rotary_workspace_bytes
    long long tokens, all;  // of a sequence, of the batch
    int dim, turned, layout;
    int element, weight_element;
    int norm;
    float epsilon, amplitude;
    int cus;
};
// By element (rotary_f32.hip, ...). back: the gradients.
int launch_rotary_f32(const RotaryArgs& a, hipStream_t s, bool back);
int launch_rotary_f16(const RotaryArgs& a, hipStream_t s, bool back);
int launch_rotary_bf16(const RotaryArgs& a, hipStream_t s, bool back);
// A row of sums for each block of the backward pass, up to 4 a CU.
inline size_t rotary_workspace_bytes(int dim, int cus) { return (size_t)cus * 4 * (size_t)dim * sizeof(float); }

// ------------------------------------------------------- gated recurrence

constexpr int kSpan = 16;  // tokens between saved states

struct RecurrenceSide {
    const void* p;
    long long batch, token;  // element strides
};
struct RecurrenceArgs {
    RecurrenceSide x, gate;
    RecurrenceSide dy;      // backward
    RecurrenceSide y;       // backward: dx
    RecurrenceSide dgate;   // backward
    const int* lengths;     // null: tokens
    const float* state_in;  // null: zeros; backward: dstate_out
    float* state_out;       // null: not wanted; backward: dstate_in
    float* saved;           // null: not wanted; backward: read
    float* work;            // recurrence_workspace_bytes
    long long tokens, channels;
    int batch;
    int element, gate_kind, complement;
    int cus;
};
// By element (recurrence_f32.hip, ...). back: the gradients.
int launch_recurrence_f32(const RecurrenceArgs& a, hipStream_t s, bool back);
int launch_recurrence_f16(const RecurrenceArgs& a, hipStream_t s, bool back);
int launch_recurrence_bf16(const RecurrenceArgs& a, hipStream_t s, bool back);

// Most channels of all sequences that run as chains of blocks: 64 to 128 channels a
// block, in up to 3 rounds of the CUs' number. A chain has 64; its counter has a
// line of kChainLine words. A launch has words_of 64-bit words for its chains.
constexpr int kChainLine = 32;
inline long long most_chained(int cus) { return (long long)cus * 128 * 3; }
inline long long words_of(int cus) { return (long long)cus * 4096; }
inline size_t recurrence_workspace_bytes(int cus) {
    return (size_t)(most_chained(cus) / 64 * kChainLine + most_chained(cus)) * sizeof(float) + (size_t)words_of(cus) * sizeof(uint64_t);
}

}  // namespace vkfx
