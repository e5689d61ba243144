// rotary_plan.cpp -- plans and C ABI of rotary positions and head norms.
// Arguments are checked here, before anything is launched; the kernels rely on
// it.
#include <cfloat>
#include <cmath>
#include <memory>
#include <string>
#include <vector>

#include "sequence.hpp"
#include "sequence_checks.hpp"

using namespace vkfx;

struct vkfx_rotary {
    vkfx_context* ctx = nullptr;
    vkfx_rotary_desc desc{};
    DevBuf turns;  // [rotary_dim / 2] 2^-64 turns a position
    DevBuf work;
};

namespace {

constexpr uint64_t kMostTokens = 0x7fffffffull;

// Radians as a fraction of a turn in 64 bits: multiples of it by whole numbers
// wrap as angles do.
uint64_t turn_of(double radians) {
    constexpr long double two_pi = 6.283185307179586476925286766559005768L;
    long double t = (long double)radians / two_pi;
    t -= floorl(t);
    t = rintl(t * 0x1p64L);
    return t >= 0x1p64L ? 0 : (uint64_t)t;
}

// One of the two tensors of a call and its result.
struct Pair {
    const char *in, *out;
    const vkfx_sequence &from, &to;
    uint64_t heads;
    bool wanted() const { return from.data && heads; }
    bool in_place() const { return from.data == to.data; }
};

int check_pair(const Pair& p, uint64_t batch, uint64_t tokens, uint64_t dim) {
    if (!p.wanted()) return VKFX_OK;
    if (int rc = check_sequence(p.in, p.from, batch, tokens, p.heads, dim, false)) return rc;
    if (int rc = check_sequence(p.out, p.to, batch, tokens, p.heads, dim, true)) return rc;
    const auto same = [](int64_t a, int64_t b, uint64_t extent) { return extent <= 1 || a == b; };
    if (p.in_place() && !(same(p.from.batch_stride, p.to.batch_stride, batch) && same(p.from.token_stride, p.to.token_stride, tokens) &&
                          same(p.from.head_stride, p.to.head_stride, p.heads)))
        return bad(std::string(p.out) + " may be " + p.in + " only with its strides");
    return VKFX_OK;
}

RotarySide side(const vkfx_sequence& s) { return RotarySide{s.data, s.batch_stride, s.token_stride, s.head_stride}; }

// What a forward and a backward call have in common.
int common(const vkfx_rotary* plan, uint64_t batch, uint64_t tokens, const int32_t* positions, const int32_t* starts,
           const int32_t* lengths, const void* q_weight, const void* k_weight, RotaryArgs* a) {
    const vkfx_rotary_desc& d = plan->desc;
    uint64_t all;
    if (positions && starts) return bad("positions and starts exclude each other");
    if (!d.norm && (q_weight || k_weight)) return bad("the plan was made without the norm: it has no weights");
    if (batch > kMostTokens || tokens > kMostTokens || (all = batch * tokens) > kMostTokens)
        return fail(VKFX_ERR_RESOURCE_LIMIT, "more than 2^31 - 1 tokens");
    a->rows[0].weight = q_weight;
    a->rows[1].weight = k_weight;
    a->turns = (const uint64_t*)plan->turns.p;
    a->positions = positions;
    a->starts = starts;
    a->lengths = lengths;
    a->tokens = (long long)tokens;
    a->all = (long long)all;
    a->dim = (int)d.head_dim;
    a->turned = (int)d.rotary_dim;
    a->layout = d.layout;
    a->element = d.element;
    a->weight_element = d.weight_element;
    a->norm = d.norm;
    a->epsilon = (float)d.epsilon;
    a->amplitude = (float)d.amplitude;
    a->cus = (int)plan->ctx->profile.compute_units;
    return VKFX_OK;
}

int launch(const RotaryArgs& a, hipStream_t s, bool back) {
    if (a.element == VKFX_ELEMENT_F32) return launch_rotary_f32(a, s, back);
    if (a.element == VKFX_ELEMENT_F16) return launch_rotary_f16(a, s, back);
    return launch_rotary_bf16(a, s, back);
}

}  // namespace

extern "C" {

int vkfx_rotary_create(vkfx_context* ctx, const vkfx_rotary_desc* desc, vkfx_rotary** out) {
    if (!ctx || !desc || !out) return bad("null argument");
    *out = nullptr;
    return guarded([&]() -> int {
        const vkfx_rotary_desc& d = *desc;
        if (d.heads < 1 || d.heads > 65535) return bad("heads must be 1 .. 65535");
        if (d.kv_heads > 65535) return bad("kv_heads must be 0 .. 65535");
        if (d.head_dim < 1 || d.head_dim > 256) return bad("head_dim must be 1 .. 256");
        if (d.rotary_dim > d.head_dim || d.rotary_dim % 2) return bad("rotary_dim must be even and at most head_dim");
        if (d.layout != VKFX_ROTARY_INTERLEAVED && d.layout != VKFX_ROTARY_HALF) return bad("unknown layout");
        if (!known_element(d.element)) return fail(VKFX_ERR_UNSUPPORTED_PRECISION, "element must be F32, F16 or BF16");
        if (d.weight_element != d.element && d.weight_element != VKFX_ELEMENT_F32)
            return fail(VKFX_ERR_UNSUPPORTED_PRECISION, "weights must be F32 or of the rows' element");
        if (d.norm != 0 && d.norm != 1) return bad("norm must be 0 or 1");
        if (d.norm && !((float)d.epsilon >= FLT_MIN && (float)d.epsilon <= FLT_MAX))
            return bad("epsilon must be a normal number of 32 bits");
        if (!std::isfinite((float)d.amplitude)) return bad("amplitude must be finite in 32 bits");
        if (d.rotary_dim && !d.frequencies) return bad("null frequencies");
        std::vector<uint64_t> turns(d.rotary_dim / 2);
        for (uint32_t i = 0; i < d.rotary_dim / 2; ++i) {
            if (!(std::fabs(d.frequencies[i]) <= 6.283185307179587)) return bad("frequencies must be within 2 pi: pair " + std::to_string(i));
            turns[i] = turn_of(d.frequencies[i]);
        }
        auto p = std::make_unique<vkfx_rotary>();
        p->ctx = ctx;
        p->desc = d;
        p->desc.frequencies = nullptr;
        OnDevice on(ctx);
        const size_t bytes = turns.size() * sizeof(uint64_t);
        if (int rc = allocate(p->turns, bytes)) return rc;
        if (bytes) {
            const hipError_t e = hipMemcpy(p->turns.p, turns.data(), bytes, hipMemcpyHostToDevice);
            if (e != hipSuccess) return hip_fail(e, "hipMemcpy frequencies");
        }
        if (d.norm)
            if (int rc = allocate(p->work, rotary_workspace_bytes((int)d.head_dim, (int)ctx->profile.compute_units))) return rc;
        retain(ctx);
        *out = p.release();
        return VKFX_OK;
    });
}

int vkfx_rotary_destroy(vkfx_rotary* plan) { return destroy(plan); }

int vkfx_rotary_workspace_bytes(const vkfx_rotary* plan, uint64_t* out) {
    if (!plan || !out) return bad("null argument");
    *out = plan->work.bytes;
    return VKFX_OK;
}

int vkfx_rotary_forward(vkfx_rotary* plan, const vkfx_rotary_forward_args* args, void* stream) {
    if (!plan || !args) return bad("null argument");
    return guarded([&]() -> int {
        const vkfx_rotary_desc& d = plan->desc;
        const uint64_t b = args->batch, t = args->tokens;
        RotaryArgs a{};
        if (int rc = common(plan, b, t, args->positions, args->starts, args->lengths, args->q_weight, args->k_weight, &a)) return rc;
        if (!a.all) return VKFX_OK;
        const Pair q{"q", "q_out", args->q, args->q_out, d.heads}, k{"k", "k_out", args->k, args->k_out, d.kv_heads};
        for (const Pair* p : {&q, &k})
            if (int rc = check_pair(*p, b, t, d.head_dim)) return rc;
        static const vkfx_sequence none{};
        const vkfx_sequence &qi = q.wanted() ? q.from : none, &qo = q.wanted() ? q.to : none;
        const vkfx_sequence &ki = k.wanted() ? k.from : none, &ko = k.wanted() ? k.to : none;
        const uint64_t weights = d.head_dim * bytes_of(d.weight_element);
        if (int rc = check_apart({sequence_of(q.out, qo, b, t, d.heads, d.head_dim, d.element, true),
                                  sequence_of(k.out, ko, b, t, d.kv_heads, d.head_dim, d.element, true),
                                  sequence_of(q.in, qi, b, t, d.heads, d.head_dim, d.element, false),
                                  sequence_of(k.in, ki, b, t, d.kv_heads, d.head_dim, d.element, false),
                                  flat("q_weight", args->q_weight, weights, false), flat("k_weight", args->k_weight, weights, false),
                                  flat("positions", args->positions, b * t * 4, false), flat("starts", args->starts, b * 4, false),
                                  flat("lengths", args->lengths, b * 4, false)},
                                 q.in_place() ? q.out : nullptr, q.in, k.in_place() ? k.out : nullptr, k.in))
            return rc;
        const Pair* pairs[2] = {&q, &k};
        for (int i = 0; i < 2; ++i) {
            if (!pairs[i]->wanted()) continue;
            a.rows[i].x = side(pairs[i]->from);
            a.rows[i].out = side(pairs[i]->to);
            a.rows[i].heads = (int)pairs[i]->heads;
        }
        OnDevice on(plan->ctx);
        const int e = launch(a, stream_of(plan->ctx, stream), false);
        return e == hipSuccess ? VKFX_OK : hip_fail((hipError_t)e, "launch rotary positions");
    });
}

int vkfx_rotary_backward(vkfx_rotary* plan, const vkfx_rotary_backward_args* args, void* d_work, void* stream) {
    if (!plan || !args) return bad("null argument");
    return guarded([&]() -> int {
        const vkfx_rotary_desc& d = plan->desc;
        const uint64_t b = args->batch, t = args->tokens;
        RotaryArgs a{};
        if (int rc = common(plan, b, t, args->positions, args->starts, args->lengths, args->q_weight, args->k_weight, &a)) return rc;
        if (!d.norm && (args->dq_weight || args->dk_weight)) return bad("the plan was made without the norm: it has no weights");
        if (d.norm)
            if (int rc = check_work(d_work)) return rc;
        const Pair q{"dq_out", "dq", args->dq_out, args->dq, d.heads}, k{"dk_out", "dk", args->dk_out, args->dk, d.kv_heads};
        const vkfx_sequence* inputs[2] = {&args->q, &args->k};
        const Pair* pairs[2] = {&q, &k};
        static const vkfx_sequence none{};
        const vkfx_sequence *from[2] = {&none, &none}, *to[2] = {&none, &none}, *in[2] = {&none, &none};
        for (int i = 0; i < 2 && a.all; ++i) {
            if (int rc = check_pair(*pairs[i], b, t, d.head_dim)) return rc;
            if (!pairs[i]->wanted()) continue;
            from[i] = &pairs[i]->from;
            to[i] = &pairs[i]->to;
            if (!d.norm) continue;
            if (int rc = check_sequence(i ? "k" : "q", *inputs[i], b, t, pairs[i]->heads, d.head_dim, false)) return rc;
            in[i] = inputs[i];
        }
        const uint64_t weights = d.head_dim * bytes_of(d.weight_element);
        if (int rc = check_apart({sequence_of(q.out, *to[0], b, t, d.heads, d.head_dim, d.element, true),
                                  sequence_of(k.out, *to[1], b, t, d.kv_heads, d.head_dim, d.element, true),
                                  flat("dq_weight", args->dq_weight, weights, true), flat("dk_weight", args->dk_weight, weights, true),
                                  flat("work", d_work, plan->work.bytes, true),
                                  sequence_of(q.in, *from[0], b, t, d.heads, d.head_dim, d.element, false),
                                  sequence_of(k.in, *from[1], b, t, d.kv_heads, d.head_dim, d.element, false),
                                  sequence_of("q", *in[0], b, t, d.heads, d.head_dim, d.element, false),
                                  sequence_of("k", *in[1], b, t, d.kv_heads, d.head_dim, d.element, false),
                                  flat("q_weight", args->q_weight, weights, false), flat("k_weight", args->k_weight, weights, false),
                                  flat("positions", args->positions, b * t * 4, false), flat("starts", args->starts, b * 4, false),
                                  flat("lengths", args->lengths, b * 4, false)},
                                 q.in_place() ? q.out : nullptr, q.in, k.in_place() ? k.out : nullptr, k.in))
            return rc;
        a.rows[0].dweight = args->dq_weight;
        a.rows[1].dweight = args->dk_weight;
        a.partial = (float*)(d_work ? d_work : plan->work.p);
        for (int i = 0; i < 2; ++i) {
            if (!from[i]->data) continue;
            a.rows[i].x = side(*from[i]);
            a.rows[i].in = side(*in[i]);
            a.rows[i].out = side(*to[i]);
            a.rows[i].heads = (int)pairs[i]->heads;
        }
        OnDevice on(plan->ctx);
        const int e = launch(a, stream_of(plan->ctx, stream), true);
        return e == hipSuccess ? VKFX_OK : hip_fail((hipError_t)e, "launch rotary gradients");
    });
}

}  // extern "C"
