// recurrence_plan.cpp -- plans and C ABI of the gated recurrence. Arguments are
// checked here, before anything is launched; the kernels rely on it.
#include <memory>
#include <string>

#include "sequence.hpp"
#include "sequence_checks.hpp"

using namespace vkfx;

static_assert(kSpan == VKFX_RECURRENCE_SPAN);

struct vkfx_gated_recurrence {
    vkfx_context* ctx = nullptr;
    vkfx_gated_recurrence_desc desc{};
    DevBuf work;
};

namespace {

constexpr uint64_t kMostSequences = 65535, kMostTokens = 0x7fffffffull - 65535;

vkfx_sequence as_sequence(const vkfx_channels& c) { return vkfx_sequence{c.data, c.batch_stride, c.token_stride, 0}; }

int check_channels(const char* name, const vkfx_channels& c, uint64_t batch, uint64_t tokens, uint64_t channels, bool written) {
    return check_sequence(name, as_sequence(c), batch, tokens, 1, channels, written);
}

Tensor channels_of(const char* name, const vkfx_channels& c, uint64_t batch, uint64_t tokens, uint64_t channels, int32_t element,
                   bool written) {
    return sequence_of(name, as_sequence(c), batch, tokens, 1, channels, element, written);
}

// An output that stands in an input's place has its strides.
int check_in_place(const char* out, const vkfx_channels& o, const char* in, const vkfx_channels& i, uint64_t batch, uint64_t tokens) {
    if (o.data == i.data && ((batch > 1 && o.batch_stride != i.batch_stride) || (tokens > 1 && o.token_stride != i.token_stride)))
        return bad(std::string(out) + " may be " + in + " only with its strides");
    return VKFX_OK;
}

int check_counts(uint64_t batch, uint64_t tokens) {
    if (batch > kMostSequences) return fail(VKFX_ERR_RESOURCE_LIMIT, "more than 65535 sequences");
    if (tokens > kMostTokens) return fail(VKFX_ERR_RESOURCE_LIMIT, "more than 2^31 - 65536 tokens");
    return VKFX_OK;
}

RecurrenceSide side(const vkfx_channels& c) { return RecurrenceSide{c.data, c.batch_stride, c.token_stride}; }

RecurrenceArgs common(const vkfx_gated_recurrence* plan, uint64_t batch, uint64_t tokens, const int32_t* lengths, void* d_work) {
    RecurrenceArgs a{};
    a.lengths = lengths;
    a.work = (float*)(d_work ? d_work : plan->work.p);
    a.tokens = (long long)tokens;
    a.channels = (long long)plan->desc.channels;
    a.batch = (int)batch;
    a.element = plan->desc.element;
    a.gate_kind = plan->desc.gate;
    a.complement = plan->desc.complement;
    a.cus = (int)plan->ctx->profile.compute_units;
    return a;
}

int launch(const RecurrenceArgs& a, hipStream_t s, bool back) {
    if (a.element == VKFX_ELEMENT_F32) return launch_recurrence_f32(a, s, back);
    if (a.element == VKFX_ELEMENT_F16) return launch_recurrence_f16(a, s, back);
    return launch_recurrence_bf16(a, s, back);
}

}  // namespace

extern "C" {

int vkfx_gated_recurrence_create(vkfx_context* ctx, const vkfx_gated_recurrence_desc* desc, vkfx_gated_recurrence** out) {
    if (!ctx || !desc || !out) return bad("null argument");
    *out = nullptr;
    return guarded([&]() -> int {
        const vkfx_gated_recurrence_desc& d = *desc;
        if (d.channels < 1 || d.channels > (1u << 28)) return bad("channels must be 1 .. 2^28");
        if (!known_element(d.element)) return fail(VKFX_ERR_UNSUPPORTED_PRECISION, "element must be F32, F16 or BF16");
        if (d.gate != VKFX_GATE_SIGMOID && d.gate != VKFX_GATE_EXP) return bad("unknown gate");
        if (d.complement != 0 && d.complement != 1) return bad("complement must be 0 or 1");
        if (d.reserved) return bad("reserved must be 0");
        auto p = std::make_unique<vkfx_gated_recurrence>();
        p->ctx = ctx;
        p->desc = d;
        OnDevice on(ctx);
        const size_t bytes = recurrence_workspace_bytes((int)ctx->profile.compute_units);
        if (int rc = allocate(p->work, bytes)) return rc;
        retain(ctx);
        *out = p.release();
        return VKFX_OK;
    });
}

int vkfx_gated_recurrence_destroy(vkfx_gated_recurrence* plan) { return destroy(plan); }

int vkfx_gated_recurrence_workspace_bytes(const vkfx_gated_recurrence* plan, uint64_t* out) {
    if (!plan || !out) return bad("null argument");
    *out = plan->work.bytes;
    return VKFX_OK;
}

int vkfx_gated_recurrence_forward(vkfx_gated_recurrence* plan, const vkfx_gated_recurrence_forward_args* args, void* d_work,
                                  void* stream) {
    if (!plan || !args) return bad("null argument");
    return guarded([&]() -> int {
        const vkfx_gated_recurrence_desc& d = plan->desc;
        const uint64_t b = args->batch, t = args->tokens, c = d.channels;
        if (int rc = check_counts(b, t)) return rc;
        if (int rc = check_work(d_work)) return rc;
        if (!b) return VKFX_OK;
        if (t) {
            if (int rc = check_channels("x", args->x, b, t, c, false)) return rc;
            if (int rc = check_channels("gate", args->gate, b, t, c, false)) return rc;
            if (int rc = check_channels("y", args->y, b, t, c, true)) return rc;
            if (int rc = check_in_place("y", args->y, "x", args->x, b, t)) return rc;
        }
        const uint64_t states = b * c * 4;
        uint64_t saved;
        if (!mul(states, (t + kSpan - 1) / kSpan, &saved)) return fail(VKFX_ERR_ARITHMETIC_OVERFLOW, "saved states reach past 2^60 bytes");
        const char *in = "state_in", *after = "state_out", *x = "x", *y = "y";
        if (int rc = check_apart({channels_of(y, args->y, b, t, c, d.element, true), flat(after, args->state_out, states, true),
                                  flat("saved", args->saved, saved, true), flat("work", d_work, plan->work.bytes, true),
                                  flat(in, args->state_in, states, false), flat("lengths", args->lengths, b * 4, false),
                                  channels_of(x, args->x, b, t, c, d.element, false),
                                  channels_of("gate", args->gate, b, t, c, d.element, false)},
                                 args->state_in == args->state_out ? after : nullptr, in, args->y.data == args->x.data ? y : nullptr, x))
            return rc;
        RecurrenceArgs a = common(plan, b, t, args->lengths, d_work);
        a.x = side(args->x);
        a.gate = side(args->gate);
        a.y = side(args->y);
        a.state_in = args->state_in;
        a.state_out = args->state_out;
        a.saved = args->saved;
        OnDevice on(plan->ctx);
        const int e = launch(a, stream_of(plan->ctx, stream), false);
        return e == hipSuccess ? VKFX_OK : hip_fail((hipError_t)e, "launch gated recurrence");
    });
}

int vkfx_gated_recurrence_backward(vkfx_gated_recurrence* plan, const vkfx_gated_recurrence_backward_args* args, void* d_work,
                                   void* stream) {
    if (!plan || !args) return bad("null argument");
    return guarded([&]() -> int {
        const vkfx_gated_recurrence_desc& d = plan->desc;
        const uint64_t b = args->batch, t = args->tokens, c = d.channels;
        if (int rc = check_counts(b, t)) return rc;
        if (int rc = check_work(d_work)) return rc;
        if (!b) return VKFX_OK;
        if (t) {
            if (!args->saved) return bad("null saved");
            if (int rc = check_channels("x", args->x, b, t, c, false)) return rc;
            if (int rc = check_channels("gate", args->gate, b, t, c, false)) return rc;
            if (int rc = check_channels("dy", args->dy, b, t, c, false)) return rc;
            if (int rc = check_channels("dx", args->dx, b, t, c, true)) return rc;
            if (int rc = check_channels("dgate", args->dgate, b, t, c, true)) return rc;
            if (int rc = check_in_place("dx", args->dx, "dy", args->dy, b, t)) return rc;
        }
        const uint64_t states = b * c * 4;
        uint64_t saved;
        if (!mul(states, (t + kSpan - 1) / kSpan, &saved)) return fail(VKFX_ERR_ARITHMETIC_OVERFLOW, "saved states reach past 2^60 bytes");
        const char *dx = "dx", *dy = "dy", *in = "dstate_out", *after = "dstate_in";
        if (int rc = check_apart({channels_of(dx, args->dx, b, t, c, d.element, true),
                                  channels_of("dgate", args->dgate, b, t, c, d.element, true),
                                  flat(after, args->dstate_in, states, true), flat("work", d_work, plan->work.bytes, true),
                                  flat(in, args->dstate_out, states, false), flat("saved", args->saved, saved, false),
                                  flat("lengths", args->lengths, b * 4, false),
                                  channels_of("x", args->x, b, t, c, d.element, false),
                                  channels_of("gate", args->gate, b, t, c, d.element, false),
                                  channels_of(dy, args->dy, b, t, c, d.element, false)},
                                 args->dstate_in == args->dstate_out ? after : nullptr, in, args->dx.data == args->dy.data ? dx : nullptr, dy))
            return rc;
        RecurrenceArgs a = common(plan, b, t, args->lengths, d_work);
        a.x = side(args->x);
        a.gate = side(args->gate);
        a.dy = side(args->dy);
        a.y = side(args->dx);
        a.dgate = side(args->dgate);
        a.state_in = args->dstate_out;
        a.state_out = args->dstate_in;
        a.saved = (float*)args->saved;
        OnDevice on(plan->ctx);
        const int e = launch(a, stream_of(plan->ctx, stream), true);
        return e == hipSuccess ? VKFX_OK : hip_fail((hipError_t)e, "launch gated recurrence gradients");
    });
}

}  // extern "C"
