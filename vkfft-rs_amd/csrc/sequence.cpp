// sequence.cpp -- plans and C ABI of the sequence operators: layer norm and
// linear attention. Arguments are checked here, before anything is launched;
// the kernels rely on it.
#include <algorithm>
#include <cfloat>
#include <cmath>
#include <memory>
#include <string>
#include <vector>

#include "sequence.hpp"
#include "sequence_checks.hpp"

using namespace vkfx;

struct vkfx_layer_norm {
    vkfx_context* ctx = nullptr;
    vkfx_layer_norm_desc desc{};
    DevBuf work;
};

struct vkfx_linear_attention {
    vkfx_context* ctx = nullptr;
    vkfx_linear_attention_desc desc{};
    DevBuf powers;  // [heads][kDecayPowers] floats
    DevBuf work;  // states between segments, then a shared head's gradients for each query head
    uint64_t state_floats = 0;
};

namespace {

ScanSide side(const vkfx_sequence& s, int group) {
    return ScanSide{s.data, s.batch_stride, s.token_stride, s.head_stride, group};
}

// Floats that calls of the scans need for states between segments.
uint64_t state_floats(const vkfx_linear_attention_desc& d) {
    // backward: the state for dq, its gradient for dk and dv
    return scan_work_floats((int)d.key_dim, (int)d.value_dim, (int)d.heads, d.gradient ? 2 : 1, (long long)d.max_batch,
                            (long long)d.max_tokens);
}

// Floats of the gradients of k and v for each query head, summed over a shared
// head's query heads afterwards.
bool group_floats(const vkfx_linear_attention_desc& d, uint64_t batch, uint64_t tokens, uint64_t* out) {
    *out = 0;
    if (d.heads == d.kv_heads) return true;
    uint64_t n;
    return mul(batch, tokens, &n) && mul(n, d.heads, &n) && mul(n, d.key_dim + d.value_dim, out);
}

}  // namespace

extern "C" {

int vkfx_layer_norm_create(vkfx_context* ctx, const vkfx_layer_norm_desc* desc, vkfx_layer_norm** out) {
    if (!ctx || !desc || !out) return bad("null argument");
    *out = nullptr;
    return guarded([&]() -> int {
        if (desc->width < 1 || desc->width > (1u << 30)) return bad("width must be 1 .. 2^30");
        if (!known_element(desc->element)) return fail(VKFX_ERR_UNSUPPORTED_PRECISION, "element must be F32, F16 or BF16");
        if (desc->weight_element != desc->element && desc->weight_element != VKFX_ELEMENT_F32)
            return fail(VKFX_ERR_UNSUPPORTED_PRECISION, "weights must be F32 or of the rows' element");
        if (!(desc->epsilon > 0) || !std::isfinite((float)desc->epsilon) || (float)desc->epsilon == 0.f)
            return bad("epsilon must be positive and finite in 32 bits");
        auto p = std::make_unique<vkfx_layer_norm>();
        p->ctx = ctx;
        p->desc = *desc;
        (void)hipSetDevice(ctx->device);
        if (int rc = allocate(p->work, norm_workspace_bytes(desc->element, (int)desc->width, (int)ctx->profile.compute_units))) return rc;
        retain(ctx);
        *out = p.release();
        return VKFX_OK;
    });
}

int vkfx_layer_norm_destroy(vkfx_layer_norm* plan) { return destroy(plan); }

int vkfx_layer_norm_workspace_bytes(const vkfx_layer_norm* plan, uint64_t* out) {
    if (!plan || !out) return bad("null argument");
    *out = plan->work.bytes;
    return VKFX_OK;
}

int vkfx_layer_norm_forward(vkfx_layer_norm* plan, uint64_t rows, const void* x, int64_t x_row_stride, const void* weight,
                            const void* bias, void* y, int64_t y_row_stride, float* stats, void* stream) {
    if (!plan) return bad("null plan");
    return guarded([&]() -> int {
        if (!rows) return VKFX_OK;
        const int64_t w = (int64_t)plan->desc.width;
        if (!x || !y) return bad("null device buffer");
        if (rows > 0x7fffffffull) return fail(VKFX_ERR_RESOURCE_LIMIT, "more than 2^31 - 1 rows");
        uint64_t reach;
        if (x_row_stride < 0 || (x_row_stride && x_row_stride < w && rows > 1)) return bad("x: rows overlap");
        if (y_row_stride < w && rows > 1) return bad("y: rows overlap");
        if (x == y && x_row_stride != y_row_stride && rows > 1) return bad("y may be x only with x's stride");
        if (!mul((uint64_t)x_row_stride, rows, &reach) || (rows > 1 && !mul((uint64_t)y_row_stride, rows, &reach)))
            return fail(VKFX_ERR_ARITHMETIC_OVERFLOW, "row strides reach past 2^60 elements");
        const int32_t element = plan->desc.element;
        const uint64_t weights = (uint64_t)w * bytes_of(plan->desc.weight_element);
        const char *nx = "x", *ny = "y";
        if (int rc = check_apart({rows_of(ny, y, rows, y_row_stride, w, element, true), flat("stats", stats, rows * 8, true),
                                  rows_of(nx, x, rows, x_row_stride, w, element, false), flat("weight", weight, weights, false),
                                  flat("bias", bias, weights, false)},
                                 x == y ? ny : nullptr, nx))
            return rc;
        NormArgs a{};
        a.x = x;
        a.weight = weight;
        a.bias = bias;
        a.y = y;
        a.stats_out = stats;
        a.rows = (long long)rows;
        a.x_stride = x_row_stride;
        a.y_stride = y_row_stride;
        a.width = (int)w;
        a.element = plan->desc.element;
        a.weight_element = plan->desc.weight_element;
        a.epsilon = (float)plan->desc.epsilon;
        a.cus = (int)plan->ctx->profile.compute_units;
        (void)hipSetDevice(plan->ctx->device);
        const int e = launch_norm_forward(a, stream_of(plan->ctx, stream));
        return e == hipSuccess ? VKFX_OK : hip_fail((hipError_t)e, "launch layer norm");
    });
}

int vkfx_layer_norm_backward(vkfx_layer_norm* plan, uint64_t rows, const void* x, int64_t x_row_stride, const void* weight,
                             const float* stats, const void* dy, int64_t dy_row_stride, void* dx, int64_t dx_row_stride,
                             void* dweight, void* dbias, void* d_work, void* stream) {
    if (!plan) return bad("null plan");
    return guarded([&]() -> int {
        const int64_t w = (int64_t)plan->desc.width;
        if (rows && (!x || !dy || !stats)) return bad("null device buffer");
        if (rows > 0x7fffffffull) return fail(VKFX_ERR_RESOURCE_LIMIT, "more than 2^31 - 1 rows");
        uint64_t reach;
        if (x_row_stride < 0 || (x_row_stride && x_row_stride < w && rows > 1)) return bad("x: rows overlap");
        if (dy_row_stride < 0 || (dy_row_stride && dy_row_stride < w && rows > 1)) return bad("dy: rows overlap");
        if (dx && dx_row_stride < w && rows > 1) return bad("dx: rows overlap");
        if (dx && dx == dy && dx_row_stride != dy_row_stride && rows > 1) return bad("dx may be dy only with dy's stride");
        if (!mul((uint64_t)x_row_stride, rows, &reach) || !mul((uint64_t)dy_row_stride, rows, &reach) ||
            (dx && rows > 1 && !mul((uint64_t)dx_row_stride, rows, &reach)))
            return fail(VKFX_ERR_ARITHMETIC_OVERFLOW, "row strides reach past 2^60 elements");
        const int32_t element = plan->desc.element;
        const uint64_t weights = (uint64_t)w * bytes_of(plan->desc.weight_element);
        const char *nx = "dx", *ny = "dy";
        if (int rc = check_apart({rows_of(nx, dx, rows, dx_row_stride, w, element, true), flat("dweight", dweight, weights, true),
                                  flat("dbias", dbias, weights, true), flat("work", d_work, plan->work.bytes, true),
                                  rows_of(ny, dy, rows, dy_row_stride, w, element, false),
                                  rows_of("x", x, rows, x_row_stride, w, element, false), flat("weight", weight, weights, false),
                                  flat("stats", stats, rows * 8, false)},
                                 dx == dy ? nx : nullptr, ny))
            return rc;
        NormArgs a{};
        a.x = x;
        a.weight = weight;
        a.stats_in = stats;
        a.dy = dy;
        a.y = dx;
        a.dweight = dweight;
        a.dbias = dbias;
        a.partial = (float*)(d_work ? d_work : plan->work.p);
        a.rows = (long long)rows;
        a.x_stride = x_row_stride;
        a.dy_stride = dy_row_stride;
        a.y_stride = dx_row_stride;
        a.width = (int)w;
        a.element = plan->desc.element;
        a.weight_element = plan->desc.weight_element;
        a.cus = (int)plan->ctx->profile.compute_units;
        (void)hipSetDevice(plan->ctx->device);
        const int e = launch_norm_backward(a, stream_of(plan->ctx, stream));
        return e == hipSuccess ? VKFX_OK : hip_fail((hipError_t)e, "launch layer norm gradients");
    });
}

int vkfx_linear_attention_create(vkfx_context* ctx, const vkfx_linear_attention_desc* desc, vkfx_linear_attention** out) {
    if (!ctx || !desc || !out) return bad("null argument");
    *out = nullptr;
    return guarded([&]() -> int {
        const vkfx_linear_attention_desc& d = *desc;
        if (d.heads < 1 || d.heads > 65535) return bad("heads must be 1 .. 65535");
        if (d.kv_heads < 1 || d.heads % d.kv_heads) return bad("kv_heads must divide heads");
        if (d.key_dim < 1 || d.key_dim > 256 || d.value_dim < 1 || d.value_dim > 256)
            return bad("key_dim and value_dim must be 1 .. 256");
        if (!known_element(d.element)) return fail(VKFX_ERR_UNSUPPORTED_PRECISION, "element must be F32, F16 or BF16");
        if (!std::isfinite(d.scale) || !std::isfinite((float)d.scale)) return bad("scale must be finite in 32 bits");
        if (!d.decay) return bad("null decay");
        if (d.max_batch < 1 || d.max_batch > 65535) return bad("max_batch must be 1 .. 65535");
        if (d.max_tokens < 1 || d.max_tokens > 0x7fffffffull - 4095) return bad("max_tokens must be 1 .. 2^31 - 4096");
        std::vector<float> powers((size_t)d.heads * kDecayPowers);
        for (uint32_t h = 0; h < d.heads; ++h) {
            if (!(d.decay[h] >= 0 && d.decay[h] <= 1)) return bad("decay must be in [0, 1]: head " + std::to_string(h));
            float* row = powers.data() + (size_t)h * kDecayPowers;
            for (int n = 0; n < kDecayHigh; ++n) row[n] = (float)std::pow(d.decay[h], n);
            float high = (float)d.decay[h];
            if ((double)high > d.decay[h]) high = std::nextafter(high, 0.f);
            row[kDecayHigh] = high;
            row[kDecayLow] = (float)(d.decay[h] - (double)high);
            if (d.decay[h] > 0 && row[kDecayLow] == 0.f) row[kDecayLow] = std::max(high * 0x1p-60f, FLT_TRUE_MIN);
        }
        uint64_t floats = 0;
        if (d.gradient && !group_floats(d, d.max_batch, d.max_tokens, &floats))
            return fail(VKFX_ERR_ARITHMETIC_OVERFLOW, "workspace size");
        auto p = std::make_unique<vkfx_linear_attention>();
        p->ctx = ctx;
        p->desc = d;
        p->desc.decay = nullptr;
        (void)hipSetDevice(ctx->device);
        if (int rc = allocate(p->powers, powers.size() * sizeof(float))) return rc;
        const hipError_t e = hipMemcpy(p->powers.p, powers.data(), powers.size() * sizeof(float), hipMemcpyHostToDevice);
        if (e != hipSuccess) return hip_fail(e, "hipMemcpy decays");
        p->state_floats = state_floats(d);
        if (int rc = allocate(p->work, (p->state_floats + floats) * sizeof(float))) return rc;
        retain(ctx);
        *out = p.release();
        return VKFX_OK;
    });
}

int vkfx_linear_attention_destroy(vkfx_linear_attention* plan) { return destroy(plan); }

int vkfx_linear_attention_workspace_bytes(const vkfx_linear_attention* plan, uint64_t* out) {
    if (!plan || !out) return bad("null argument");
    *out = plan->work.bytes;
    return VKFX_OK;
}

int vkfx_linear_attention_forward(vkfx_linear_attention* plan, const vkfx_linear_attention_forward_args* args, void* d_work,
                                  void* stream) {
    if (!plan || !args) return bad("null argument");
    return guarded([&]() -> int {
        const vkfx_linear_attention_desc& d = plan->desc;
        if (args->batch > d.max_batch || args->tokens > d.max_tokens)
            return fail(VKFX_ERR_INPUT_LENGTH_MISMATCH, "more sequences or tokens than the plan's capacity");
        if (!args->batch) return VKFX_OK;
        if (args->tokens) {
            if (int rc = check_sequence("q", args->q, args->batch, args->tokens, d.heads, d.key_dim, false)) return rc;
            if (int rc = check_sequence("k", args->k, args->batch, args->tokens, d.kv_heads, d.key_dim, false)) return rc;
            if (int rc = check_sequence("v", args->v, args->batch, args->tokens, d.kv_heads, d.value_dim, false)) return rc;
            if (int rc = check_sequence("out", args->out, args->batch, args->tokens, d.heads, d.value_dim, true)) return rc;
        }
        const uint64_t b = args->batch, t = args->tokens, states = b * d.heads * d.key_dim * d.value_dim * 4;
        const char *in = "state_in", *after = "state_out";
        if (int rc = check_apart({sequence_of("out", args->out, b, t, d.heads, d.value_dim, d.element, true),
                                  flat(after, args->state_out, states, true), flat("work", d_work, plan->work.bytes, true),
                                  flat(in, args->state_in, states, false), flat("lengths", args->lengths, b * 4, false),
                                  sequence_of("q", args->q, b, t, d.heads, d.key_dim, d.element, false),
                                  sequence_of("k", args->k, b, t, d.kv_heads, d.key_dim, d.element, false),
                                  sequence_of("v", args->v, b, t, d.kv_heads, d.value_dim, d.element, false)},
                                 args->state_in == args->state_out ? after : nullptr, in))
            return rc;
        const int group = (int)(d.heads / d.kv_heads);
        ScanArgs s{};
        s.a = side(args->q, 1);
        s.b = side(args->k, group);
        s.c = side(args->v, group);
        s.out = (void*)args->out.data;
        s.out_batch = args->out.batch_stride;
        s.out_token = args->out.token_stride;
        s.out_head = args->out.head_stride;
        s.lengths = args->lengths;
        s.state_in = args->state_in;
        s.state_out = args->state_out;
        s.state_row = (int)d.value_dim;
        s.state_col = 1;
        s.tokens = (long long)args->tokens;
        s.batch = (int)args->batch;
        s.heads = (int)d.heads;
        s.dk = (int)d.key_dim;
        s.dv = (int)d.value_dim;
        s.scale_in = (float)d.scale;
        s.scale_update = 1.f;
        s.like = -1;
        (void)hipSetDevice(plan->ctx->device);
        float* work = (float*)(d_work ? d_work : plan->work.p);
        const int e = launch_scans(d.element, &s, 1, (const float*)plan->powers.p, work, (int)plan->ctx->profile.compute_units,
                                   stream_of(plan->ctx, stream));
        return e == hipSuccess ? VKFX_OK : hip_fail((hipError_t)e, "launch linear attention");
    });
}

int vkfx_linear_attention_backward(vkfx_linear_attention* plan, const vkfx_linear_attention_backward_args* args, void* d_work,
                                   void* stream) {
    if (!plan || !args) return bad("null argument");
    return guarded([&]() -> int {
        const vkfx_linear_attention_desc& d = plan->desc;
        if (args->batch > d.max_batch || args->tokens > d.max_tokens)
            return fail(VKFX_ERR_INPUT_LENGTH_MISMATCH, "more sequences or tokens than the plan's capacity");
        if (!d.gradient) return bad("the plan was made without gradient");
        if (!args->batch) return VKFX_OK;
        const uint64_t b = args->batch, t = args->tokens;
        if (t) {
            if (int rc = check_sequence("q", args->q, b, t, d.heads, d.key_dim, false)) return rc;
            if (int rc = check_sequence("k", args->k, b, t, d.kv_heads, d.key_dim, false)) return rc;
            if (int rc = check_sequence("v", args->v, b, t, d.kv_heads, d.value_dim, false)) return rc;
            if (int rc = check_sequence("dout", args->dout, b, t, d.heads, d.value_dim, false)) return rc;
            if (int rc = check_sequence("dq", args->dq, b, t, d.heads, d.key_dim, true)) return rc;
            if (int rc = check_sequence("dk", args->dk, b, t, d.kv_heads, d.key_dim, true)) return rc;
            if (int rc = check_sequence("dv", args->dv, b, t, d.kv_heads, d.value_dim, true)) return rc;
        }
        const uint64_t states = b * d.heads * d.key_dim * d.value_dim * 4;
        if (int rc = check_apart({sequence_of("dq", args->dq, b, t, d.heads, d.key_dim, d.element, true),
                                  sequence_of("dk", args->dk, b, t, d.kv_heads, d.key_dim, d.element, true),
                                  sequence_of("dv", args->dv, b, t, d.kv_heads, d.value_dim, d.element, true),
                                  flat("dstate_in", args->dstate_in, states, true), flat("work", d_work, plan->work.bytes, true),
                                  flat("state_in", args->state_in, states, false),
                                  flat("dstate_out", args->dstate_out, states, false), flat("lengths", args->lengths, b * 4, false),
                                  sequence_of("q", args->q, b, t, d.heads, d.key_dim, d.element, false),
                                  sequence_of("k", args->k, b, t, d.kv_heads, d.key_dim, d.element, false),
                                  sequence_of("v", args->v, b, t, d.kv_heads, d.value_dim, d.element, false),
                                  sequence_of("dout", args->dout, b, t, d.heads, d.value_dim, d.element, false)}))
            return rc;
        const int group = (int)(d.heads / d.kv_heads);
        const int dk = (int)d.key_dim, dv = (int)d.value_dim;
        float* work = (float*)(d_work ? d_work : plan->work.p);
        ScanArgs base{};
        base.lengths = args->lengths;
        base.tokens = (long long)t;
        base.batch = (int)b;
        base.heads = (int)d.heads;
        const auto scan = [&](const vkfx_sequence& x, int gx, const vkfx_sequence& y, int gy, const vkfx_sequence& z, int gz) {
            ScanArgs s = base;
            s.a = side(x, gx);
            s.b = side(y, gy);
            s.c = side(z, gz);
            return s;
        };
        // dq: the forward scan of (dout, v, k) from the state's transpose
        ScanArgs scans[3] = {scan(args->dout, 1, args->v, group, args->k, group), scan(args->k, group, args->q, 1, args->dout, 1),
                             scan(args->v, group, args->dout, 1, args->q, 1)};
        ScanArgs &q = scans[0], &v = scans[1], &k = scans[2];
        q.like = v.like = -1;
        k.like = 1;
        q.dk = dv, q.dv = dk, q.state_row = 1, q.state_col = dv, q.state_in = args->state_in;
        q.scale_in = (float)d.scale, q.scale_update = 1.f;
        v.dk = dk, v.dv = dv, v.state_row = dv, v.state_col = 1, v.state_in = args->dstate_out, v.state_out = args->dstate_in;
        k.dk = dv, k.dv = dk, k.state_row = 1, k.state_col = dv, k.state_in = args->dstate_out;
        v.reverse = k.reverse = 1;
        v.scale_in = k.scale_in = 1.f;
        v.scale_update = k.scale_update = (float)d.scale;
        const auto to = [&](ScanArgs& s, const vkfx_sequence& o) {
            s.out = (void*)o.data;
            s.out_batch = o.batch_stride, s.out_token = o.token_stride, s.out_head = o.head_stride;
        };
        to(q, args->dq);
        float *wk = work + plan->state_floats, *wv = wk + b * t * d.heads * d.key_dim;
        if (group > 1) {  // floats of every query head, [batch][token][head][dim]
            to(k, vkfx_sequence{wk, (int64_t)(t * d.heads * dk), (int64_t)d.heads * dk, dk});
            to(v, vkfx_sequence{wv, (int64_t)(t * d.heads * dv), (int64_t)d.heads * dv, dv});
            k.out_f32 = v.out_f32 = 1;
        } else {
            to(k, args->dk);
            to(v, args->dv);
        }
        (void)hipSetDevice(plan->ctx->device);
        hipStream_t st = stream_of(plan->ctx, stream);
        int e = launch_scans(d.element, scans, 3, (const float*)plan->powers.p, work, (int)plan->ctx->profile.compute_units, st);
        if (e == hipSuccess && group > 1 && t) {
            e = launch_group_sum(d.element, GroupSum{wk, side(args->dk, 1), dk}, GroupSum{wv, side(args->dv, 1), dv},
                                 (long long)b, (long long)t, (int)d.kv_heads, group, st);
        }
        return e == hipSuccess ? VKFX_OK : hip_fail((hipError_t)e, "launch linear attention gradients");
    });
}

}  // extern "C"
