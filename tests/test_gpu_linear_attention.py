"""Linear attention with a decay for each head: prompts, single tokens and
gradients against the recurrence in 64 bits."""
import numpy as np
import pytest

import sequence_reference as ref
import vkfft_amd as vk

pytestmark = pytest.mark.gpu

ELEMENT = {"f32": vk.Element.F32, "f16": vk.Element.F16, "bf16": vk.Element.BF16}
ELEMENTS = list(ELEMENT)


def _types():
    import torch
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _decays(heads):
    return [(0.5, 0.9375, 0.998, 1.0, 0.0, 0.99)[h % 6] for h in range(heads)]


def _plan(ctx, batch, tokens, heads, kv, dk, dv, element, gradient=False, decay=None, scale=None):
    c = vk.LinearAttentionConfig.new(heads, dk, dv).with_kv_heads(kv).with_element(ELEMENT[element]).with_gradient(gradient)
    c.with_decay(decay or _decays(heads)).with_capacity(max(1, batch), max(1, tokens))
    if scale is not None:
        c.with_scale(scale)
    return vk.LinearAttentionPlan(ctx, c)


def _tensor(seed, shape, element, layout="bthd", pad=0, offset=0):
    """[batch][token][head][dim], laid out "bthd" or "bhtd" with `pad` unused elements after each row."""
    import torch
    b, t, h, d = shape
    g = torch.Generator(device="cuda").manual_seed(seed)
    p = d + pad
    flat = torch.full((offset + b * t * h * p + 8,), float("nan"), device="cuda", dtype=_types()[element])
    strides = (t * h * p, h * p, p, 1) if layout == "bthd" else (t * h * p, p, t * p, 1)
    x = flat.as_strided(shape, strides, offset)
    x.copy_(torch.randn(shape, generator=g, device="cuda", dtype=torch.float32))
    return x


def _state(seed, *shape):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32) * 2


def _np(*xs):
    return [None if x is None else x.double().cpu().numpy() for x in xs]




def _run(ctx, element, b, t, h, kv, dk, dv, lengths=None, gradient=True, layout="bthd", pad=0, offset=0, decay=None, states=True):
    import torch
    kw = {"layout": layout, "pad": pad, "offset": offset}
    plan = _plan(ctx, b, t, h, kv, dk, dv, element, gradient, decay)
    decay = decay or _decays(h)
    q, k, v = _tensor(1, (b, t, h, dk), element, **kw), _tensor(2, (b, t, kv, dk), element, **kw), _tensor(3, (b, t, kv, dv), element, **kw)
    state = _state(4, b, h, dk, dv) if states else None
    n = torch.tensor(lengths, device="cuda", dtype=torch.int32) if lengths is not None else None
    ln = np.clip(np.array(lengths if lengths is not None else [t] * b), 0, t)
    if lengths is not None:  # what lies past a sequence's end is not read
        for i, m in enumerate(ln):
            for x in (q, k, v):
                x[i, m:] = float("nan")
    out = _tensor(5, (b, t, h, dv), element, **kw)
    state_out = torch.full((b, h, dk, dv), float("nan"), device="cuda")
    plan.forward_tensors(q, k, v, out, state_in=state, state_out=state_out, lengths=n)
    qn, kn, vn = (np.nan_to_num(x) for x in _np(q, k, v))
    sn = _np(state)[0] if states else np.zeros((b, h, dk, dv))
    scale = np.float64(np.float32(dk ** -0.5))
    args = (decay, scale, ln)
    want, total = ref.attention(qn, kn, vn, sn, *args), ref.attention(*map(np.abs, (qn, kn, vn, sn)), *args)
    ref.check("out", out, want[0], total[0], element, ref.TERM[element])
    ref.check("state", state_out, want[1], total[1], "f32", ref.STATE_TERM)
    if pad:
        rows = out.as_strided(out.shape[:3] + (pad,), out.stride(), out.storage_offset() + dv)
        assert torch.isnan(rows).all()
    if not gradient:
        return
    dout = _tensor(6, (b, t, h, dv), element, **kw)
    for i, m in enumerate(ln):
        dout[i, m:] = float("nan")
    dstate = _state(7, b, h, dk, dv) if states else None
    dq, dkk, dvv = (_tensor(8, x.shape, element, **kw) for x in (q, k, v))
    dstate_in = torch.full((b, h, dk, dv), float("nan"), device="cuda")
    plan.backward_tensors(q, k, v, dout, dq, dkk, dvv, state_in=state, dstate_out=dstate, dstate_in=dstate_in, lengths=n)
    don, = (np.nan_to_num(x) for x in _np(dout))
    dsn = _np(dstate)[0] if states else np.zeros((b, h, dk, dv))
    want = ref.attention_gradients(qn, kn, vn, sn, don, dsn, *args)
    total = ref.attention_gradients(*map(np.abs, (qn, kn, vn, sn, don, dsn)), *args)
    for name, got, w, a in zip(("dq", "dk", "dv"), (dq, dkk, dvv), want, total):
        ref.check(name, got, w, a, element, ref.TERM[element])
    ref.check("dstate_in", dstate_in, want[3], total[3], "f32", ref.STATE_TERM)


@pytest.mark.parametrize("element", ELEMENTS)
@pytest.mark.parametrize("t", [1, 2, 3, 8, 9, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 130, 300])
def test_lengths_of_time(hip_ctx, element, t):
    _run(hip_ctx, element, 2, t, 3, 3, 64, 64)


@pytest.mark.parametrize("element", ELEMENTS)
@pytest.mark.parametrize("dk,dv", [(1, 1), (1, 64), (64, 1), (3, 5), (16, 32), (17, 33), (32, 96), (77, 80), (80, 96), (96, 112), (100, 130),
                                   (128, 128), (128, 64), (129, 127), (192, 64), (64, 192), (200, 24), (256, 256)])
def test_widths(hip_ctx, element, dk, dv):
    _run(hip_ctx, element, 1, 150, 2, 2, dk, dv)


@pytest.mark.parametrize("element", ELEMENTS)
@pytest.mark.parametrize("h,kv", [(4, 1), (6, 2), (12, 4), (1, 1)])
def test_shared_heads(hip_ctx, element, h, kv):
    _run(hip_ctx, element, 2, 100, h, kv, 48, 64)


@pytest.mark.parametrize("element", ELEMENTS)
@pytest.mark.parametrize("dk,dv", [(1, 3), (5, 6), (30, 129), (254, 255)])
def test_shared_heads_of_any_width(hip_ctx, element, dk, dv):
    _run(hip_ctx, element, 2, 37, 6, 2, dk, dv, pad=3, offset=1)


@pytest.mark.parametrize("element", ELEMENTS)
@pytest.mark.parametrize("t,lengths", [(5, [0, 1, 5, 3]), (1, [0, 1, 1, 0]), (130, [130, 0, 64, 65]), (200, [1, 63, 199, 200]),
                                       (70, [-3, 71, 2 ** 31 - 1, 7])])
def test_uneven_lengths(hip_ctx, element, t, lengths):
    _run(hip_ctx, element, 4, t, 4, 2, 40, 72, lengths=lengths)


@pytest.mark.parametrize("element", ELEMENTS)
@pytest.mark.parametrize("layout,pad,offset", [("bhtd", 0, 0), ("bthd", 8, 0), ("bhtd", 3, 1), ("bthd", 1, 5)])
def test_layouts(hip_ctx, element, layout, pad, offset):
    _run(hip_ctx, element, 2, 90, 4, 2, 64, 80, layout=layout, pad=pad, offset=offset)
    _run(hip_ctx, element, 2, 1, 4, 2, 64, 80, layout=layout, pad=pad, offset=offset, gradient=False)


@pytest.mark.parametrize("element", ELEMENTS)
def test_without_states(hip_ctx, element):
    _run(hip_ctx, element, 2, 100, 2, 1, 32, 48, states=False)


@pytest.mark.parametrize("element", ELEMENTS)
@pytest.mark.parametrize("decay", [0.0, 1.0, 1e-30, 0.999999])
def test_decays_at_the_ends(hip_ctx, element, decay):
    _run(hip_ctx, element, 1, 140, 2, 2, 32, 32, decay=[decay, 0.75])


@pytest.mark.parametrize("element", ELEMENTS)
@pytest.mark.parametrize("t,lengths", [(4100, None), (4100, [4100, 77]), (5000, [4097, 0])])
def test_long_sequences_of_few_heads(hip_ctx, element, t, lengths):
    """Split over the tokens where one sequence's heads cannot fill the GPU."""
    _run(hip_ctx, element, 2, t, 2, 1, 64, 48, lengths=lengths, decay=[0.998, 0.99])


@pytest.mark.parametrize("element", ELEMENTS)
@pytest.mark.parametrize("b,h,dk,dv", [(70, 8, 128, 128), (3, 5, 100, 36), (1, 1, 256, 256), (300, 2, 16, 16)])
@pytest.mark.parametrize("t", [1, 4])
def test_single_tokens(hip_ctx, element, b, h, dk, dv, t):
    _run(hip_ctx, element, b, t, h, h, dk, dv, gradient=False)


@pytest.mark.parametrize("element", ELEMENTS)
def test_token_by_token_gives_the_prompts_outputs(hip_ctx, element):
    """A prompt in one call, in two parts, and token by token in place."""
    import torch
    b, t, h, d = 2, 97, 2, 64
    plan = _plan(hip_ctx, b, t, h, h, d, d, element)
    q, k, v = (_tensor(i, (b, t, h, d), element) for i in (1, 2, 3))
    outs, states = [], []
    for parts in ([97], [40, 57], [1] * 97):
        state, out, at = _state(4, b, h, d, d), torch.empty_like(v), 0
        for n in parts:
            plan.forward_tensors(*(x[:, at:at + n] for x in (q, k, v, out)), state_in=state, state_out=state)
            at += n
        outs.append(out.double())
        states.append(state.double())
    for o, s in zip(outs[1:], states[1:]):
        # each way is within its own bound of the definition: twice that apart
        assert (o - outs[0]).norm() <= 2 * (ref.UNIT[element] + ref.TERM[element]) * outs[0].norm()
        assert (s - states[0]).norm() <= 2 * ref.STATE_TERM * states[0].norm()


def test_an_exponential_filter_is_a_convolution(hip_ctx):
    """With q = k = 1 a head is the causal filter decay^t, which a zero-padded convolution plan computes."""
    import torch
    n, decay = 500, 0.97
    x = _tensor(1, (1, n, 1, 1), "f32")
    one = torch.ones_like(x)
    out = torch.empty_like(x)
    _plan(hip_ctx, 1, n, 1, 1, 1, 1, "f32", decay=[decay], scale=1.0).forward_tensors(one, one, x, out)
    h = np.zeros(1024)
    h[:n] = decay ** np.arange(n)
    conv = vk.ConvolutionIr.build(vk.FftConfig.new([1024]).with_convolution(True), np.fft.fft(h).astype(np.complex64))
    padded = np.zeros(1024, np.complex64)
    padded[:n] = x.flatten().cpu().numpy()
    y = hip_ctx.execute_convolution(conv, padded)[:n].real
    got = out.flatten().cpu().numpy()
    # both in 32 bits: the convolution's error is 1e-6 of the output's norm
    assert np.linalg.norm(got - y) <= 4e-6 * np.linalg.norm(y)


def test_gradients_against_differences(hip_ctx):
    """<out, dout> + <state_out, dstate> is linear in each input alone: its difference along a direction is its slope."""
    import torch
    b, t, h, kv, dk, dv = 2, 150, 4, 2, 24, 40
    plan = _plan(hip_ctx, b, t, h, kv, dk, dv, "f32", True)
    at = [_tensor(1, (b, t, h, dk), "f32"), _tensor(2, (b, t, kv, dk), "f32"), _tensor(3, (b, t, kv, dv), "f32"), _state(4, b, h, dk, dv)]
    dout, dstate = _tensor(5, (b, t, h, dv), "f32"), _state(6, b, h, dk, dv)
    n = torch.tensor([150, 91], device="cuda", dtype=torch.int32)
    got = [torch.empty_like(x) for x in at]
    plan.backward_tensors(*at[:3], dout, *got[:3], state_in=at[3], dstate_out=dstate, dstate_in=got[3], lengths=n)

    def loss(xs):
        out, state = torch.empty_like(dout), torch.empty_like(dstate)
        plan.forward_tensors(*xs[:3], out, state_in=xs[3], state_out=state, lengths=n)
        terms = [(out.double() * dout.double()).flatten(), (state.double() * dstate.double()).flatten()]
        return sum(x.sum().item() for x in terms), sum(x.abs().sum().item() for x in terms)

    for i, g in enumerate(got):
        d = torch.randn(at[i].shape, generator=torch.Generator(device="cuda").manual_seed(40 + i), device="cuda")
        up, down = list(at), list(at)
        up[i], down[i] = at[i] + d, at[i] - d
        (lu, au), (ld, ad) = loss(up), loss(down)
        # both losses round in 32 bits; so does the gradient
        assert abs((g.double() * d.double()).sum().item() - (lu - ld) / 2) <= ref.TERM["f32"] * (au + ad)


def test_no_tokens_and_no_sequences(hip_ctx):
    import torch
    plan = _plan(hip_ctx, 2, 8, 2, 1, 16, 24, "bf16", True)
    for b in (2, 0):
        q, k, v = (torch.empty(b, 0, h, d, device="cuda", dtype=torch.bfloat16) for h, d in ((2, 16), (1, 16), (1, 24)))
        out = torch.empty(b, 0, 2, 24, device="cuda", dtype=torch.bfloat16)
        state = _state(1, b, 2, 16, 24)
        after = torch.full_like(state, 7)
        plan.forward_tensors(q, k, v, out, state_in=state, state_out=after)
        assert torch.equal(state, after)
        back = torch.full_like(state, 7)
        plan.backward_tensors(q, k, v, out, q.clone(), k.clone(), v.clone(), state_in=state, dstate_out=state, dstate_in=back)
        assert torch.equal(state, back)


def test_capacity_is_an_upper_bound(hip_ctx):
    """One plan serves every size up to its capacity, and its workspace holds what one call left there."""
    import torch
    plan = _plan(hip_ctx, 3, 4096, 2, 1, 64, 64, "bf16", True, decay=[0.99, 0.9])
    for b, t in ((1, 4096), (3, 70), (1, 1), (2, 1000)):
        one = _plan(hip_ctx, b, t, 2, 1, 64, 64, "bf16", True, decay=[0.99, 0.9])
        q, k, v, dout = (_tensor(i, (b, t, h, 64), "bf16") for i, h in ((1, 2), (2, 1), (3, 1), (4, 2)))
        runs = []
        for p in (plan, one):
            o = [torch.full_like(x, float("nan")) for x in (dout, q, k, v)]
            p.forward_tensors(q, k, v, o[0])
            p.backward_tensors(q, k, v, dout, *o[1:])
            runs.append(o)
        assert all(torch.equal(x, y) for x, y in zip(*runs))


def test_broadcast_inputs(hip_ctx):
    """Keys and values of one sequence and one head for all, without copies."""
    import torch
    q = _tensor(1, (3, 80, 4, 32), "f32")
    k, v = _tensor(2, (1, 80, 1, 32), "f32"), _tensor(3, (1, 80, 1, 32), "f32")
    plan = _plan(hip_ctx, 3, 80, 4, 4, 32, 32, "f32")
    a, b = torch.empty_like(q), torch.empty_like(q)
    plan.forward_tensors(q, k.expand(3, 80, 4, 32), v.expand(3, 80, 4, 32), a)
    plan.forward_tensors(q, k.expand(3, 80, 4, 32).contiguous(), v.expand(3, 80, 4, 32).contiguous(), b)
    assert torch.equal(a, b)


def test_offsets_past_32_bits(hip_ctx):
    """Rows of a buffer whose offsets pass 2^32 elements."""
    import torch
    far = torch.zeros((1 << 32) + (1 << 20), device="cuda", dtype=torch.bfloat16)
    t, h, d = 96, 1, 64
    step = (1 << 32) // (t - 1) // 64 * 64 + 64
    x = [far.as_strided((1, t, h, d), (far.numel(), step, d, 1), 0), far.as_strided((1, t, h, d), (far.numel(), step, d, 1), 128),
         far.as_strided((1, t, h, d), (far.numel(), step, d, 1), 256), far.as_strided((1, t, h, d), (far.numel(), step, d, 1), 384)]
    near = [_tensor(i, (1, t, h, d), "bf16") for i in range(4)]
    for f, n in zip(x[:3], near):
        f.copy_(n)
    plan = _plan(hip_ctx, 1, t, h, h, d, d, "bf16", decay=[0.95])
    plan.forward_tensors(*x)
    plan.forward_tensors(*near)
    assert torch.equal(x[3], near[3])


@pytest.mark.parametrize("where", ["past the length", "another sequence", "another head"])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_bad_values_stay_where_they_belong(hip_ctx, where, value):
    import torch
    plan = _plan(hip_ctx, 2, 100, 2, 2, 32, 32, "bf16", True)
    x = [_tensor(i, (2, 100, 2, 32), "bf16") for i in range(4)]
    n = torch.tensor([40, 100], device="cuda", dtype=torch.int32)

    def run():
        o = [torch.full_like(x[0], 3) for _ in range(4)]
        plan.forward_tensors(*x[:3], o[0], lengths=n)
        plan.backward_tensors(*x, *o[1:], lengths=n)
        return o

    want = run()
    for y in x:
        if where == "past the length":
            y[0, 40:] = value
        elif where == "another sequence":
            y[1, 50] = value
        else:
            y[0, 20, 1] = value
    got = run()
    at = (slice(0, 1), slice(None), slice(0, 1)) if where == "another head" else (slice(0, 1),)
    assert all(torch.equal(p[at], q[at]) for p, q in zip(want, got))


def test_streams_workspaces_and_repeats(hip_ctx):
    import torch
    shape = (2, 3000, 2, 64)
    plan = _plan(hip_ctx, 2, 3000, 2, 1, 64, 64, "f16", True)
    q, dout = _tensor(1, shape, "f16"), _tensor(2, shape, "f16")
    k, v = _tensor(3, (2, 3000, 1, 64), "f16"), _tensor(4, (2, 3000, 1, 64), "f16")
    want = [torch.empty_like(x) for x in (dout, q, k, v)]
    plan.forward_tensors(q, k, v, want[0])
    plan.backward_tensors(q, k, v, dout, *want[1:])
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = [[torch.empty_like(x) for x in want] for _ in streams]
    work = [torch.empty(max(1, plan.workspace_bytes), device="cuda", dtype=torch.uint8) for _ in streams]
    torch.cuda.synchronize()
    for s, o, w in zip(streams, got, work):
        with torch.cuda.stream(s):
            plan.forward_tensors(q, k, v, o[0], work=w)
            plan.backward_tensors(q, k, v, dout, *o[1:], work=w)
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for o in got for x, y in zip(want, o))


def test_graph_replays(hip_ctx):
    import torch
    b, t, h, d = 1, 2050, 2, 64
    plan = _plan(hip_ctx, b, t, h, 1, d, d, "bf16", True)
    q, dout = _tensor(1, (b, t, h, d), "bf16"), _tensor(2, (b, t, h, d), "bf16")
    k, v = _tensor(3, (b, t, 1, d), "bf16"), _tensor(4, (b, t, 1, d), "bf16")
    state = _state(5, b, h, d, d)
    outs = [torch.empty_like(x) for x in (dout, state, q, k, v, state)]

    def step():
        plan.forward_tensors(q, k, v, outs[0], state_in=state, state_out=outs[1])
        plan.backward_tensors(q, k, v, dout, *outs[2:5], state_in=state, dstate_in=outs[5])
        plan.forward_tensors(q[:, :1], k[:, :1], v[:, :1], outs[0][:, :1], state_in=outs[1], state_out=outs[1])

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step()
    for seed in (11, 12, 13):
        q.copy_(_tensor(seed, (b, t, h, d), "bf16"))
        step()
        torch.cuda.synchronize()
        want = [o.clone() for o in outs]
        for o in outs:
            o.fill_(5)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(want, outs))


def test_refusals(hip_ctx):
    import torch

    def refused(kind, f, *a, **kw):
        with pytest.raises(vk.VkFftError) as e:
            f(*a, **kw)
        assert e.value.kind == kind, e.value

    def config(heads=2, dk=16, dv=16):
        return vk.LinearAttentionConfig.new(heads, dk, dv)

    for c in (config(0), config(2, 0), config(2, 257), config(2, 16, 257), config().with_kv_heads(0), config(3).with_kv_heads(2),
              config().with_decay([0.5, 1.5]), config().with_decay([0.5, -0.1]), config().with_decay([0.5, float("nan")]),
              config().with_scale(float("inf")), config().with_capacity(0, 1), config().with_capacity(1, 0), config().with_capacity(65536, 1)):
        refused("InvalidArgument", vk.LinearAttentionPlan, hip_ctx, c)
    refused("InputLengthMismatch", vk.LinearAttentionPlan, hip_ctx, config().with_decay([0.5]))

    plan = _plan(hip_ctx, 2, 8, 4, 2, 16, 24, "f32", True)
    q, k, v = (torch.zeros(2, 8, h, d, device="cuda") for h, d in ((4, 16), (2, 16), (2, 24)))
    out, st = torch.zeros(2, 8, 4, 24, device="cuda"), torch.zeros(2, 4, 16, 24, device="cuda")
    f = plan.forward_tensors
    refused("InvalidArgument", f, q.cpu(), k, v, out)
    refused("InvalidArgument", f, q, k.cpu(), v, out)
    refused("UnsupportedPrecision", f, q, k.half(), v, out)
    refused("InputLengthMismatch", f, q, k[:, :7], v, out)
    refused("InputLengthMismatch", f, q[0], k, v, out)
    refused("InputLengthMismatch", f, q, q, v, out)
    refused("InputLengthMismatch", f, q, k, v, out, state_in=st[:1])
    refused("UnsupportedPrecision", f, q, k, v, out, state_in=st.half())
    refused("InvalidArgument", f, q, k, v, out, state_in=st.transpose(0, 1).contiguous().transpose(0, 1))
    refused("UnsupportedPrecision", f, q, k, v, out, lengths=torch.zeros(2, device="cuda", dtype=torch.int64))
    refused("InputLengthMismatch", f, q, k, v, out, lengths=torch.zeros(3, device="cuda", dtype=torch.int32))
    refused("InvalidArgument", f, q, k, v, out[:, :, :1].expand(2, 8, 4, 24))
    refused("InvalidArgument", f, torch.zeros(2, 8, 16, 4, device="cuda").transpose(2, 3), k, v, out)
    wide = torch.zeros(2, 9, 4, 16, device="cuda")
    refused("InputLengthMismatch", f, wide, torch.zeros(2, 9, 2, 16, device="cuda"), torch.zeros(2, 9, 2, 24, device="cuda"),
            torch.zeros(2, 9, 4, 24, device="cuda"))
    same = _plan(hip_ctx, 2, 8, 4, 4, 16, 16, "f32", True)
    refused("InvalidArgument", same.forward_tensors, q, q, q, q)
    g = same.backward_tensors
    a, b, c = (torch.zeros_like(q) for _ in range(3))
    square = torch.zeros(2, 4, 16, 16, device="cuda")
    refused("InvalidArgument", g, q, q, q, q, q, b, c)
    refused("InvalidArgument", g, q, q, q, q, a, a, c)
    refused("InvalidArgument", g, q, q, q, q, a, b, c, dstate_out=square, dstate_in=square)
    refused("InvalidArgument", _plan(hip_ctx, 2, 8, 4, 4, 16, 16, "f32").backward_tensors, q, q, q, q, a, b, c)
    if plan.workspace_bytes:
        refused("InputLengthMismatch", f, q, k, v, out, work=torch.zeros(1, device="cuda"))


def test_plans_hold_their_context(hip_ctx):
    ctx = vk.HipExecutionContext(0)
    plan = _plan(ctx, 1, 1, 1, 1, 8, 8, "f32")
    assert ctx._L.vkfx_context_destroy(ctx.handle) == -2
    plan.close()
    ctx.close()


@pytest.mark.parametrize("lengths", [None, [4200, 700]])
def test_long_prompts_update_a_state_in_place(hip_ctx, lengths):
    """The tokens are split over blocks: none of them may read what another one has already written."""
    import torch
    b, t, h, d = 2, 4200, 2, 64
    plan = _plan(hip_ctx, b, t, h, h, d, d, "bf16", decay=[0.998, 0.9])
    q, k, v = (_tensor(i, (b, t, h, d), "bf16") for i in (1, 2, 3))
    n = torch.tensor(lengths, device="cuda", dtype=torch.int32) if lengths else None
    state, out, again = _state(4, b, h, d, d), torch.empty_like(v), torch.empty_like(v)
    after = torch.empty_like(state)
    plan.forward_tensors(q, k, v, out, state_in=state, state_out=after, lengths=n)
    plan.forward_tensors(q, k, v, again, state_in=state, state_out=state, lengths=n)
    assert torch.equal(out, again) and torch.equal(after, state)


@pytest.mark.parametrize("element", ELEMENTS)
@pytest.mark.parametrize("dk,dv", [(32, 32), (64, 100), (5, 6)])
def test_bad_values_do_not_reach_the_tokens_before(hip_ctx, element, dk, dv):
    """An infinity or a NaN in a token changes that token and later ones; backwards, keys and values of that token and earlier ones."""
    import torch
    t, at = 100, 43
    plan = _plan(hip_ctx, 1, t, 2, 2, dk, dv, element, True)
    x = [_tensor(i, (1, t, 2, d), element) for i, d in ((1, dk), (2, dk), (3, dv), (4, dv))]

    def run():
        o = [torch.full_like(x[i], 3) for i in (3, 0, 1, 2)]
        plan.forward_tensors(*x[:3], o[0])
        plan.backward_tensors(*x, *o[1:])
        return o

    want = run()
    for i, value in ((0, float("nan")), (1, float("inf")), (2, float("nan")), (2, float("inf")), (3, float("-inf"))):
        keep = x[i].clone()
        x[i][0, at, 0, 0] = value
        out, dq, dk_, dv_ = run()
        x[i].copy_(keep)
        forward, backward = i != 3, i in (0, 3)
        assert torch.equal(out[:, :at], want[0][:, :at])
        assert torch.equal(dq[:, :at], want[1][:, :at])
        assert torch.equal(out[:, :, 1], want[0][:, :, 1])
        if backward:  # q and dout enter the state's gradient from their token backwards
            assert torch.equal(dk_[:, at + 1:], want[2][:, at + 1:]) and torch.equal(dv_[:, at + 1:], want[3][:, at + 1:])
        if forward:
            assert not torch.isfinite(out[:, at, 0]).all()
        if not backward:
            assert torch.equal(dv_ if i == 2 else dk_, want[3 if i == 2 else 2])  # dv does not depend on v, dk not on k


def test_more_blocks_than_32_bits_count_threads(hip_ctx):
    """65535 heads of 300 sequences: more than 2^32 threads, one block a state."""
    import torch
    b, t, h = 300, 9, 65535
    plan = _plan(hip_ctx, b, t, h, 1, 1, 1, "f32", decay=[0.5] * h, scale=1.0)
    q, k, v = (_tensor(i, (b, t, 1, 1), "f32") for i in (1, 2, 3))
    out = torch.full((b, t, h, 1), float("nan"), device="cuda")
    state = torch.full((b, h, 1, 1), float("nan"), device="cuda")
    plan.forward_tensors(q.expand(b, t, h, 1), k, v, out, state_out=state)
    assert torch.equal(out, out[:, :, :1].expand_as(out)) and torch.equal(state, state[:, :1].expand_as(state))
    qn, kn, vn = _np(q, k, v)
    args = ([0.5], 1.0, np.full(b, t))
    zero = np.zeros((b, 1, 1, 1))
    want, total = ref.attention(qn, kn, vn, zero, *args), ref.attention(*map(np.abs, (qn, kn, vn, zero)), *args)
    ref.check("out", out[:, :, :1], want[0], total[0], "f32", ref.TERM["f32"])
    ref.check("state", state[:, :1], want[1], total[1], "f32", ref.STATE_TERM)


@pytest.mark.parametrize("element", ELEMENTS)
@pytest.mark.parametrize("decay", [0.99995, 0.999997])
def test_slow_decays_over_many_chunks(hip_ctx, element, decay):
    """With nothing added the states are powers of the decay alone, in the order of the tokens and backwards; enough
    heads that no sequence is split over its tokens."""
    import torch
    t, h, d = 16384, 520, 8
    plan = _plan(hip_ctx, 1, t, h, 1, d, d, element, True, decay=[decay] * h)
    one = lambda heads: torch.ones(1, 1, 1, d, device="cuda", dtype=_types()[element]).expand(1, t, heads, d)  # noqa: E731
    none = lambda heads: torch.zeros(1, 1, 1, d, device="cuda", dtype=_types()[element]).expand(1, t, heads, d)  # noqa: E731
    state = _state(1, 1, h, d, d).abs_()
    after = torch.empty_like(state)
    out = torch.empty(1, t, h, d, device="cuda", dtype=_types()[element])
    plan.forward_tensors(one(h), one(1), none(1), out, state_in=state, state_out=after)
    sn, = _np(state)
    want = decay ** t * sn
    ref.check("state", after, want, want, "f32", ref.STATE_TERM)
    for i in (0, 31, 32, t // 2, t - 1):
        want = np.float64(np.float32(d ** -0.5)) * decay ** (i + 1) * sn[0].sum(1)
        ref.check(f"out {i}", out[0, i], want, want, element, ref.TERM[element])
    back = torch.empty_like(state)
    dq = torch.empty_like(out)
    dk, dv = torch.empty(1, t, 1, d, device="cuda", dtype=out.dtype), torch.empty(1, t, 1, d, device="cuda", dtype=out.dtype)
    plan.backward_tensors(none(h), one(1), one(1), none(h), dq, dk, dv, state_in=state, dstate_out=state, dstate_in=back)
    want = decay ** t * sn
    ref.check("dstate_in", back, want, want, "f32", ref.STATE_TERM)
    for i in (0, 1, t // 2, t - 32, t - 1):
        power = decay ** (t - 1 - i)
        # dk sums 520 heads of 8 terms in 32 bits
        for name, got, axes in (("dk", dk, (0, 1, 3)), ("dv", dv, (0, 1, 2))):
            want = power * sn.sum(axes)
            ref.check(f"{name} {i}", got[0, i, 0], want, want, element, ref.TERM[element])


@pytest.mark.parametrize("element", ["f32", "bf16"])
def test_states_near_the_largest_number(hip_ctx, element):
    """States of 1e37 and their gradients, which 32 bits hold, over a prompt's chunks."""
    import torch
    b, t, h, d = 1, 96, 2, 32
    plan = _plan(hip_ctx, b, t, h, h, d, d, element, True, decay=[0.9, 0.99], scale=1.0)
    q, k, v, dout = (_tensor(i, (b, t, h, d), element).abs_() for i in range(4))
    k, v = (k * 1e18).to(q.dtype), (v * 1e18).to(q.dtype)
    q, dout = (q * 1e-2).to(q.dtype), (dout * 1e-2).to(q.dtype)
    out, state = torch.empty_like(v), torch.empty(b, h, d, d, device="cuda")
    plan.forward_tensors(q, k, v, out, state_out=state)
    qn, kn, vn, dn = _np(q, k, v, dout)
    zero = np.zeros((b, h, d, d))
    args = ([0.9, 0.99], 1.0, np.array([t]))
    want, want_state = ref.attention(qn, kn, vn, zero, *args)
    assert 1e36 < np.abs(want_state).max() < 3e38 and want.max() < 3e38
    ref.check("state", state, want_state, want_state, "f32", ref.STATE_TERM)
    ref.check("out", out, want, want, element, ref.TERM[element])
    dq, dk, dv = (torch.empty_like(x) for x in (q, k, v))
    plan.backward_tensors(q, k, v, dout, dq, dk, dv)
    wants = ref.attention_gradients(qn, kn, vn, zero, dn, zero, *args)
    for name, got, w in zip(("dq", "dk", "dv"), (dq, dk, dv), wants):
        ref.check(name, got, w, w, element, ref.TERM[element])


@pytest.mark.parametrize("dk", [5, 33, 64, 100, 128, 200])
@pytest.mark.parametrize("batch", [1, 40])
def test_an_infinite_state_row_gives_infinite_outputs_of_a_token(hip_ctx, dk, batch):
    """The state's last row, which the rows that pad a block must not meet with zeros."""
    import torch
    h, dv = 4, 24
    q, k, v = (_tensor(i, (batch, 1, h, d), "f32").abs_() + 0.1 for i, d in ((1, dk), (2, dk), (3, dv)))
    state = _state(4, batch, h, dk, dv)
    state[:, :, dk - 1, 3] = float("inf")
    state[:, 3, dk - 1, 5] = float("-inf")
    plan = _plan(hip_ctx, batch, 1, h, h, dk, dv, "f32", decay=[0.5, 0.9375, 0.998, 1.0])
    out = torch.empty(batch, 1, h, dv, device="cuda")
    plan.forward_tensors(q, k, v, out, state_in=state, state_out=state)
    assert torch.isposinf(out[:, 0, :, 3]).all() and torch.isneginf(out[:, 0, 3, 5]).all()
    out[:, :, :, 3] = 0
    out[:, :, 3, 5] = 0
    assert torch.isfinite(out).all()


@pytest.mark.parametrize("dk", [5, 33, 64, 100, 200])
@pytest.mark.parametrize("batch", [1, 40])
def test_an_infinite_value_of_a_token_gives_an_infinite_output(hip_ctx, dk, batch):
    """The same for the token itself: an infinity in v enters every row of the state's column, and no other column."""
    import torch
    h, dv = 4, 24
    q, k, v = (_tensor(i, (batch, 3, h, d), "f32").abs_() + 0.1 for i, d in ((1, dk), (2, dk), (3, dv)))
    v[:, 1, :, 3] = float("inf")
    plan = _plan(hip_ctx, batch, 3, h, h, dk, dv, "f32", decay=[0.5, 0.9375, 0.998, 1.0])
    out, state = torch.empty(batch, 3, h, dv, device="cuda"), torch.empty(batch, h, dk, dv, device="cuda")
    plan.forward_tensors(q, k, v, out, state_out=state)
    assert torch.isposinf(out[:, 1:, :, 3]).all() and torch.isposinf(state[:, :, :, 3]).all()
    out[:, 1:, :, 3] = 0
    state[:, :, :, 3] = 0
    assert torch.isfinite(out).all() and torch.isfinite(state).all()


def test_partial_overlaps_are_refused_and_packed_tensors_are_not(hip_ctx):
    import torch
    b, t, h, d = 2, 40, 4, 16
    plan = _plan(hip_ctx, b, t, h, h, d, d, "f32", True)
    n = b * t * h * d

    def at(flat, i):
        return flat[i:i + n].view(b, t, h, d)

    def refused(f, *a, **kw):
        with pytest.raises(vk.VkFftError) as e:
            f(*a, **kw)
        assert e.value.kind == "InvalidArgument" and "overlap" in str(e.value)

    flat = torch.zeros(9 * n, device="cuda")
    q, k, v, out = (at(flat, i * n) for i in range(4))
    states = torch.zeros(2 * b * h * d * d, device="cuda")
    size = b * h * d * d
    s, s2 = states[:size].view(b, h, d, d), states[d:size + d].view(b, h, d, d)
    f, g = plan.forward_tensors, plan.backward_tensors
    for i in range(3):
        refused(f, q, k, v, at(flat, i * n + 1 if i < 2 else 3 * n - 5))
    refused(f, q, k, v, at(flat, n // 2))
    refused(f, q, k, v, out, state_in=s, state_out=s2)
    refused(f, q, k, v, out, state_out=flat[4 * n - size:4 * n].view(b, h, d, d))
    refused(f, q, k, v, out, state_out=s, lengths=states[:b].view(torch.int32))
    dq, dk, dv = (at(flat, i * n) for i in (4, 5, 6))
    for i, name in enumerate((dq, dk, dv)):
        for j in (0, 1, 2, 3):
            moved = [dq, dk, dv]
            moved[i] = at(flat, j * n + 3)
            refused(g, q, k, v, out, *moved)
    refused(g, q, k, v, out, dq, at(flat, 5 * n - 1), dv)
    refused(g, q, k, v, out, dq, dk, dv, state_in=s, dstate_in=s2)
    refused(g, q, k, v, out, dq, dk, dv, dstate_out=s, dstate_in=s2)
    # views of one projection, and of one buffer for its gradients
    packed, grads = (torch.zeros(b, t, 3, h, d, device="cuda") for _ in range(2))
    packed.copy_(_tensor(1, (b, t, 3 * h, d), "f32").view(b, t, 3, h, d))
    dout = _tensor(2, (b, t, h, d), "f32")
    wide = torch.zeros(b, t, 2, h, d, device="cuda")  # out beside dout
    wide[:, :, 1] = dout
    f(*packed.unbind(2), wide[:, :, 0])
    g(*packed.unbind(2), wide[:, :, 1], *grads.unbind(2))
    want = [torch.empty(b, t, h, d, device="cuda") for _ in range(4)]
    apart = [x.contiguous() for x in packed.unbind(2)]
    f(*apart, want[0])
    g(*apart, dout, *want[1:])
    assert torch.equal(wide[:, :, 0], want[0])
    assert all(torch.equal(x, y) for x, y in zip(grads.unbind(2), want[1:]))


@pytest.mark.parametrize("element", ELEMENTS)
@pytest.mark.parametrize("dk,dv", [(64, 64), (100, 130), (130, 61), (200, 256), (256, 33)])
@pytest.mark.parametrize("t", [1, 5, 8])
def test_few_tokens_of_many_states(hip_ctx, element, dk, dv, t):
    """Enough states for blocks of 64 columns, whose gradients read their states transposed."""
    _run(hip_ctx, element, 8, t, 8, 8, dk, dv, lengths=[t, 0, 1, t, t // 2, t, t - 1, t])


@pytest.mark.parametrize("element", ELEMENTS)
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_bad_values_in_a_split_sequence(hip_ctx, element, value):
    """A token of a middle segment: what comes before it, the other heads and the other sequence stay as they are; the
    state after the last token, and backwards the gradient of the first state, do not."""
    import torch
    b, t, h, dk, dv, at = 2, 4200, 2, 64, 48, 2049
    plan = _plan(hip_ctx, b, t, h, h, dk, dv, element, True, decay=[0.998, 0.99])
    x = [_tensor(i, (b, t, h, d), element) for i, d in ((1, dk), (2, dk), (3, dv), (4, dv))]
    s, ds = _state(5, b, h, dk, dv), _state(6, b, h, dk, dv)

    def run():
        o = [torch.full_like(x[i], 3) for i in (3, 0, 1, 2)] + [torch.empty_like(s), torch.empty_like(s)]
        plan.forward_tensors(*x[:3], o[0], state_in=s, state_out=o[4])
        plan.backward_tensors(*x, *o[1:4], state_in=s, dstate_out=ds, dstate_in=o[5])
        return o

    want = run()
    assert all(torch.isfinite(o).all() for o in want)
    for i in range(4):
        keep = x[i].clone()
        x[i][0, at, 0, 7] = value
        out, dq, dk_, dv_, after, back = run()
        x[i].copy_(keep)
        for got, w in zip((out, dq, dk_, dv_, after, back), want):
            assert torch.equal(got[1], w[1])
        for got, w in zip((out, dq, dk_, dv_), want):
            assert torch.equal(got[0, :, 1], w[0, :, 1])
        for got, w in zip((after, back), want[4:]):
            assert torch.equal(got[0, 1], w[0, 1])
        assert torch.equal(out[0, :at], want[0][0, :at]) and torch.equal(dq[0, :at], want[1][0, :at])
        if i in (0, 3):  # q and dout reach the state's gradient alone
            assert torch.equal(dk_[0, at + 1:], want[2][0, at + 1:]) and torch.equal(dv_[0, at + 1:], want[3][0, at + 1:])
            assert torch.equal(after, want[4]) and not torch.isfinite(back[0, 0]).all()
        else:  # k and v reach the state alone, and the other one's gradient at their own token
            assert torch.equal(back, want[5]) and not torch.isfinite(after[0, 0]).all()
            same, other = ((dk_, want[2]), (dv_, want[3]))[::1 if i == 1 else -1]
            assert torch.equal(*same)
            rest = torch.arange(t, device="cuda") != at
            assert torch.equal(other[0][:, rest], other[1][:, rest])
            assert not torch.isfinite(other[0][0, at, 0]).all()


@pytest.mark.parametrize("element", ELEMENTS)
@pytest.mark.parametrize("dk,dv", [(32, 32), (64, 100), (5, 6)])
@pytest.mark.parametrize("sign", [1, -1])
def test_the_largest_numbers_do_not_reach_the_tokens_before(hip_ctx, element, dk, dv, sign):
    """The type's largest and lowest numbers in a token: not infinite, but near enough that a rounding makes them so."""
    import torch
    t, at = 100, 43
    plan = _plan(hip_ctx, 1, t, 2, 2, dk, dv, element, True)
    x = [_tensor(i, (1, t, 2, d), element) for i, d in ((1, dk), (2, dk), (3, dv), (4, dv))]
    value = sign * torch.finfo(x[0].dtype).max

    def run():
        o = [torch.full_like(x[i], 3) for i in (3, 0, 1, 2)]
        plan.forward_tensors(*x[:3], o[0])
        plan.backward_tensors(*x, *o[1:])
        return o

    want = run()
    for i in range(4):
        keep = x[i].clone()
        x[i][0, at, 0, 0] = value
        out, dq, dk_, dv_ = run()
        x[i].copy_(keep)
        for got, w in zip((out, dq, dk_, dv_), want):
            assert torch.equal(got[:, :, 1], w[:, :, 1])
        assert torch.equal(out[:, :at], want[0][:, :at]) and torch.equal(dq[:, :at], want[1][:, :at])
        if i in (0, 3):
            assert torch.equal(dk_[:, at + 1:], want[2][:, at + 1:]) and torch.equal(dv_[:, at + 1:], want[3][:, at + 1:])
        else:
            same, other = ((dk_, want[2]), (dv_, want[3]))[::1 if i == 1 else -1]
            assert torch.equal(*same)
            rest = torch.arange(t, device="cuda") != at
            assert torch.equal(other[0][:, rest], other[1][:, rest])
