"""The gated recurrence and its gradients against the definition in 64 bits."""
import numpy as np
import pytest

import mixer_reference as ref
import vkfft_amd as vk

pytestmark = pytest.mark.gpu

ELEMENT = {"f32": vk.Element.F32, "f16": vk.Element.F16, "bf16": vk.Element.BF16}
ELEMENTS = list(ELEMENT)
GATES = {"sigmoid": vk.Gate.Sigmoid, "exp": vk.Gate.Exp}


def _types():
    import torch
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _plan(ctx, channels, element, gate="sigmoid", complement=True):
    return vk.GatedRecurrencePlan(ctx, vk.GatedRecurrenceConfig.new(channels).with_element(ELEMENT[element]).with_gate(GATES[gate])
                                  .with_complement(complement))


def _tensor(seed, shape, element, layout="btc", pad=0, offset=0, scale=1.0):
    """Normal numbers, the last dimension padded, `offset` elements into an allocation of NaN."""
    import torch
    b, t, c = shape
    order = (b, t) if layout == "btc" else (t, b)
    flat = torch.full((offset + b * t * (c + pad) + 8,), float("nan"), device="cuda", dtype=_types()[element])
    x = flat[offset:offset + b * t * (c + pad)].view(*order, c + pad)[..., :c]
    g = torch.Generator(device="cuda").manual_seed(seed)
    x.copy_(torch.randn(*order, c, generator=g, device="cuda") * scale)
    return x if layout == "btc" else x.transpose(0, 1)


def _gate(seed, shape, element, gate, slow=6.0, **kw):
    """Logits of memories of 2 to e^slow tokens over the channels, or logarithms of such decays."""
    import torch
    x = _tensor(seed, shape, "f32", **kw) + torch.linspace(0.5, slow, shape[2], device="cuda")
    y = _tensor(seed, shape, element, **kw)
    y.copy_(x if gate == "sigmoid" else -torch.exp(-x))
    return y


def _state(seed, *shape):
    import torch
    return torch.randn(shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


def _np(*xs):
    out = [x.double().cpu().numpy() for x in xs]
    return out[0] if len(out) == 1 else out


def _check(ctx, element, x, gate, dy, states=True, lengths=None, kind="sigmoid", complement=True, in_place=False, gradient=True, like=None):
    """Runs both passes on the given tensors and compares all that they give."""
    import torch
    b, t, c = x.shape
    plan = _plan(ctx, c, element, kind, complement)
    s0, ds = (_state(21, b, c), _state(22, b, c)) if states else (None, None)
    n = np.full(b, t) if lengths is None else np.clip(np.asarray(lengths), 0, t)
    ln = None if lengths is None else torch.tensor(lengths, device="cuda", dtype=torch.int32)
    xn, gn, dyn = _np(x, gate, dy)
    zero = np.zeros((b, c))
    y, ye, h, e, before = ref.recurrence(xn, gn, _np(s0) if states else zero, n, kind == "sigmoid", complement)
    like = like or (lambda z: torch.full_like(z, 7))
    kept = x.clone()
    yt = x if in_place else like(x)
    so, saved = torch.full((b, c), float("nan"), device="cuda"), torch.full(plan.saved_shape(b, t), float("nan"), device="cuda")
    plan.forward_tensors(x, gate, yt, state_in=s0, state_out=so, saved=saved, lengths=ln)
    ref.check_bound("y", yt, y, ye, element)
    ref.check_bound("state", so, h, e, "f32")
    if not gradient:
        return yt
    dx, dg = dy if in_place else like(dy), like(gate)
    ds0 = torch.full((b, c), float("nan"), device="cuda")
    plan.backward_tensors(kept, gate, saved, dy, dx, dg, dstate_out=ds, dstate_in=ds0, lengths=ln)
    wants = ref.recurrence_gradients(xn, gn, before, dyn, _np(ds) if states else zero, n, kind == "sigmoid", complement)
    for i, (name, got, el) in enumerate((("dx", dx, element), ("dgate", dg, element), ("dstate", ds0, "f32"))):
        ref.check_bound(name, got, wants[2 * i], wants[2 * i + 1], el)
    return yt, dx, dg


def _run(ctx, element, b, t, c, kind="sigmoid", complement=True, slow=6.0, layout="btc", pad=0, offset=0, **kw):
    tensor = lambda seed: _tensor(seed, (b, t, c), element, layout, pad, offset)  # noqa: E731
    gate = _gate(2, (b, t, c), element, kind, slow, layout=layout, pad=pad, offset=offset)
    return _check(ctx, element, tensor(1), gate, tensor(3), kind=kind, complement=complement, **kw)


@pytest.mark.parametrize("element", ELEMENTS)
@pytest.mark.parametrize("kind", list(GATES))
@pytest.mark.parametrize("complement", [False, True])
@pytest.mark.parametrize("t", [1, 2, 3, 8, 15, 16, 17, 31, 33, 64, 100, 127, 128, 129, 255, 256, 257, 700])
def test_lengths_of_time(hip_ctx, element, kind, complement, t):
    _run(hip_ctx, element, 2, t, 70, kind, complement)


@pytest.mark.parametrize("element", ELEMENTS)
@pytest.mark.parametrize("c", [1, 2, 3, 31, 63, 64, 65, 127, 128, 129, 255, 257, 1000, 1001, 4099])
def test_channels(hip_ctx, element, c):
    _run(hip_ctx, element, 3, 37, c)


@pytest.mark.parametrize("element", ELEMENTS)
@pytest.mark.parametrize("b,t,c", [(1, 5000, 64), (1, 9011, 33), (2, 3000, 130), (1, 1500, 1000), (5, 2049, 7)])
def test_long_sequences_of_few_channels(hip_ctx, element, b, t, c):
    _run(hip_ctx, element, b, t, c)


@pytest.mark.parametrize("element", ELEMENTS)
@pytest.mark.parametrize("b,t,c", [(64, 20, 4096), (300, 17, 520), (9, 100, 2050)])
def test_many_channels(hip_ctx, element, b, t, c):
    _run(hip_ctx, element, b, t, c)


@pytest.mark.parametrize("element", ELEMENTS)
@pytest.mark.parametrize("kind", list(GATES))
@pytest.mark.parametrize("t,lengths", [(5, [0, 1, 5, 3]), (1, [0, 1, 1, 0]), (130, [130, 0, 64, 65]), (300, [1, -4, 999, 255]),
                                       (3000, [3000, 0, 1333, 16])])
def test_uneven_lengths(hip_ctx, element, kind, t, lengths):
    _run(hip_ctx, element, 4, t, 50, kind, lengths=lengths)


@pytest.mark.parametrize("element", ELEMENTS)
@pytest.mark.parametrize("layout,pad,offset", [("tbc", 0, 0), ("btc", 8, 0), ("tbc", 3, 1), ("btc", 1, 5)])
@pytest.mark.parametrize("t", [1, 40, 2500])
def test_layouts(hip_ctx, element, layout, pad, offset, t):
    import torch
    made = []

    def like(z):
        made.append(_tensor(9, (2, t, 35), element, layout, pad, offset))
        made[-1].fill_(7)
        return made[-1]

    _run(hip_ctx, element, 2, t, 35, layout=layout, pad=pad, offset=offset, like=like)
    for z in made:  # what lies between the rows stays as it was
        z0 = z if layout == "btc" else z.transpose(0, 1)
        if pad and t > 1:
            assert torch.isnan(z0.as_strided((2 * t - 1, pad), (35 + pad, 1), z0.storage_offset() + 35)).all()


@pytest.mark.parametrize("element", ELEMENTS)
@pytest.mark.parametrize("t", [1, 50, 2500])
def test_without_states(hip_ctx, element, t):
    _run(hip_ctx, element, 2, t, 40, states=False)


@pytest.mark.parametrize("element", ELEMENTS)
@pytest.mark.parametrize("b,t,c", [(2, 1, 40), (2, 50, 40), (1, 3000, 40), (40, 45, 4096)])
def test_in_place(hip_ctx, element, b, t, c):
    _run(hip_ctx, element, b, t, c, in_place=True, lengths=[t - i % t for i in range(b)])


@pytest.mark.parametrize("kind", list(GATES))
@pytest.mark.parametrize("complement", [False, True])
@pytest.mark.parametrize("t", [40, 3000])
def test_gates_at_the_ends(hip_ctx, kind, complement, t):
    """Gates that forget all, keep all, or nearly so: infinities, the largest numbers, zeros and the smallest."""
    import torch
    ends = [float("-inf"), -3e38, -200.0, -88.0, -1.0, -0.6931472, -0.5, -1e-3, -1e-7, -1e-30, -1e-45, -0.0, 0.0, 1e-30, 1e-3, 1.0, 20.0, 90.0, 3e38,
            float("inf")]
    c = len(ends) * 2
    # half of the channels keep one gate, the others change theirs
    fixed = torch.tensor(ends, device="cuda").expand(2, t, len(ends))
    at = torch.randint(0, len(ends), (2, t, len(ends)), device="cuda", generator=torch.Generator(device="cuda").manual_seed(4))
    gate = torch.cat([fixed, torch.tensor(ends, device="cuda")[at]], 2)
    _check(hip_ctx, "f32", _tensor(1, (2, t, c), "f32"), gate, _tensor(3, (2, t, c), "f32"), kind=kind, complement=complement)


@pytest.mark.parametrize("element", ELEMENTS)
@pytest.mark.parametrize("kind", list(GATES))
def test_slow_decays_do_not_drift(hip_ctx, element, kind):
    """Memories of a thousand to a million tokens, each channel's gate the same at every token."""
    import torch
    t, c = 20000, 12
    logits = torch.linspace(7.0, 14.0, c, device="cuda").expand(1, t, c)
    gate = (logits if kind == "sigmoid" else -torch.exp(-logits)).to(_types()[element]).contiguous()
    x = torch.zeros(1, t, c, device="cuda", dtype=_types()[element])
    plan = _plan(hip_ctx, c, element, kind)
    s = torch.full((1, c), 1.0, device="cuda")
    plan.forward_tensors(x, gate, torch.empty_like(x), state_in=s, state_out=s)
    a = ref.gates(_np(gate)[0, 0], kind == "sigmoid", True)
    want = np.exp(t * np.log1p(-a[1]))
    # the decay's own error, 2^-21 of 1 - a at each of t tokens, and the state's rounding, 2^-24 at each, all to one side
    assert (np.abs(_np(s)[0] - want) <= want * (t * a[1] * 2.0 ** -21 + t * 2.0 ** -24)).all()


def test_a_reset_forgets_the_sequence_before(hip_ctx):
    """Documents packed one after the other: a gate of -inf at the first token of each."""
    import torch
    for kind in GATES:
        plan = _plan(hip_ctx, 50, "bf16", kind)
        x, gate = _tensor(1, (1, 900, 50), "bf16"), _gate(2, (1, 900, 50), "bf16", kind)
        gate[:, 300] = float("-inf")
        y, z = torch.empty_like(x), torch.empty_like(x[:, 300:])
        plan.forward_tensors(x, gate, y)
        plan.forward_tensors(x[:, 300:], gate[:, 300:], z)
        # the same sums in another order: a step of the output's type
        assert (y[:, 300:].float() - z.float()).abs().max() <= 2.0 ** -8 * z.abs().max().float()
        x[:, :300] = 1e30
        plan.forward_tensors(x, gate, y)
        assert (y[:, 300:].float() - z.float()).abs().max() <= 2.0 ** -8 * z.abs().max().float()


@pytest.mark.parametrize("element", ELEMENTS)
@pytest.mark.parametrize("b,t,prompt", [(3, 60, 41), (1, 5010, 5000)])
def test_token_by_token_gives_the_prompts_outputs(hip_ctx, element, b, t, prompt):
    import torch
    c = 48
    plan = _plan(hip_ctx, c, element)
    x, gate = _tensor(1, (b, t, c), element), _gate(2, (b, t, c), element, "sigmoid")
    s = _state(3, b, c)
    want, ye, h, e, _ = ref.recurrence(*_np(x, gate, s), np.full(b, t), True, True)
    parts = [slice(0, prompt)] + [slice(i, i + 1) for i in range(prompt, t - 4)] + [slice(t - 4, t)]
    y = torch.empty_like(x)
    for p in parts:
        plan.forward_tensors(x[:, p], gate[:, p], y[:, p], state_in=s, state_out=s)
    ref.check_bound("y", y, want, ye, element)
    ref.check_bound("state", s, h, e, "f32")


def test_a_constant_gate_is_an_exponential_filter(hip_ctx):
    """What a zero-padded convolution plan gives with the taps a^t."""
    import torch
    t, c, n, a = 300, 3, 1024, 0.9375
    plan = _plan(hip_ctx, c, "f32", "exp", False)
    x = _tensor(1, (1, t, c), "f32")
    y = torch.empty_like(x)
    plan.forward_tensors(x, torch.full_like(x, float(np.log(a))), y)
    taps = np.zeros(n)
    taps[:t] = a ** np.arange(t)
    rows = np.zeros((c, n), np.complex64)
    rows[:, :t] = x[0].T.cpu().numpy()
    config = vk.FftConfig.new([n]).with_batch_count(c).with_convolution(True)
    z = hip_ctx.execute_convolution(vk.ConvolutionIr.build(config, np.fft.fft(taps).astype(np.complex64)), rows)
    z = z.reshape(c, n)[:, :t].real.T
    assert np.abs(y[0].cpu().numpy() - z).max() <= 1e-5 * np.abs(z).max()


@pytest.mark.parametrize("kind", list(GATES))
@pytest.mark.parametrize("complement", [False, True])
def test_gradients_against_differences(hip_ctx, kind, complement):
    """d(<y, dy> + <state, dstate>) along a direction of x, gate and state, by central differences in 64 bits."""
    import torch
    b, t, c = 2, 37, 9
    plan = _plan(hip_ctx, c, "f32", kind, complement)
    x, gate, dy = _tensor(1, (b, t, c), "f32"), _gate(2, (b, t, c), "f32", kind, 3.0), _tensor(3, (b, t, c), "f32")
    s, ds = _state(4, b, c), _state(5, b, c)
    y, saved = torch.empty_like(x), torch.empty(plan.saved_shape(b, t), device="cuda")
    got = [torch.empty_like(v) for v in (x, gate, s)]
    plan.forward_tensors(x, gate, y, state_in=s, saved=saved)
    plan.backward_tensors(x, gate, saved, dy, got[0], got[1], dstate_out=ds, dstate_in=got[2])

    def f(*v):
        y, _, h, _, _ = ref.recurrence(*v, np.full(b, t), kind == "sigmoid", complement)
        return (y * _np(dy)).sum() + (h * _np(ds)).sum()

    at, rng = _np(x, gate, s), np.random.default_rng(5)
    for i, g in enumerate(got):
        v = rng.standard_normal(at[i].shape)
        up, down = list(at), list(at)
        up[i], down[i] = at[i] + 1e-5 * v, at[i] - 1e-5 * v
        slope = (f(*up) - f(*down)) / 2e-5
        # 32-bit gradients: c of their largest size times the direction's; the difference's own error is 1e-9 of it
        assert abs((_np(g) * v).sum() - slope) <= 2.0 ** -16 * (np.abs(_np(g)) * np.abs(v)).sum()


def test_no_tokens_and_no_sequences(hip_ctx):
    import torch
    plan = _plan(hip_ctx, 5, "bf16")
    e = torch.empty(3, 0, 5, device="cuda", dtype=torch.bfloat16)
    s = _state(1, 3, 5)
    o = torch.full_like(s, 7)
    plan.forward_tensors(e, e, e.clone(), state_in=s, state_out=o)
    assert torch.equal(s, o)
    plan.forward_tensors(e, e, e.clone(), state_out=o)
    assert not o.any()
    saved = torch.empty(plan.saved_shape(3, 0), device="cuda")
    plan.backward_tensors(e, e, saved, e.clone(), e.clone(), e.clone(), dstate_out=s, dstate_in=o)
    assert torch.equal(s, o)
    e = torch.empty(0, 4, 5, device="cuda", dtype=torch.bfloat16)
    plan.forward_tensors(e, e, e.clone())


def test_broadcast_inputs(hip_ctx):
    """One sequence's gates for all, one gate for all tokens, and a gradient of one row."""
    import torch
    for t in (70, 5000):
        x, dy = _tensor(1, (3, t, 40), "f32"), _tensor(2, (3, 1, 40), "f32").expand(3, t, 40)
        plan = _plan(hip_ctx, 40, "f32")
        for g in (_gate(3, (1, t, 40), "f32", "sigmoid").expand(3, t, 40), _gate(3, (1, 1, 40), "f32", "sigmoid").expand(3, t, 40)):
            outs = []
            for gate, d in ((g, dy), (g.contiguous(), dy.contiguous())):
                o = [torch.empty_like(x) for _ in range(3)]
                saved = torch.empty(plan.saved_shape(3, t), device="cuda")
                plan.forward_tensors(x, gate, o[0], saved=saved)
                plan.backward_tensors(x, gate, saved, d, o[1], o[2])
                outs.append(o + [saved])
            assert all(torch.equal(p, q) for p, q in zip(*outs))


def test_offsets_past_32_bits(hip_ctx):
    import torch
    far = torch.zeros((1 << 32) + (1 << 21), device="cuda", dtype=torch.bfloat16)
    for t, c in ((96, 70), (5000, 33)):
        step = (1 << 32) // (t - 1) // 64 * 64 + 64
        x = [far.as_strided((1, t, c), (far.numel(), step, 1), 128 * i) for i in range(6)]
        near = [_tensor(i, (1, t, c), "bf16") for i in range(6)]
        for f, n in zip(x[:3], near):
            f.copy_(n)
        plan = _plan(hip_ctx, c, "bf16")
        saved = torch.empty(plan.saved_shape(1, t), device="cuda")
        for v in (x, near):
            plan.forward_tensors(v[0], v[1], v[3], saved=saved)
            plan.backward_tensors(v[0], v[1], saved, v[2], v[4], v[5])
        assert all(torch.equal(f, n) for f, n in zip(x[3:], near[3:]))


@pytest.mark.parametrize("t", [100, 6000])
@pytest.mark.parametrize("where", ["past the length", "another sequence", "another channel", "later tokens"])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), 3e38])
def test_bad_values_stay_where_they_belong(hip_ctx, t, where, value):
    import torch
    plan = _plan(hip_ctx, 70, "bf16")
    x, gate, dy = _tensor(1, (2, t, 70), "bf16"), _gate(2, (2, t, 70), "bf16", "sigmoid"), _tensor(3, (2, t, 70), "bf16")
    m = t * 2 // 5
    n = torch.tensor([m, t], device="cuda", dtype=torch.int32)
    saved = torch.empty(plan.saved_shape(2, t), device="cuda")

    def run():
        o = [torch.full_like(x, 3) for _ in range(3)] + [torch.empty(2, 70, device="cuda") for _ in range(2)]
        plan.forward_tensors(x, gate, o[0], state_out=o[3], saved=saved, lengths=n)
        plan.backward_tensors(x, gate, saved, dy, o[1], o[2], dstate_in=o[4], lengths=n)
        return o

    want = run()
    for y in (x, gate, dy):
        if where == "past the length":
            y[0, m:] = value
        elif where == "another sequence":
            y[1, 50] = value
        elif where == "another channel":
            y[0, 20, 9] = value
        elif y is not dy:
            y[0, m // 2] = value
    got = run()
    if where == "later tokens":
        assert torch.equal(want[0][0, :m // 2], got[0][0, :m // 2])
        return
    if where == "another channel":
        for p, q in zip(want, got):
            p[..., 9], q[..., 9] = 0, 0
    assert all(torch.equal(p[:1], q[:1]) for p, q in zip(want, got))


@pytest.mark.parametrize("t", [1, 40, 6000])
def test_an_infinite_state_stays_in_its_channel(hip_ctx, t):
    import torch
    plan = _plan(hip_ctx, 20, "f32")
    x, gate = _tensor(1, (1, t, 20), "f32"), _gate(2, (1, t, 20), "f32", "sigmoid")
    s = _state(3, 1, 20)
    y, z, o = torch.empty_like(x), torch.empty_like(x), torch.empty_like(s)
    plan.forward_tensors(x, gate, y, state_in=s)
    s[0, 7] = float("inf")
    plan.forward_tensors(x, gate, z, state_in=s, state_out=o)
    assert not torch.isfinite(z[0, 0, 7])
    y[..., 7], z[..., 7] = 0, 0
    assert torch.equal(y, z)
    plan.forward_tensors(x, gate, z, state_in=s, state_out=o, lengths=torch.zeros(1, device="cuda", dtype=torch.int32))
    assert torch.equal(s, o)  # past the length a state stays as it is


@pytest.mark.parametrize("t,lengths", [(700, None), (9000, [9000, 3000])])
def test_streams_workspaces_and_repeats(hip_ctx, t, lengths):
    import torch
    plan = _plan(hip_ctx, 90, "f16")
    x, gate, dy = _tensor(1, (2, t, 90), "f16"), _gate(2, (2, t, 90), "f16", "sigmoid"), _tensor(3, (2, t, 90), "f16")
    n = None if lengths is None else torch.tensor(lengths, device="cuda", dtype=torch.int32)

    def make():
        return [torch.empty_like(x) for _ in range(3)] + [torch.empty(2, 90, device="cuda") for _ in range(2)] \
            + [torch.full(plan.saved_shape(2, t), 7.0, device="cuda")]

    def run(o, **kw):
        plan.forward_tensors(x, gate, o[0], state_out=o[3], saved=o[5], lengths=n, **kw)
        plan.backward_tensors(x, gate, o[5], dy, o[1], o[2], dstate_in=o[4], lengths=n, **kw)

    want = make()
    run(want)
    torch.cuda.synchronize()
    for i, m in enumerate(lengths or []):  # saved states end with their sequence
        assert (want[5][i, -(-m // plan.SPAN):] == 7).all()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = [make() for _ in streams]
    work = [torch.empty(max(1, plan.workspace_bytes), device="cuda", dtype=torch.uint8) for _ in streams]
    torch.cuda.synchronize()
    for s, o, w in zip(streams, got, work):
        with torch.cuda.stream(s):
            run(o, work=w)
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for o in got for x, y in zip(want, o))


@pytest.mark.parametrize("t", [60, 9000])
def test_graph_replays(hip_ctx, t):
    import torch
    plan = _plan(hip_ctx, 50, "bf16")
    x, gate = _tensor(1, (1, t, 50), "bf16"), _gate(2, (1, t, 50), "bf16", "sigmoid")
    s = _state(3, 1, 50)
    outs = [torch.empty_like(x) for _ in range(3)] + [torch.empty_like(s) for _ in range(2)] + [torch.empty(plan.saved_shape(1, t), device="cuda")]

    def step():
        plan.forward_tensors(x, gate, outs[0], state_in=s, state_out=outs[3], saved=outs[5])
        plan.backward_tensors(x, gate, outs[5], outs[0], outs[1], outs[2], dstate_out=outs[3], dstate_in=outs[4])

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step()
    for seed in (11, 12, 13):
        x.copy_(_tensor(seed, x.shape, "bf16"))
        s.add_(1)
        step()
        torch.cuda.synchronize()
        want = [o.clone() for o in outs]
        for o in outs:
            o.fill_(5)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(want, outs))


def test_refusals(hip_ctx):
    import torch

    def refused(kind, f, *a, **kw):
        with pytest.raises(vk.VkFftError) as e:
            f(*a, **kw)
        assert e.value.kind == kind, e.value

    for n in (0, 1 << 31):
        refused("InvalidArgument", vk.GatedRecurrencePlan, hip_ctx, vk.GatedRecurrenceConfig.new(n))
    plan = _plan(hip_ctx, 16, "f32")
    x, g, y = (torch.zeros(2, 40, 16, device="cuda") for _ in range(3))
    s, saved = torch.zeros(2, 16, device="cuda"), torch.zeros(plan.saved_shape(2, 40), device="cuda")
    n = torch.zeros(2, device="cuda", dtype=torch.int32)
    f, back = plan.forward_tensors, plan.backward_tensors
    refused("InvalidArgument", f, x.cpu(), g, y)
    refused("InvalidArgument", f, x, g.cpu(), y)
    refused("InvalidArgument", f, x, None, y)
    refused("InvalidArgument", f, x, g, y, state_in=s.cpu())
    refused("InputLengthMismatch", f, x[0], g, y)
    refused("InputLengthMismatch", f, x, g[:, :39], y)
    refused("InputLengthMismatch", f, x, g, y, state_in=s[:1])
    refused("InputLengthMismatch", f, x, g, y, saved=saved[:, :2])
    refused("InputLengthMismatch", f, x, g, y, lengths=n[:1])
    refused("InputLengthMismatch", f, x, g, y, work=torch.zeros(0, device="cuda"))
    refused("InvalidArgument", f, x, g, y, work=torch.zeros(plan.workspace_bytes + 16, device="cuda", dtype=torch.uint8)[1:])
    refused("UnsupportedPrecision", f, x.half(), g, y)
    refused("UnsupportedPrecision", f, x, g.half(), y)
    refused("UnsupportedPrecision", f, x, g, y, lengths=n.long())
    refused("UnsupportedPrecision", f, x, g, y, state_out=s.double())
    refused("InvalidArgument", f, x, g, torch.zeros(2, 16, 40, device="cuda").transpose(1, 2))
    refused("InvalidArgument", f, x, g, torch.zeros(1, 40, 16, device="cuda").expand(2, 40, 16))
    refused("InvalidArgument", f, x, g, g)
    refused("InvalidArgument", f, x, g, x.view(-1).as_strided((2, 40, 16), (16, 32, 1)))
    refused("InvalidArgument", f, x, g, y, state_out=y.view(-1)[:32].view(2, 16))
    refused("InvalidArgument", f, x, g, y, state_out=s, lengths=s.view(-1)[:2].view(torch.int32))
    flat = torch.zeros(4000, device="cuda")
    refused("InvalidArgument", f, flat[:1280].view(2, 40, 16), g, flat[16:1296].view(2, 40, 16))
    refused("InvalidArgument", back, x, g, None, y, torch.zeros_like(x), torch.zeros_like(x))
    refused("InvalidArgument", back, x, g, saved, y, x, torch.zeros_like(x))
    refused("InvalidArgument", back, x, g, saved, y, y, y)
    refused("InvalidArgument", back, x, g, saved, y, torch.zeros_like(x), g)
    refused("InputLengthMismatch", back, x, g, saved[:, :1], y, torch.zeros_like(x), torch.zeros_like(x))
    big = torch.zeros(1, 1, 16, device="cuda")
    refused("ResourceLimitExceeded", f, big.expand(70000, 1, 16), big.expand(70000, 1, 16), torch.zeros(70000, 1, 16, device="cuda"))


def test_plans_hold_their_context(hip_ctx):
    ctx = vk.HipExecutionContext(0)
    plan = _plan(ctx, 8, "f32")
    assert ctx._L.vkfx_context_destroy(ctx.handle) == -2
    plan.close()
    ctx.close()


@pytest.mark.parametrize("lengths", [None, [5300]])
def test_many_long_chains_take_several_launches(hip_ctx, lengths):
    """More tokens of more channels than one launch's workspace holds; a part of the channels alone takes one."""
    import torch
    t, c, part = 5400, 20000, 640
    plan, alone = _plan(hip_ctx, c, "bf16"), _plan(hip_ctx, part, "bf16")
    x, gate, dy = _tensor(1, (1, t, c), "bf16"), _gate(2, (1, t, c), "bf16", "sigmoid"), _tensor(3, (1, t, c), "bf16")
    s, ds = _state(4, 1, c), _state(5, 1, c)
    n = None if lengths is None else torch.tensor(lengths, device="cuda", dtype=torch.int32)
    outs = []
    for p, at in ((plan, slice(0, c)), (alone, slice(c - part, c))):
        v = [z[..., at] for z in (x, gate, dy)]
        o = [torch.full(v[0].shape, 7, device="cuda", dtype=torch.bfloat16) for _ in range(3)]
        states = [s[:, at].clone(), ds[:, at].clone()]
        saved = torch.empty(p.saved_shape(1, t), device="cuda")
        p.forward_tensors(v[0], v[1], o[0], state_in=states[0], state_out=states[0], saved=saved, lengths=n)
        p.backward_tensors(v[0], v[1], saved, v[2], o[1], o[2], dstate_out=states[1], dstate_in=states[1], lengths=n)
        outs.append([z[..., -part:] for z in o + states])
    for name, a, b in zip(("y", "dx", "dgate", "state", "dstate"), *outs):
        # The same sums joined in other places, about 2^-20 of them apart; where a 16-bit rounding falls between, each is
        # half a step, 2^-8, from it, on two sides: 2^-7 apart. Few of them are.
        step = 2.0 ** -7 if a.dtype is torch.bfloat16 else 2.0 ** -18
        far = (a.double() - b.double()).abs()
        over = (far - step * b.double().abs() - 2.0 ** -18 * b.double().abs().max()).max().item()
        assert over <= 0, (name, over)
        if a.dtype is torch.bfloat16:
            assert (far > 0).double().mean().item() <= 2.0 ** -6, name


def test_calls_side_by_side_on_streams_of_chains_and_others(hip_ctx):
    """Chains wait for their own blocks only: several calls' chains share the machine, beside calls that fill it."""
    import torch
    plan, wide = _plan(hip_ctx, 100, "bf16"), _plan(hip_ctx, 8192, "bf16")
    x, gate = _tensor(1, (1, 20000, 100), "bf16"), _gate(2, (1, 20000, 100), "bf16", "sigmoid")
    xw, gw = _tensor(3, (8, 300, 8192), "bf16"), _gate(4, (8, 300, 8192), "bf16", "sigmoid")
    want, want_wide = torch.empty_like(x), torch.empty_like(xw)
    plan.forward_tensors(x, gate, want)
    wide.forward_tensors(xw, gw, want_wide)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(6)]
    got = [torch.empty_like(x) for _ in streams]
    got_wide = [torch.empty_like(xw) for _ in streams]
    work = [torch.empty(plan.workspace_bytes, device="cuda", dtype=torch.uint8) for _ in streams]
    torch.cuda.synchronize()
    for _ in range(3):
        for s, o, ow, w in zip(streams, got, got_wide, work):
            with torch.cuda.stream(s):
                plan.forward_tensors(x, gate, o, work=w)
                wide.forward_tensors(xw, gw, ow, work=w)
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in got) and all(torch.equal(o, want_wide) for o in got_wide)


# Blocks of 64 words of channels go along their sequences where there are enough for three quarters of the 256 CUs, 8 waves
# of 16 tokens at a time.
WIDE = [(6, 4096, "f16"), (6, 4098, "bf16"), (3, 4099, "f32"), (3, 4099, "bf16")]


@pytest.mark.parametrize("b,c,element", WIDE)
@pytest.mark.parametrize("t,kind,complement", [(129, "exp", False), (256, "sigmoid", True), (257, "exp", True), (385, "sigmoid", False)])
def test_wide_sequences_of_several_tiles(hip_ctx, b, c, element, t, kind, complement):
    _run(hip_ctx, element, b, t, c, kind, complement)


@pytest.mark.parametrize("b,c,element", WIDE)
def test_wide_sequences_of_uneven_lengths(hip_ctx, b, c, element):
    """Lengths that end in the first, a middle and the last tile, at their ends and with none; in place, and strided."""
    _run(hip_ctx, element, b, 270, c, in_place=True, lengths=[270, 5, 256, 0, 200, 129, 128, 17][:b])
    _run(hip_ctx, element, b, 260, c, "exp", lengths=[140, 260, 257, 999, -1, 127, 16, 258][:b], layout="tbc", pad=2, offset=2)


@pytest.mark.parametrize("b,c,element", WIDE)
def test_wide_sequences_keep_their_states_in_one_buffer(hip_ctx, b, c, element):
    """state_out that is state_in, dstate_in that is dstate_out, and a prompt in two calls."""
    import torch
    t, cut = 300, 140
    plan = _plan(hip_ctx, c, element)
    x, gate, dy = _tensor(1, (b, t, c), element), _gate(2, (b, t, c), element, "sigmoid"), _tensor(3, (b, t, c), element)
    s0, ds0 = _state(4, b, c), _state(5, b, c)
    outs = []
    for shared in (False, True):
        s, ds = s0.clone(), ds0.clone()
        so, dso = (s, ds) if shared else (torch.empty_like(s), torch.empty_like(ds))
        o, saved = [torch.empty_like(x) for _ in range(3)], torch.empty(plan.saved_shape(b, t), device="cuda")
        plan.forward_tensors(x, gate, o[0], state_in=s, state_out=so, saved=saved)
        plan.backward_tensors(x, gate, saved, dy, o[1], o[2], dstate_out=ds, dstate_in=dso)
        outs.append(o + [so, dso])
    assert all(torch.equal(p, q) for p, q in zip(*outs))
    want, ye, h, e, _ = ref.recurrence(*_np(x, gate, s0), np.full(b, t), True, True)
    y, s = torch.empty_like(x), s0.clone()
    for p in (slice(0, cut), slice(cut, t)):
        plan.forward_tensors(x[:, p], gate[:, p], y[:, p], state_in=s, state_out=s)
    ref.check_bound("y", y, want, ye, element)
    ref.check_bound("state", s, h, e, "f32")
