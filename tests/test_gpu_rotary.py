"""Rotary positions, head norms and their gradients against the definition in 64 bits."""
import numpy as np
import pytest

import mixer_reference as ref
import vkfft_amd as vk

pytestmark = pytest.mark.gpu

ELEMENT = {"f32": vk.Element.F32, "f16": vk.Element.F16, "bf16": vk.Element.BF16}
ELEMENTS = list(ELEMENT)
HALF, PAIRS = vk.RotaryLayout.Half, vk.RotaryLayout.Interleaved
EPSILON = 1e-6


def _types():
    import torch
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _tensor(seed, shape, element, layout="bthd", pad=0, offset=0, scale=1.0, shift=0.0):
    """Normal numbers, the last dimension padded, `offset` elements into an allocation of NaN."""
    import torch
    b, t, h, d = shape
    order = (b, t, h) if layout == "bthd" else (b, h, t)
    flat = torch.full((offset + b * t * h * (d + pad) + 8,), float("nan"), device="cuda", dtype=_types()[element])
    x = flat[offset:offset + b * t * h * (d + pad)].view(*order, d + pad)[..., :d]
    g = torch.Generator(device="cuda").manual_seed(seed)
    x.copy_(torch.randn(*order, d, generator=g, device="cuda") * scale + shift)
    return x if layout == "bthd" else x.transpose(1, 2)


def _vector(seed, n, element, scale=0.3, shift=1.0):
    return _tensor(seed, (1, 1, 1, n), element, scale=scale, shift=shift).reshape(n).clone()


def _np(*xs):
    out = [x.double().cpu().numpy() for x in xs]
    return out[0] if len(out) == 1 else out


def _config(element, h, kv, d, r=None, layout=HALF, norm=False, weight_element=None, **kw):
    c = vk.RotaryConfig.new(h, d).with_kv_heads(kv).with_element(ELEMENT[element]).with_layout(layout)
    if r is not None:
        c.with_rotary_dim(r)
    if norm:
        c.with_norm(EPSILON)
    if weight_element:
        c.with_weight_element(ELEMENT[weight_element])
    for name, value in kw.items():
        getattr(c, "with_" + name)(value)
    return c


def _positions(b, t, positions, starts):
    if positions is not None:
        return positions.cpu().numpy().astype(np.int64)
    p = np.arange(t, dtype=np.int64)[None].repeat(b, 0)
    return p if starts is None else p + starts.cpu().numpy().astype(np.int64)[:, None]


def _run(ctx, element, b, t, h, kv, d, r=None, layout=HALF, norm=False, weight_element=None, weights=True, positions=None, starts=None,
         lengths=None, storage="bthd", pad=0, offset=0, in_place=False, scale=(2.0, 0.5), **kw):
    import torch
    config = _config(element, h, kv, d, r, layout, norm, weight_element, **kw)
    plan = vk.RotaryPlan(ctx, config)
    r = d if r is None else r
    we = weight_element or element
    cos, sin = ref.angles(_positions(b, t, positions, starts), config.turns())
    amplitude = config.amplitude
    n = np.full(b, t) if lengths is None else np.clip(np.asarray(lengths), 0, t)
    live = (np.arange(t)[None] < n[:, None])[:, :, None, None]
    where = {"positions": positions, "starts": starts,
             "lengths": None if lengths is None else torch.tensor(lengths, device="cuda", dtype=torch.int32)}
    make = lambda seed, heads, **k: _tensor(seed, (b, t, heads, d), element, storage, pad, offset, **k)  # noqa: E731
    names = ("q", "k") if kv else ("q",)
    heads = {"q": h, "k": kv}
    x = {f: make(i + 1, heads[f], scale=scale[i]) for i, f in enumerate(names)}
    dy = {f: make(i + 3, heads[f]) for i, f in enumerate(names)}
    w = {f: _vector(5 + i, d, we) if norm and weights else None for i, f in enumerate(names)}
    w.setdefault("k"), x.setdefault("k"), dy.setdefault("k")
    values = {f: _np(x[f], dy[f]) for f in names}
    y, dx = ({f: source[f] if in_place else make(7, heads[f], scale=0) for f in names} for source in (x, dy))
    if not in_place:
        for f in names:
            y[f].fill_(7), dx[f].fill_(7)
    y.setdefault("k"), dx.setdefault("k")
    kept = {f: x[f].clone() for f in names}
    kept.setdefault("k")
    plan.forward_tensors(x["q"], x["k"], y["q"], y["k"], q_weight=w["q"], k_weight=w["k"], **where)
    dw = {f: torch.full((d,), float("nan"), device="cuda", dtype=_types()[we]) if norm else None for f in ("q", "k")}
    plan.backward_tensors(dy["q"], dy["k"], dx["q"], dx["k"], q=kept["q"] if norm else None, k=kept["k"] if norm else None, q_weight=w["q"],
                          k_weight=w["k"], dq_weight=dw["q"], dk_weight=dw["k"], **where)
    for f in names:
        xn, dyn = values[f]
        wn = np.ones(d) if w[f] is None else _np(w[f])
        u = ref.rms(xn, wn, EPSILON)[1] if norm else xn
        term = ref.NORM_TERM if norm else ref.TURN_TERM
        want, total = ref.turn(u, cos, sin, r, layout == HALF, amplitude)
        ref.check(f, y[f], want * live, total * live, element, term)
        du, size = ref.turn_back(dyn, cos, sin, r, layout == HALF, amplitude)
        if norm:
            du, size, dwn, dws = ref.rms_gradients(xn, wn, EPSILON, du, size, live)
            ref.check("dw" + f, dw[f], dwn, dws, we, ref.NORM_TERM)
        ref.check("d" + f, dx[f], du * live, size * live, element, term)
        if pad and t > 1:  # what lies between the rows stays as it was
            for z in (y[f], dx[f]):
                z0 = z if storage == "bthd" else z.transpose(1, 2)
                flat = z0.as_strided((b * t * heads[f] - 1, pad), (d + pad, 1), z0.storage_offset() + d)
                assert torch.isnan(flat).all()
    return {f: y[f] for f in names}


@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("element", ELEMENTS)
@pytest.mark.parametrize("layout", [HALF, PAIRS])
@pytest.mark.parametrize("d,r", [(1, 0), (2, 2), (3, 2), (6, 6), (7, 4), (16, 16), (20, 10), (32, 8), (63, 62), (64, 64), (80, 40), (96, 96), (100, 26),
                                 (112, 112), (128, 128), (128, 2), (130, 66), (192, 128), (200, 198), (255, 254), (256, 256)])
def test_heads_of_every_width(hip_ctx, norm, element, layout, d, r):
    _run(hip_ctx, element, 2, 5, 3, 2, d, r, layout, norm)


@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("element", ELEMENTS)
@pytest.mark.parametrize("b,t,h,kv", [(1, 1, 1, 1), (1, 1, 32, 8), (300, 1, 4, 1), (3, 67, 12, 4), (2, 500, 5, 0), (1, 3000, 2, 6), (5, 7, 40, 40)])
def test_counts(hip_ctx, norm, element, b, t, h, kv):
    _run(hip_ctx, element, b, t, h, kv, 64, norm=norm)


@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("layout", [HALF, PAIRS])
@pytest.mark.parametrize("element", ELEMENTS)
@pytest.mark.parametrize("lengths", [[0, 9, 4], [9, 0, 1], [-3, 20, 9]])
def test_uneven_lengths(hip_ctx, norm, layout, element, lengths):
    _run(hip_ctx, element, 3, 9, 4, 2, 48, 32, layout, norm, lengths=lengths)


@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("layout", [HALF, PAIRS])
@pytest.mark.parametrize("element", ELEMENTS)
@pytest.mark.parametrize("storage,pad,offset", [("bhtd", 0, 0), ("bthd", 8, 0), ("bhtd", 3, 1), ("bthd", 1, 5)])
@pytest.mark.parametrize("d,r", [(64, 64), (40, 12)])
def test_layouts(hip_ctx, norm, layout, element, storage, pad, offset, d, r):
    _run(hip_ctx, element, 2, 11, 4, 2, d, r, layout, norm, storage=storage, pad=pad, offset=offset)


@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("layout", [HALF, PAIRS])
@pytest.mark.parametrize("element", ELEMENTS)
@pytest.mark.parametrize("d,r", [(128, 128), (50, 22)])
def test_in_place(hip_ctx, norm, layout, element, d, r):
    _run(hip_ctx, element, 2, 33, 6, 3, d, r, layout, norm, in_place=True, lengths=[33, 20])


@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("layout", [HALF, PAIRS])
@pytest.mark.parametrize("where", ["table", "starts"])
def test_far_positions(hip_ctx, norm, layout, where):
    """Up to the ends of 32 bits, whose angles 32 bits do not hold; starts may reach past them."""
    import torch
    b, t = 4, 6
    ends = torch.tensor([2 ** 31 - 1, -2 ** 31, 2 ** 30 + 12345, 98765], device="cuda", dtype=torch.int64)
    if where == "starts":
        _run(hip_ctx, "f32", b, t, 2, 2, 64, None, layout, norm, starts=ends.int())
    else:
        table = (ends[:, None] - torch.arange(t, device="cuda") * 1000003 * ends.sign()[:, None]).int()
        _run(hip_ctx, "f32", b, t, 2, 2, 64, None, layout, norm, positions=table)


@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("element", ["f32", "bf16"])
@pytest.mark.parametrize("scaling", [("linear_scaling", (8.0,)), ("base_scaling", (4.0,)), ("blended_scaling", (16.0, 512)), ("base", (500000.0,)),
                                     ("frequencies", ([0.0, -1.0, 6.2, 1e-9, -6.28, 3.14159265358979, 1e-30, 0.5],)), ("amplitude", (1.37,))])
def test_scalings(hip_ctx, norm, element, scaling):
    import torch
    name, args = scaling
    c = _config(element, 3, 2, 16, norm=norm)
    getattr(c, "with_" + name)(*args)
    starts = torch.tensor([70000, 5], device="cuda", dtype=torch.int32)
    kw = {"frequencies": c.turns()} if name != "amplitude" else {"amplitude": args[0]}
    _run(hip_ctx, element, 2, 9, 3, 2, 16, norm=norm, starts=starts, **kw)


@pytest.mark.parametrize("element", ["f16", "bf16"])
@pytest.mark.parametrize("d", [64, 90])
def test_weights_in_32_bits(hip_ctx, element, d):
    _run(hip_ctx, element, 2, 40, 6, 2, d, norm=True, weight_element="f32")


@pytest.mark.parametrize("element", ELEMENTS)
def test_without_weights(hip_ctx, element):
    _run(hip_ctx, element, 2, 12, 3, 1, 72, norm=True, weights=False)


@pytest.mark.parametrize("layout", [HALF, PAIRS])
@pytest.mark.parametrize("norm", [False, True])
def test_many_tokens(hip_ctx, layout, norm):
    """More rows than the launch has waves, many times over."""
    _run(hip_ctx, "bf16", 3, 4001, 12, 4, 64, None, layout, norm)


def test_one_tensor_alone(hip_ctx):
    import torch
    for norm in (False, True):
        plan = vk.RotaryPlan(hip_ctx, _config("f32", 4, 2, 32, norm=norm))
        q, k = _tensor(1, (2, 10, 4, 32), "f32"), _tensor(2, (2, 10, 2, 32), "f32")
        both, alone = [torch.empty_like(q), torch.empty_like(k)], [torch.empty_like(q), torch.empty_like(k)]
        plan.forward_tensors(q, k, *both)
        plan.forward_tensors(q, None, alone[0], None)
        plan.forward_tensors(None, k, None, alone[1])
        assert all(torch.equal(x, y) for x, y in zip(both, alone))
        w = [torch.full((32,), 3.0, device="cuda") if norm else None for _ in range(4)]
        plan.backward_tensors(q, k, *both, q=k.new_ones(q.shape), k=k, dq_weight=w[0], dk_weight=w[1])
        plan.backward_tensors(q, None, alone[0], None, q=k.new_ones(q.shape), dq_weight=w[2], dk_weight=w[3])
        assert torch.equal(both[0], alone[0])
        if norm:
            assert torch.equal(w[0], w[2]) and not w[3].any() and w[1].any()
            for i in range(2):  # dx alone, without gradients of the weights
                dx = torch.empty_like(q)
                plan.backward_tensors(q, None, dx, None, q=k.new_ones(q.shape), dq_weight=w[0] if i else None)
                assert torch.equal(dx, both[0])


def test_scores_depend_on_the_distance(hip_ctx):
    """q turned by p and k by p - n: the same product wherever p is."""
    import torch
    plan = vk.RotaryPlan(hip_ctx, _config("f32", 1, 1, 64))
    q, k = _tensor(1, (1, 1, 1, 64), "f32").expand(1, 50, 1, 64), _tensor(2, (1, 1, 1, 64), "f32").expand(1, 50, 1, 64)
    p = torch.randint(0, 1 << 30, (1, 50), device="cuda", dtype=torch.int32)
    a, b = torch.empty(1, 50, 1, 64, device="cuda"), torch.empty(1, 50, 1, 64, device="cuda")
    plan.forward_tensors(q, None, a, None, positions=p)
    plan.forward_tensors(None, k, None, b, positions=p - 37)
    scores = (a.double() * b.double()).sum((2, 3))
    # two turns' errors, 2^-21 of the sizes each
    assert (scores - scores[0, 0]).abs().max() <= 2.0 ** -19 * (q.abs().double() * 2).mul(k.abs().double() * 2).sum((2, 3)).max()


def test_gradients_against_differences(hip_ctx):
    """d<y, dy> along a direction of x and weight, by central differences of the definition in 64 bits."""
    import torch
    b, t, h, d, r = 2, 5, 3, 24, 16
    config = _config("f32", h, 0, d, r, PAIRS, True)
    plan = vk.RotaryPlan(hip_ctx, config)
    x, dy, w = _tensor(1, (b, t, h, d), "f32"), _tensor(2, (b, t, h, d), "f32"), _vector(3, d, "f32")
    dx, dw = torch.empty_like(x), torch.empty_like(w)
    plan.backward_tensors(dy, None, dx, None, q=x, q_weight=w, dq_weight=dw)
    cos, sin = ref.angles(_positions(b, t, None, None), config.turns())
    f = lambda x, w: (ref.turn(ref.rms(x, w, EPSILON)[1], cos, sin, r, False)[0] * _np(dy)).sum()  # noqa: E731
    at, rng = _np(x, w), np.random.default_rng(5)
    for i, g in enumerate((dx, dw)):
        v = rng.standard_normal(at[i].shape)
        up, down = list(at), list(at)
        up[i], down[i] = at[i] + 1e-5 * v, at[i] - 1e-5 * v
        slope = (f(*up) - f(*down)) / 2e-5
        # 32-bit gradients: c of their largest size times the direction's; the difference's own error is 1e-10 of it
        assert abs((_np(g) * v).sum() - slope) <= 2.0 ** -16 * (np.abs(_np(g)) * np.abs(v)).sum()


@pytest.mark.parametrize("element", ["f32", "bf16"])
@pytest.mark.parametrize("size", [1e-18, 1e18, 3e38])
def test_sizes_at_the_ends(hip_ctx, element, size):
    """Squares that leave 32 bits: the norm of what is finite is finite. Small rows are epsilon's."""
    import torch
    plan = vk.RotaryPlan(hip_ctx, _config(element, 2, 0, 64, 0, norm=True))
    unit = torch.rand(1, 4, 2, 64, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)) * 2 - 1
    x = (unit * size).to(_types()[element])
    y = torch.empty_like(x)
    plan.forward_tensors(x, None, y, None)
    want = ref.rms(_np(x), 1.0, EPSILON)[0]
    ref.check("y", y, want, np.abs(want), element, ref.NORM_TERM)


@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_bad_values_stay_in_their_row(hip_ctx, norm, value):
    import torch
    plan = vk.RotaryPlan(hip_ctx, _config("bf16", 3, 2, 48, 32, PAIRS, norm))
    q, k, dq, dk = (_tensor(i, (2, 20, h, 48), "bf16") for i, h in enumerate((3, 2, 3, 2)))
    n = torch.tensor([12, 20], device="cuda", dtype=torch.int32)

    def run():
        o = [torch.full_like(x, 3) for x in (q, k, q, k)]
        plan.forward_tensors(q, k, *o[:2], lengths=n)
        plan.backward_tensors(dq, dk, *o[2:], q=q, k=k, lengths=n)
        return o

    want = run()
    for x in (q, k, dq, dk):
        x[0, 12:] = value  # not read
    assert all(torch.equal(a, b) for a, b in zip(want, run()))
    for x in (q, k, dq, dk):
        x[1, 7, 1, 5] = value
    for a, b in zip(want, run()):
        assert not torch.isfinite(b[1, 7, 1]).all()
        b[1, 7, 1] = a[1, 7, 1]
        assert torch.equal(a, b)


def test_equal_rows_keep_their_sums(hip_ctx):
    """The weights' gradients over many equal rows: each addition of 32 bits would round to the same side."""
    import torch
    b, t, h, d = 8, 8192, 16, 32
    plan = vk.RotaryPlan(hip_ctx, _config("f32", h, 0, d, 0, norm=True))
    x, dy = _tensor(1, (1, 1, 1, d), "f32"), _tensor(2, (1, 1, 1, d), "f32")
    dx, dw = torch.empty(b, t, h, d, device="cuda"), torch.empty(d, device="cuda")
    plan.backward_tensors(dy.expand(b, t, h, d), None, dx, None, q=x.expand(b, t, h, d), dq_weight=dw)
    n = ref.rms(_np(x), 1.0, EPSILON)[0]
    want = b * t * h * (_np(dy) * n).reshape(d)
    ref.check("dw", dw, want, np.abs(want), "f32", ref.NORM_TERM)


def test_broadcast_and_packed_tensors(hip_ctx):
    """Views of one projection, in place and apart; one head for all."""
    import torch
    for norm in (False, True):
        plan = vk.RotaryPlan(hip_ctx, _config("f16", 4, 4, 64, 48, norm=norm))
        packed = _tensor(1, (2, 30, 12, 64), "f16").view(2, 30, 3, 4, 64)
        q, k, v = packed.unbind(2)
        want = [torch.empty(2, 30, 4, 64, device="cuda", dtype=torch.float16) for _ in range(2)]
        plan.forward_tensors(q, k, *want)
        kept = v.clone()
        plan.forward_tensors(q, k, q, k)
        assert torch.equal(q, want[0]) and torch.equal(k, want[1]) and torch.equal(v, kept)
        one = _tensor(2, (1, 30, 1, 64), "f16")
        a, b = torch.empty_like(want[0]), torch.empty_like(want[0])
        plan.forward_tensors(one.expand(2, 30, 4, 64), None, a, None)
        plan.forward_tensors(one.expand(2, 30, 4, 64).contiguous(), None, b, None)
        assert torch.equal(a, b)


def test_offsets_past_32_bits(hip_ctx):
    import torch
    far = torch.zeros((1 << 32) + (1 << 20), device="cuda", dtype=torch.bfloat16)
    t, d = 96, 64
    step = (1 << 32) // (t - 1) // 64 * 64 + 64
    x, y = (far.as_strided((1, t, 1, d), (far.numel(), step, d, 1), 128 * i) for i in range(2))
    near = _tensor(1, (1, t, 1, d), "bf16")
    x.copy_(near)
    for norm in (False, True):
        plan = vk.RotaryPlan(hip_ctx, _config("bf16", 1, 0, d, norm=norm))
        plan.forward_tensors(x, None, y, None)
        want = torch.empty_like(near)
        plan.forward_tensors(near, None, want, None)
        assert torch.equal(y, want)
        plan.backward_tensors(x, None, y, None, q=x)
        plan.backward_tensors(near, None, want, None, q=near)
        assert torch.equal(y, want)


def test_streams_workspaces_and_repeats(hip_ctx):
    import torch
    plan = vk.RotaryPlan(hip_ctx, _config("bf16", 8, 2, 128, norm=True))
    q, k, dq, dk = (_tensor(i, (2, 700, h, 128), "bf16") for i, h in enumerate((8, 2, 8, 2)))
    w = [_vector(i, 128, "bf16") for i in (5, 6)]

    def run(o, **kw):
        plan.backward_tensors(dq, dk, o[0], o[1], q=q, k=k, q_weight=w[0], k_weight=w[1], dq_weight=o[2], dk_weight=o[3], **kw)

    want = [torch.empty_like(x) for x in (q, k, *w)]
    run(want)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = [[torch.empty_like(x) for x in want] for _ in streams]
    work = [torch.empty(plan.workspace_bytes, device="cuda", dtype=torch.uint8) for _ in streams]
    torch.cuda.synchronize()
    for s, o, wk in zip(streams, got, work):
        with torch.cuda.stream(s):
            run(o, work=wk)
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for o in got for x, y in zip(want, o))
    run(got[0], stream=streams[0])
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(want, got[0]))


def test_graph_replays(hip_ctx):
    import torch
    plan = vk.RotaryPlan(hip_ctx, _config("bf16", 8, 2, 64, norm=True))
    q, k = _tensor(1, (3, 200, 8, 64), "bf16"), _tensor(2, (3, 200, 2, 64), "bf16")
    starts = torch.tensor([5, 900, 0], device="cuda", dtype=torch.int32)
    outs = [torch.empty_like(x) for x in (q, k, q, k)] + [torch.empty(64, device="cuda", dtype=torch.bfloat16) for _ in range(2)]

    def step():
        plan.forward_tensors(q, k, *outs[:2], starts=starts)
        plan.backward_tensors(*outs[:2], *outs[2:4], q=q, k=k, dq_weight=outs[4], dk_weight=outs[5], starts=starts)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step()
    for seed in (11, 12, 13):
        q.copy_(_tensor(seed, q.shape, "bf16"))
        starts += 1000
        step()
        torch.cuda.synchronize()
        want = [o.clone() for o in outs]
        for o in outs:
            o.fill_(5)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(want, outs))


def test_no_tokens(hip_ctx):
    import torch
    plan = vk.RotaryPlan(hip_ctx, _config("f32", 2, 1, 16, norm=True))
    for b, t in ((0, 5), (3, 0)):
        q, k = torch.empty(b, t, 2, 16, device="cuda"), torch.empty(b, t, 1, 16, device="cuda")
        w = [torch.full((16,), 7.0, device="cuda") for _ in range(2)]
        plan.forward_tensors(q, k, q.clone(), k.clone())
        plan.backward_tensors(q, k, q.clone(), k.clone(), q=q, k=k, dq_weight=w[0], dk_weight=w[1])
        assert not w[0].any() and not w[1].any()


def test_refusals(hip_ctx):
    import torch

    def refused(kind, f, *a, **kw):
        with pytest.raises(vk.VkFftError) as e:
            f(*a, **kw)
        assert e.value.kind == kind, e.value

    def config(**kw):
        c = vk.RotaryConfig.new(2, 16)
        for name, value in kw.items():
            setattr(c, name, value)
        return c

    make = lambda c: vk.RotaryPlan(hip_ctx, c)  # noqa: E731
    for c in (config(heads=65536), config(kv_heads=65536), config(head_dim=257), config(rotary_dim=15), config(rotary_dim=18), config(epsilon=0.0),
              config(epsilon=float("nan")), config(epsilon=1e-39), config(epsilon=1e39), config(amplitude=1e39), config(amplitude=float("nan")),
              config(frequencies=[float("inf")] * 8), config(frequencies=[float("nan")] * 8), config(frequencies=[6.3] * 8)):
        refused("InvalidArgument", make, c)
    refused("UnsupportedPrecision", make, config(weight_element=vk.Element.F16))
    refused("InputLengthMismatch", make, config(frequencies=[1.0]))
    plan = make(config(epsilon=1e-6))
    plain = make(config())
    q, k = torch.zeros(2, 4, 2, 16, device="cuda"), torch.zeros(2, 4, 2, 16, device="cuda")
    a, b = torch.zeros_like(q), torch.zeros_like(q)
    w = torch.zeros(16, device="cuda")
    n = torch.zeros(2, device="cuda", dtype=torch.int32)
    p = torch.zeros(2, 4, device="cuda", dtype=torch.int32)
    f, g = plan.forward_tensors, plan.backward_tensors
    refused("InvalidArgument", f, q.cpu(), k, a, b)
    refused("InvalidArgument", f, None, None, None, None)
    refused("InvalidArgument", f, q, None, a, b)
    refused("InvalidArgument", f, q, k, a, None)
    refused("InvalidArgument", f, q, k, a, b, positions=p, starts=n)
    refused("InvalidArgument", f, q, k, a, b, positions=p.cpu())
    refused("InputLengthMismatch", f, q[0], k, a, b)
    refused("InputLengthMismatch", f, q, k[:, :3], a, b)
    refused("InputLengthMismatch", f, q, k, a, b, positions=n)
    refused("InputLengthMismatch", f, q, k, a, b, starts=n[:1])
    refused("InputLengthMismatch", f, q, k, a, b, q_weight=w[:8])
    refused("UnsupportedPrecision", f, q, k, a, b, lengths=n.long())
    refused("UnsupportedPrecision", f, q.half(), k, a, b)
    refused("UnsupportedPrecision", f, q, k, a, b, k_weight=w.half())
    refused("InvalidArgument", f, q, k, torch.zeros(1, 1, 1, 16, device="cuda").expand(2, 4, 2, 16), b)
    refused("InvalidArgument", f, q, k, torch.zeros(2, 4, 16, 2, device="cuda").transpose(2, 3), b)
    refused("InvalidArgument", f, q, k, a, a)
    refused("InvalidArgument", f, q, k, k, b)
    refused("InvalidArgument", f, q, k, q.transpose(0, 1).reshape(4, 2, 2, 16).transpose(0, 1)[:], q)
    refused("InvalidArgument", f, q, k, q.view(-1).as_strided((2, 4, 2, 16), (16, 64, 32, 1)), b)  # q in another order
    refused("InvalidArgument", plain.forward_tensors, q, k, a, b, q_weight=w)
    refused("InvalidArgument", plain.backward_tensors, q, k, a, b, dk_weight=w)
    refused("InvalidArgument", g, q, k, a, b)  # the norm needs q and k
    refused("InvalidArgument", g, q, k, a, b, q=a, k=k)
    refused("InvalidArgument", g, q, k, a, b, q=q, k=k, dq_weight=w, dk_weight=w)
    refused("InvalidArgument", g, q, k, a, b, q=q, k=k, q_weight=w, dk_weight=w)
    refused("InputLengthMismatch", g, q, k, a, b, q=q, k=k, work=torch.zeros(4, device="cuda"))
    flat = torch.zeros(2 * q.numel(), device="cuda")
    x = flat[:q.numel()].view(q.shape)
    refused("InvalidArgument", f, x, k, flat[16:16 + q.numel()].view(q.shape), b)


def test_plans_hold_their_context(hip_ctx):
    ctx = vk.HipExecutionContext(0)
    plan = vk.RotaryPlan(ctx, vk.RotaryConfig.new(2, 16))
    assert ctx._L.vkfx_context_destroy(ctx.handle) == -2
    plan.close()
    ctx.close()


def test_more_rows_than_a_launch_has_groups(hip_ctx):
    """Blocks go on to further tokens; the last ones are turned by their own positions."""
    import torch
    t = (1 << 28) + (1 << 18) + 5
    plan = vk.RotaryPlan(hip_ctx, _config("f16", 1, 0, 2))
    x = torch.empty(1, t, 1, 2, device="cuda", dtype=torch.float16)
    x[:] = _tensor(1, (1, 1, 1, 2), "f16")
    y = torch.empty_like(x)
    plan.forward_tensors(x, None, y, None)
    for at in (0, (1 << 28) - 500, t - 1000):
        z = torch.empty(1, 1000, 1, 2, device="cuda", dtype=torch.float16)
        plan.forward_tensors(x[:, at:at + 1000], None, z, None, starts=torch.tensor([at], device="cuda", dtype=torch.int32))
        assert torch.equal(y[:, at:at + 1000], z)


@pytest.mark.parametrize("layout", [HALF, PAIRS])
@pytest.mark.parametrize("element", ELEMENTS)
@pytest.mark.parametrize("b,t,h,kv", [(2, 9, 3, 2), (2, 9000, 5, 3), (3, 12000, 2, 1)])
@pytest.mark.parametrize("d,r", [(48, 32), (50, 22), (128, 2), (37, 30)])
def test_what_does_not_turn_passes(hip_ctx, layout, element, b, t, h, kv, d, r):
    """Elements from rotary_dim on are the row's, to the bit; what is not finite among them reaches no other."""
    import torch
    bits = torch.int32 if element == "f32" else torch.int16
    plan = vk.RotaryPlan(hip_ctx, _config(element, h, kv, d, r, layout, amplitude=0.5))
    q, k = _tensor(1, (b, t, h, d), element), _tensor(2, (b, t, kv, d), element)
    runs = []
    for bad in (False, True):
        if bad:
            for x in (q, k):
                most = torch.finfo(x.dtype).max
                for i, v in enumerate((float("inf"), -0.0, float("-inf"), most, float("nan"))):
                    x[:, i::6, 1 % x.size(2), r + i % (d - r)] = v
                x[:, 5::6, 0, r:] = float("inf")
        o = [torch.full_like(x, 3) for x in (q, k, q, k)]
        plan.forward_tensors(q, k, *o[:2])
        plan.backward_tensors(q, k, *o[2:])
        runs.append(o)
        for x, y in zip((q, k, q, k), o):
            x, y = x[..., r:], y[..., r:]
            assert torch.equal(torch.isnan(x), torch.isnan(y))
            assert torch.equal(x.nan_to_num(9.0, 8.0, 7.0).contiguous().view(bits), y.nan_to_num(9.0, 8.0, 7.0).contiguous().view(bits))
    assert all(torch.equal(x[..., :r], y[..., :r]) for x, y in zip(*runs))


@pytest.mark.parametrize("element", ELEMENTS)
def test_what_does_not_turn_passes_the_norm(hip_ctx, element):
    """Behind the norm it is what a plan that turns none of the row gives; zeros keep their signs."""
    import torch
    h, d, r = 3, 48, 32
    x, w = _tensor(1, (2, 40, h, d), element), _vector(3, d, element, scale=0.05)
    x[:, ::2, :, r + 1::2] = -0.0
    bits = torch.int32 if element == "f32" else torch.int16
    outs = []
    for turned in (r, 0):
        plan = vk.RotaryPlan(hip_ctx, _config(element, h, 0, d, turned, PAIRS, True))
        y = torch.empty_like(x)
        plan.forward_tensors(x, None, y, None, q_weight=w)
        assert (w > 0).all() and torch.equal(torch.signbit(y[..., r:]), torch.signbit(x[..., r:]))
        outs.append(y[..., r:].contiguous().view(bits))
    assert torch.equal(*outs)


@pytest.mark.parametrize("element", ["f32", "bf16"])
@pytest.mark.parametrize("size,epsilon,d", [(1e19, 1e37, 64), (3e19, 1e38, 64), (2e19, 3e38, 64), (1e38, 3e38, 200), (1.2e19, 3.3e38, 2), (3e38, 1e-6, 64),
                                            (1e18, 3e38, 64)])
def test_large_epsilons(hip_ctx, element, size, epsilon, d):
    """An epsilon that is no less than rows whose squares pass 32 bits, alone or with it, counts beside them."""
    import torch
    plan = vk.RotaryPlan(hip_ctx, vk.RotaryConfig.new(2, d).with_kv_heads(0).with_rotary_dim(0).with_element(ELEMENT[element]).with_norm(epsilon))
    unit = torch.rand(1, 4, 2, d, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)) * 0.5 + 0.5
    x, dy = (unit * size).to(_types()[element]), _tensor(2, (1, 4, 2, d), element)
    y, dw = torch.empty_like(x), torch.empty(d, device="cuda", dtype=x.dtype)
    plan.forward_tensors(x, None, y, None)
    want = ref.rms(_np(x), 1.0, epsilon)[0]
    ref.check("y", y, want, np.abs(want), element, ref.NORM_TERM)
    plan.backward_tensors(dy, None, torch.empty_like(x), None, q=x, dq_weight=dw)
    _, _, want, total = ref.rms_gradients(_np(x), np.ones(d), epsilon, _np(dy), np.abs(_np(dy)), 1.0)
    ref.check("dw", dw, want, total, element, ref.NORM_TERM)


@pytest.mark.parametrize("size,weight,epsilon", [(3e38, 1e-3, 1e-6), (1e30, 1e-12, 1e-6), (1e-20, 1e25, 2e-38), (1e-19, 1e-25, 2e-38)])
def test_weights_beside_rows_at_the_ends(hip_ctx, size, weight, epsilon):
    """The row's factor times the weight may leave 32 bits, or their normal numbers, where the result does not."""
    import torch
    d = 64
    plan = vk.RotaryPlan(hip_ctx, _config("f32", 2, 0, d, 0).with_norm(epsilon))
    g = torch.Generator(device="cuda").manual_seed(1)
    x, w = ((torch.rand(n, device="cuda", generator=g) * 0.5 + 0.5) * s for n, s in (((1, 4, 2, d), size), ((d,), weight)))
    y = torch.empty_like(x)
    plan.forward_tensors(x, None, y, None, q_weight=w)
    want = ref.rms(_np(x), _np(w), epsilon)[1]
    ref.check("y", y, want, np.abs(want), "f32", ref.NORM_TERM)


@pytest.mark.parametrize("frequency", [1.0, 0.01, -2.5, 1e-4])
def test_cosines_and_sines(hip_ctx, frequency):
    """(1, 0) turns to (cos, sin): what is above 2^-0.5 within 2^-21.9 of itself, the other within 2^-21.6."""
    import torch
    t = 1 << 21
    plan = vk.RotaryPlan(hip_ctx, _config("f32", 1, 0, 2, frequencies=[frequency]))
    x = torch.tensor([1.0, 0.0], device="cuda").expand(1, t, 1, 2)
    y = torch.empty(1, t, 1, 2, device="cuda")
    plan.forward_tensors(x, None, y, None)
    a = np.arange(t, dtype=np.longdouble) * np.longdouble(frequency)
    got = _np(y).reshape(t, 2)
    # In 2^-24 of each: t's two roundings, that of r and of 2 pi 3.5 (r tan r <= 0.79 of them for the cosine), the sine's
    # last product 1 and the sum in it 0.6; the cosine's last sum 0.7 and the squares in it 0.5: 5.1 and 4. A near quarter
    # turn gives either from the other's series.
    for i, want in enumerate((np.cos(a), np.sin(a))):
        size = np.abs(want)
        # the frequency is a multiple of 2^-64 turns, and the angle here of 64 bits: 2^-40 at these positions
        over = np.abs(got[:, i] - want) - np.where(size > 2.0 ** -0.5, 2.0 ** -21.9, 2.0 ** -21.6) * size - 2.0 ** -40
        assert over.max() <= 0, (i, int(np.argmax(over)), float(over.max()))


def test_a_workspace_at_an_odd_place_is_refused(hip_ctx):
    """Its sums are floats; the plan without the norm uses none."""
    import torch
    plan, plain = (vk.RotaryPlan(hip_ctx, _config("f32", 2, 0, 16, norm=n)) for n in (True, False))
    x, y = torch.ones(1, 4, 2, 16, device="cuda"), torch.empty(1, 4, 2, 16, device="cuda")
    room = torch.zeros(plan.workspace_bytes + 16, device="cuda", dtype=torch.uint8)
    for at in (1, 4, 8):
        with pytest.raises(vk.VkFftError) as e:
            plan.backward_tensors(x, None, y, None, q=x, work=room[at:])
        assert e.value.kind == "InvalidArgument" and "aligned" in str(e.value)
        plain.backward_tensors(x, None, y, None, work=room[at:])
    assert not room.any()
    plan.backward_tensors(x, None, y, None, q=x, work=room[16:])


# From 8 waves a CU on, 2048 of the 256 CUs here, a lane takes several heads of its token: four, two where there are
# no more, two in the gradients behind the norm. Tokens are as many as that takes with each width's lanes.
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("element", ELEMENTS)
@pytest.mark.parametrize("b,t,h,kv,d,r,layout", [
    (2, 8203, 5, 3, 64, 64, HALF), (2, 4099, 5, 3, 128, 128, HALF), (3, 8200, 2, 1, 128, 128, PAIRS), (2, 4111, 7, 0, 90, 90, HALF),
    (2, 4111, 3, 2, 90, 90, PAIRS), (2, 4111, 5, 1, 128, 32, HALF), (2, 8231, 6, 2, 100, 50, HALF), (2, 8229, 5, 3, 80, 40, PAIRS),
    (2, 2063, 4, 1, 256, 256, HALF), (1, 4101, 5, 3, 256, 66, HALF), (1, 4101, 1, 6, 255, 254, PAIRS), (2, 33001, 2, 1, 20, 10, HALF)])
def test_several_heads_a_lane(hip_ctx, norm, element, b, t, h, kv, d, r, layout):
    _run(hip_ctx, element, b, t, h, kv, d, r, layout, norm)


@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("element", ELEMENTS)
@pytest.mark.parametrize("layout,d,r", [(HALF, 128, 128), (HALF, 90, 26), (PAIRS, 110, 50)])
def test_several_heads_a_lane_in_place_and_ragged(hip_ctx, norm, element, layout, d, r):
    """In place, with rows past their length, positions of their own and rows at odd places."""
    import torch
    starts = torch.tensor([5, 1 << 20, -3], device="cuda", dtype=torch.int32)
    _run(hip_ctx, element, 3, 4011, 7, 3, d, r, layout, norm, in_place=True, lengths=[4011, 0, 1999], starts=starts, pad=3, offset=1, amplitude=1.25)
    _run(hip_ctx, element, 3, 4011, 9, 3, d, r, layout, norm, lengths=[1, 2000, 4010], storage="bhtd",
         positions=torch.randint(0, 1 << 20, (3, 4011), device="cuda", dtype=torch.int32), weight_element="f32" if norm else None)
