"""Layer norm and its gradients against the definition in 64 bits."""
import numpy as np
import pytest

import sequence_reference as ref
import vkfft_amd as vk

pytestmark = pytest.mark.gpu

ELEMENT = {"f32": vk.Element.F32, "f16": vk.Element.F16, "bf16": vk.Element.BF16}


def _types():
    import torch
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _normal(seed, shape, element, scale=1.0, shift=0.0):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(shape, generator=g, device="cuda", dtype=torch.float32) * scale + shift
    return x.to(_types()[element])


def _np(*xs):
    return [x.double().cpu().numpy() for x in xs]


def _plan(ctx, width, element, weight_element=None, epsilon=1e-5):
    c = vk.LayerNormConfig.new(width).with_element(ELEMENT[element]).with_epsilon(epsilon)
    if weight_element:
        c.with_weight_element(ELEMENT[weight_element])
    return vk.LayerNormPlan(ctx, c)


def _rows(seed, rows, width, element, pitch=None, offset=0, **kw):
    """Rows at a pitch of their own, `offset` elements into an allocation."""
    import torch
    pitch = pitch or width
    flat = torch.full((offset + rows * pitch + 8,), float("nan"), device="cuda", dtype=_types()[element])
    x = flat[offset:offset + rows * pitch].view(rows, pitch)[:, :width]
    x.copy_(_normal(seed, (rows, width), element, **kw))
    return x


def _run(ctx, rows, width, element, weight_element=None, pitch=None, offset=0, scale=1.5, shift=0.4):
    import torch
    we = weight_element or element
    plan = _plan(ctx, width, element, weight_element)
    x = _rows(1, rows, width, element, pitch, offset, scale=scale, shift=shift)
    w, b = _normal(2, (width,), we, 0.2, 1.0), _normal(3, (width,), we, 0.2)
    y = _rows(4, rows, width, element, pitch, offset)
    stats = torch.full((rows, 2), float("nan"), device="cuda")
    plan.forward_tensors(x, w, b, y, stats)
    xn, wn, bn = _np(x, w, b)
    want, want_stats = ref.norm(xn, wn, bn, 1e-5)
    ref.check("y", y, want, ref.norm_bound(xn, wn, bn, want_stats), element, ref.NORM_TERM)
    total = np.concatenate([np.abs(xn).mean(1, keepdims=True), want_stats[:, 1:]], 1)
    # the variance keeps a few units of its squared distances; with a mean far from zero also of the mean's rounding
    ref.check("stats", stats, want_stats, total * (1 + np.abs(want_stats[:, :1]) * want_stats[:, 1:]), "f32", ref.NORM_TERM)

    dy = _rows(5, rows, width, element, pitch, offset)
    dx = _rows(6, rows, width, element, pitch, offset)
    dw, db = torch.full_like(w, float("nan")), torch.full_like(b, float("nan"))
    plan.backward_tensors(x, w, stats, dy, dx, dw, db)
    sn, dyn = _np(stats, dy)
    wants, totals = ref.norm_gradients(xn, wn, sn, dyn), ref.norm_gradients_bound(xn, wn, sn, dyn)
    for name, got, want, total, e in zip(("dx", "dw", "db"), (dx, dw, db), wants, totals, (element, we, we)):
        ref.check(name, got, want, total, e, ref.NORM_TERM)
    if pitch and pitch > width:  # what lies between the rows stays as it was
        for t in (y, dx):
            assert torch.isnan(t.as_strided((rows - 1, pitch - width), (pitch, 1), t.storage_offset() + width)).all()


@pytest.mark.parametrize("element", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,width", [(1, 1), (3, 2), (5, 7), (1, 64), (17, 100), (257, 128), (33, 129), (4, 511), (9, 512), (2, 513),
                                        (31, 1000), (6, 1001), (3, 1024), (7, 2049), (130, 4096), (2, 5000), (2, 8193), (3, 16384),
                                        (2, 20011), (1, 32768), (2, 40001), (1, 70003), (4099, 96)])
def test_norm_of_every_width(hip_ctx, element, rows, width):
    _run(hip_ctx, rows, width, element)


@pytest.mark.parametrize("element", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,width,pitch,offset", [(9, 128, 136, 0), (9, 128, 131, 1), (5, 1001, 1003, 3), (3, 4096, 4100, 5),
                                                     (2, 33000, 33001, 7)])
def test_strides_and_alignments(hip_ctx, element, rows, width, pitch, offset):
    _run(hip_ctx, rows, width, element, pitch=pitch, offset=offset)


@pytest.mark.parametrize("element", ["f16", "bf16"])
@pytest.mark.parametrize("rows,width", [(13, 768), (3, 1003)])
def test_weights_in_32_bits(hip_ctx, element, rows, width):
    _run(hip_ctx, rows, width, element, weight_element="f32")


def test_a_mean_far_from_zero_keeps_the_variance(hip_ctx):
    """Squares of x itself would leave no digits of the variance here."""
    _run(hip_ctx, 5, 1000, "f32", scale=1.0, shift=3000.0)


def test_without_weight_bias_and_stats(hip_ctx):
    import torch
    x = _normal(1, (5, 300), "f32")
    y = torch.empty_like(x)
    plan = _plan(hip_ctx, 300, "f32")
    plan.forward_tensors(x, None, None, y)
    xn, = _np(x)
    one = np.ones(300)
    want, st = ref.norm(xn, one, 0 * one, 1e-5)
    ref.check("y", y, want, ref.norm_bound(xn, one, 0 * one, st), "f32", ref.NORM_TERM)
    stats = torch.from_numpy(st).float().cuda()
    dy = _normal(2, (5, 300), "f32")
    dx, dw, db = torch.empty_like(x), torch.empty(300, device="cuda"), torch.empty(300, device="cuda")
    wants = ref.norm_gradients(xn, one, _np(stats)[0], _np(dy)[0])
    totals = ref.norm_gradients_bound(xn, one, _np(stats)[0], _np(dy)[0])
    for only in range(3):  # each gradient alone
        outs = [t if i == only else None for i, t in enumerate((dx, dw, db))]
        plan.backward_tensors(x, None, stats, dy, *outs)
        ref.check(str(only), (dx, dw, db)[only], wants[only], totals[only], "f32", ref.NORM_TERM)


@pytest.mark.parametrize("width", [128, 1001, 16384, 40001])
def test_in_place(hip_ctx, width):
    import torch
    plan = _plan(hip_ctx, width, "f32")
    x, w = _normal(1, (6, width), "f32"), _normal(2, (width,), "f32")
    y, stats = torch.empty_like(x), torch.empty(6, 2, device="cuda")
    plan.forward_tensors(x, w, w, y, stats)
    z = x.clone()
    plan.forward_tensors(z, w, w, z)
    assert torch.equal(y, z)
    dy = _normal(3, (6, width), "f32")
    dx, dw, db = torch.empty_like(x), torch.empty_like(w), torch.empty_like(w)
    plan.backward_tensors(x, w, stats, dy, dx, dw, db)
    dx2, dw2, db2 = dy.clone(), torch.empty_like(w), torch.empty_like(w)
    plan.backward_tensors(x, w, stats, dx2, dx2, dw2, db2)
    assert torch.equal(dx, dx2) and torch.equal(dw, dw2) and torch.equal(db, db2)


def test_no_rows(hip_ctx):
    import torch
    plan = _plan(hip_ctx, 100, "bf16")
    x = torch.empty(0, 100, device="cuda", dtype=torch.bfloat16)
    w = _normal(2, (100,), "bf16")
    plan.forward_tensors(x, w, w, x.clone(), torch.empty(0, 2, device="cuda"))
    dw, db = torch.full_like(w, 7), torch.full_like(w, 7)
    plan.backward_tensors(x, w, torch.empty(0, 2, device="cuda"), x, x.clone(), dw, db)
    assert not dw.any() and not db.any()


def test_broadcast_gradient(hip_ctx):
    """dy of one row for all, as a sum's backward pass gives it."""
    import torch
    x, w = _normal(1, (70, 200), "f32"), _normal(2, (200,), "f32")
    plan = _plan(hip_ctx, 200, "f32")
    y, stats = torch.empty_like(x), torch.empty(70, 2, device="cuda")
    plan.forward_tensors(x, w, w, y, stats)
    dy = _normal(3, (1, 200), "f32").expand(70, 200)
    a, b = ([torch.empty_like(x), torch.empty_like(w), torch.empty_like(w)] for _ in range(2))
    plan.backward_tensors(x, w, stats, dy, *a)
    plan.backward_tensors(x, w, stats, dy.contiguous(), *b)
    assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_a_nan_stays_in_its_row(hip_ctx):
    import torch
    for width in (40, 1001, 16384):
        x = _normal(1, (9, width), "f32")
        x[4, width // 2] = float("nan")
        x[6, 0] = float("inf")
        y, stats = torch.empty_like(x), torch.empty(9, 2, device="cuda")
        _plan(hip_ctx, width, "f32").forward_tensors(x, None, None, y, stats)
        finite = torch.isfinite(y).all(1).cpu().tolist()
        assert finite == [i not in (4, 6) for i in range(9)]
        assert torch.isnan(y[4]).all()


def test_gradients_against_differences(hip_ctx):
    """d<y, dy> along a direction of x, weight and bias, by central differences of the definition in 64 bits."""
    import torch
    rows, width = 7, 130
    plan = _plan(hip_ctx, width, "f32")
    x, w, b, dy = _normal(1, (rows, width), "f32"), _normal(2, (width,), "f32", 0.2, 1.0), _normal(3, (width,), "f32"), _normal(4, (rows, width), "f32")
    y, stats = torch.empty_like(x), torch.empty(rows, 2, device="cuda")
    plan.forward_tensors(x, w, b, y, stats)
    got = [torch.empty_like(x), torch.empty_like(w), torch.empty_like(b)]
    plan.backward_tensors(x, w, stats, dy, *got)
    at = _np(x, w, b)
    dyn, = _np(dy)
    rng = np.random.default_rng(5)
    for i, g in enumerate(got):
        d = rng.standard_normal(at[i].shape)
        up, down = list(at), list(at)
        up[i], down[i] = at[i] + 1e-5 * d, at[i] - 1e-5 * d
        slope = ((ref.norm(*up, 1e-5)[0] - ref.norm(*down, 1e-5)[0]) * dyn).sum() / 2e-5
        gn, = _np(g)
        # 32-bit gradients: c of their largest size times the direction's; the difference's own error is 1e-10 of it
        assert abs((gn * d).sum() - slope) <= 2.0 ** -16 * (np.abs(gn) * np.abs(d)).sum()


def test_sums_over_rows_are_repeatable(hip_ctx):
    import torch
    x, w, dy = _normal(1, (5000, 260), "bf16"), _normal(2, (260,), "bf16"), _normal(3, (5000, 260), "bf16")
    plan = _plan(hip_ctx, 260, "bf16")
    y, stats = torch.empty_like(x), torch.empty(5000, 2, device="cuda")
    plan.forward_tensors(x, w, w, y, stats)
    runs = []
    for _ in range(3):
        o = [torch.empty_like(x), torch.empty_like(w), torch.empty_like(w)]
        plan.backward_tensors(x, w, stats, dy, *o)
        runs.append(o)
    assert all(torch.equal(p, q) for o in runs[1:] for p, q in zip(runs[0], o))


def test_another_stream_and_a_workspace_of_the_callers(hip_ctx):
    import torch
    x, w, dy = _normal(1, (300, 520), "f32"), _normal(2, (520,), "f32"), _normal(3, (300, 520), "f32")
    plan = _plan(hip_ctx, 520, "f32")
    y, stats = torch.empty_like(x), torch.empty(300, 2, device="cuda")
    plan.forward_tensors(x, w, w, y, stats)
    want = [torch.empty_like(x), torch.empty_like(w), torch.empty_like(w)]
    plan.backward_tensors(x, w, stats, dy, *want)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = [[torch.empty_like(t) for t in want] for _ in streams]
    work = [torch.empty(plan.workspace_bytes, device="cuda", dtype=torch.uint8) for _ in streams]
    torch.cuda.synchronize()
    for s, o, wk in zip(streams, got, work):
        with torch.cuda.stream(s):
            plan.backward_tensors(x, w, stats, dy, *o, work=wk)
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for o in got for p, q in zip(want, o))


def test_graph_replays(hip_ctx):
    import torch
    x, w, dy = _normal(1, (600, 392), "bf16"), _normal(2, (392,), "bf16"), _normal(3, (600, 392), "bf16")
    plan = _plan(hip_ctx, 392, "bf16")
    outs = [torch.empty_like(x), torch.empty(600, 2, device="cuda"), torch.empty_like(x), torch.empty_like(w), torch.empty_like(w)]

    def step():
        plan.forward_tensors(x, w, w, outs[0], outs[1])
        plan.backward_tensors(x, w, outs[1], dy, *outs[2:])

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step()
    for seed in (11, 12, 13):
        x.copy_(_normal(seed, (600, 392), "bf16"))
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

    for c in (vk.LayerNormConfig.new(0), vk.LayerNormConfig.new(1 << 31), vk.LayerNormConfig.new(8).with_epsilon(0),
              vk.LayerNormConfig.new(8).with_epsilon(float("nan")), vk.LayerNormConfig.new(8).with_epsilon(1e-60)):
        refused("InvalidArgument", vk.LayerNormPlan, hip_ctx, c)
    refused("UnsupportedPrecision", vk.LayerNormPlan, hip_ctx,
            vk.LayerNormConfig.new(8).with_element(vk.Element.F32).with_weight_element(vk.Element.F16))
    plan = _plan(hip_ctx, 64, "f32")
    x, w = torch.zeros(4, 64, device="cuda"), torch.zeros(64, device="cuda")
    y, st = torch.zeros_like(x), torch.zeros(4, 2, device="cuda")
    refused("InvalidArgument", plan.forward_tensors, x.cpu(), w, w, y)
    refused("InvalidArgument", plan.forward_tensors, x, w.cpu(), w, y)
    refused("InputLengthMismatch", plan.forward_tensors, x, w[:32], w, y)
    refused("InputLengthMismatch", plan.forward_tensors, x, w, w, y[:3])
    refused("InputLengthMismatch", plan.forward_tensors, x, w, w, y, st[:, :1])
    refused("UnsupportedPrecision", plan.forward_tensors, x.half(), w, w, y)
    refused("InvalidArgument", plan.forward_tensors, torch.zeros(64, 4, device="cuda").t(), w, w, y)
    refused("InvalidArgument", plan.forward_tensors, x, w, w, torch.zeros(64, device="cuda").expand(4, 64))
    refused("InvalidArgument", plan.forward_tensors, x, w, w, torch.zeros(300, device="cuda").as_strided((4, 64), (32, 1)))
    refused("InvalidArgument", plan.backward_tensors, x, w, None, y, y, w, w)
    refused("InvalidArgument", plan.backward_tensors, x, w, st, y, x, w, w)
    refused("InputLengthMismatch", plan.backward_tensors, x, w, st, y, y, w, w, work=torch.zeros(4, device="cuda"))


def test_an_epsilon_past_32_bits_is_refused(hip_ctx):
    """Its square root would make every row the bias."""
    with pytest.raises(vk.VkFftError) as e:
        vk.LayerNormPlan(hip_ctx, vk.LayerNormConfig.new(8).with_epsilon(1e39))
    assert e.value.kind == "InvalidArgument"


@pytest.mark.parametrize("width", [1 << 20, (1 << 20) + 77])
def test_long_rows_of_one_value_keep_their_sums(hip_ctx, width):
    """Equal elements round to the same side at every addition: a thread's long sums would drift."""
    import torch
    plan = _plan(hip_ctx, width, "f32")
    x = torch.full((2, width), 0.1, device="cuda")
    w, b = _normal(2, (width,), "f32", 0.2, 1.0), _normal(3, (width,), "f32", 0.2)
    y, stats = torch.empty_like(x), torch.empty(2, 2, device="cuda")
    plan.forward_tensors(x, w, b, y, stats)
    xn, wn, bn = _np(x, w, b)
    want, want_stats = ref.norm(xn, wn, bn, 1e-5)
    ref.check("mean", stats[:, :1], want_stats[:, :1], np.abs(want_stats[:, :1]), "f32", ref.NORM_TERM)
    ref.check("y", y, want, ref.norm_bound(xn, wn, bn, want_stats), "f32", ref.NORM_TERM)
    # gradients: the rows of a usual input, dy weight the same everywhere
    x = _normal(4, (2, width), "f32", 1.5, 0.4)
    xn, = _np(x)
    stats = torch.from_numpy(ref.norm(xn, 1.0, 0.0, 1e-5)[1]).float().cuda()
    dy = torch.full((2, width), 0.1, device="cuda")
    dx = torch.empty_like(x)
    plan.backward_tensors(x, None, stats, dy, dx)
    one, (sn, dyn) = np.ones(width), _np(stats, dy)
    ref.check("dx", dx, ref.norm_gradients(xn, one, sn, dyn)[0], ref.norm_gradients_bound(xn, one, sn, dyn)[0], "f32", ref.NORM_TERM)


def test_plans_of_every_width_that_is_promised(hip_ctx):
    """The workspace follows what a width's kernels write, so that the widest plan fits beside its rows."""
    import torch
    for width in (32769, 1 << 17, 1 << 20, 1 << 27):
        plan = _plan(hip_ctx, width, "f16")
        assert plan.workspace_bytes <= max(1 << 26, 8 * width)
        plan.close()
    width = 1 << 30
    plan = _plan(hip_ctx, width, "f16")
    x = torch.zeros(1, width, device="cuda", dtype=torch.float16)
    x[:, ::2] = 1
    y, stats = torch.full_like(x, 7), torch.empty(1, 2, device="cuda")
    plan.forward_tensors(x, None, None, y, stats)
    # a mean of 1/2, and 1 in 16 bits as what lies around it
    assert stats[0, 0].item() == 0.5 and (y[:, 1::2] == -1).all() and (y[:, ::2] == 1).all()
    dw, db = torch.full_like(x[0], 7), torch.full_like(x[0], 7)
    plan.backward_tensors(x, None, stats, x, y, dw, db)
    assert torch.equal(db, x[0]) and torch.equal(dw, x[0])
    # dx = rstd (g - mean g - n mean(g n)) with g = x: 4 epsilon, and a few roundings of 1/2
    assert y.abs().max().item() <= 4.2e-5
    plan.close()


@pytest.mark.parametrize("element", ["f32", "bf16"])
@pytest.mark.parametrize("rows,width", [(70, 65536), (9, 300001), (5, 1 << 22), (3, (1 << 22) + 1)])
def test_rows_split_over_fewer_sums_where_they_are_wide(hip_ctx, element, rows, width):
    _run(hip_ctx, rows, width, element)


def test_partial_overlaps_are_refused_and_interleaved_rows_are_not(hip_ctx):
    import torch
    plan = _plan(hip_ctx, 64, "f32")
    buf = torch.zeros(40, 128, device="cuda")
    w, b, st = torch.ones(64, device="cuda"), torch.zeros(64, device="cuda"), torch.zeros(8, 2, device="cuda")
    flat = buf.view(-1)
    x = flat[:512].view(8, 64)

    def refused(f, *a, **kw):
        with pytest.raises(vk.VkFftError) as e:
            f(*a, **kw)
        assert e.value.kind == "InvalidArgument" and "overlap" in str(e.value)

    for at in (1, 64, 511):
        refused(plan.forward_tensors, x, w, b, flat[at:at + 512].view(8, 64))
    refused(plan.forward_tensors, x, w, b, buf[:8, 64:])  # rows of another pitch
    refused(plan.forward_tensors, buf[:8, :64], w, b, buf[2:10, 32:96])
    refused(plan.forward_tensors, x, w, b, buf[20:28, :64], flat[500:516].view(8, 2))
    refused(plan.forward_tensors, buf[20:28, :64], flat[:64], b, x)
    refused(plan.forward_tensors, buf[20:28, :64], w, flat[448:512], x)
    dy, dx, dw, db = buf[10:18, :64], buf[20:28, :64], torch.zeros_like(w), torch.zeros_like(w)
    refused(plan.backward_tensors, x, w, st, dy, flat[64:576].view(8, 64), dw, db)
    refused(plan.backward_tensors, x, w, st, dy, buf[11:19, :64], dw, db)
    refused(plan.backward_tensors, x, w, st, dy, dx, dw, dw)
    refused(plan.backward_tensors, x, w, st, dy, dx, buf[20, :64], db)
    refused(plan.backward_tensors, x, w, st, dy, dx, dw, x[3])
    work = torch.zeros(plan.workspace_bytes // 4 + 64, device="cuda")
    refused(plan.backward_tensors, x, w, st, dy, dx, dw, work[-128:-64], work=work[:-64])

    # the two halves of every row of one buffer, and the same rows
    buf.copy_(_normal(1, (40, 128), "f32"))
    want = torch.empty(8, 64, device="cuda")
    plan.forward_tensors(buf[:8, :64], w, b, want, st)
    plan.forward_tensors(buf[:8, :64], w, b, buf[:8, 64:], st)
    assert torch.equal(buf[:8, 64:], want)
    plan.backward_tensors(buf[:8, :64], w, st, buf[10:18, :64], buf[10:18, 64:], dw, db)
    plan.backward_tensors(buf[:8, :64], w, st, buf[10:18, :64], buf[10:18, :64], dw, db)
    assert torch.equal(buf[10:18, :64], buf[10:18, 64:])


@pytest.mark.parametrize("element", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,width", [(20011, 40), (40009, 100), (9001, 512), (2500, 1001), (2100, 2049), (1100, 4100), (600, 8200), (600, 20011),
                                        (520, 33000), (517, 70003)])
def test_blocks_that_take_several_rows(hip_ctx, element, rows, width):
    """More rows than the blocks that a launch has, in no multiple of them: rows read ahead, a last turn in which only
    some of a block's groups have a row, and sums carried from row to row."""
    _run(hip_ctx, rows, width, element)


@pytest.mark.parametrize("element", ["f16", "bf16"])
@pytest.mark.parametrize("width", [200, 16385, 20011, 33000])
def test_gradients_in_place_of_their_input_in_16_bits(hip_ctx, element, width):
    import torch
    plan = _plan(hip_ctx, width, element)
    x, w, dy = _normal(1, (300, width), element), _normal(2, (width,), element), _normal(3, (300, width), element)
    y, stats = torch.empty_like(x), torch.empty(300, 2, device="cuda")
    plan.forward_tensors(x, w, w, y, stats)
    dx, dw, db = torch.empty_like(x), torch.empty_like(w), torch.empty_like(w)
    plan.backward_tensors(x, w, stats, dy, dx, dw, db)
    dw2, db2 = torch.empty_like(w), torch.empty_like(w)
    plan.backward_tensors(x, w, stats, dy, dy, dw2, db2)
    assert torch.equal(dx, dy) and torch.equal(dw, dw2) and torch.equal(db, db2)


def test_a_transform_and_a_norm_are_ordered_by_default(hip_ctx):
    """The context's stream, where transforms run by default, and torch's default stream, where norms then run, wait for
    each other."""
    import torch
    n, batch = 4096, 4096
    fft = hip_ctx.plan(vk.TransformIr.build(vk.FftConfig.new([n]).with_batch_count(batch), vk.Direction.Forward))
    plan = _plan(hip_ctx, 2 * n, "f32")
    x = _normal(1, (batch, 2 * n), "f32")

    def run(wait):
        a, b, c = (torch.full_like(x, float("nan")) for _ in range(3))
        wait()
        for _ in range(4):  # transforms take longer than the norm that reads the last one
            fft.execute_tensors(x, a)
        wait()
        plan.forward_tensors(a, None, None, b)
        wait()
        fft.execute_tensors(b, c)
        wait()
        torch.cuda.synchronize()
        return a, b, c

    want = run(torch.cuda.synchronize)
    for _ in range(3):
        assert all(torch.equal(p, q) for p, q in zip(want, run(lambda: None)))


@pytest.mark.parametrize("element,rows,width", [("f32", 262147, 2100), ("bf16", 1 << 24, 16), ("bf16", 1 << 22, 1001), ("f16", 1 << 19, 5000),
                                                ("bf16", 65537, 20000), ("f32", 65537, 16385)])
def test_sums_over_many_rows_of_one_value(hip_ctx, element, rows, width):
    """The gradient of a mean is the same in every row: weight and bias gradients add equal numbers, which round to one
    side where they are added one by one."""
    import torch
    plan = _plan(hip_ctx, width, element, "f32")
    x, dy = _normal(1, (1, width), element), torch.full((1, width), 0.1, device="cuda", dtype=_types()[element])
    xn, dyn = _np(x, dy)
    st = ref.norm(xn, 1.0, 0.0, 1e-5)[1].astype(np.float32)
    stats = torch.from_numpy(st).cuda().expand(rows, 2).contiguous()
    dw, db = torch.empty(width, device="cuda"), torch.empty(width, device="cuda")
    plan.backward_tensors(x.expand(rows, width), None, stats, dy.expand(rows, width), None, dw, db)
    one, sn = np.ones(width), st.astype(np.float64)
    wants, totals = ref.norm_gradients(xn, one, sn, dyn), ref.norm_gradients_bound(xn, one, sn, dyn)
    for name, got, i in (("dw", dw, 1), ("db", db, 2)):
        ref.check(name, got, rows * wants[i], rows * totals[i], "f32", ref.NORM_TERM)
