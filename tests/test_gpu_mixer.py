"""The sequence operators one behind the other, as a layer runs them: norm, queries and keys normed and turned,
linear attention, gated recurrence. A prompt at once, token by token, and gradients of the whole."""
import numpy as np
import pytest

import mixer_reference as ref
import sequence_reference as seq
import vkfft_amd as vk

pytestmark = pytest.mark.gpu

B, T, H, KV, D, WIDTH, EPS = 2, 45, 4, 2, 16, 64, 1e-6
DECAYS = [0.5, 0.875, 0.96875, 0.9921875]


class Layer:
    def __init__(self, ctx):
        import torch
        g = torch.Generator(device="cuda").manual_seed(3)
        rand = lambda *s, scale=1.0: torch.randn(s, generator=g, device="cuda") * scale  # noqa: E731
        self.w = {"norm": rand(WIDTH, scale=0.2) + 1, "bias": rand(WIDTH, scale=0.2), "qkv": rand(WIDTH, (H + 2 * KV) * D, scale=WIDTH ** -0.5),
                  "q": rand(D, scale=0.2) + 1, "k": rand(D, scale=0.2) + 1, "gate": rand(WIDTH, H * D, scale=WIDTH ** -0.5)}
        self.norm = vk.LayerNormPlan(ctx, vk.LayerNormConfig.new(WIDTH).with_epsilon(EPS))
        self.config = vk.RotaryConfig.new(H, D).with_kv_heads(KV).with_rotary_dim(8).with_norm(EPS)
        self.rotary = vk.RotaryPlan(ctx, self.config)
        self.mix = vk.LinearAttentionPlan(ctx, vk.LinearAttentionConfig.new(H, D, D).with_kv_heads(KV).with_decay(DECAYS)
                                          .with_capacity(B, T).with_gradient())
        self.recur = vk.GatedRecurrencePlan(ctx, vk.GatedRecurrenceConfig.new(H * D).with_complement())

    def forward(self, x, states, starts=None, keep=None):
        """y for the next tokens; the states are updated in place."""
        import torch
        b, t = x.shape[:2]
        w, rows = self.w, x.reshape(-1, WIDTH)
        n, stats = torch.empty_like(rows), torch.empty(rows.shape[0], 2, device="cuda")
        self.norm.forward_tensors(rows, w["norm"], w["bias"], n, stats)
        packed = (n @ w["qkv"]).view(b, t, H + 2 * KV, D)
        q, k, v = packed[:, :, :H], packed[:, :, H:H + KV], packed[:, :, H + KV:]
        qr, kr = torch.empty(b, t, H, D, device="cuda"), torch.empty(b, t, KV, D, device="cuda")
        self.rotary.forward_tensors(q, k, qr, kr, q_weight=w["q"], k_weight=w["k"], starts=starts)
        o = torch.empty(b, t, H, D, device="cuda")
        self.mix.forward_tensors(qr, kr, v, o, state_in=states[0], state_out=states[0])
        gate = (n @ w["gate"]).view(b, t, H * D)
        y = torch.empty_like(gate)
        saved = torch.empty(self.recur.saved_shape(b, t), device="cuda") if keep is not None else None
        self.recur.forward_tensors(o.view(b, t, H * D), gate, y, state_in=states[1], state_out=states[1], saved=saved)
        if keep is not None:
            keep.update(rows=rows, stats=stats, n=n, q=q, k=k, v=v, qr=qr, kr=kr, o=o.view(b, t, H * D), gate=gate, saved=saved)
        return y

    def backward(self, dy, kept):
        import torch
        b, t = dy.shape[:2]
        w, z = self.w, kept
        do, dgate = torch.empty_like(z["o"]), torch.empty_like(z["gate"])
        self.recur.backward_tensors(z["o"], z["gate"], z["saved"], dy, do, dgate)
        packed = torch.empty(b, t, H + 2 * KV, D, device="cuda")
        dq, dk, dv = packed[:, :, :H], packed[:, :, H:H + KV], packed[:, :, H + KV:]
        self.mix.backward_tensors(z["qr"], z["kr"], z["v"], do.view(b, t, H, D), dq, dk, dv)
        dqw, dkw = torch.empty_like(w["q"]), torch.empty_like(w["k"])
        self.rotary.backward_tensors(dq, dk, dq, dk, q=z["q"], k=z["k"], q_weight=w["q"], k_weight=w["k"], dq_weight=dqw, dk_weight=dkw)
        dn = packed.view(b * t, -1) @ w["qkv"].t() + dgate.view(b * t, -1) @ w["gate"].t()
        dx, dw, db = torch.empty_like(dn), torch.empty_like(w["norm"]), torch.empty_like(w["bias"])
        self.norm.backward_tensors(z["rows"], w["norm"], z["stats"], dn, dx, dw, db)
        return {"x": dx.view(b, t, WIDTH), "norm": dw, "bias": db, "q": dqw, "k": dkw}


def _states():
    import torch
    return [torch.zeros(B, H, D, D, device="cuda"), torch.zeros(B, H * D, device="cuda")]


def _definition(layer, x, w):
    b, t = x.shape[:2]
    n = seq.norm(x.reshape(-1, WIDTH), w["norm"], w["bias"], EPS)[0]
    packed = (n @ w["qkv"]).reshape(b, t, H + 2 * KV, D)
    cos, sin = ref.angles(np.arange(t)[None].repeat(b, 0), layer.config.turns())
    q, k = (ref.turn(ref.rms(z, w[f], EPS)[1], cos, sin, 8, True)[0] for z, f in ((packed[:, :, :H], "q"), (packed[:, :, H:H + KV], "k")))
    o, s = seq.attention(q, k, packed[:, :, H + KV:], np.zeros((b, H, D, D)), DECAYS, D ** -0.5, np.full(b, t))
    y, _, h, _, _ = ref.recurrence(o.reshape(b, t, -1), (n @ w["gate"]).reshape(b, t, -1), np.zeros((b, H * D)), np.full(b, t), True, True)
    return y, s, h


def _np(x):
    return x.double().cpu().numpy()


# A step of a 32-bit product over 64 terms, of the attention's (2^-18 a term) or a norm moves what follows by a few
# times its own error: 2^-13 of a result's size over the five operators.
WHOLE = 2.0 ** -13


def test_a_prompt_and_token_by_token(hip_ctx):
    import torch
    layer = Layer(hip_ctx)
    x = torch.randn(B, T, WIDTH, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")
    y, s, h = _definition(layer, _np(x), {f: _np(v) for f, v in layer.w.items()})
    states = _states()
    whole = layer.forward(x, states)
    for name, got, want in (("y", whole, y), ("attention", states[0], s), ("recurrence", states[1], h)):
        assert np.abs(_np(got) - want).max() <= WHOLE * np.abs(want).max(), name
    states = _states()
    parts = [layer.forward(x[:, :20], states)]
    for t in range(20, T):
        parts.append(layer.forward(x[:, t:t + 1], states, starts=torch.full((B,), t, device="cuda", dtype=torch.int32)))
    assert np.abs(_np(torch.cat(parts, 1)) - y).max() <= WHOLE * np.abs(y).max()


def test_gradients_of_the_whole(hip_ctx):
    import torch
    layer = Layer(hip_ctx)
    g = torch.Generator(device="cuda").manual_seed(2)
    x, dy = (torch.randn(B, T, n, generator=g, device="cuda") for n in (WIDTH, H * D))
    kept = {}
    layer.forward(x, _states(), keep=kept)
    got = layer.backward(dy, kept)
    at = {"x": _np(x), **{f: _np(v) for f, v in layer.w.items()}}
    rng = np.random.default_rng(5)

    def f(v):
        return (_definition(layer, v["x"], v)[0] * _np(dy)).sum()

    for name, grad in got.items():
        d = rng.standard_normal(at[name].shape)
        slope = (f({**at, name: at[name] + 1e-5 * d}) - f({**at, name: at[name] - 1e-5 * d})) / 2e-5
        assert abs((_np(grad) * d).sum() - slope) <= WHOLE * (np.abs(_np(grad)) * np.abs(d)).sum(), name


def test_a_step_in_a_graph(hip_ctx):
    """One new token of each sequence, captured once and replayed: states and positions move on."""
    import torch
    layer = Layer(hip_ctx)
    x = torch.randn(B, 6, WIDTH, generator=torch.Generator(device="cuda").manual_seed(4), device="cuda")
    token, starts, states = torch.empty(B, 1, WIDTH, device="cuda"), torch.zeros(B, device="cuda", dtype=torch.int32), _states()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        token.copy_(x[:, :1])
        layer.forward(token, states, starts)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        y = layer.forward(token, states, starts)
    for s in states:
        s.zero_()
    eager = _states()
    for t in range(6):
        token.copy_(x[:, t:t + 1])
        starts.fill_(t)
        want = layer.forward(token, eager, starts)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want) and all(torch.equal(a, b) for a, b in zip(states, eager))
