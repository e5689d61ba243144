"""Performance cases of the operators around linear attention: rotary positions of queries and keys, the same with a norm of each head in front, and the
gated linear recurrence; forward, backward and token by token.

A program makes a plan for its heads or channels once, keeps it with its buffers, and calls it for every new input; so `prepare` makes the inputs, the
output buffers and (for the framework's own operators) the plan, and `run` makes the calls of one pass. The "kind"s:

  rotate            queries and keys of a batch of sequences rotated by their positions: q and k
  rotate_grad       its backward pass: gradients of q and k
  norm_rotate       each head of q and k divided by its root mean square and scaled by a weight, then rotated
  norm_rotate_grad  its backward pass: gradients of q, k and both weights
  recur             the gated recurrence over a prompt, from a state to the next: outputs and the state after the last token
  recur_step        the same for one new token of each sequence (a few with speculation): the state is updated in place
  recur_grad        a training step's two passes: outputs and the last state, then gradients of x, gate and the initial state

Rotation of a head of d elements at position p: the first r of them form r / 2 pairs, (2i, 2i + 1) interleaved or (i, i + r / 2) by halves; pair i turns
by p f[i], f[i] = base^(-2i / r). For contexts `stretch` times as long as the trained one, a pair that turns less than once in the trained context turns
`stretch` times slower, one that turns 32 times or more as before, in between by a share of both that goes with the turns.

Recurrence of one channel, a = sigmoid(gate) or exp(min(gate, 0)), m = 1 - a ("complement") or 1:
  h[t] = a[t] h[t-1] + m[t] x[t]        y[t] = h[t]
Sequences of a batch may be shorter than the batch's tokens ("ragged"): rows from a sequence's length on give zeros and leave its state alone.
"""
import math
import os
import sys

import torch

own = False

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_BASE, _TRAINED, _FAST, _SLOW, _EPSILON = 10000.0, 4096, 32.0, 1.0, 1e-6
_context = None


def _vk():
    sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "vkfft-rs_amd"))
    import vkfft_amd
    return vkfft_amd


def _ctx(vk):
    global _context
    if _context is None:
        torch.cuda.init()  # torch's HIP runtime is the one the library binds to
        _context = vk.HipExecutionContext(0)
    return _context


def _rotate(name, kind, batch, tokens, heads, kv_heads, head_dim, element, rotary_dim=None, layout="half", positions="none", far=0, stretch=1, ragged=False):
    return {"name": name, "kind": kind, "batch": batch, "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim,
            "rotary_dim": rotary_dim or head_dim, "layout": layout, "positions": positions, "far": far, "stretch": stretch, "element": element, "ragged": ragged}


def _recur(name, kind, batch, tokens, channels, element, gate="sigmoid", complement=True, ragged=False):
    return {"name": name, "kind": kind, "batch": batch, "tokens": tokens, "channels": channels, "gate": gate, "complement": complement,
            "element": element, "ragged": ragged}


def listed():
    return [
        # one sequence answering token by token, deep in its context: latency
        _rotate("rotate_1_h32_8_128_bf16", "rotate", 1, 1, 32, 8, 128, "bf16", positions="starts", far=32768),
        # prompts of a serving batch
        _rotate("rotate_8x2048_h32_8_128_bf16", "rotate", 8, 2048, 32, 8, 128, "bf16"),
        # half of an uneven head in neighbouring pairs, full precision, packed documents at far positions of a stretched context, uneven lengths
        _rotate("rotate_3x1001_h12_4_80_f32", "rotate", 3, 1001, 12, 4, 80, "f32", 40, "interleaved", "table", 1 << 20, 8, True),
        # a training batch's backward pass
        _rotate("rotate_grad_4x4096_h16_4_128_f16", "rotate_grad", 4, 4096, 16, 4, 128, "f16", layout="interleaved"),
        # a full serving batch answering token by token
        _rotate("norm_rotate_256_h32_8_128_bf16", "norm_rotate", 256, 1, 32, 8, 128, "bf16", positions="starts", far=8192),
        # prompts of a serving batch, each query head with a key head of its own
        _rotate("norm_rotate_8x2048_h16_128_bf16", "norm_rotate", 8, 2048, 16, 16, 128, "bf16"),
        # a training batch's backward pass
        _rotate("norm_rotate_grad_4x4096_h16_4_128_bf16", "norm_rotate_grad", 4, 4096, 16, 4, 128, "bf16"),
        # prompts of a serving batch: channels enough to fill the machine
        _recur("recur_8x2048_4096_bf16", "recur", 8, 2048, 4096, "bf16"),
        # one long document: little to run side by side but the sequence itself
        _recur("recur_1x65536_1024_bf16", "recur", 1, 65536, 1024, "bf16"),
        # a serving batch answering token by token
        _recur("recur_step_64_4096_bf16", "recur_step", 64, 1, 4096, "bf16"),
        # a training batch
        _recur("recur_grad_4x4096_2048_bf16", "recur_grad", 4, 4096, 2048, "bf16"),
        # odd counts, an odd width and uneven lengths in full precision, decays given by their logarithms
        _recur("recur_grad_3x1001_1001_f32", "recur_grad", 3, 1001, 1001, "f32", "exp", False, True),
    ]


def _near(rng, low, high):
    """A whole number in [low, high], uniform over its logarithm: a power of two, a round number or an odd one."""
    at = math.exp(rng.uniform(math.log(low), math.log(high)))
    which = rng.random()
    n = 2 ** round(math.log2(at)) if which < 0.3 else 10 * round(at / 10) if which < 0.6 else 2 * round((at - 1) / 2) + 1
    return max(low, min(high, int(n)))


def draw(rng):
    element = rng.choice(["bf16", "bf16", "f16", "f32"])
    wide = 2 if element == "f32" else 1
    if rng.random() < 0.55:
        kind = rng.choice(["rotate", "rotate_grad", "norm_rotate", "norm_rotate", "norm_rotate_grad"])
        heads = rng.choice([1, 2, 4, 6, 8, 12, 16, 32])
        kv_heads = rng.choice([h for h in (1, 2, 4, 6, 8, 12, 16, 32) if heads % h == 0])
        d = rng.choice([32, 64, 64, 80, 96, 128, 128, 192, 256, 2 * rng.randint(5, 64)])
        r = d if rng.random() < 0.6 else 2 * rng.randint(1, d // 2)
        most = (63 << 20) // (wide * (heads + kv_heads) * d * (2 if kind == "norm_rotate_grad" else 1))
        tokens = 1 if rng.random() < 0.25 else _near(rng, 2, max(2, min(32768, most)))
        batch = _near(rng, 1, max(1, min(256, most // tokens)))
        positions = rng.choice(["none", "starts", "starts", "table"])
        far = 0 if positions == "none" else _near(rng, 64, 1 << 20)
        c = _rotate("", kind, batch, tokens, heads, kv_heads, d, element, r, rng.choice(["half", "interleaved"]), positions, far, rng.choice([1, 1, 4, 16]),
                    batch > 1 and rng.random() < 0.3)
    else:
        kind = rng.choice(["recur", "recur", "recur_step", "recur_grad"])
        channels = _near(rng, 16, 8192)
        most = (63 << 20) // (wide * channels * (2 if kind == "recur_grad" else 1))
        tokens = rng.choice([1, 1, 1, 2, 4]) if kind == "recur_step" else _near(rng, 5, min(65536, most))
        batch = _near(rng, 1, max(1, min(256 if kind == "recur_step" else 64, most // tokens)))
        c = _recur("", kind, batch, tokens, channels, element, rng.choice(["sigmoid", "exp"]), rng.random() < 0.6, batch > 1 and rng.random() < 0.4)
    del c["name"]
    return c


def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t, b, n = _TYPES[case["element"]], case["batch"], case["tokens"]

    def normal(*shape, scale=1.0, shift=0.0, dtype=t):
        return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).mul_(scale).add_(shift).to(dtype)

    # lengths from none to all of the tokens
    s = {"lengths": torch.randint(0, n + 1, (b,), generator=g, device="cuda", dtype=torch.int32) if case["ragged"] else None}
    if case["kind"].startswith("recur"):
        c = case["channels"]
        s["x"] = normal(b, n, c)
        # memories of 2 to about a thousand tokens over the channels, moved by the data: logits, or logarithms of the decay
        slow = torch.linspace(0.5, 6.0, c, device="cuda")
        logits = torch.randn((b, n, c), generator=g, device="cuda", dtype=torch.float32).add_(slow)
        s["gate"] = (logits if case["gate"] == "sigmoid" else torch.exp(-logits).mul_(-1.0)).to(t)
        s["state"] = normal(b, c, dtype=torch.float32)
        if case["kind"] == "recur_grad":
            s["dy"] = normal(b, n, c)
            s["dstate"] = normal(b, c, dtype=torch.float32)
        return s
    h, kv, d = case["heads"], case["kv_heads"], case["head_dim"]
    s["starts"] = torch.randint(0, case["far"], (b,), generator=g, device="cuda", dtype=torch.int32) if case["positions"] == "starts" else None
    s["table"] = None
    if case["positions"] == "table":  # documents of about 200 tokens one after the other, each from a position of its own
        at = torch.randint(0, case["far"], (b, n // 200 + 1), generator=g, device="cuda", dtype=torch.int32)
        i = torch.arange(n, device="cuda")
        s["table"] = (at[:, i // 200] + (i % 200)).to(torch.int32)
    norm, grad = case["kind"].startswith("norm"), case["kind"].endswith("grad")
    if norm or not grad:
        s["q"], s["k"] = normal(b, n, h, d, scale=2.0), normal(b, n, kv, d, scale=0.5)
    if norm:
        s["q_weight"], s["k_weight"] = (normal(d, scale=0.2, shift=1.0) for _ in range(2))
    if grad:
        s["dq_out"], s["dk_out"] = normal(b, n, h, d), normal(b, n, kv, d)
    return s


def _frequencies(case):
    """Radians a position for each pair, in 64 bits."""
    r, out = case["rotary_dim"], []
    for i in range(r // 2):
        f = _BASE ** (-2.0 * i / r)
        share = min(1.0, max(0.0, (_TRAINED * f / (2 * math.pi) - _SLOW) / (_FAST - _SLOW)))
        out.append(f * (share + (1 - share) / case["stretch"]))
    return out


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    kind = case["kind"]
    if kind.startswith("recur"):
        s["y"] = torch.empty_like(s["x"])
        s["state_out"] = s["state"] if kind == "recur_step" else torch.empty_like(s["state"])
        if kind == "recur_grad":
            s["dx"], s["dgate"], s["dstate_in"] = (torch.empty_like(s[f]) for f in ("x", "gate", "state"))
    else:
        ends = ("dq_out", "dk_out") if kind.endswith("grad") else ("q", "k")
        s["to_q"], s["to_k"] = (torch.empty_like(s[f]) for f in ends)
        if kind == "norm_rotate_grad":
            s["dq_weight"], s["dk_weight"] = (torch.empty_like(s[f]) for f in ("q_weight", "k_weight"))
        s["frequencies"] = torch.tensor(_frequencies(case), device="cuda", dtype=torch.float64)
    if own:
        vk = _vk()
        element = {"f32": vk.Element.F32, "f16": vk.Element.F16, "bf16": vk.Element.BF16}[case["element"]]
        if kind.startswith("recur"):
            c = vk.GatedRecurrenceConfig.new(case["channels"]).with_element(element).with_complement(case["complement"])
            c.with_gate(vk.Gate.Sigmoid if case["gate"] == "sigmoid" else vk.Gate.Exp)
            s["plan"] = vk.GatedRecurrencePlan(_ctx(vk), c)
            if kind == "recur_grad":
                s["saved"] = torch.empty(s["plan"].saved_shape(case["batch"], case["tokens"]), device="cuda", dtype=torch.float32)
        else:
            c = vk.RotaryConfig.new(case["heads"], case["head_dim"]).with_kv_heads(case["kv_heads"]).with_rotary_dim(case["rotary_dim"]).with_element(element)
            c.with_layout(vk.RotaryLayout.Half if case["layout"] == "half" else vk.RotaryLayout.Interleaved).with_base(_BASE)
            if case["stretch"] != 1:
                c.with_blended_scaling(case["stretch"], _TRAINED, _FAST, _SLOW)
            if kind.startswith("norm"):
                c.with_norm(_EPSILON)
            s["plan"] = vk.RotaryPlan(_ctx(vk), c)
    return s


# ---------------------------------------------------------------- plain forms: elementary operations in 32 bits, angles in 64

def _inside(s, like):
    """1 for rows before a sequence's length, 0 from there on."""
    if s["lengths"] is None:
        return None
    at = torch.arange(like.shape[1], device=like.device, dtype=torch.int32)
    return (at[None] < s["lengths"][:, None]).reshape(list(like.shape[:2]) + [1] * (like.dim() - 2)).float()


def _turns(s, like):
    """Cosine and sine of every token and pair."""
    at = torch.arange(like.shape[1], device=like.device)[None].double()
    if s["table"] is not None:
        at = s["table"].double()
    elif s["starts"] is not None:
        at = s["starts"].double()[:, None] + at
    angle = at[..., None, None] * s["frequencies"]
    return angle.cos().float(), angle.sin().float()


def _turn(x, s, cos, sin):
    r, half = s["case"]["rotary_dim"], s["case"]["layout"] == "half"
    if half:
        a, b = x[..., :r // 2], x[..., r // 2:r]
        return torch.cat([a * cos - b * sin, a * sin + b * cos, x[..., r:]], -1)
    a, b = x[..., 0:r:2], x[..., 1:r:2]
    return torch.cat([torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2), x[..., r:]], -1)


def _only(y, inside, t):
    return (y if inside is None else y * inside).to(t)


def _plain_rotate(s):
    cos, sin = _turns(s, s["q"])
    inside, norm, out = _inside(s, s["q"]), s["case"]["kind"] == "norm_rotate", []
    for x, weight in (("q", "q_weight"), ("k", "k_weight")):
        y = s[x].float()
        if norm:
            y = y * (y.square().mean(-1, keepdim=True) + _EPSILON).rsqrt() * s[weight].float()
        out.append(_only(_turn(y, s, cos, sin), inside, s[x].dtype))
    return out


def _plain_rotate_grad(s):
    cos, sin = _turns(s, s["dq_out"])
    inside = _inside(s, s["dq_out"])
    if s["case"]["kind"] == "rotate_grad":
        return [_only(_turn(s[f].float(), s, cos, -sin), inside, s[f].dtype) for f in ("dq_out", "dk_out")]
    out, weights = [], []
    for x, weight, dy in (("q", "q_weight", "dq_out"), ("k", "k_weight", "dk_out")):
        n = s[x].float()
        rstd = (n.square().mean(-1, keepdim=True) + _EPSILON).rsqrt()
        n = n * rstd
        du = _turn(s[dy].float(), s, cos, -sin)
        du = du if inside is None else du * inside
        g = du * s[weight].float()
        out.append(((g - n * (g * n).mean(-1, keepdim=True)) * rstd).to(s[x].dtype))
        weights.append((du * n).sum((0, 1, 2)).to(s[weight].dtype))
    return out + weights


def _gates(s):
    """a and m for every token; 1 and 0 past a sequence's length."""
    g = s["gate"].float()
    small = torch.exp(-g.abs())
    a = torch.where(g > 0, 1 / (1 + small), small / (1 + small)) if s["case"]["gate"] == "sigmoid" else torch.exp(g.clamp(max=0))
    m = torch.ones_like(a)
    if s["case"]["complement"]:
        m = torch.where(g > 0, small / (1 + small), 1 / (1 + small)) if s["case"]["gate"] == "sigmoid" else -torch.expm1(g.clamp(max=0))
    inside = _inside(s, g)
    return (a, m, None) if inside is None else (1 + (a - 1) * inside, m * inside, inside)


def _scan(a, b):
    """h[t] = a[t] h[t-1] + b[t], h[-1] = 0: twice as many tokens joined each time."""
    n, step = a.shape[1], 1
    while step < n:
        b = torch.cat([b[:, :step], torch.addcmul(b[:, step:], a[:, step:], b[:, :-step])], 1)
        step, a = 2 * step, torch.cat([a[:, :step], a[:, step:] * a[:, :-step]], 1)
    return b


def _plain_recur(s):
    a, m, inside = _gates(s)
    b = m * s["x"].float()
    b[:, 0] += a[:, 0] * s["state"]
    h = _scan(a, b)
    y = _only(h, inside, s["x"].dtype)
    if s["case"]["kind"] == "recur_step":
        s["state"].copy_(h[:, -1])
        return [y, s["state"]]
    if s["case"]["kind"] == "recur":
        return [y, h[:, -1].clone()]
    d = s["dy"].float()
    d = d.clone() if inside is None else d * inside
    d[:, -1] += s["dstate"]
    # D[t] = dy[t] + a[t+1] D[t+1]
    d = _scan(torch.cat([torch.zeros_like(a[:, :1]), a.flip(1)[:, :-1]], 1), d.flip(1)).flip(1)
    da = d * (torch.cat([s["state"][:, None], h[:, :-1]], 1) - (s["x"].float() if s["case"]["complement"] else 0))
    g = s["gate"].float()
    slope = torch.exp(-g.abs()) / (1 + torch.exp(-g.abs())).square() if s["case"]["gate"] == "sigmoid" else a * (g <= 0)
    dg = da * slope
    return [y, h[:, -1].clone(), (m * d).to(s["x"].dtype), _only(dg, inside, s["gate"].dtype), a[:, 0] * d[:, 0]]


_PLAIN = {"rotate": _plain_rotate, "norm_rotate": _plain_rotate, "rotate_grad": _plain_rotate_grad, "norm_rotate_grad": _plain_rotate_grad,
          "recur": _plain_recur, "recur_step": _plain_recur, "recur_grad": _plain_recur}


def run(state):
    s, kind = state, state["case"]["kind"]
    if not own:
        return _PLAIN[kind](s)
    plan = s["plan"]
    if kind in ("recur", "recur_step"):
        plan.forward_tensors(s["x"], s["gate"], s["y"], state_in=s["state"], state_out=s["state_out"], lengths=s["lengths"])
        return [s["y"], s["state_out"]]
    if kind == "recur_grad":
        plan.forward_tensors(s["x"], s["gate"], s["y"], state_in=s["state"], state_out=s["state_out"], saved=s["saved"], lengths=s["lengths"])
        plan.backward_tensors(s["x"], s["gate"], s["saved"], s["dy"], s["dx"], s["dgate"], dstate_out=s["dstate"], dstate_in=s["dstate_in"],
                              lengths=s["lengths"])
        return [s["y"], s["state_out"], s["dx"], s["dgate"], s["dstate_in"]]
    where = {"positions": s["table"], "starts": s["starts"], "lengths": s["lengths"]}
    if kind == "rotate":
        plan.forward_tensors(s["q"], s["k"], s["to_q"], s["to_k"], **where)
    elif kind == "norm_rotate":
        plan.forward_tensors(s["q"], s["k"], s["to_q"], s["to_k"], q_weight=s["q_weight"], k_weight=s["k_weight"], **where)
    elif kind == "rotate_grad":
        plan.backward_tensors(s["dq_out"], s["dk_out"], s["to_q"], s["to_k"], **where)
    else:
        plan.backward_tensors(s["dq_out"], s["dk_out"], s["to_q"], s["to_k"], q=s["q"], k=s["k"], q_weight=s["q_weight"], k_weight=s["k_weight"],
                              dq_weight=s["dq_weight"], dk_weight=s["dk_weight"], **where)
        return [s["to_q"], s["to_k"], s["dq_weight"], s["dk_weight"]]
    return [s["to_q"], s["to_k"]]


def work(case):
    """Every input is read once and every output written once (a training step's two passes as if x and gate stayed at hand between them).
    A rotated element costs 3 operations, its norm 4, the gradients of both 12; a recurrence's channel costs about 10 a token, its gradients 15 more."""
    size, b, n = 4 if case["element"] == "f32" else 2, case["batch"], case["tokens"]
    if case["kind"].startswith("recur"):
        c = case["channels"]
        grad = case["kind"] == "recur_grad"
        return {"bytes": size * b * n * c * (6 if grad else 3) + 4 * b * c * (4 if grad else 2), "flops": (25.0 if grad else 10.0) * b * n * c}
    e, d = b * n * (case["heads"] + case["kv_heads"]) * case["head_dim"], case["head_dim"]
    more = {"none": 0, "starts": 4 * b, "table": 4 * b * n}[case["positions"]]
    if case["kind"] == "norm_rotate_grad":
        return {"bytes": size * (3 * e + 4 * d) + more, "flops": 15.0 * e}
    return {"bytes": size * 2 * e + (2 * size * d if case["kind"] == "norm_rotate" else 0) + more, "flops": (7.0 if case["kind"] == "norm_rotate" else 3.0) * e}


# ---------------------------------------------------------------- the definitions in 64 bits: turns as complex numbers, the recurrence token by token

def exact(case, seed):
    s = {f: x.double() if torch.is_tensor(x) and x.is_floating_point() else x for f, x in _inputs(case, seed).items()}
    return _exact_recur(case, s) if case["kind"].startswith("recur") else _exact_rotate(case, s)


def _exact_rotate(case, s):
    r, d, b, n = case["rotary_dim"], case["head_dim"], case["batch"], case["tokens"]
    i = torch.arange(r // 2, device="cuda", dtype=torch.float64)
    f = torch.pow(torch.tensor(_BASE, device="cuda", dtype=torch.float64), -2 * i / r)
    share = ((f * _TRAINED / (2 * math.pi) - _SLOW) / (_FAST - _SLOW)).clamp(0, 1)
    f = f * share + f * (1 - share) / case["stretch"]
    p = torch.arange(n, device="cuda", dtype=torch.float64).expand(b, n)
    if case["positions"] == "table":
        p = s["table"].double()
    elif case["positions"] == "starts":
        p = p + s["starts"].double().unsqueeze(1)
    turn = torch.polar(torch.ones(b, n, r // 2, device="cuda", dtype=torch.float64), p.unsqueeze(2) * f).unsqueeze(2)
    live = torch.ones(b, n, 1, 1, device="cuda", dtype=torch.float64)
    if s["lengths"] is not None:
        live = (torch.arange(n, device="cuda").unsqueeze(0) < s["lengths"].unsqueeze(1)).double().reshape(b, n, 1, 1)
    first, second = (slice(0, r // 2), slice(r // 2, r)) if case["layout"] == "half" else (slice(0, r, 2), slice(1, r, 2))

    def by(x, z):
        out = x.clone()
        c = torch.complex(x[..., first].contiguous(), x[..., second].contiguous()) * z
        out[..., first], out[..., second] = c.real, c.imag
        return out

    pairs = (("q", "q_weight", "dq_out"), ("k", "k_weight", "dk_out"))
    if case["kind"] == "rotate":
        return [by(s[x], turn) * live for x, _, _ in pairs]
    if case["kind"] == "rotate_grad":
        return [by(s[dy], turn.conj()) * live for _, _, dy in pairs]
    out, weights = [], []
    for x, w, dy in pairs:
        root = torch.sqrt((s[x] ** 2).sum(3, keepdim=True) / d + _EPSILON)
        if case["kind"] == "norm_rotate":
            out.append(by(s[x] / root * s[w], turn) * live)
            continue
        du = by(s[dy], turn.conj()) * live
        out.append(du * s[w] / root - s[x] / root ** 3 * (du * s[w] * s[x]).sum(3, keepdim=True) / d)
        weights.append((du * s[x] / root).flatten(0, 2).sum(0))
    return out + weights


def _exact_recur(case, s):
    b, n, c = case["batch"], case["tokens"], case["channels"]
    lengths = [n] * b if s["lengths"] is None else s["lengths"].tolist()
    last = torch.tensor(lengths, device="cuda").reshape(b, 1)
    sigmoid, whole = case["gate"] == "sigmoid", min(lengths) == n

    def gates(t):
        g = s["gate"][:, t]
        a = torch.special.expit(g) if sigmoid else torch.exp(torch.clamp(g, max=0))
        return g, a, 1 - a if case["complement"] else torch.ones_like(a)

    h, y = s["state"].clone(), torch.zeros(b, n, c, device="cuda", dtype=torch.float64)
    before = torch.zeros_like(y) if case["kind"] == "recur_grad" else None
    for t in range(max(lengths)):
        _, a, m = gates(t)
        if before is not None:
            before[:, t] = h
        new = a * h + m * s["x"][:, t]
        h = new if whole else torch.where(t < last, new, h)
        y[:, t] = new if whole else torch.where(t < last, new, 0.0)
    if case["kind"] != "recur_grad":
        return [y, h]
    dx, dg, back = torch.zeros_like(y), torch.zeros_like(y), s["dstate"].clone()  # of the state after token t, then before it
    for t in reversed(range(max(lengths))):
        g, a, m = gates(t)
        total = back + s["dy"][:, t]
        da = total * (before[:, t] - s["x"][:, t] if case["complement"] else before[:, t])
        slope = a * torch.special.expit(-g) if sigmoid else torch.where(g > 0, 0.0, a)
        here = (t < last).expand(b, c)
        dx[:, t] = torch.where(here, m * total, 0.0)
        dg[:, t] = torch.where(here, da * slope, 0.0)
        back = torch.where(here, a * total, back)
    return [y, h, dx, dg, back]
