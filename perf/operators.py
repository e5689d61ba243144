"""Performance cases of the sequence operators: layer norm and linear attention with a decay for each head, forward, backward and token by token.

A program makes a plan for its widths and heads once, keeps it with its buffers, and calls it for every new input; so `prepare` makes the inputs,
the output buffers and (for the framework's own operators) the plan, and `run` makes one call. The five "kind"s:

  norm           layer norm of rows: y, and each row's mean and reciprocal deviation for a later backward pass
  norm_grad      its backward pass: gradients of x, weight and bias
  attention      linear attention over a prompt of a batch of sequences, from a state to the next: outputs and the state after the last token
  step           the same for one new token of each sequence (a few with speculation): the state is updated in place
  attention_grad its backward pass: gradients of q, k, v and of the initial state, with a gradient arriving at the final state

Linear attention of one head with decay g, keys of dk and values of dv elements, state S (dk x dv):
  S[t] = g S[t-1] + k[t] v[t]^T        o[t] = scale q[t] S[t]
Query heads share key and value heads in groups of heads / kv_heads; each query head has its own decay and state. A sequence of a batch may be
shorter than the batch's tokens ("ragged"): its rows from its length on give zeros and leave the state alone.
"""
import math
import os
import sys

import torch

own = False

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
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


def _norm(name, rows, width, element, grad=False):
    return {"name": name, "kind": "norm_grad" if grad else "norm", "rows": rows, "width": width, "element": element}


def _attention(name, kind, batch, tokens, heads, kv_heads, key_dim, value_dim, element, ragged=False):
    return {"name": name, "kind": kind, "batch": batch, "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "key_dim": key_dim,
            "value_dim": value_dim, "element": element, "ragged": ragged}


def listed():
    return [
        # the rows of four sequences that each get one token: latency
        _norm("norm_4x1024_bf16", 4, 1024, "bf16"),
        # the rows of a prompt or a training batch
        _norm("norm_8192x4096_bf16", 8192, 4096, "bf16"),
        # prime counts and an odd width in full precision: rows that start at any alignment
        _norm("norm_4099x1001_f32", 4099, 1001, "f32"),
        # a training batch's backward pass
        _norm("norm_grad_8192x4096_bf16", 8192, 4096, "bf16", True),
        # many short rows, as in a norm over each head's output
        _norm("norm_grad_65537x128_f16", 65537, 128, "f16", True),
        # prompts of a serving batch
        _attention("attention_8x2048_h16_128_bf16", "attention", 8, 2048, 16, 16, 128, 128, "bf16"),
        # one long document with shared key and value heads: little to run side by side but the sequence itself
        _attention("attention_1x65536_h16_4_64_bf16", "attention", 1, 65536, 16, 4, 64, 64, "bf16"),
        # uneven heads, sequences of uneven lengths, full precision
        _attention("attention_3x1001_h12_4_80x96_f32", "attention", 3, 1001, 12, 4, 80, 96, "f32", True),
        # one sequence answering token by token: latency
        _attention("step_1_h16_128_bf16", "step", 1, 1, 16, 16, 128, 128, "bf16"),
        # a full serving batch answering token by token: the states' bytes
        _attention("step_256_h16_128_bf16", "step", 256, 1, 16, 16, 128, 128, "bf16"),
        # a training batch's backward pass
        _attention("attention_grad_4x4096_h16_128_bf16", "attention_grad", 4, 4096, 16, 16, 128, 128, "bf16"),
        # the same with shared heads, uneven widths and uneven lengths
        _attention("attention_grad_6x1215_h8_2_64x112_f16", "attention_grad", 6, 1215, 8, 2, 64, 112, "f16", True),
    ]


def _near(rng, low, high):
    """A whole number in [low, high], uniform over its logarithm: a power of two, a round number or an odd one."""
    at = math.exp(rng.uniform(math.log(low), math.log(high)))
    which = rng.random()
    n = 2 ** round(math.log2(at)) if which < 0.3 else 10 * round(at / 10) if which < 0.6 else 2 * round((at - 1) / 2) + 1
    return max(low, min(high, int(n)))


def draw(rng):
    element = rng.choice(["bf16", "bf16", "f16", "f32"])
    if rng.random() < 0.4:
        width = _near(rng, 16, 16384)
        most = (1 << 25) // (width * (2 if element == "f32" else 1))
        c = _norm("", _near(rng, 1, max(1, min(65537, most))), width, element, rng.random() < 0.5)
    else:
        kind = rng.choice(["attention", "attention", "step", "attention_grad"])
        heads = rng.choice([1, 2, 4, 6, 8, 12, 16, 32])
        kv_heads = rng.choice([h for h in (1, 2, 4, 6, 8, 12, 16, 32) if heads % h == 0])
        key_dim, value_dim = (rng.choice([16, 32, 64, 64, 80, 96, 128, 128, 192, 256, rng.randint(9, 127)]) for _ in range(2))
        if kind == "step":
            tokens = rng.choice([1, 1, 1, 2, 4])
            batch = _near(rng, 1, max(1, min(256, (1 << 26) // (heads * key_dim * value_dim))))
        else:
            tokens = _near(rng, 5, 65536)
            most = (1 << (25 if element == "f32" else 26)) // (heads * (key_dim + value_dim))
            most = min(most, (1 << 32) // (heads * key_dim * value_dim))
            tokens = max(1, min(tokens, most // (2 if kind == "attention_grad" else 1)))
            batch = _near(rng, 1, max(1, min(64, most // (tokens * (2 if kind == "attention_grad" else 1)))))
        c = _attention("", kind, batch, tokens, heads, kv_heads, key_dim, value_dim, element, batch > 1 and rng.random() < 0.4)
    del c["name"]
    return c


def _decays(case):
    """1 - 2^-a, memories of 8 to 512 tokens over the heads: numbers that 32 bits hold exactly."""
    h = case["heads"]
    return [1.0 - 2.0 ** -(3 + (6 * i) // max(1, h - 1)) for i in range(h)]


def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = _TYPES[case["element"]]

    def normal(*shape, scale=1.0, shift=0.0, dtype=t):
        return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).mul_(scale).add_(shift).to(dtype)

    if case["kind"] in ("norm", "norm_grad"):
        n, d = case["rows"], case["width"]
        s = {"x": normal(n, d, scale=1.5, shift=0.4), "weight": normal(d, scale=0.2, shift=1.0), "bias": normal(d, scale=0.2)}
        if case["kind"] == "norm_grad":
            x = s["x"].double()
            s["stats"] = torch.stack([x.mean(1), (x.var(1, unbiased=False) + 1e-5).rsqrt()], 1).float()
            s["dy"] = normal(n, d)
        return s
    b, n, h, kv, dk, dv = (case[f] for f in ("batch", "tokens", "heads", "kv_heads", "key_dim", "value_dim"))
    s = {"q": normal(b, n, h, dk), "k": normal(b, n, kv, dk), "v": normal(b, n, kv, dv), "state": normal(b, h, dk, dv, scale=3.0, dtype=torch.float32)}
    # lengths from none to all of the tokens
    s["lengths"] = torch.randint(0, n + 1, (b,), generator=g, device="cuda", dtype=torch.int32) if case["ragged"] else None
    if case["kind"] == "attention_grad":
        s["dout"] = normal(b, n, h, dv)
        s["dstate"] = normal(b, h, dk, dv, dtype=torch.float32)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    norm = case["kind"] in ("norm", "norm_grad")
    if case["kind"] == "norm":
        s["y"] = torch.empty_like(s["x"])
        s["stats"] = torch.empty(case["rows"], 2, device="cuda", dtype=torch.float32)
    elif case["kind"] == "norm_grad":
        s["dx"], s["dweight"], s["dbias"] = (torch.empty_like(s[f]) for f in ("x", "weight", "bias"))
    elif case["kind"] == "attention_grad":
        s["dq"], s["dk"], s["dv"], s["dstate_in"] = (torch.empty_like(s[f]) for f in ("q", "k", "v", "state"))
    else:
        s["out"] = torch.empty(case["batch"], case["tokens"], case["heads"], case["value_dim"], device="cuda", dtype=_TYPES[case["element"]])
        s["state_out"] = s["state"] if case["kind"] == "step" else torch.empty_like(s["state"])
    if not norm:
        s["decay"] = torch.tensor(_decays(case), device="cuda", dtype=torch.float32)
        s["scale"] = 1.0 / math.sqrt(case["key_dim"])
    if own:
        vk = _vk()
        element = {"f32": vk.Element.F32, "f16": vk.Element.F16, "bf16": vk.Element.BF16}[case["element"]]
        if norm:
            s["plan"] = vk.LayerNormPlan(_ctx(vk), vk.LayerNormConfig.new(case["width"]).with_element(element).with_epsilon(1e-5))
        else:
            c = vk.LinearAttentionConfig.new(case["heads"], case["key_dim"], case["value_dim"]).with_kv_heads(case["kv_heads"]).with_element(element)
            c.with_decay(_decays(case)).with_scale(s["scale"]).with_capacity(case["batch"], case["tokens"])
            c.with_gradient(case["kind"] == "attention_grad")
            s["plan"] = vk.LinearAttentionPlan(_ctx(vk), c)
    return s


# ---------------------------------------------------------------- plain forms: elementary operations in 32 bits

def _plain_norm(s):
    x = s["x"].float()
    mean = x.mean(1, keepdim=True)
    x = x - mean
    rstd = (x.square().mean(1, keepdim=True) + 1e-5).rsqrt()
    return [(x * rstd * s["weight"].float() + s["bias"].float()).to(s["x"].dtype), torch.cat([mean, rstd], 1)]


def _plain_norm_grad(s):
    mean, rstd = s["stats"][:, :1], s["stats"][:, 1:]
    x = (s["x"].float() - mean) * rstd
    dy = s["dy"].float()
    g = dy * s["weight"].float()
    dx = (g - g.mean(1, keepdim=True) - x * (g * x).mean(1, keepdim=True)) * rstd
    return [dx.to(s["x"].dtype), (dy * x).sum(0).to(s["weight"].dtype), dy.sum(0).to(s["bias"].dtype)]


def _heads(x, heads):
    """[batch][token][head][dim] in 32 bits with the heads in front, shared ones repeated."""
    return x.float().transpose(1, 2).repeat_interleave(heads // x.shape[2], 1)


def _steps(n, s):
    return torch.arange(n, device=s["q"].device, dtype=torch.float32)


def _power(decay, exponent):
    """decay^exponent for each head, 0 for negative exponents."""
    at = exponent.clamp(min=0)
    return torch.where(exponent >= 0, decay.reshape([-1] + [1] * (exponent.dim() - 1)).pow(at), torch.zeros_like(at))


def _scan(q, k, v, s, state=None):
    """sum over j <= i of decay^(i-j) (q[i] k[j]) v[j], plus decay^(i+1) q[i] state, in chunks of about the square root of the length."""
    n, decay = q.shape[2], s["decay"]
    c = 1 << max(0, math.ceil(math.log2(max(1, n)) / 2))
    m = -(-n // c)
    q, k, v = (torch.nn.functional.pad(x, (0, 0, 0, m * c - n)).reshape(x.shape[0], x.shape[1], m, c, x.shape[3]) for x in (q, k, v))
    i, r = _steps(c, s)[None], _steps(m, s)[None]
    out = (q @ k.transpose(3, 4) * _power(decay, i[:, :, None] - i[:, None])[:, None]) @ v
    sums = (k * _power(decay, c - 1 - i)[:, None, :, None]).transpose(3, 4) @ v
    before = (_power(decay, c * (r[:, :, None] - 1 - r[:, None])) @ sums.flatten(3)).reshape(sums.shape)
    if state is not None:
        before = before + _power(decay, c * r)[:, :, None, None] * state[:, :, None]
    out = out + _power(decay, i + 1)[:, None, :, None] * (q @ before)
    return out.flatten(2, 3)[:, :, :n]


def _lengths(s):
    b, n = s["q"].shape[:2]
    length = s["lengths"].float() if s["lengths"] is not None else torch.full((b,), float(n), device=s["q"].device)
    return length, (_steps(n, s)[None] < length[:, None])[:, None, :, None]


def _rows(x, t):
    return x.transpose(1, 2).to(t)


def _plain_attention(s):
    heads, decay = s["q"].shape[2], s["decay"]
    length, inside = _lengths(s)
    q, k, v = (_heads(s[f], heads) * inside for f in ("q", "k", "v"))
    out = _scan(q, k, v, s, s["state"]) * s["scale"] * inside
    left = _power(decay, (length[:, None] - 1 - _steps(q.shape[2], s)[None])[None])  # head, batch, token
    state = (k * left.transpose(0, 1)[..., None]).transpose(2, 3) @ v + _power(decay, length[None]).T[:, :, None, None] * s["state"]
    return [_rows(out, s["q"].dtype), state]


def _plain_step(s):
    """The recurrence itself where there is one token; the state is updated in place."""
    if s["q"].shape[1] > 1 or s["lengths"] is not None:
        out, state = _plain_attention(s)
        s["state"].copy_(state)
        return [out, s["state"]]
    heads = s["q"].shape[2]
    q, k, v = (_heads(s[f], heads) for f in ("q", "k", "v"))
    s["state"].mul_(s["decay"][:, None, None]).add_(k.transpose(2, 3) * v)
    return [_rows(q @ s["state"] * s["scale"], s["q"].dtype), s["state"]]


def _shared(x, kv_heads):
    """Gradients of the query heads' copies of a shared head, summed."""
    return x.reshape(x.shape[0], kv_heads, -1, x.shape[2], x.shape[3]).sum(2)


def _plain_attention_grad(s):
    heads, kv, decay, t = s["q"].shape[2], s["k"].shape[2], s["decay"], s["q"].dtype
    length, inside = _lengths(s)
    q, k, v, do = (_heads(s[f], heads) * inside for f in ("q", "k", "v", "dout"))
    do = do * s["scale"]
    at = _steps(q.shape[2], s)[None]
    dq = _scan(do, v, k, s, s["state"].transpose(2, 3))
    left = _power(decay, (length[:, None] - 1 - at)[None]).transpose(0, 1)[..., None]  # from each token to the end of its sequence
    qr, kr, vr, dor = (x.flip(2) for x in (q, k, v, do))
    dk = _scan(vr, dor, qr, s).flip(2) + left * (v @ s["dstate"].transpose(2, 3))
    dv = _scan(kr, qr, dor, s).flip(2) + left * (k @ s["dstate"])
    dstate = (q * _power(decay, at + 1)[None, :, :, None]).transpose(2, 3) @ do + _power(decay, length[None]).T[:, :, None, None] * s["dstate"]
    return [_rows(dq * inside, t), _rows(_shared(dk * inside, kv), t), _rows(_shared(dv * inside, kv), t), dstate]


_PLAIN = {"norm": _plain_norm, "norm_grad": _plain_norm_grad, "attention": _plain_attention, "step": _plain_step, "attention_grad": _plain_attention_grad}


def run(state):
    s, kind = state, state["case"]["kind"]
    if not own:
        return _PLAIN[kind](s)
    if kind == "norm":
        s["plan"].forward_tensors(s["x"], s["weight"], s["bias"], s["y"], s["stats"])
        return [s["y"], s["stats"]]
    if kind == "norm_grad":
        s["plan"].backward_tensors(s["x"], s["weight"], s["stats"], s["dy"], s["dx"], s["dweight"], s["dbias"])
        return [s["dx"], s["dweight"], s["dbias"]]
    if kind == "attention_grad":
        s["plan"].backward_tensors(s["q"], s["k"], s["v"], s["dout"], s["dq"], s["dk"], s["dv"], state_in=s["state"], dstate_out=s["dstate"],
                                   dstate_in=s["dstate_in"], lengths=s["lengths"])
        return [s["dq"], s["dk"], s["dv"], s["dstate_in"]]
    s["plan"].forward_tensors(s["q"], s["k"], s["v"], s["out"], state_in=s["state"], state_out=s["state_out"], lengths=s["lengths"])
    return [s["out"], s["state_out"]]


def work(case):
    """Every input is read once and every output written once. A token of a head costs a multiplication and an addition for each element of the
    state to update it and as many to read it; backwards, the state is formed again and read, and its gradient formed and read twice."""
    size = 4 if case["element"] == "f32" else 2
    if case["kind"] in ("norm", "norm_grad"):
        n, d = case["rows"], case["width"]
        if case["kind"] == "norm":
            return {"bytes": size * (2 * n * d + 2 * d) + 8 * n, "flops": 8.0 * n * d}
        return {"bytes": size * (3 * n * d + 3 * d) + 8 * n, "flops": 13.0 * n * d}
    b, n, h, kv, dk, dv = (case[f] for f in ("batch", "tokens", "heads", "kv_heads", "key_dim", "value_dim"))
    state = 4 * b * h * dk * dv
    if case["kind"] == "attention_grad":
        return {"bytes": size * b * n * (h * (2 * dk + dv) + 2 * kv * (dk + dv)) + 3 * state, "flops": 10.0 * b * n * h * dk * dv}
    return {"bytes": size * b * n * (h + kv) * (dk + dv) + 2 * state, "flops": 4.0 * b * n * h * dk * dv}


# ---------------------------------------------------------------- the definition in 64 bits, token by token

def exact(case, seed):
    s = {f: x.double() if torch.is_tensor(x) and x.is_floating_point() else x for f, x in _inputs(case, seed).items()}
    if case["kind"] == "norm":
        mean, var = s["x"].mean(1), s["x"].var(1, unbiased=False)
        rstd = 1.0 / torch.sqrt(var + 1e-5)
        return [torch.addcmul(s["bias"], (s["x"] - mean[:, None]) * rstd[:, None], s["weight"]), torch.stack([mean, rstd], 1)]
    if case["kind"] == "norm_grad":
        rstd = s["stats"][:, 1].unsqueeze(1)
        n = (s["x"] - s["stats"][:, 0].unsqueeze(1)) * rstd
        dn = s["dy"] * s["weight"]
        d = case["width"]
        return [rstd * (dn - dn.sum(1, keepdim=True) / d - n * (dn * n).sum(1, keepdim=True) / d), (n * s["dy"]).sum(0), s["dy"].sum(0)]
    b, n, h, kv, dk, dv = (case[f] for f in ("batch", "tokens", "heads", "kv_heads", "key_dim", "value_dim"))
    if n * b * h * dk * dv > 1 << 35:
        return None
    group, scale = h // kv, 1.0 / math.sqrt(dk)
    decay = torch.tensor(_decays(case), device="cuda", dtype=torch.float64).reshape(1, h, 1, 1)
    lengths = [n] * b if s["lengths"] is None else s["lengths"].tolist()
    length = torch.tensor(lengths, device="cuda").reshape(b, 1, 1, 1)
    whole = min(lengths) == n
    wide = [torch.arange(h, device="cuda") // group]
    state = s["state"].clone()
    if case["kind"] == "attention_grad":
        return _exact_grad(s, b, n, h, kv, group, scale, decay, length, lengths, state)
    out = torch.zeros(b, n, h, dv, device="cuda", dtype=torch.float64)
    for t in range(max(lengths)):
        k, v = s["k"][:, t][:, wide[0]], s["v"][:, t][:, wide[0]]
        new = decay * state + k[..., :, None] * v[..., None, :]
        o = scale * (s["q"][:, t][..., None, :] @ new)[..., 0, :]
        if whole:
            state, out[:, t] = new, o
        else:
            here = t < length
            state, out[:, t] = torch.where(here, new, state), torch.where(here[..., 0], o, torch.zeros_like(o))
    return [out, state]


def _exact_grad(s, b, n, h, kv, group, scale, decay, length, lengths, state):
    at = torch.arange(h, device="cuda") // group
    dq, dk, dv = (torch.zeros_like(s[f]) for f in ("q", "k", "v"))
    for t in range(max(lengths)):
        here = t < length
        state = torch.where(here, decay * state + s["k"][:, t][:, at][..., :, None] * s["v"][:, t][:, at][..., None, :], state)
        dq[:, t] = torch.where(here[..., 0], scale * (state @ s["dout"][:, t][..., None])[..., 0], 0.0)
    grad = s["dstate"].clone()  # of the state after token t, then before it
    for t in reversed(range(max(lengths))):
        here = t < length
        grad = torch.where(here, grad + scale * s["q"][:, t][..., :, None] * s["dout"][:, t][..., None, :], grad)
        a = (grad @ s["v"][:, t][:, at][..., None])[..., 0]
        c = (s["k"][:, t][:, at][..., None, :] @ grad)[..., 0, :]
        dk[:, t] = torch.where(here[..., 0], a, 0.0).reshape(b, kv, group, -1).sum(2)
        dv[:, t] = torch.where(here[..., 0], c, 0.0).reshape(b, kv, group, -1).sum(2)
        grad = torch.where(here, decay * grad, grad)
    return [dq, dk, dv, grad]
