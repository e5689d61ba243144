"""The sequence operators' definitions in 64 bits, token by token on the host,
and how far a result may be from them.

A result's bound is u |y| for its one rounding to the element type plus c A,
where A is the same formula over the absolute values of every term (what a sum
can lose to cancellation) and c the relative error of the terms:

  linear attention: products of 16-bit inputs are exact in 32-bit sums; scores
  and states enter the second product in two 8-bit parts, so a term keeps 2^-17
  and, with weights and sums in 32 bits, c = 2^-15. In full precision every
  factor has 24 bits and a sum of some hundred terms c = 2^-18. States and
  their gradients take three parts, c = 2^-18 for every element type.
  layer norm: all in 32 bits, a few roundings on each term, c = 2^-19.
"""
import numpy as np

UNIT = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
SUBNORMAL = {"f32": 2.0 ** -149, "f16": 2.0 ** -25, "bf16": 2.0 ** -134}
TERM = {"f32": 2.0 ** -18, "f16": 2.0 ** -15, "bf16": 2.0 ** -15}
STATE_TERM = 2.0 ** -18
NORM_TERM = 2.0 ** -19


def attention(q, k, v, state, decay, scale, lengths):
    """q [b][t][h][dk], k and v [b][t][kv][.], state [b][h][dk][dv] -> out, state."""
    b, t, h, _ = q.shape
    k, v = (np.repeat(x, h // k.shape[2], axis=2) for x in (k, v))
    decay = np.asarray(decay, np.float64).reshape(1, h, 1, 1)
    s = state.copy()
    out = np.zeros((b, t, h, v.shape[3]))
    for i in range(t):
        here = i < lengths
        if not here.any():
            break
        n = decay * s + k[:, i, :, :, None] * v[:, i, :, None, :]
        s[here] = n[here]
        out[here, i] = scale * (q[:, i, :, None, :] @ n)[here, :, 0]
    return out, s


def attention_gradients(q, k, v, state, dout, dstate, decay, scale, lengths):
    """-> dq, dk, dv (summed over a shared head's query heads), dstate_in."""
    b, t, h, _ = q.shape
    kv = k.shape[2]
    k, v = (np.repeat(x, h // kv, axis=2) for x in (k, v))
    decay = np.asarray(decay, np.float64).reshape(1, h, 1, 1)
    dq, dk, dv = np.zeros_like(q), np.zeros_like(k), np.zeros_like(v)
    s = state.copy()
    for i in range(t):
        here = i < lengths
        s[here] = (decay * s + k[:, i, :, :, None] * v[:, i, :, None, :])[here]
        dq[here, i] = scale * (s @ dout[:, i, :, :, None])[here, :, :, 0]
    g = dstate.copy()
    for i in reversed(range(t)):
        here = i < lengths
        g[here] += scale * (q[:, i, :, :, None] * dout[:, i, :, None, :])[here]
        dk[here, i] = (g @ v[:, i, :, :, None])[here, :, :, 0]
        dv[here, i] = (k[:, i, :, None, :] @ g)[here, :, 0]
        g[here] = (decay * g)[here]
    dk, dv = (x.reshape(b, t, kv, h // kv, -1).sum(3) for x in (dk, dv))
    return dq, dk, dv, g


def norm(x, weight, bias, epsilon):
    mean = x.mean(1, keepdims=True)
    rstd = 1 / np.sqrt(x.var(1, keepdims=True) + epsilon)
    return (x - mean) * rstd * weight + bias, np.concatenate([mean, rstd], 1)


def norm_bound(x, weight, bias, stats):
    """A of y: every summand of (x - mean) rstd weight + bias, x and mean apart."""
    big = np.abs(x) + np.abs(x).mean(1, keepdims=True)
    return big * stats[:, 1:] * np.abs(weight) + np.abs(bias)


def norm_gradients(x, weight, stats, dy):
    n = (x - stats[:, :1]) * stats[:, 1:]
    g = dy * weight
    dx = stats[:, 1:] * (g - g.mean(1, keepdims=True) - n * (g * n).mean(1, keepdims=True))
    return dx, (dy * n).sum(0), dy.sum(0)


def norm_gradients_bound(x, weight, stats, dy):
    n = (np.abs(x) + np.abs(stats[:, :1])) * stats[:, 1:]
    g = np.abs(dy * weight)
    dx = stats[:, 1:] * (g + g.mean(1, keepdims=True) + n * (g * n).mean(1, keepdims=True))
    return dx, (np.abs(dy) * n).sum(0), np.abs(dy).sum(0)


def check(name, got, want, total, element, term):
    """got: a torch tensor; want and total (A): arrays in 64 bits."""
    y = got.detach().double().cpu().numpy()
    assert y.shape == want.shape, (name, y.shape, want.shape)
    assert np.isfinite(y).all(), f"{name}: not finite"
    allowed = UNIT[element] * np.abs(want) + (1 + UNIT[element]) * term * total + SUBNORMAL[element]
    over = np.abs(y - want) - allowed
    at = np.unravel_index(np.argmax(over), over.shape) if over.size else ()
    assert not over.size or over[at] <= 0, f"{name}{list(map(int, at))}: {y[at]} for {want[at]}, allowed {allowed[at]}"
