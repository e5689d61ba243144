"""Rotary positions, head norms and the gated recurrence in 64 bits on the host,
and how far a result in 32-bit arithmetic may be from them.

Rotary: y1 = u1 c - u2 s. The products, their sum, cosine and sine (each off by
at most 2^-22.5 of itself) and the amplitude's rounding: 2^-21 of |u1 c| + |u2 s|.
Angles are whole multiples of 2^-64 turns: at positions up to 2^31 off by 2^-31
radians, and rounded to 24 bits; both 2^-29 of |u1| + |u2| at most. In front of
the norm, as for layer norm: a few roundings on each term, 2^-19 of the terms.
Sums over rows are formed in 64 bits from such terms.

Recurrence: bounds that follow the recurrence itself. With A the same formula
over absolute values, a step rounds at most four times, 2^-24 of A each; the
smaller of a and 1 - a is off by at most 2^-21 of itself (its exponential 2^-22.5,
a sum, a quotient and a product 2^-24 each), and so is m. An error e of the state
decays as the state does: e[t] = a e[t-1] + 2^-22 A[t] + 2^-21 (min(a, 1 - a) A[t-1] + m |x|).
"""
import numpy as np

from sequence_reference import SUBNORMAL, UNIT, check  # noqa: F401

TURN_TERM, ANGLE, NORM_TERM = 2.0 ** -21, 2.0 ** -8, 2.0 ** -19
STEP, GATE = 2.0 ** -22, 2.0 ** -21


def angles(positions, frequencies):
    """Cosine and sine of [b][t][pair]; long doubles keep far angles."""
    a = np.asarray(positions, np.longdouble)[..., None] * np.asarray(frequencies, np.longdouble)
    return np.cos(a).astype(np.float64), np.sin(a).astype(np.float64)


def halves(x, r, half):
    return (x[..., :r // 2], x[..., r // 2:r]) if half else (x[..., 0:r:2], x[..., 1:r:2])


def turn(x, cos, sin, r, half, amplitude=1.0):
    """x [b][t][h][d] turned, and the sizes of its terms, angles' errors among them."""
    y, total = x.copy(), np.abs(x)
    a, b = halves(x, r, half)
    c, s = cos[:, :, None] * amplitude, sin[:, :, None] * amplitude
    y1, y2 = halves(y, r, half)
    t1, t2 = halves(total, r, half)
    more = ANGLE * abs(amplitude) * (np.abs(a) + np.abs(b))
    y1[...], y2[...] = a * c - b * s, a * s + b * c
    t1[...], t2[...] = np.abs(a * c) + np.abs(b * s) + more, np.abs(a * s) + np.abs(b * c) + more
    return y, total


def rms(x, weight, epsilon):
    """n, u = n weight, rstd."""
    rstd = 1 / np.sqrt((x * x).mean(-1, keepdims=True) + epsilon)
    return x * rstd, x * rstd * weight, rstd


def turn_back(dy, cos, sin, r, half, amplitude=1.0):
    return turn(dy, cos, -sin, r, half, amplitude)


def rms_gradients(x, weight, epsilon, du, size, live):
    """dx and dweight for du (of terms `size`), and their terms' sizes; rows outside `live` have none."""
    n, _, rstd = rms(x, weight, epsilon)
    du, size = du * live, size * live
    g, gs = du * weight, size * np.abs(weight)
    dx = rstd * (g - n * (g * n).mean(-1, keepdims=True))
    dxs = rstd * (gs + np.abs(n) * (gs * np.abs(n)).mean(-1, keepdims=True))
    return dx, dxs, (du * n).sum((0, 1, 2)), (size * np.abs(n)).sum((0, 1, 2))


def gates(gate, sigmoid, complement):
    """a, 1 - a, m and da/dgate."""
    with np.errstate(over="ignore", under="ignore"):
        e = np.exp(-np.abs(gate))
        if sigmoid:
            a, w = np.where(gate > 0, 1 / (1 + e), e / (1 + e)), np.where(gate > 0, e / (1 + e), 1 / (1 + e))
            slope = e / (1 + e) ** 2
        else:
            g = np.minimum(gate, 0)
            a, w = np.exp(g), -np.expm1(g)
            slope = np.where(gate > 0, 0.0, a)
    return a, w, w if complement else np.ones_like(a), slope


def recurrence(x, gate, state, lengths, sigmoid, complement):
    """y and the last state with their bounds, and h, A and e before every token."""
    b, t, c = x.shape
    a, w, m, _ = gates(gate, sigmoid, complement)
    h, A, e = state.copy(), np.abs(state), np.zeros_like(state)
    y, ye = np.zeros_like(x), np.zeros_like(x)
    before = [np.zeros_like(x) for _ in range(3)]
    for i in range(t):
        here = (i < lengths)[:, None]
        for k, v in zip(before, (h, A, e)):
            k[:, i] = v
        size = m[:, i] * np.abs(x[:, i])
        An = a[:, i] * A + size
        en = a[:, i] * e + STEP * An + GATE * (np.minimum(a, w)[:, i] * A + size)
        h, e, A = (np.where(here, n, o) for n, o in ((a[:, i] * h + m[:, i] * x[:, i], h), (en, e), (An, A)))
        y[:, i], ye[:, i] = np.where(here, h, 0), np.where(here, e, 0)
    return y, ye, h, e, before


def recurrence_gradients(x, gate, before, dy, dstate, lengths, sigmoid, complement):
    """dx, dgate and the first state's gradient, each with its bound."""
    b, t, c = x.shape
    a, w, m, slope = gates(gate, sigmoid, complement)
    h, H, he = before
    E, A, e = dstate.copy(), np.abs(dstate), np.zeros_like(dstate)
    dx, dxe, dg, dge = (np.zeros_like(x) for _ in range(4))
    for i in reversed(range(t)):
        here = (i < lengths)[:, None]
        D, S = dy[:, i] + E, np.abs(dy[:, i]) + A
        De = e + STEP * S
        dx[:, i], dxe[:, i] = np.where(here, m[:, i] * D, 0), np.where(here, m[:, i] * (De + GATE * S), 0)
        v = x[:, i] if complement else 0.0
        p, ps = h[:, i] - v, H[:, i] + np.abs(v)
        dg[:, i] = np.where(here, D * p * slope[:, i], 0)
        dge[:, i] = np.where(here, slope[:, i] * (De * ps + S * he[:, i] + 2 * GATE * S * ps), 0)
        E, e, A = (np.where(here, n, o) for n, o in ((a[:, i] * D, E), (a[:, i] * De + GATE * np.minimum(a, w)[:, i] * S + STEP * a[:, i] * S, e),
                                                     (a[:, i] * S, A)))
    return dx, dxe, dg, dge, E, e


def check_bound(name, got, want, bound, element):
    """|got - want| within half a step of the element's rounding and the bound before it."""
    check(name, got, want, bound, element, 1.0)
