"""Float64 oracle of a recurrent language model's operators, from their formulas (numpy).

They have no counterpart in the reference; the definitions are those of include/gdn2.h."""
from __future__ import annotations

import numpy as np

SMALLEST = 2.0 ** -126  # a gate whose exp is below it empties the state


def decays(g, valid=None, reset=None):
    """exp(g) per token and channel as the recurrence uses it: 1 at padding, 0 at a reset and where it
    would be below 2^-126, at most 2^127."""
    with np.errstate(over="ignore"):
        a = np.exp(g)
    a = np.where(a < SMALLEST, 0.0, np.minimum(a, 2.0 ** 127))
    if reset is not None:
        a = np.where((reset != 0)[..., None], 0.0, a)
    if valid is not None:
        a = np.where((valid != 0)[..., None], a, 1.0)
    return a


def _times(a, h):
    """a h, with 0 where a is."""
    with np.errstate(invalid="ignore"):
        return np.where(a == 0, 0.0, a * h)


def recurrence(x, g, valid=None, reset=None, initial=None):
    """x, g [B, T, W] -> (y [B, T, W], final [B, W], carried [B, T, W] = a_t h_{t-1})."""
    B, T, W = x.shape
    on = np.ones((B, T), bool) if valid is None else valid != 0
    a = decays(g, valid, reset)
    h = np.zeros((B, W)) if initial is None else np.asarray(initial, float)
    y, carried = np.zeros((B, T, W)), np.zeros((B, T, W))
    for t in range(T):
        carried[:, t] = _times(a[:, t], h)
        h = carried[:, t] + np.where(on[:, t, None], x[:, t], 0.0)
        y[:, t] = np.where(on[:, t, None], h, 0.0)
    return y, h, carried


def recurrence_backward(x, g, valid, reset, initial, dy, d_final=None):
    """(dx, dg, d_initial)."""
    B, T, W = x.shape
    on = np.ones((B, T), bool) if valid is None else valid != 0
    a = decays(g, valid, reset)
    carried = recurrence(x, g, valid, reset, initial)[2]
    E = np.zeros((B, W)) if d_final is None else np.asarray(d_final, float)
    dx, dg = np.zeros((B, T, W)), np.zeros((B, T, W))
    for t in range(T - 1, -1, -1):
        o = on[:, t, None]
        e = E + np.where(o, dy[:, t], 0.0)
        dx[:, t] = np.where(o, e, 0.0)
        with np.errstate(invalid="ignore"):
            dg[:, t] = np.where(o & (a[:, t] != 0), carried[:, t] * e, 0.0)
        E = _times(a[:, t], e)
    return dx, dg, E


def scores(x, target, temperature=1.0):
    """Rows x [R, N] (-inf is probability 0), target [R]: (log p [R, N], log_probs [R], entropy [R])."""
    with np.errstate(invalid="ignore", divide="ignore"):
        z = x / temperature
        z = z - z.max(1, keepdims=True)
        lp = z - np.log(np.exp(z).sum(1, keepdims=True))
        p = np.exp(lp)
        entropy = -np.where(p > 0, p * np.where(p > 0, lp, 0), 0 * lp.max(1, keepdims=True)).sum(1)
    return lp, lp[np.arange(len(x)), target], entropy


def scores_backward(x, target, d_lp, d_entropy, temperature=1.0):
    lp, _, entropy = scores(x, target, temperature)
    p = np.exp(lp)
    dx = -p * (d_lp[:, None] + d_entropy[:, None] * np.where(p > 0, lp + entropy[:, None], 0))
    dx[np.arange(len(x)), target] += d_lp
    return dx / temperature


def top(x, k):
    """Indices of the k largest of each row: the lower first among equal ones, NaN before all."""
    key = np.where(np.isnan(x), np.inf, x)
    order = [sorted(range(x.shape[1]), key=lambda i: (not np.isnan(row[i]), -k_row[i], i))
             for row, k_row in zip(x, key)]
    return np.array(order, dtype=np.int64)[:, :k]


COEFFICIENTS = (3.4445, -4.7750, 2.0315)


def orthogonalize(u, steps=5, coefficients=COEFFICIENTS, epsilon=1e-7, product=np.matmul):
    """One matrix [rows, cols]; product(L, R^T) forms the products."""
    a, b, c = coefficients
    tall = u.shape[0] > u.shape[1]
    x = u.T if tall else u
    x = x / (np.sqrt((x ** 2).sum()) + epsilon)
    for _ in range(steps):
        gram = product(x, x.T)
        x = product(a * np.eye(len(x)) + b * gram + c * product(gram, gram), x)
    return x.T if tall else x


def split_product(left, right):
    """A product of float16 pairs that are scaled to 2^13 .. 2^14, summed in float32 by 32 columns: the
    arithmetic of the library's products."""
    def split(x):
        top = np.abs(x).max()
        by = 2.0 ** (14 - np.frexp(top)[1]) if top > 0 else 1.0
        hi = (x * by).astype(np.float16).astype(float)
        return hi, (x * by - hi).astype(np.float16).astype(float), by

    (lh, ll, lb), (rh, rl, rb) = split(left), split(right)
    total = np.zeros((left.shape[0], right.shape[1]), np.float32)
    for k in range(0, left.shape[1], 32):
        s = slice(k, k + 32)
        for a, b in ((lh, rh), (lh, rl), (ll, rh)):
            total = (total + (a[:, s] @ b[s])).astype(np.float32)
    return total.astype(float) / (lb * rb)


def muon(x, g, m, lr, beta=0.95, nesterov=True, decay=0.0, steps=5, coefficients=COEFFICIENTS,
         epsilon=1e-7, product=np.matmul):
    """(x, m) after one update."""
    m = beta * m + g
    o = orthogonalize(g + beta * m if nesterov else m, steps, coefficients, epsilon, product)
    return (1 - lr * decay) * x - lr * np.sqrt(max(1.0, x.shape[0] / x.shape[1])) * o, m
