"""float64 restatement of the linear-attention block's operators, token by token and value by value:
linear attention with a decay for each head, layer norm, and the 8-bit form of a SwiGLU's input."""
import numpy as np


def attention(q, k, v, g, valid=None, reset=None, initial=None):
    """q, k [B,T,H,K], v [B,T,H,V], g [B,T,H]; returns (output, final_state, states), states [T+1]
    arrays [B,H,K,V] before every token and after the last."""
    q, k, v, g = (np.asarray(x, np.float64) for x in (q, k, v, g))
    B, T, H, K = q.shape
    V = v.shape[3]
    S = np.zeros((B, H, K, V)) if initial is None else np.array(initial, np.float64)
    out = np.zeros((B, T, H, V))
    states = [S]
    for t in range(T):
        S = S.copy()
        for b in range(B):
            if valid is not None and not valid[b, t]:
                continue
            cut = reset is not None and reset[b, t]
            for h in range(H):
                a = 0.0 if cut else np.exp(g[b, t, h])
                old = np.zeros((K, V)) if a == 0 else a * S[b, h]
                S[b, h] = old + np.outer(k[b, t, h], v[b, t, h])
                out[b, t, h] = q[b, t, h] @ S[b, h]
        states.append(S)
    return out, S, states


def attention_backward(q, k, v, g, valid, reset, initial, d_output, d_final=None):
    """Returns a dict of dq, dk, dv, dg, dinitial by the adjoint recurrence."""
    q, k, v, g, do = (np.asarray(x, np.float64) for x in (q, k, v, g, d_output))
    B, T, H, K = q.shape
    V = v.shape[3]
    _, _, states = attention(q, k, v, g, valid, reset, initial)
    D = np.zeros((B, H, K, V)) if d_final is None else np.array(d_final, np.float64)
    dq, dk, dv, dg = np.zeros_like(q), np.zeros_like(k), np.zeros_like(v), np.zeros_like(g)
    for t in reversed(range(T)):
        for b in range(B):
            if valid is not None and not valid[b, t]:
                continue
            cut = reset is not None and reset[b, t]
            for h in range(H):
                a = 0.0 if cut else np.exp(g[b, t, h])
                D[b, h] += np.outer(q[b, t, h], do[b, t, h])
                dq[b, t, h] = states[t + 1][b, h] @ do[b, t, h]
                dk[b, t, h] = D[b, h] @ v[b, t, h]
                dv[b, t, h] = k[b, t, h] @ D[b, h]
                if a == 0:
                    D[b, h] = 0
                    continue
                D[b, h] *= a
                dg[b, t, h] = np.sum(D[b, h] * states[t][b, h])
    return dict(dq=dq, dk=dk, dv=dv, dg=dg, dinitial=D)


def layer_norm(x, weight, bias, epsilon):
    """x [rows, W]; returns (y, mean, inverse)."""
    x = np.asarray(x, np.float64)
    mean = x.mean(1)
    inv = 1 / np.sqrt(np.mean((x - mean[:, None]) ** 2, 1) + epsilon)
    y = (x - mean[:, None]) * inv[:, None] * weight
    return (y if bias is None else y + bias), mean, inv


def layer_norm_backward(x, weight, epsilon, dy):
    """Returns (dx, dweight, dbias)."""
    x, dy = np.asarray(x, np.float64), np.asarray(dy, np.float64)
    _, mean, inv = layer_norm(x, weight, None, epsilon)
    xh = (x - mean[:, None]) * inv[:, None]
    c = dy * weight
    dx = inv[:, None] * (c - c.mean(1, keepdims=True) - xh * (c * xh).mean(1, keepdims=True))
    return dx, (dy * xh).sum(0), dy.sum(0)


def q8(h, block=32):
    """codes int8 [rows, 2 M] and exponents uint8 [rows, 2 ceil(M / block)] of h = [gate | up]."""
    h = np.asarray(h, np.float64)
    rows, M = h.shape[0], h.shape[1] // 2
    codes, exps = np.zeros(h.shape, np.int8), []
    for half in range(2):
        for c in range(0, M, block):
            at = np.s_[:, half * M + c:half * M + min(M, c + block)]
            x = h[at]
            e = np.zeros(rows, np.int64)
            for r in range(rows):
                top = np.abs(x[r]).max() if np.isfinite(x[r]).all() else np.inf
                if not np.isfinite(top):
                    e[r] = 128
                    continue
                e[r] = -126
                while top > 127 * 2.0 ** e[r] and e[r] < 121:  # at 122 a value could round to 2^128
                    e[r] += 1
            ok = e < 128
            code = np.rint(np.where(ok[:, None], x, 0) * 2.0 ** -e[:, None])
            codes[at] = np.where(ok[:, None], np.clip(code, -127, 127), 0)
            exps.append((e + 127).astype(np.uint8))
    return codes, np.stack(exps, 1)


def q8_values(codes, exps, block=32):
    rows, M = codes.shape[0], codes.shape[1] // 2
    scale = np.where(exps == 255, np.nan, 2.0 ** (exps.astype(np.float64) - 127))
    scale = np.repeat(scale.reshape(rows, 2, -1), block, 2)[:, :, :M].reshape(rows, 2 * M)
    return codes * scale


def swiglu(h):
    h = np.asarray(h, np.float64)
    gate, up = np.split(h, 2, 1)
    return gate / (1 + np.exp(-gate)) * up


def swiglu_backward(h, da):
    """dh at the values h."""
    gate, up = np.split(np.asarray(h, np.float64), 2, 1)
    s = 1 / (1 + np.exp(-gate))
    return np.concatenate([da * up * s * (1 + gate * (1 - s)), da * gate * s], 1)
