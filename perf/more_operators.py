"""Measured calls of the operators of a recurrent language model.

Kinds:
  recurrence   gated linear recurrence, a state for each channel: forward + backward (the raw calls
               of a fused training block, or the autograd function), or the forward alone (a prompt)
  step         its single-token form, on carried states
  score        log probabilities of given tokens, entropy and top alternatives: with the gradient of
               the first two, or the forward alone
  update       one Muon update of a group of matrices: momentum, Newton-Schulz products, decay
  orthogonal   the Newton-Schulz products alone

listed() holds the named cases, draw() gives more of the same ranges, prepare() makes what the
caller has in hand, run() is one pass (plain torch operations in float32, or the framework's
operators where `own` is true) and exact() the same results in float64.
"""
import math
import os
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
COEFFICIENTS = (3.4445, -4.7750, 2.0315)  # the quintic's, as published with Muon
EPSILON = 1e-7
_PACKAGE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                        "delta-block-lm_amd")


def listed():
    return [
        # One layer of the lm512 model's size in training: 16 x 512 tokens, 512 channels, the
        # log decays in bfloat16 like the values.
        dict(name="recurrence_lm512", kind="recurrence", dtype="bf16", gates="bf16", batch=16,
             time=512, width=512, mode="raw"),
        # Long-context training: 4 x 8192 tokens of 2048 channels.
        dict(name="recurrence_long8k", kind="recurrence", dtype="bf16", gates="bf16", batch=4,
             time=8192, width=2048, mode="raw"),
        # float32 training of padded, packed sequences of a ragged length and an odd width on a
        # carried state, with a gradient of the final state.
        dict(name="recurrence_f32", kind="recurrence", dtype="f32", gates="f32", batch=8, time=509,
             width=1001, mode="grad", masks=True, initial=True, final_grad=True),
        # One long prompt, continued from a state, without gradients: few channels, a long axis.
        dict(name="recurrence_prompt", kind="recurrence", dtype="bf16", gates="f32", batch=1,
             time=30001, width=512, mode="forward", initial=True),
        # Serving: one token on 256 sequences of the lm512 width.
        dict(name="step_serving", kind="step", dtype="bf16", gates="bf16", batch=256, width=512),
        # A policy or distillation loss over a training batch: 16 x 512 rows of the lm512
        # vocabulary, gradients of the log probabilities and of the entropy.
        dict(name="score_lm512", kind="score", dtype="bf16", rows=8192, width=32768, top=0,
             mode="raw"),
        # Serving: eight sequences' next tokens with eight alternatives each.
        dict(name="score_decode", kind="score", dtype="bf16", rows=8, width=32768, top=8,
             mode="forward"),
        # float32 logits of an odd vocabulary at a temperature, padded rows and ruled-out tokens
        # among them, with gradients and twenty alternatives.
        dict(name="score_odd", kind="score", dtype="f32", rows=333, width=10007, top=20,
             mode="grad", temperature=0.7, masked=True, padded=True),
        # The update of the eight layers' feed-forward inputs of the lm512 model.
        dict(name="update_lm512", kind="update", dtype="f32", matrices=8, rows=2816, cols=512),
        # One square matrix, the smallest of that model's.
        dict(name="update_single", kind="update", dtype="f32", matrices=1, rows=512, cols=512),
        # Three matrices of odd sizes.
        dict(name="orthogonal_odd", kind="orthogonal", dtype="f32", matrices=3, rows=333,
             cols=1001),
        # A wide model's square projection, in bfloat16.
        dict(name="orthogonal_wide", kind="orthogonal", dtype="bf16", matrices=1, rows=4096,
             cols=4096),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["recurrence", "recurrence", "recurrence", "step", "score", "score", "score",
                       "update", "orthogonal", "orthogonal"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    if kind in ("recurrence", "step"):
        gates = rng.choice([dtype, dtype, "f32"])
        width = rng.choice([256, 512, 1024, _log(rng, 16, 4096)])
        if kind == "step":
            return dict(kind=kind, dtype=dtype, gates=gates, batch=_log(rng, 1, 1024), width=width)
        time = _log(rng, 1, 32768)
        most = (1 << 26 if dtype == "bf16" else 1 << 25) // (time * width)
        case = dict(kind=kind, dtype=dtype, gates=gates, batch=_log(rng, 1, max(1, min(64, most))),
                    time=time, width=width, mode=rng.choice(["raw", "grad", "forward"]))
        if case["batch"] * time * width > 1 << 26:  # a long axis of a wide state
            case["time"] = (1 << 26) // (case["batch"] * width)
        for name, share in (("masks", 0.4), ("initial", 0.5), ("final_grad", 0.3)):
            if rng.random() < share:
                case[name] = True
        return case
    if kind == "score":
        width = rng.choice([32768, _log(rng, 50, 200000)])
        case = dict(kind=kind, dtype=dtype, width=width,
                    rows=_log(rng, 1, max(1, min(16384, (1 << 27) // width))),
                    top=min(width // 4, rng.choice([0, 1, 8, 20, 32])),
                    mode=rng.choice(["raw", "grad", "forward"]))
        if rng.random() < 0.4:
            case["temperature"] = round(rng.uniform(0.3, 2.0), 2)
        for name, share in (("masked", 0.4), ("padded", 0.4)):
            if rng.random() < share:
                case[name] = True
        return case
    rows, cols = rng.choice([(512, 512), (512, 1408), (2048, 512),
                             (_log(rng, 8, 3000), _log(rng, 8, 3000))])
    small, large = min(rows, cols), max(rows, cols)
    most = int(2e11 / (small * small * (3 * large + small)))  # an eighth of orthogonal_wide's
    return dict(kind=kind, dtype="f32" if kind == "update" else dtype, rows=rows, cols=cols,
                matrices=_log(rng, 1, max(1, min(16, most))))


# ---- inputs --------------------------------------------------------------------------------


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed & 0x7fffffff)

    def normal(*size):
        return torch.randn(size, generator=gen, device="cuda")

    def uniform(*size):
        return torch.rand(size, generator=gen, device="cuda")

    dt = DTYPES[case["dtype"]]
    s = dict(kind=case["kind"], mode=case.get("mode", "raw"))
    if case["kind"] in ("update", "orthogonal"):
        n, rows, cols = case["matrices"], case["rows"], case["cols"]
        # gradients: some strong directions, the rest noise whose rows differ in size
        rank = min(8, rows, cols)
        g = normal(n, rows, rank) @ normal(n, rank, cols) * (0.3 / rank ** 0.5) \
            + normal(n, rows, cols) * (0.2 + uniform(n, rows, 1))
        g = g * 1e-3
        if case["kind"] == "orthogonal":
            s["g"] = g.to(dt)
            return s
        s["g"] = list(g.unbind())
        s["m"] = list((5e-3 * normal(n, rows, cols) + 3 * g).unbind())
        s["p"] = list((normal(n, rows, cols) * cols ** -0.5).unbind())
        s["lr"], s["decay"] = 0.02, 0.01
        return s
    if case["kind"] == "score":
        rows, width = case["rows"], case["width"]
        # logits of a model that is sure of some tokens: a few large ones a row
        x = normal(rows, width) * 1.5
        x += 6 * (uniform(rows, width) < 4 / width)
        tokens = torch.randint(0, width, (rows,), generator=gen, device="cuda")
        if case.get("masked"):
            out = uniform(width) < 0.5  # a part of the vocabulary is ruled out, the given tokens not
            keep = x.gather(1, tokens[:, None])
            x = x.masked_fill(out, -math.inf).scatter_(1, tokens[:, None], keep)
        s["x"], s["tokens"] = x.to(dt), tokens
        s["valid"] = (uniform(rows) < 0.8).float() if case.get("padded") else None
        s["top"], s["temperature"] = case["top"], case.get("temperature", 1.0)
        if s["mode"] != "forward":
            s["d_log_probs"] = normal(rows) / rows
            s["d_entropy"] = 0.1 * normal(rows) / rows
        if s["mode"] == "grad":
            s["x"].requires_grad_(True)
        return s
    B, T, W = case["batch"], case.get("time", 1), case["width"]
    s["x"] = normal(B, T, W).to(dt)
    # a memory of some 2 to 500 tokens over the channels, changed by each token's gate
    rate = torch.exp(-0.7 - 5.5 * uniform(W))
    s["g"] = (-rate * 2 * torch.sigmoid(normal(B, T, W))).to(DTYPES[case["gates"]])
    if case["kind"] == "step":
        s["state"] = normal(B, W)
        return s
    s["valid"] = s["reset"] = s["initial"] = s["d_final"] = None
    if case.get("masks"):
        # sequences padded at the end, of documents that begin about every 100 tokens
        length = (T * (0.6 + 0.4 * uniform(B, 1))).ceil()
        s["valid"] = (torch.arange(T, device="cuda") < length).float()
        s["reset"] = (uniform(B, T) < 0.01).float()
    if case.get("initial"):
        s["initial"] = normal(B, W)
    if s["mode"] != "forward":
        s["dy"] = normal(B, T, W).to(dt)
        if case.get("final_grad"):
            s["d_final"] = normal(B, W)
    if s["mode"] == "grad":
        for n in ("x", "g", "initial"):
            if s[n] is not None:
                s[n].requires_grad_(True)
    return s


# ---- the framework's operators -------------------------------------------------------------


def _operators():
    if _PACKAGE not in sys.path:
        sys.path.insert(0, _PACKAGE)
    import delta_kernels
    return delta_kernels


def _own_recurrence(s):
    dk = _operators()
    inputs = [s[n] for n in ("x", "g", "valid", "reset", "initial")]
    if s["mode"] == "forward":
        y, final = dk.gated_recurrence(*inputs)
        return dict(y=y, final=final)
    if s["mode"] == "raw":
        y, final, checkpoint = dk.gated_recurrence_forward(*inputs)
        dx, dg, di = dk.gated_recurrence_backward(*inputs, checkpoint, s["dy"], s["d_final"])
        out = dict(y=y, final=final, dx=dx, dg=dg)
        return out if di is None else dict(out, dinitial=di)
    y, final = dk.gated_recurrence(*inputs)
    names = [n for n in ("x", "g", "initial") if s[n] is not None]
    outs, ups = ([y], [s["dy"]]) if s["d_final"] is None else ([y, final], [s["dy"], s["d_final"]])
    grads = torch.autograd.grad(outs, [s[n] for n in names], ups)
    return dict(y=y.detach(), final=final.detach(), **{"d" + n: d for n, d in zip(names, grads)})


def _own_score(s):
    dk = _operators()
    args = (s["x"], s["tokens"], s["top"], s["valid"], s["temperature"])
    if s["mode"] == "raw":
        r, stats = dk.token_log_probs_forward(*args)
        dx = dk.token_log_probs_backward(s["x"], s["tokens"], s["valid"], s["temperature"], stats,
                                         s["d_log_probs"], s["d_entropy"])
        out = dict(log_probs=r.log_probs, entropy=r.entropy, dx=dx)
    else:
        r = dk.token_log_probs(*args)
        out = dict(log_probs=r.log_probs.detach(), entropy=r.entropy.detach())
        if s["mode"] == "grad":
            (out["dx"],) = torch.autograd.grad([r.log_probs, r.entropy], [s["x"]],
                                               [s["d_log_probs"], s["d_entropy"]])
    if s["top"]:
        out.update(top_log_probs=r.top_log_probs, top_tokens=r.top_tokens)
    return out


# ---- the plain forms -----------------------------------------------------------------------


def _scan(a, x, dim=1):
    """h_t = a_t h_{t-1} + x_t along dim from h = 0, by doubling steps."""
    T, step = a.shape[dim], 1
    while step < T:
        def shifted(t, fill):
            head = torch.full_like(t.narrow(dim, 0, step), fill)
            return torch.cat([head, t.narrow(dim, 0, T - step)], dim)
        x = x + a * shifted(x, 0.0)
        a = a * shifted(a, 1.0)
        step *= 2
    return x


def _masks(s, B, T):
    on = None if s["valid"] is None else (s["valid"] != 0)[..., None]
    cut = None if s["reset"] is None else (s["reset"] != 0)[..., None]
    if cut is not None and on is not None:
        cut = cut & on
    return on, cut


def _plain_recurrence(s):
    x, g = s["x"].detach().float(), s["g"].detach().float()
    B, T, W = x.shape
    on, cut = _masks(s, B, T)
    a = g.exp()
    if on is not None:
        x, a = x * on, torch.where(on, a, 1.0)
    if cut is not None:
        a = torch.where(cut, 0.0, a)
    first = torch.zeros((B, W), device=x.device) if s["initial"] is None \
        else s["initial"].detach()
    h = _scan(a, torch.cat([x[:, :1] + a[:, :1] * first[:, None], x[:, 1:]], 1))
    y = h if on is None else h * on
    out = dict(y=y.to(s["x"].dtype), final=h[:, -1].clone())
    if s["mode"] == "forward":
        return out
    d = s["dy"].float()
    if on is not None:
        d = d * on
    if s["d_final"] is not None:
        d = torch.cat([d[:, :-1], d[:, -1:] + s["d_final"][:, None]], 1)
    after = torch.cat([a[:, 1:], torch.ones_like(a[:, :1])], 1)  # the decay after each token
    e = _scan(after.flip(1), d.flip(1)).flip(1)
    dg = a * torch.cat([first[:, None], h[:, :-1]], 1) * e
    dx = e
    if on is not None:
        dx, dg = dx * on, dg * on
    out.update(dx=dx.to(s["x"].dtype), dg=dg.to(s["g"].dtype))
    if s["initial"] is not None:
        out["dinitial"] = a[:, 0] * e[:, 0]
    return out


def _plain_score(s):
    raw, t, dtype = s["x"].detach(), s["tokens"][:, None], s["x"].dtype
    x = raw.float() / s["temperature"]
    x = x - x.amax(1, keepdim=True)
    lp = x - x.exp().sum(1, keepdim=True).log()
    p = lp.exp()
    on = None if s["valid"] is None else s["valid"] != 0
    entropy = -torch.where(p > 0, p * lp, 0.0).sum(1)
    given = lp.gather(1, t)[:, 0]
    out = dict(log_probs=given, entropy=entropy)
    if s["mode"] != "forward":
        d, dh = s["d_log_probs"][:, None], s["d_entropy"][:, None]
        dx = -p * d - torch.where(p > 0, p * (lp + entropy[:, None]), 0.0) * dh
        dx = dx.scatter_add(1, t, d) / s["temperature"]
        out["dx"] = (dx if on is None else dx * on[:, None]).to(dtype)
    if s["top"]:
        order = torch.sort(raw, dim=1, descending=True, stable=True)[1][:, :s["top"]]
        out.update(top_log_probs=lp.gather(1, order), top_tokens=order)
    if on is not None:
        for n in out:
            if n != "dx":
                keep = on if out[n].dim() == 1 else on[:, None]
                out[n] = torch.where(keep, out[n], torch.zeros_like(out[n]))
    return out


def _plain_orthogonal(g, steps=5):
    a, b, c = COEFFICIENTS
    x = g.float()
    tall = x.shape[1] > x.shape[2]
    if tall:
        x = x.transpose(1, 2).contiguous()
    x = x / (x.square().sum((1, 2), keepdim=True).sqrt() + EPSILON)
    for _ in range(steps):
        gram = x @ x.transpose(1, 2).contiguous()
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return (x.transpose(1, 2).contiguous() if tall else x).to(g.dtype)


def _plain_update(s):
    g, m, beta = torch.stack(s["g"]), torch.stack(s["m"]), 0.95
    m = beta * m + g
    o = _plain_orthogonal(g + beta * m)
    rows, cols = g.shape[1:]
    scale = max(1.0, rows / cols) ** 0.5
    for p, old, new, step in zip(s["p"], s["m"], m, o):
        p.mul_(1 - s["lr"] * s["decay"]).sub_(step, alpha=s["lr"] * scale)
        old.copy_(new)
    return dict(p=s["p"], m=s["m"])


def run(state):
    s = state
    if s["kind"] == "recurrence":
        return _own_recurrence(s) if own else _plain_recurrence(s)
    if s["kind"] == "score":
        return _own_score(s) if own else _plain_score(s)
    if s["kind"] == "step":
        if own:
            y = _operators().gated_recurrence_step(s["state"], s["x"], s["g"])
        else:
            s["state"].mul_(s["g"][:, 0].float().exp()).add_(s["x"][:, 0].float())
            y = s["state"][:, None].to(s["x"].dtype)
        return dict(y=y, state=s["state"])
    if s["kind"] == "update":
        if not own:
            return _plain_update(s)
        _operators().muon_update(s["p"], s["g"], s["m"], s["lr"], decay=s["decay"])
        return dict(p=s["p"], m=s["m"])
    return _operators().orthogonalize(s["g"]) if own else _plain_orthogonal(s["g"])


# ---- what a pass cannot do without ----------------------------------------------------------


def work(case):
    es = 2 if case["dtype"] == "bf16" else 4
    if case["kind"] in ("update", "orthogonal"):
        n, m = case["rows"] * case["cols"], min(case["rows"], case["cols"])
        # the products of symmetric matrices by halves
        flops = 5 * (3 * m * n + m ** 3) * case["matrices"]
        return {"bytes": (20 if case["kind"] == "update" else 2 * es) * n * case["matrices"],
                "flops": flops}
    if case["kind"] == "score":
        n = case["rows"] * case["width"]
        rows = case["rows"] * (16 + 12 * case["top"] + (4 if case.get("padded") else 0))
        if case["mode"] == "forward":
            return {"bytes": n * es + rows, "flops": 6 * n}
        return {"bytes": 2 * n * es + rows + 8 * case["rows"], "flops": 12 * n}
    B, W, T = case["batch"], case["width"], case.get("time", 1)
    n, gs = B * T * W, 2 if case["gates"] == "bf16" else 4
    if case["kind"] == "step":
        return {"bytes": n * (8 + 2 * es + gs), "flops": 4 * n}
    states = 4 * B * W * (2 if case.get("initial") else 1)
    if case.get("masks"):
        states += 8 * B * T
    if case["mode"] == "forward":
        return {"bytes": n * (2 * es + gs) + states, "flops": 4 * n}
    states += 4 * B * W * (int(case.get("initial", False)) + int(case.get("final_grad", False)))
    return {"bytes": n * (4 * es + 2 * gs) + states, "flops": 10 * n}


# ---- the same in float64 --------------------------------------------------------------------


def _exact_recurrence(s):
    """Token by token, forwards and then backwards."""
    x, g = s["x"].detach(), s["g"].detach()
    B, T, W = x.shape
    dev, train = x.device, s["mode"] != "forward"
    h = torch.zeros((B, W), dtype=torch.float64, device=dev)
    if s["initial"] is not None:
        h = h + s["initial"].detach()
    y = torch.empty((B, T, W), dtype=torch.float64, device=dev)
    before = torch.empty_like(y) if train else None
    keep = None if s["valid"] is None else s["valid"].double()[..., None]  # 0 or 1
    stay = None if s["reset"] is None else 1 - s["reset"].double()[..., None]

    def decay(t):
        a = torch.exp(g[:, t].double())
        if stay is not None:
            a = a * stay[:, t]
        return a if keep is None else keep[:, t] * a + (1 - keep[:, t])

    for t in range(T):
        if train:
            before[:, t] = h
        u = x[:, t].double()
        if keep is None:
            h = decay(t) * h + u
            y[:, t] = h
        else:
            h = decay(t) * h + keep[:, t] * u
            y[:, t] = keep[:, t] * h
    out = dict(y=y, final=h)
    if not train:
        return out
    e = torch.zeros_like(h) if s["d_final"] is None else s["d_final"].double()
    dx, dg = torch.empty_like(y), torch.empty_like(y)
    for t in range(T - 1, -1, -1):
        up, a = s["dy"][:, t].double(), decay(t)
        on = 1.0 if keep is None else keep[:, t]
        e = e + on * up
        dx[:, t] = on * e
        dg[:, t] = on * a * before[:, t] * e
        e = a * e
    out.update(dx=dx, dg=dg)
    if s["initial"] is not None:
        out["dinitial"] = e
    return out


def _exact_score(s, rows_at_once=512):
    parts = []
    for r in range(0, s["x"].shape[0], rows_at_once):
        rows = slice(r, r + rows_at_once)
        raw, t = s["x"].detach()[rows].double(), s["tokens"][rows]
        z = raw / s["temperature"]
        total = torch.logsumexp(z, 1)
        lp = z - total[:, None]
        p = torch.softmax(z, 1)
        some = torch.nan_to_num(lp, neginf=0.0)  # where p is 0
        entropy = -(p * some).sum(1)
        i = torch.arange(len(t), device=t.device)
        part = dict(log_probs=lp[i, t], entropy=entropy)
        if s["mode"] != "forward":
            d, dh = s["d_log_probs"][rows].double(), s["d_entropy"][rows].double()
            hot = torch.zeros_like(p)
            hot[i, t] = 1
            part["dx"] = (d[:, None] * (hot - p)
                          - dh[:, None] * p * (some + entropy[:, None])) / s["temperature"]
        if s["top"]:
            # the largest first, the lower index first among equals
            found, index = [], torch.arange(raw.shape[1], device=raw.device)
            left = torch.ones_like(raw, dtype=torch.bool)
            for _ in range(s["top"]):
                best = torch.where(left, raw, -math.inf).amax(1, keepdim=True)
                at = torch.where(left & (raw == best), index, raw.shape[1]).amin(1)
                left[i, at] = False
                found.append(at)
            order = torch.stack(found, 1)
            part.update(top_log_probs=lp.gather(1, order), top_tokens=order)
        if s["valid"] is not None:
            off = s["valid"][rows] == 0
            for v in part.values():
                v[off] = 0
        parts.append(part)
    return {n: torch.cat([p[n] for p in parts]) for n in parts[0]}


def _exact_orthogonal(u, steps=5):
    """One matrix [rows, cols] of float64, on its rows whether it is tall or wide: for a wide one
    a x + (b x x^T + c (x x^T)^2) x, for a tall one the same products from the right."""
    a, b, c = COEFFICIENTS
    x = u / (torch.linalg.vector_norm(u) + EPSILON)
    for _ in range(steps):
        xt = x.t().contiguous()
        if x.shape[0] <= x.shape[1]:
            first = torch.mm(x, xt)
            third = torch.mm(first, x)
            fifth = torch.mm(first, third)
        else:
            first = torch.mm(xt, x)
            third = torch.mm(x, first)
            fifth = torch.mm(third, first)
        x = a * x + b * third + c * fifth
    return x


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "recurrence":
        return _exact_recurrence(s)
    if case["kind"] == "score":
        return _exact_score(s)
    if case["kind"] == "step":
        h = torch.exp(s["g"][:, 0].double()) * s["state"].double() + s["x"][:, 0].double()
        return dict(y=h[:, None], state=h)
    if case["kind"] == "orthogonal":
        return torch.stack([_exact_orthogonal(g.double()) for g in s["g"]])
    ps, ms = [], []
    for p, g, m in zip(s["p"], s["g"], s["m"]):
        p, g, m = p.double(), g.double(), m.double()
        m = 0.95 * m + g
        o = _exact_orthogonal(0.95 * m + g)
        step = s["lr"] * math.sqrt(max(1.0, p.shape[0] / p.shape[1]))
        ps.append(p * (1 - s["lr"] * s["decay"]) - step * o)
        ms.append(m)
    return dict(p=ps, m=ms)
