"""The operators around a mixture-of-experts block and its norms, as cases that can be timed one pass at a time.

Families (``case["op"]``):

``sort``     ``ops.moe_sort`` and ``ops.moe_dispatch``: the router's choices become rows sorted by expert
``combine``  ``ops.moe_combine``: the experts' rows back to their tokens, with the router's weights applied
``experts``  both, forward and backward: gradients of the tokens, of the experts' rows and of the weights
``norms``    ``ops.rmsnorm_add_rmsnorm``: the norm behind a block, its gate, the scaled residual stream and the norm
             in front of the next block, in one pass
``norms_bwd`` the same, forward and backward
``linear``   ``ops.linear_i8``: activations to 8-bit integers with a scale for each token, times 8-bit weights with a
             scale for each channel; with ``experts`` > 0 every expert's rows times its own weights

Sizes are the repository's: hidden 1024, 4096 and 8192, ffn 3584, 14336 and 28672, 1 to 16384 tokens, and ragged ones.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
DEVICE = "cuda"
EPS = 1e-5


def listed():
    return [
        # a decode batch of 16 sequences on its way to 64 experts
        {"name": "sort_decode", "op": "sort", "tokens": 16, "top_k": 8, "experts": 64, "ranks": 1, "dim": 8192,
         "dtype": "bf16"},
        # a prefill chunk on one of four expert-parallel ranks, which keeps the rows of its own 16 experts
        {"name": "sort_prefill_rank", "op": "sort", "tokens": 8192, "top_k": 4, "experts": 16, "ranks": 4, "dim": 4096,
         "dtype": "bf16"},
        # one token's eight rows back into one
        {"name": "combine_one_token", "op": "combine", "tokens": 1, "top_k": 8, "experts": 64, "ranks": 1, "dim": 4096,
         "dtype": "bf16"},
        # odd numbers of tokens, choices, experts and columns, some choices on another rank
        {"name": "combine_ragged_fp16", "op": "combine", "tokens": 4999, "top_k": 3, "experts": 7, "ranks": 2, "dim": 1032,
         "dtype": "fp16"},
        # a training step's 8192 tokens through 64 experts and back, with all gradients
        {"name": "experts_train", "op": "experts", "tokens": 8192, "top_k": 8, "experts": 64, "ranks": 1, "dim": 4096,
         "dtype": "bf16"},
        # one decoded token between two blocks: nothing but latency
        {"name": "norms_one_token", "op": "norms", "rows": 1, "dim": 8192, "gate": "channel", "scale": 1.0, "dtype": "bf16"},
        # a long prefill, each of its 4 sequences with a gate of its own
        {"name": "norms_prefill", "op": "norms", "rows": 16384, "dim": 8192, "gate": 4, "scale": 1.0, "dtype": "bf16"},
        # gradients with odd sizes and a gate for every element
        {"name": "norms_train_ragged_fp16", "op": "norms_bwd", "rows": 1999, "dim": 2056, "gate": "row", "scale": 0.7,
         "dtype": "fp16"},
        # gradients of a training step's tokens, one gate for each channel
        {"name": "norms_train", "op": "norms_bwd", "rows": 8192, "dim": 8192, "gate": "channel", "scale": 1.0, "dtype": "bf16"},
        # one decoded token through a down projection: the weights are read once
        {"name": "linear_one_token", "op": "linear", "m": 1, "n": 8192, "k": 3584, "experts": 0, "dtype": "bf16"},
        # a few tokens for each of 16 experts
        {"name": "linear_experts_fp16", "op": "linear", "m": 200, "n": 3584, "k": 4096, "experts": 16, "dtype": "fp16"},
        # the benchmark's headline projection in 8 bits
        {"name": "linear_headline", "op": "linear", "m": 8192, "n": 8192, "k": 28672, "experts": 0, "dtype": "bf16"},
    ]


def _log(rng, lo, hi, step=1):
    """A multiple of ``step`` in [lo, hi], spread evenly over the logarithm."""
    hi = max(lo, hi)
    x = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return int(min(hi // step, max(-(-lo // step), round(x / step))) * step)


def draw(rng):
    op = rng.choice(("sort", "combine", "experts", "norms", "norms_bwd", "linear", "linear"))
    dtype = rng.choice(("bf16", "fp16"))
    if op in ("sort", "combine", "experts"):
        ranks = rng.choice((1, 1, 2, 8))
        experts = _log(rng, 1, 256)
        top_k = rng.randint(1, min(10, experts * ranks))
        tokens = _log(rng, 1, 16384)
        dim = _log(rng, 64, min(8192, 8192 * 8 * 4096 // (tokens * top_k)), 8)
        return {"op": op, "tokens": tokens, "top_k": top_k, "experts": experts, "ranks": ranks, "dim": dim, "dtype": dtype}
    if op in ("norms", "norms_bwd"):
        rows, kind = _log(rng, 1, 16384), rng.choice(("none", "channel", "group", "row"))
        dim = _log(rng, 64, min(16384, (16384 if op == "norms" else 8192) * 8192 // rows), 8)
        if kind == "group":
            kind = rng.choice([g for g in range(1, 65) if rows % g == 0])
        return {"op": op, "rows": rows, "dim": dim, "gate": kind, "scale": rng.choice((1.0, 0.22, 1.7)), "dtype": dtype}
    experts = rng.choice((0, 0, 1, 5, 16, 64))
    m, n = _log(rng, 1, 16384), _log(rng, 64, 16384 // max(1, experts // 8), 8)
    k = _log(rng, 64, min(28672, 8192 * 8192 * 28672 // (m * n), (1 << 30) // (n * max(1, experts))), 16)
    return {"op": op, "m": m, "n": n, "k": k, "experts": experts, "dtype": dtype}


def _gen(seed):
    return torch.Generator(device=DEVICE).manual_seed(seed)


def _randn(g, *shape, dtype=torch.float32, scale=1.0):
    return torch.randn(*shape, device=DEVICE, generator=g).mul_(scale).to(dtype)


def _impl():
    from flashoverlap_b200 import ops
    impl = ops.OverlapImpl()
    impl.nccl_init(0, 1, [0] * 16)
    return impl


def prepare(case, seed):
    op, dt, g = case["op"], DTYPES[case["dtype"]], _gen(seed)
    s = {"op": op, "case": case}
    if op in ("sort", "combine", "experts"):
        tokens, top_k, dim, every = case["tokens"], case["top_k"], case["dim"], case["experts"] * case["ranks"]
        # some experts are more popular than others; the ids of other ranks' experts lie beyond this rank's
        logits = _randn(g, tokens, every) + _randn(g, every)
        best, ids = logits.topk(top_k, dim=1)
        s["ids"], s["w"] = ids.to(torch.int32), best.softmax(1)
        if op != "combine":
            s["x"] = _randn(g, tokens, dim, dtype=dt)
        if op != "sort":
            s["y"] = _randn(g, tokens * top_k, dim, dtype=dt)
        if op == "combine":
            s["order"] = _order(s["ids"], case["experts"])          # the dispatch made it
        if op == "experts":
            s["g_rows"], s["g_out"] = _randn(g, tokens * top_k, dim, dtype=dt), _randn(g, tokens, dim, dtype=dt)
    elif op in ("norms", "norms_bwd"):
        rows, dim, kind = case["rows"], case["dim"], case["gate"]
        s["x"], s["t"] = _randn(g, rows, dim, dtype=dt, scale=2.0), _randn(g, rows, dim, dtype=dt, scale=0.3)
        s["pw"], s["w"] = (1 + 0.1 * _randn(g, dim)).to(dt), (1 + 0.1 * _randn(g, dim)).to(dt)
        lines = {"none": 0, "channel": 1, "row": rows}.get(kind, kind)
        s["gate"] = (0.5 + 0.3 * _randn(g, lines, dim)).to(dt) if lines else None
        if kind == "channel":
            s["gate"] = s["gate"].view(dim)
        if op == "norms_bwd":
            s["gh"], s["gy"] = _randn(g, rows, dim, dtype=dt), _randn(g, rows, dim, dtype=dt)
    else:
        m, n, k, experts = case["m"], case["n"], case["k"], case["experts"]
        x = torch.randn(m, k, device=DEVICE, generator=g)
        x *= 1 + 7 * (torch.rand(k, device=DEVICE, generator=g) < 0.01)       # a few channels stand out
        s["x"] = x.to(dt)
        s["q"] = torch.randint(-127, 128, (max(1, experts), n, k), device=DEVICE, generator=g, dtype=torch.int8)
        s["ws"] = (0.5 + torch.rand(max(1, experts), n, device=DEVICE, generator=g)) * (0.02 / 73)
        s["offsets"], s["segments"] = None, [(0, m)]
        if experts == 0:
            s["q"], s["ws"] = s["q"][0], s["ws"][0]
        else:
            h = torch.Generator().manual_seed(seed)
            share = (torch.randn(experts, generator=h)).softmax(0)
            of = torch.multinomial(share, m, replacement=True, generator=h)
            ends = torch.bincount(of, minlength=experts).cumsum(0)
            s["offsets"] = torch.cat([torch.zeros(1, dtype=torch.int64), ends]).to(torch.int32).to(DEVICE)
            s["segments"] = list(zip([0] + ends.tolist()[:-1], ends.tolist()))
        s["impl"] = _impl() if own else None
    return s


def _order(ids, experts):
    """(slot of every choice or -1, choice of every row or -1, first row of every expert), rows stable by expert."""
    if own:
        from flashoverlap_b200 import ops
        return ops.moe_sort(ids, experts)
    flat = ids.reshape(-1).long()
    n = flat.numel()
    here = (flat >= 0) & (flat < experts)
    key = torch.where(here, flat, experts)
    ranked, choice = torch.sort(key, stable=True)
    slot = torch.empty_like(choice)
    slot[choice] = torch.arange(n, device=ids.device)
    slot = torch.where(here, slot, -1).to(torch.int32).view(ids.shape)
    source = torch.where(ranked < experts, choice, -1).to(torch.int32)
    counts = torch.zeros(experts + 1, dtype=torch.int64, device=ids.device).index_add_(0, key, torch.ones_like(key))
    offsets = torch.cat([counts[:1] * 0, counts[:experts].cumsum(0)]).to(torch.int32)
    return slot, source, offsets


def _dispatch(x, order):
    slot, source, _ = order
    rows = x[(source.long() // slot.shape[1]).clamp(min=0)]
    return rows * (source >= 0)[:, None]


def _combine(y, w, order):
    slot = order[0].long()
    rows = y[slot.clamp(min=0).reshape(-1)].view(*slot.shape, -1)
    return (rows * (w * (slot >= 0))[:, :, None]).sum(1)


def _norms(x, t, pw, w, gate, scale):
    u = t * torch.rsqrt((t * t).mean(1, keepdim=True) + EPS) * pw
    if gate is not None:
        rows, dim = x.shape
        u = (u.view(-1, rows // gate.reshape(-1, dim).shape[0], dim) * gate.reshape(-1, 1, dim)).view(rows, dim)
    h = scale * x + u
    return h, h * torch.rsqrt((h * h).mean(1, keepdim=True) + EPS) * w


def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_own(s):
    from flashoverlap_b200 import ops
    op, case = s["op"], s["case"]
    if op == "sort":
        order = ops.moe_sort(s["ids"], case["experts"])
        return [*order, ops.moe_dispatch(s["x"], order)]
    if op == "combine":
        return ops.moe_combine(s["y"], s["w"], s["order"])
    if op == "experts":
        leaves = [s[n].detach().requires_grad_() for n in ("x", "y", "w")]
        x, y, w = leaves
        order = ops.moe_sort(s["ids"], case["experts"])
        rows, out = ops.moe_dispatch(x, order), ops.moe_combine(y, w, order)
        grads = torch.autograd.grad((rows, out), leaves, (s["g_rows"], s["g_out"]))
        return [rows.detach(), out.detach(), *grads]
    if op == "norms":
        return ops.rmsnorm_add_rmsnorm(s["x"], s["t"], s["pw"], s["w"], s["gate"], case["scale"], EPS)
    if op == "norms_bwd":
        leaves = [s[n].detach().requires_grad_() for n in ("x", "t", "pw", "w", "gate") if s[n] is not None]
        x, t, pw, w, *gate = leaves
        h, y = ops.rmsnorm_add_rmsnorm(x, t, pw, w, gate[0] if gate else None, case["scale"], EPS)
        return [h.detach(), y.detach(), *torch.autograd.grad((h, y), leaves, (s["gh"], s["gy"]))]
    return ops.linear_i8(s["impl"], s["x"], s["q"], s["ws"], s["offsets"])


def _run_plain(s):
    op, case, dt = s["op"], s["case"], DTYPES[s["case"]["dtype"]]
    if op == "sort":
        order = _order(s["ids"], case["experts"])
        return [*order, _dispatch(s["x"].float(), order).to(dt)]
    if op == "combine":
        return _combine(s["y"].float(), s["w"], s["order"]).to(dt)
    if op == "experts":
        leaves = [s[n].detach().float().requires_grad_() for n in ("x", "y", "w")]
        x, y, w = leaves
        order = _order(s["ids"], case["experts"])
        rows, out = _dispatch(x, order), _combine(y, w, order)
        gx, gy, gw = torch.autograd.grad((rows, out), leaves, (s["g_rows"].float(), s["g_out"].float()))
        return [rows.detach().to(dt), out.detach().to(dt), gx.to(dt), gy.to(dt), gw]
    if op == "norms":
        return [v.to(dt) for v in _norms(*[s[n] if s[n] is None else s[n].float() for n in ("x", "t", "pw", "w", "gate")],
                                         case["scale"])]
    if op == "norms_bwd":
        leaves = [s[n].detach().float().requires_grad_() for n in ("x", "t", "pw", "w", "gate") if s[n] is not None]
        x, t, pw, w, *gate = leaves
        h, y = _norms(x, t, pw, w, gate[0] if gate else None, case["scale"])
        grads = torch.autograd.grad((h, y), leaves, (s["gh"].float(), s["gy"].float()))
        return [v.detach().to(dt) for v in (h, y, *grads)]
    x = s["x"].float()
    amax = x.abs().amax(1, keepdim=True)
    q = torch.where(amax > 0, (x * (127.0 / amax)).round(), 0.0)
    if s["offsets"] is None:
        acc = q @ s["q"].float().t()
        return (acc * (amax / 127.0) * s["ws"]).to(dt)
    parts = [q[a:b] @ s["q"][e].float().t() * (amax[a:b] / 127.0) * s["ws"][e] for e, (a, b) in enumerate(s["segments"]) if b > a]
    return torch.cat(parts).to(dt)


def work(case):
    op = case["op"]
    if op in ("sort", "combine", "experts"):
        t, k, d, e = case["tokens"], case["top_k"], case["dim"], case["experts"]
        n, here = t * k, t * k // case["ranks"]             # a rank's own experts get their share of the choices
        sort = 4 * (3 * n + e + 1)
        if op == "sort":
            return {"bytes": sort + 2 * (t * d + n * d), "flops": 0}
        if op == "combine":
            return {"bytes": 8 * n + 2 * (here * d + t * d), "flops": 2 * here * d}
        # rows sorted; the experts' rows read for the sum and again for the weights' gradients; two gradients gathered
        return {"bytes": sort + 2 * (t * d + n * d) + 2 * (2 * here * d + 2 * t * d) + 2 * n * d + 2 * (here * d + t * d) + 12 * n,
                "flops": 6 * here * d}
    if op in ("norms", "norms_bwd"):
        rows, d, kind = case["rows"], case["dim"], case["gate"]
        g = {"none": 0, "channel": 1, "row": rows}.get(kind, kind)
        fwd = 2 * (4 * rows * d + g * d + 2 * d)
        if op == "norms":
            return {"bytes": fwd, "flops": 10 * rows * d}
        # h, t, both upstream gradients and the gate in; the gradients of x, t, the gate and the weights out
        return {"bytes": fwd + 2 * (6 * rows * d + 2 * g * d + 4 * d), "flops": 40 * rows * d}
    m, n, k, e = case["m"], case["n"], case["k"], case["experts"]
    used = max(1, min(e, m))
    return {"bytes": 2 * m * k + used * n * k + 4 * used * n + 2 * m * n, "flops": 2 * m * n * k}


def exact(case, seed):
    op, f64 = case["op"], torch.float64
    s = prepare(case, seed)
    if op in ("sort", "combine", "experts"):
        ids, experts, k = s["ids"].cpu().view(-1).tolist(), case["experts"], case["top_k"]
        by = [[] for _ in range(experts)]
        for i, e in enumerate(ids):
            if 0 <= e < experts:
                by[e].append(i)
        source = [i for rows in by for i in rows]
        here = len(source)
        at = torch.tensor(source, dtype=torch.int64, device=DEVICE)
        token, n, w = at // k, len(ids), s["w"].to(f64).view(-1)
        order = [None, None, None]

        def rows_of(x):
            out = torch.zeros(n, case["dim"], dtype=f64, device=DEVICE)
            out[:here] = x[token].to(f64)
            return out

        def tokens_of(rows, weights=None):
            out = torch.zeros(case["tokens"], case["dim"], dtype=f64, device=DEVICE)
            rows = rows[:here].to(f64)
            return out.index_add_(0, token, rows if weights is None else rows * weights[at][:, None])

        if op == "sort":
            return order + [rows_of(s["x"])]
        if op == "combine":
            return tokens_of(s["y"], w)
        g = s["g_out"]
        gy = torch.zeros(n, case["dim"], dtype=f64, device=DEVICE)
        gy[:here] = g[token].to(f64) * w[at][:, None]
        gw = torch.zeros(n, dtype=f64, device=DEVICE)
        gw[at] = (g[token].to(f64) * s["y"][:here].to(f64)).sum(1)
        return [rows_of(s["x"]), tokens_of(s["y"], w), tokens_of(s["g_rows"]), gy, gw.view(case["tokens"], k)]
    if op in ("norms", "norms_bwd"):
        x, t, pw, w = (s[n].to(f64) for n in ("x", "t", "pw", "w"))
        rows, d = x.shape
        gate = s["gate"]
        lines = 1 if gate is None else gate.numel() // d
        g = torch.ones(1, d, dtype=f64, device=DEVICE) if gate is None else gate.view(lines, d).to(f64)
        g = g.repeat_interleave(rows // lines, 0) if lines > 1 else g
        r1 = 1 / (t.square().sum(1, keepdim=True) / d + EPS).sqrt()
        h = case["scale"] * x + g * pw * (t * r1)
        r2 = 1 / (h.square().sum(1, keepdim=True) / d + EPS).sqrt()
        y = h * r2 * w
        if op == "norms":
            return [h, y]
        gy, n2 = s["gy"].to(f64), h * r2
        dh = s["gh"].to(f64) + r2 * (gy * w - n2 * ((gy * w) * n2).sum(1, keepdim=True) / d)
        n1 = t * r1
        b = dh * g * pw
        dt = r1 * (b - n1 * (b * n1).sum(1, keepdim=True) / d)
        out = [h, y, case["scale"] * dh, dt, (dh * g * n1).sum(0), (gy * n2).sum(0)]
        if gate is not None:
            out.append((dh * n1 * pw).view(lines, rows // lines, d).sum(1).view(gate.shape))
        return out
    # the activations' 8-bit values are part of the definition: nearest integers, ties to even, of x * (127 / amax) in 32 bits
    x = s["x"].to(torch.float32)
    top = x.abs().max(dim=1).values
    step = torch.full_like(top, 127.0) / top
    q = torch.round(x * step[:, None]).nan_to_num(0.0).to(f64)
    out = torch.zeros(case["m"], case["n"], dtype=f64, device=DEVICE)
    weights, scales = s["q"].view(-1, case["n"], case["k"]), s["ws"].view(-1, case["n"]).to(f64)
    for e, (a, b) in enumerate(s["segments"]):
        if b > a:
            out[a:b] = q[a:b] @ weights[e].to(f64).t() * (top[a:b].to(f64) / 127)[:, None] * scales[e]
    return out
