"""The operators of a language model's training step on one GPU, as cases that a timing harness can prepare and run.

Four kinds, each through the calls that a training or scoring program makes:

* ``order``    the plan of a mixture-of-experts layer that drops no token: where every (token, pick) goes when the picks are
  sorted by expert, and where each expert's rows begin (``parallel.moe.expert_order``).  Whole numbers.
* ``experts``  products grouped by expert over such rows, groups of any length (``ops.linear_ragged`` and its gradients
  ``ops.linear_ragged_dgrad`` and ``ops.linear_ragged_wgrad``).
* ``distill``  the loss of a student against the top logits that a teacher left for every token, mixed with the cross
  entropy of the labels (``ops.distill_loss``), or that loss and the gradient of the logits (``ops.distill_loss_grad``).
* ``norm``     the residual connection of a block whose output is normalised too: norm, gate, scaled residual and the next
  block's norm (``ops.residual_norm``) and its gradients (``ops.residual_norm_bwd``).

Widths are those of the named configurations (Llama-2-7B / 70B, GPT-2-XL, Mixtral-8x7B) and of the tests and examples.
"""
from __future__ import annotations

import math

import torch

DEVICE = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}

own = False


def _order(name, tokens, k, experts):
    return {"name": name, "kind": "order", "tokens": tokens, "k": k, "experts": experts}


def _experts(name, direction, tokens, k, experts, d_in, d_out):
    return {"name": name, "kind": "experts", "dir": direction, "tokens": tokens, "k": k, "experts": experts, "d_in": d_in, "d_out": d_out}


def _distill(name, direction, rows, vocab, k, tail, temperature, alpha, dtype="bf16"):
    return {"name": name, "kind": "distill", "dir": direction, "rows": rows, "vocab": vocab, "k": k, "tail": tail,
            "temperature": temperature, "alpha": alpha, "dtype": dtype}


def _norm(name, direction, rows, d, gate_rows, dtype="bf16"):
    return {"name": name, "kind": "norm", "dir": direction, "rows": rows, "d": d, "gate_rows": gate_rows, "dtype": dtype}


def listed():
    return [
        # routing of the small mixture of experts of the tests, a ragged number of tokens
        _order("order_small", 1000, 2, 8),
        # many experts, many picks each: as many picks as a full GPU's microbatch has
        _order("order_many", 8192, 8, 64),
        # one token of a Mixtral-8x7B feed-forward block: two experts' weights are read for two rows
        _experts("experts_token", "fwd", 1, 2, 8, 4096, 28672),
        # a small mixture of experts with a ragged number of tokens
        _experts("experts_small", "fwd", 1000, 2, 8, 512, 2048),
        # the gate and up projections of a Mixtral-8x7B block, one sequence of 4096
        _experts("experts_up", "fwd", 4096, 2, 8, 4096, 28672),
        # both gradients of its down projection
        _experts("experts_down_bwd", "bwd", 4096, 2, 8, 14336, 4096),
        # scoring one short prompt against a teacher's 64 best
        _distill("distill_short", "fwd", 77, 32000, 64, True, 1.0, 1.0),
        # a microbatch of the headline shape: softened distributions, the teacher's remaining mass, half of it from labels
        _distill("distill_llama", "grad", 4096, 32000, 64, True, 2.0, 0.5),
        # a vocabulary that is no multiple of anything, teacher renormalised over its top entries
        _distill("distill_gpt2", "grad", 1024, 50257, 100, False, 1.0, 1.0),
        # the short prompt's residual stream
        _norm("norm_short", "fwd", 77, 4096, 1),
        # a microbatch of the headline shape
        _norm("norm_llama", "fwd", 4096, 4096, 1),
        # Llama-2-70B width, a gate for each of four sequences, gradients
        _norm("norm_70b_bwd", "bwd", 4096, 8192, 4),
    ]


def _log(rng, lo, hi, step=1):
    return max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))) / step)) * step)


def draw(rng):
    """One more case of the ranges above; nothing costs more than the largest listed one."""
    most_f = 0.7 * max(work(c)["flops"] for c in listed())
    most_b = max(work(c)["bytes"] for c in listed())
    while True:
        kind = rng.choice(["order", "experts", "experts", "experts", "distill", "distill", "norm", "norm"])
        if kind == "order":
            experts = rng.randint(2, 64)
            c = {"kind": kind, "tokens": _log(rng, 1, 16384), "k": rng.randint(1, min(8, experts)), "experts": experts}
        elif kind == "experts":
            experts = rng.choice([2, 4, 7, 8, 16, 33, 64])
            c = {"kind": kind, "dir": rng.choice(["fwd", "bwd"]), "tokens": _log(rng, 1, 8192), "k": rng.randint(1, min(4, experts)),
                 "experts": experts, "d_in": _log(rng, 128, 8192, 8), "d_out": _log(rng, 128, 16384, 8)}
        elif kind == "distill":
            c = {"kind": kind, "dir": rng.choice(["fwd", "grad"]), "rows": _log(rng, 1, 8192), "vocab": _log(rng, 300, 60000),
                 "k": rng.randint(1, 256), "tail": rng.random() < 0.5, "temperature": rng.choice([1.0, 1.5, 2.0, 4.0]),
                 "alpha": rng.choice([1.0, 0.5, 0.9]), "dtype": rng.choice(["bf16", "bf16", "fp32"])}
        else:
            gates = rng.choice([0, 1, 2, 4])
            c = {"kind": kind, "dir": rng.choice(["fwd", "bwd"]), "rows": max(1, gates) * _log(rng, 1, 4096), "d": _log(rng, 128, 8192, 8),
                 "gate_rows": gates, "dtype": rng.choice(["bf16", "bf16", "fp32"])}
        if kind == "distill" and c["dtype"] == "fp32" and c["rows"] * c["vocab"] > 10 ** 8:
            continue
        if work(c)["flops"] <= most_f and work(c)["bytes"] <= most_b:
            return c


# ---- inputs -----------------------------------------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device=DEVICE).manual_seed(seed * 7919 + 11)


def _randn(g, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=g, device=DEVICE) * scale).to(dtype)


def _picks(g, tokens, k, experts):
    """Experts of every token as a router picks them: distinct for a token, some experts more wanted than others."""
    logits = _randn(g, tokens, experts) + 0.5 * _randn(g, experts)
    return logits.topk(k, dim=-1).indices


def prepare(case, seed):
    g, s = _gen(seed), {"case": case}
    kind = case["kind"]
    if kind == "order":
        s["picks"] = _picks(g, case["tokens"], case["k"], case["experts"])
    elif kind == "experts":
        rows, e = case["tokens"] * case["k"], case["experts"]
        counts = torch.bincount(_picks(g, case["tokens"], case["k"], e).reshape(-1), minlength=e)
        s["offsets"] = torch.cat([counts.new_zeros(1), counts.cumsum(0)]).to(torch.int32)
        s["longest"] = int(counts.max())
        s["w"] = _randn(g, e, case["d_out"], case["d_in"], dtype=torch.bfloat16, scale=0.02)
        s["x"] = _randn(g, rows, case["d_in"], dtype=torch.bfloat16)
        if case["dir"] == "bwd":
            s["dy"] = _randn(g, rows, case["d_out"], dtype=torch.bfloat16, scale=0.1)
    elif kind == "distill":
        rows, vocab, k, t = case["rows"], case["vocab"], min(case["k"], case["vocab"]), case["temperature"]
        # a few tokens of every row are likely, the rest is a long tail
        teacher = _randn(g, rows, vocab, scale=2.0)
        likely = torch.randint(0, vocab, (rows, 8), generator=g, device=DEVICE)
        teacher.scatter_add_(1, likely, 14 * torch.rand(rows, 8, generator=g, device=DEVICE))
        s["logits"] = (0.8 * teacher + _randn(g, rows, vocab)).to(TYPES[case["dtype"]])
        top, ids = teacher.topk(k, dim=-1)
        s["ids"], s["top"] = ids.to(torch.int32), top.to(TYPES[case["dtype"]])
        s["lse"] = torch.logsumexp(teacher / t, -1) if case["tail"] else None
        # the label is often what the teacher says; prompt tokens (one row in ten) carry neither label nor teacher
        other = torch.randint(0, vocab, (rows,), generator=g, device=DEVICE)
        coin = torch.rand(2, rows, generator=g, device=DEVICE)
        labels = torch.where(coin[0] < 0.6, ids[:, 0], other)
        s["labels"] = torch.where(coin[1] < 0.1, -1, labels) if case["alpha"] < 1 else None
        s["ids"].masked_fill_((coin[1] < 0.1)[:, None], -1)
        s["dloss"] = torch.where(coin[1] < 0.1, 0.0, 1.0 + coin[0])
    else:
        rows, d, dt = case["rows"], case["d"], TYPES[case["dtype"]]
        s["scale"], s["eps"] = 0.9, 1e-5
        s["x"], s["y"] = _randn(g, rows, d, dtype=dt, scale=3.0), _randn(g, rows, d, dtype=dt, scale=0.5)
        s["w_post"], s["w_pre"] = (1 + _randn(g, d, scale=0.1)).to(dt), (1 + _randn(g, d, scale=0.1)).to(dt)
        shape = (case["gate_rows"], d) if case["gate_rows"] > 1 else (d,)
        s["gate"] = _randn(g, *shape, dtype=dt, scale=0.3) if case["gate_rows"] else None
        if case["dir"] == "bwd":
            s["dr"], s["dh"] = _randn(g, rows, d, dtype=dt, scale=0.1), _randn(g, rows, d, dtype=dt, scale=0.1)
            r = _residual(s, s["x"].double(), s["y"].double(), torch.float64)
            s["rstd_post"], s["rstd_pre"] = r["rstd_post"].float().squeeze(-1), r["rstd_pre"].float().squeeze(-1)
    return s


# ---- the calls of a user's program, and the same from elementary operations ----------------------------------------------
def run(state):
    kind = state["case"]["kind"]
    if own:
        return _own(state, kind)
    return {"order": _plain_order, "experts": _plain_experts, "distill": _plain_distill, "norm": _plain_norm}[kind](state)


def _own(s, kind):
    from jaxpp_b200.ops import core as ops

    c = s["case"]
    if kind == "order":
        from jaxpp_b200.parallel import moe

        return moe.expert_order(s["picks"], c["experts"])
    if kind == "experts":
        if c["dir"] == "fwd":
            return ops.linear_ragged(s["x"], s["w"], s["offsets"])
        return ops.linear_ragged_dgrad(s["dy"], s["w"], s["offsets"]), ops.linear_ragged_wgrad(s["dy"], s["x"], s["offsets"])
    if kind == "distill":
        args = (s["logits"], s["ids"], s["top"], s["lse"], s["labels"], c["temperature"], c["alpha"])
        return ops.distill_loss(*args) if c["dir"] == "fwd" else ops.distill_loss_grad(s["dloss"], *args)
    if c["dir"] == "fwd":
        return ops.residual_norm(s["x"], s["y"], s["w_post"], s["gate"], s["w_pre"], s["scale"], s["eps"])[:2]
    grads = ops.residual_norm_bwd(s["dr"], s["dh"], s["x"], s["y"], s["w_post"], s["gate"], s["w_pre"], s["rstd_post"], s["rstd_pre"], s["scale"])
    return grads if s["gate"] is not None else (grads[0], grads[1], grads[2], grads[4])


def _plain_order(s):
    experts = s["case"]["experts"]
    flat = s["picks"].reshape(-1)
    hit = flat[None, :] == torch.arange(experts, device=flat.device)[:, None]
    running = hit.cumsum(1, dtype=torch.int32)
    offsets = torch.cat([running.new_zeros(1), running[:, -1].cumsum(0, dtype=torch.int32)])
    dest = offsets[flat] + running.gather(0, flat[None, :])[0] - 1
    inv = torch.empty_like(dest)
    inv[dest] = torch.arange(flat.numel(), device=flat.device, dtype=torch.int32)
    return dest.long(), inv, offsets


def _plain_experts(s):
    w, offsets, x = s["w"].float(), s["offsets"].long(), s["x"]
    # [experts, longest] row numbers of every group, and the group and place of every row
    at = offsets[:-1, None] + torch.arange(s["longest"], device=x.device)[None, :]
    live = at < offsets[1:, None]
    at = torch.where(live, at, 0)
    row = torch.arange(x.shape[0], device=x.device)
    group = torch.searchsorted(offsets[1:].contiguous(), row, right=True)
    place = row - offsets[group]

    def gather(t):
        return torch.where(live[..., None], t[at].float(), 0.0)

    def scatter(t, like):
        return t[group, place].to(like.dtype)

    if s["case"]["dir"] == "fwd":
        return scatter(torch.bmm(gather(s["x"]), w.transpose(1, 2)), s["x"])
    dy = gather(s["dy"])
    dx = scatter(torch.bmm(dy, w), s["x"])
    return dx, torch.bmm(dy.transpose(1, 2), gather(s["x"])).to(s["w"].dtype)


def _plain_distill(s):
    c = s["case"]
    t, alpha, z = c["temperature"], c["alpha"], s["logits"].float()
    valid = s["ids"] >= 0
    ids = torch.where(valid, s["ids"], 0).long()
    teacher = torch.where(valid, s["top"].float() / t, -math.inf)
    some = valid.any(-1)

    def log_softmax(v):
        v = v - v.amax(-1, keepdim=True)
        return v - v.exp().sum(-1, keepdim=True).log()

    logp_t = log_softmax(z / t)
    if c["tail"]:
        logq = teacher - s["lse"][:, None]
    else:
        logq = log_softmax(torch.where(some[:, None], teacher, 0.0))
    q = torch.where(valid, logq.exp(), 0.0)
    soft = torch.where(q > 0, q * (logq - logp_t.gather(-1, ids)), 0.0).sum(-1)
    ratio, mass = torch.zeros_like(soft), q.sum(-1)
    if c["tail"]:
        # what the teacher and the student leave outside of the listed entries
        q_rest = (1.0 - q.double().sum(-1)).clamp(min=0).float()
        inside = torch.zeros_like(z, dtype=torch.bool).scatter_(-1, ids, valid)
        p_rest = torch.where(inside, 0.0, logp_t.exp()).sum(-1)
        rest = (q_rest > 0) & (p_rest > 0)
        soft = soft + torch.where(rest, q_rest * (q_rest.log() - p_rest.log()), 0.0)
        ratio = torch.where(rest, q_rest / p_rest, 0.0)
        mass = mass + torch.where(rest, q_rest, 0.0)
    loss = torch.where(some, alpha * t * t * soft, 0.0)
    labelled = None
    if alpha < 1:
        labelled = s["labels"] >= 0
        label = torch.where(labelled, s["labels"], 0)[:, None]
        logp = log_softmax(z)
        loss = loss + torch.where(labelled, -(1 - alpha) * logp.gather(-1, label)[:, 0], 0.0)
    if c["dir"] == "fwd":
        return loss
    p = logp_t.exp() * mass[:, None]           # the mass is 1 but for roundings of the teacher's logits
    if c["tail"]:
        p = torch.where(inside, p, p - logp_t.exp() * ratio[:, None])
    dz = torch.where(some[:, None], alpha * t * p.scatter_add(-1, ids, -q), 0.0)
    if alpha < 1:
        d = logp.exp().scatter_add(-1, label, -torch.ones_like(logp[:, :1]))
        dz = dz + torch.where(labelled[:, None], (1 - alpha) * d, 0.0)
    return loss, (dz * s["dloss"][:, None]).to(s["logits"].dtype)


def _residual(s, x, y, dt):
    """The forward formulas in the given type."""
    out = {"rstd_post": torch.rsqrt((y * y).mean(-1, keepdim=True) + s["eps"])}
    out["p"] = y * out["rstd_post"]
    out["n"] = out["p"] * s["w_post"].to(dt)
    out["gate"] = torch.ones((), dtype=dt, device=x.device)
    if s["gate"] is not None:
        gate = s["gate"].to(dt).reshape(-1, x.shape[1])
        out["gate"] = gate.repeat_interleave(x.shape[0] // gate.shape[0], 0)
    out["r"] = s["scale"] * x + out["gate"] * out["n"]
    out["rstd_pre"] = torch.rsqrt((out["r"] * out["r"]).mean(-1, keepdim=True) + s["eps"])
    return out


def _plain_norm(s):
    x, y, dt = s["x"].float(), s["y"].float(), s["x"].dtype
    f = _residual(s, x, y, torch.float32)
    hat, w_pre = f["r"] * f["rstd_pre"], s["w_pre"].float()
    if s["case"]["dir"] == "fwd":
        return f["r"].to(dt), (hat * w_pre).to(dt)
    dr, dh, d = s["dr"].float(), s["dh"].float(), x.shape[1]
    u = dh * w_pre
    dr = dr + f["rstd_pre"] * (u - hat * (u * hat).mean(-1, keepdim=True))
    dn = dr * f["gate"]
    v = dn * s["w_post"].float()
    dy = f["rstd_post"] * (v - f["p"] * (v * f["p"]).mean(-1, keepdim=True))
    out = [s["scale"] * dr, dy, (dn * f["p"]).sum(0)]
    if s["gate"] is not None:
        groups = max(1, s["case"]["gate_rows"])
        out.append((dr * f["n"]).reshape(groups, -1, d).sum(1).reshape(s["gate"].shape))
    return tuple(o.to(dt) for o in (*out, (dh * hat).sum(0)))


# ---- what a pass cannot do without -----------------------------------------------------------------------------------------
def work(case):
    kind = case["kind"]
    if kind == "order":
        n = case["tokens"] * case["k"]
        return {"bytes": n * (8 + 8 + 4) + 4 * (case["experts"] + 1), "flops": 0}
    if kind == "experts":
        rows, e, i, o = case["tokens"] * case["k"], case["experts"], case["d_in"], case["d_out"]
        touched = e * (1 - (1 - case["k"] / e) ** case["tokens"])   # experts that some token picks
        w = touched * i * o * 2
        if case["dir"] == "fwd":
            return {"bytes": int(w + rows * (i + o) * 2 + 4 * (e + 1)), "flops": 2 * rows * i * o}
        return {"bytes": int(w + e * i * o * 2 + rows * (2 * i + o) * 2 + 4 * (e + 1)), "flops": 4 * rows * i * o}
    size = 4 if case["dtype"] == "fp32" else 2
    if kind == "distill":
        rows, vocab, k = case["rows"], case["vocab"], min(case["k"], case["vocab"])
        small = rows * (k * (4 + size) + 4 + (4 if case["tail"] else 0) + (8 if case["alpha"] < 1 else 0))
        exps = 2 if case["alpha"] < 1 and case["temperature"] != 1.0 else 1
        if case["dir"] == "fwd":
            return {"bytes": rows * vocab * size + small, "flops": rows * vocab * (3 + 2 * exps)}
        return {"bytes": 2 * rows * vocab * size + small + 4 * rows, "flops": rows * vocab * (5 + 5 * exps)}
    rows, d, g = case["rows"], case["d"], case["gate_rows"]
    if case["dir"] == "fwd":
        return {"bytes": (4 * rows * d + (2 + g) * d) * size, "flops": 11 * rows * d}
    return {"bytes": (6 * rows * d + 2 * (2 + g) * d) * size + 8 * rows, "flops": 28 * rows * d}


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------------------
def exact(case, seed):
    s, kind = prepare(case, seed), case["kind"]
    if kind == "order":
        return None
    if kind == "experts":
        ends = s["offsets"].tolist()
        x = s["x"]
        if case["dir"] == "fwd":
            out = torch.zeros(x.shape[0], case["d_out"], dtype=torch.float64, device=x.device)
            for e, (a, b) in enumerate(zip(ends, ends[1:])):
                out[a:b] = x[a:b].double() @ s["w"][e].double().t()
            return out
        dx = torch.zeros(x.shape, dtype=torch.float64, device=x.device)
        dw = torch.zeros(s["w"].shape, dtype=torch.float64, device=x.device)
        for e, (a, b) in enumerate(zip(ends, ends[1:])):
            dy = s["dy"][a:b].double()
            dx[a:b] = dy @ s["w"][e].double()
            dw[e] = dy.t() @ x[a:b].double()
        return dx, dw
    if kind == "distill":
        return _exact_distill(s)
    return _exact_norm(s)


def _exact_distill(s):
    """From the definition of the loss, differentiated by autograd, 256 rows at a time."""
    c = s["case"]
    t, alpha, losses, grads = c["temperature"], c["alpha"], [], []
    for a in range(0, c["rows"], 256):
        cut = slice(a, a + 256)
        z = s["logits"][cut].double().requires_grad_(True)
        ids, top = s["ids"][cut].long(), s["top"][cut].double()
        has = ids[:, 0] >= 0                       # a row has all its entries or none
        ids = ids.clamp(min=0)
        p = torch.softmax(z / t, -1)
        p_in = p.gather(-1, ids)
        if c["tail"]:
            q_in = torch.exp(top / t - s["lse"][cut].double()[:, None])
            q_out = (1 - q_in.sum(-1)).clamp(min=0)
            outside = torch.ones_like(p).scatter(-1, ids, 0.0)
            kl = (q_in * (q_in / p_in).log()).sum(-1)
            p_out = (p * outside).sum(-1)
            live = (q_out > 0) & (p_out > 0)
            kl = kl + torch.where(live, q_out * (torch.where(live, q_out, 1.0) / torch.where(live, p_out, 1.0)).log(), 0.0)
        else:
            q_in = torch.softmax(top / t, -1)
            kl = (q_in * (q_in / p_in).log()).sum(-1)
        loss = torch.where(has, alpha * t ** 2 * kl, 0.0)
        if alpha < 1:
            y = s["labels"][cut]
            nll = torch.logsumexp(z, -1) - z.gather(-1, y.clamp(min=0)[:, None])[:, 0]
            loss = loss + torch.where(y >= 0, (1 - alpha) * nll, 0.0)
        losses.append(loss.detach())
        if c["dir"] == "grad":
            grads.append(torch.autograd.grad((loss * s["dloss"][cut].double()).sum(), z)[0])
    loss = torch.cat(losses)
    return loss if c["dir"] == "fwd" else (loss, torch.cat(grads))


def _exact_norm(s):
    """From the definition; the gradients by autograd, with the parameters' sums over all rows."""
    bwd = s["case"]["dir"] == "bwd"
    names = ["x", "y", "w_post"] + (["gate"] if s["gate"] is not None else []) + ["w_pre"]
    v = {k: s[k].double().requires_grad_(bwd) for k in names}
    rows, d = v["x"].shape

    def unit(t):
        return t / (t.square().sum(-1, keepdim=True) / d + s["eps"]).sqrt()

    n = unit(v["y"]) * v["w_post"]
    if "gate" in v:
        groups = v["gate"].numel() // d
        n = (n.view(groups, rows // groups, d) * v["gate"].view(groups, 1, d)).view(rows, d)
    r = s["scale"] * v["x"] + n
    h = unit(r) * v["w_pre"]
    if not bwd:
        return r, h
    total = (r * s["dr"].double()).sum() + (h * s["dh"].double()).sum()
    return torch.autograd.grad(total, [v[k] for k in names])
