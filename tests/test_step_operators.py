"""Residual norm, distillation loss and the order of expert picks against plain 64-bit implementations, on the CPU (the
reference implementations of the ops) and on the GPU (the kernels).

Tolerances: a result is rounded once to its type, which is half a step (``finfo.eps / 2`` of its value), and comes from fp32
arithmetic, whose part is derived beside each test as a number of roundings of 2^-24 of the size of the terms."""
import math
import os
import subprocess
import sys

import pytest
import torch

import jaxpp_b200 as jp  # noqa: F401  (registers the ops)
from jaxpp_b200.ops import core as ops
from jaxpp_b200.parallel import moe

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
U = 2.0 ** -24   # half a step of fp32


@pytest.fixture(autouse=True)
def status():
    yield
    if torch.cuda.is_available():
        from jaxpp_b200.ops import native

        if native.is_available():
            torch.cuda.synchronize()
            assert native.read_status() == 0, "a kernel reported a time-out or a bad argument"


def rnd(seed, *shape, scale=1.0, dtype=torch.float32, device="cpu"):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype).to(device)


def within(got, want, slack):
    """|got - want| <= half a step of got's type, plus ``slack`` (a number or a tensor)."""
    got, want = got.detach().double().cpu(), want.detach().double().cpu()
    half = torch.finfo(GOT[0]).eps / 2
    slack = slack.double().cpu() if isinstance(slack, torch.Tensor) else slack
    off = (got - want).abs() - (half * want.abs() * (1 + 2 ** -7) + slack)
    assert got.shape == want.shape
    assert not torch.isnan(got).any()
    assert (off <= 0).all(), f"off by {off.max().item():.3g} more than allowed at {off.argmax().item()}"


GOT = [torch.float32]


def check(got, want, slack):
    GOT[0] = got.dtype
    within(got, want, slack)


# ---- residual norm -------------------------------------------------------------------------------------------------------
def norm_inputs(rows, d, gates, post, pre, dtype, device, seed=0):
    x, y = rnd(seed, rows, d, scale=2.0, dtype=dtype, device=device), rnd(seed + 1, rows, d, scale=0.5, dtype=dtype, device=device)
    w_post = (1 + rnd(seed + 2, d, scale=0.2)).to(dtype).to(device) if post else None
    w_pre = (1 + rnd(seed + 3, d, scale=0.2)).to(dtype).to(device) if pre else None
    gate = None if gates is None else rnd(seed + 4, *((gates, d) if gates else (d,)), dtype=dtype, device=device)
    return x, y, w_post, gate, w_pre


def norm_exact(x, y, w_post, gate, w_pre, scale, eps):
    rows, d = x.numel() // x.shape[-1], x.shape[-1]
    n = y
    if w_post is not None:
        n = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + eps) * w_post
    if gate is not None:
        g = gate.reshape(-1, 1, d)
        n = (n.reshape(g.shape[0], rows // g.shape[0], d) * g).reshape(x.shape)
    r = scale * x + n
    return r, None if w_pre is None else r * torch.rsqrt(r.square().mean(-1, keepdim=True) + eps) * w_pre


NORMS = [  # rows, d, gate rows (0: one vector; None: no gate), post, pre
    (1, 8, 0, True, True), (5, 8, None, True, True), (3, 264, 0, True, False), (4, 1024, None, False, True), (6, 40, 2, True, True),
    (7, 4096, 7, True, True), (130, 1600, 0, True, True), (64, 512, 4, False, True), (2, 8192, 0, True, True),
    (9, 136, 3, True, False), (40, 2000, 0, True, True), (0, 64, 0, True, True), (300, 128, 0, False, False), (40, 16384, 2, True, True),
    (300, 1024, 4, True, True), (160, 2048, 40, True, True), (97, 512, 0, True, True), (320, 5120, None, True, True), (64, 256, 64, True, True),
    (300, 1024, 4, True, False), (160, 2048, None, False, True), (97, 512, 0, False, True), (65, 8192, 0, True, False), (8, 16384, 4, False, True),
]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,d,gates,post,pre", NORMS)
def test_residual_norm(device, dtype, rows, d, gates, post, pre):
    if device == "cuda" and dtype == torch.float32 and d > 8192:
        pytest.skip("rows of at most 8192 float32 elements")
    x, y, w_post, gate, w_pre = norm_inputs(rows, d, gates, post, pre, dtype, device)
    scale, eps = 0.75, 1e-5
    r, h, rstd_post, rstd_pre = ops.residual_norm(x, y, w_post, gate, w_pre, scale, eps)
    ins = [None if t is None else t.double().cpu().requires_grad_(True) for t in (x, y, w_post, gate, w_pre)]
    er, eh = norm_exact(*ins, scale, eps)
    # r: the mean square is a sum of d positive terms in a tree of at most 16 + log2(d) roundings each, halved by the root;
    # then a handful of products.  h: the same once more, and r's error over its root mean square
    depth = 32 + math.log2(d)
    gsize = 1.0 if gate is None else float(gate.float().abs().max()) if gate.numel() else 0.0
    nmax = (ins[1].abs().amax(-1, keepdim=True) * 3 if w_post is None else 3 * math.sqrt(d)) if rows else 0.0
    part = (ins[0].abs() * scale + gsize * nmax).detach() if rows else 0.0
    check(r, er, depth * U * part)
    if pre:
        check(h, eh, 3 * depth * U * (eh.detach().abs() + part * 2 / er.detach().square().mean(-1, keepdim=True).sqrt()) if rows else 0.0)
    else:
        assert h.numel() == 0 and rstd_pre.numel() == 0
    assert rstd_post.numel() == (rows if post else 0)
    # gradients, through autograd and by the op with fp32 sums
    dr, dh = rnd(11, rows, d, dtype=dtype, device=device), rnd(12, rows, d, dtype=dtype, device=device)
    total = (er * dr.double().cpu()).sum() + ((eh * dh.double().cpu()).sum() if pre else 0.0)
    live = [t for t in ins if t is not None]
    want = dict(zip([i for i, t in enumerate(ins) if t is not None], torch.autograd.grad(total, live)))
    leaves = [None if t is None else t.clone().requires_grad_(True) for t in (x, y, w_post, gate, w_pre)]
    r2, h2, _, _ = ops.residual_norm(*leaves, scale, eps)
    got = torch.autograd.grad([r2] + ([h2] if pre else []), [t for t in leaves if t is not None], [dr] + ([dh] if pre else []))
    got = dict(zip(want, got))
    # terms: |dr| + rstd_pre (|u| + |hat| mean|u hat|) all of unit size, times gate, weights and rstd_post
    inv = 1.0 if not rows or not pre else 1 / er.detach().square().mean(-1, keepdim=True).add(eps).sqrt()
    size = (dr.double().cpu().abs() + (inv * (2 * dh.double().cpu().abs() + 4 * er.detach().abs() * inv) if pre else 0)) if rows else torch.zeros(rows, d)
    rp = 1.0 if not post or not rows else 1 / ins[1].detach().square().mean(-1, keepdim=True).add(eps).sqrt()
    top = size.amax(-1, keepdim=True) if rows else 0.0
    slack = {0: 4 * depth * U * size, 1: 8 * depth * U * rp * gsize * 2 * (top if rows else 0.0)}
    for i in (2, 3, 4):   # sums over rows of products of unit-size terms, each with the error of its terms
        slack[i] = 0.0 if not rows else 8 * (depth + math.log2(rows + 1) + 8) * U * rows * float(top.max()) * max(1.0, gsize) * 4
    for i in want:
        check(got[i], want[i], slack[i])
    back = ops.residual_norm_bwd(dr, dh if pre else None, x, y, w_post, gate, w_pre, rstd_post, rstd_pre, scale, torch.float32)
    assert all(back[i].dtype == torch.float32 for i in want if i >= 2)
    for i in want:
        if i >= 2:
            check(back[i], want[i], slack[i] + 1e-30)
        else:
            assert torch.equal(back[i], got[i])


@pytest.mark.parametrize("device", DEVICES)
def test_residual_norm_absent_gradients(device):
    """dr or dh None is a gradient of zeros."""
    x, y, w_post, gate, w_pre = norm_inputs(6, 72, 3, True, True, torch.float32, device)
    _, _, a, b = ops.residual_norm(x, y, w_post, gate, w_pre, 1.0, 1e-6)
    g, zero = rnd(5, 6, 72, device=device), torch.zeros(6, 72, device=device)
    for dr, dh in ((g, None), (None, g)):
        got = ops.residual_norm_bwd(dr, dh, x, y, w_post, gate, w_pre, a, b, 1.0)
        want = ops.residual_norm_bwd(zero if dr is None else dr, zero if dh is None else dh, x, y, w_post, gate, w_pre, a, b, 1.0)
        for p, q in zip(got, want):
            assert torch.equal(p, q)
    leaves = [t.clone().requires_grad_(True) for t in (x, y, w_post, gate, w_pre)]
    r, h, _, _ = ops.residual_norm(*leaves, 1.0, 1e-6)
    grads = torch.autograd.grad(r.sum(), leaves, allow_unused=True)     # nothing arrives over h
    assert grads[4] is None or not grads[4].any()
    assert torch.allclose(grads[0], torch.ones_like(x))


@pytest.mark.parametrize("device", DEVICES)
def test_residual_norm_differences(device):
    """The gradient against central differences of the forward, fp32 inputs, along random directions: the truncation is the
    third derivative times step^2 / 6 (terms of unit size, a few dozen at most: 1e-4 of the sum of squares at step 1e-2), the
    rounding 2^-24 of the sum of sizes over the step."""
    args = norm_inputs(4, 64, 2, True, True, torch.float32, device, seed=3)
    dr, dh = rnd(7, 4, 64, device=device), rnd(8, 4, 64, device=device)
    _, _, a, b = ops.residual_norm(*args, 0.9, 1e-5)
    grads = ops.residual_norm_bwd(dr, dh, *args, a, b, 0.9)
    value = lambda t: sum((o.double() * g.double()).sum() for o, g in zip(ops.residual_norm(*t, 0.9, 1e-5)[:2], (dr, dh)))
    for i in range(5):
        step = rnd(20 + i, *args[i].shape, device=device)
        up, down = list(args), list(args)
        up[i], down[i] = args[i] + 1e-2 * step, args[i] - 1e-2 * step
        want = (value(up) - value(down)).item() / 2e-2
        got = (grads[i].double() * step.double()).sum().item()
        assert abs(got - want) <= 2e-3 * (1 + grads[i].double().norm().item() * step.double().norm().item() / 8)


@pytest.mark.parametrize("device", DEVICES)
def test_residual_norm_views(device):
    """Strided, transposed and unaligned operands give what their copies give."""
    big = rnd(1, 6, 3, 80, dtype=torch.bfloat16, device=device)
    flat = rnd(2, 6 * 80 + 1, dtype=torch.bfloat16, device=device)
    x, y = big[:, 1, :], flat[1:].view(6, 80)
    w = flat[3:83]
    got = ops.residual_norm(x, y, w, None, w, 1.0, 1e-5)
    want = ops.residual_norm(x.clone(), y.clone(), w.clone(), None, w.clone(), 1.0, 1e-5)
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    dt = rnd(4, 80, 6, dtype=torch.bfloat16, device=device).t()
    got = ops.residual_norm_bwd(dt, dt, x, y, w, None, w, got[2], got[3])
    want = ops.residual_norm_bwd(dt.contiguous(), dt.contiguous(), x.clone(), y.clone(), w.clone(), None, w.clone(), want[2], want[3])
    assert all(torch.equal(p, q) for p, q in zip(got, want))


def test_residual_norm_refusals():
    x, y, w, gate, _ = norm_inputs(6, 16, 0, True, True, torch.float32, "cpu")
    for bad in ((x, y[:5], w, gate, w), (x, y.bfloat16(), w, gate, w), (x, y, w[:8], gate, w), (x, y, w, gate[:8], w),
                (x, y, w, gate.expand(4, 16), w), (x, y, w, gate, w.bfloat16()), (x, y, w, gate.expand(1, 1, 16), w)):
        with pytest.raises((ValueError, RuntimeError)):
            ops.residual_norm(*bad, 1.0, 1e-5)
    with pytest.raises((ValueError, RuntimeError)):
        ops.residual_norm_bwd(x[:5], None, x, y, w, gate, w, x[:, 0], x[:, 0])
    with pytest.raises((ValueError, RuntimeError)):
        ops.residual_norm_bwd(x, x, x, y, w, gate, w, x[:, 0], x[:3, 0])


@pytest.mark.gpu
def test_residual_norm_refusals_gpu():
    from jaxpp_b200.ops import native

    args = norm_inputs(3, 16, 0, True, True, torch.float32, "cuda")
    for bad in (norm_inputs(3, 12, None, True, True, torch.bfloat16, "cuda"), norm_inputs(3, 8200, None, True, True, torch.float32, "cuda"),
                norm_inputs(3, 16, None, True, True, torch.float16, "cuda"), (*args[:2], args[2].cpu(), *args[3:])):
        with pytest.raises(native.NativeError):
            ops.residual_norm(*bad, 1.0, 1e-5)


# ---- distillation loss -----------------------------------------------------------------------------------------------------
def distill_inputs(rows, V, K, device, dtype=torch.float32, tail=True, labels=True, t=1.0, ids_dtype=torch.int32, seed=0, scale=2.0):
    teacher = rnd(seed, rows, V, scale=scale)
    teacher[:, : min(V, 3)] += 4.0
    logits = (0.8 * teacher + rnd(seed + 1, rows, V)).to(dtype).to(device)
    top, ids = teacher.topk(min(K, V), dim=-1)
    top = top.to(dtype)
    if K > V:   # more places than entries: the others hold none
        top, ids = torch.nn.functional.pad(top, (0, K - V)), torch.nn.functional.pad(ids, (0, K - V), value=-1)
    lse = torch.logsumexp(teacher / t, -1).to(device) if tail else None
    lab = None
    if labels:
        lab = torch.randint(0, V, (rows,), generator=torch.Generator().manual_seed(seed + 2)).to(device)
    return logits, ids.to(ids_dtype).to(device), top.to(device), lse, lab


def distill_exact(dloss, logits, ids, top, lse, labels, t, alpha):
    """Row by row and entry by entry from the definition, in 64 bits.  Returns losses, gradients and, for the tolerances, the
    sizes of the gradient's terms."""
    V = logits.shape[-1]
    losses, grads, sizes = [], [], []
    for r in range(logits.shape[0]):
        z = logits[r].double().cpu()
        p, p1 = torch.softmax(z / t, 0), torch.softmax(z, 0)
        ent = [(int(i), float(v)) for i, v in zip(ids[r].tolist(), top[r].double().tolist()) if 0 <= i < V and v != -math.inf]
        loss, grad, size = 0.0, torch.zeros(V, dtype=torch.float64), torch.zeros(V, dtype=torch.float64)
        if ent:
            q = torch.tensor([v / t for _, v in ent], dtype=torch.float64)
            logq = q - float(lse[r]) if lse is not None else torch.log_softmax(q, 0)
            q, where = logq.exp(), torch.tensor([i for i, _ in ent])
            kl = float((q * (logq - torch.log_softmax(z / t, 0)[where]))[q > 0].sum())
            mass, ratio = float(q.sum()), 0.0
            inside = torch.zeros(V, dtype=torch.bool)
            inside[where] = True
            if lse is not None:
                q_o, p_o = max(0.0, 1.0 - mass), float(p[~inside].sum())
                if q_o > 0 and p_o >= 2.0 ** -126:
                    ratio = q_o / p_o
                    kl += q_o * math.log(ratio)
                    mass += q_o
            loss += alpha * t * t * kl
            d = torch.where(inside, p * mass, p * (mass - ratio)).index_add(0, where, -q)
            grad += alpha * t * d
            size += alpha * t * (p * (mass + ratio)).index_add(0, where, q)
        if labels is not None and 0 <= int(labels[r]) < V:
            y = int(labels[r])
            loss += (1 - alpha) * -float(torch.log_softmax(z, 0)[y])
            d = p1.clone()
            d[y] -= 1
            grad += (1 - alpha) * d
            size += (1 - alpha) * d.abs()
            size[y] += 2 * (1 - alpha)
        w = float(dloss[r])
        losses.append(loss)
        grads.append(grad * w if w else torch.zeros_like(grad))
        sizes.append(size * abs(w) if w else torch.zeros_like(size))
    stack = lambda v: torch.stack(v) if v else torch.zeros(0, V, dtype=torch.float64)
    return torch.tensor(losses, dtype=torch.float64), stack(grads), stack(sizes)


def distill_slack(logits, t):
    """Roundings of a logarithm of a probability: the argument (z - m) / t of an exponential has three, each half a step of
    its size, the exponential is good to 2^-22, sums of positive terms to 16 roundings, and the logarithm's own value is as
    large as the argument; a probability is off by the same relative amount."""
    span = float((logits.float().amax(-1) - logits.float().clamp(min=-1e4).amin(-1)).max()) / min(t, 1.0) if logits.numel() else 0.0
    return U * (4 * 5 + 16 + 6 * span)


def check_distill(device, logits, ids, top, lse, labels, t, alpha, seed=9):
    rows = logits.shape[0]
    dloss = rnd(seed, rows, device=device)
    if rows > 2:
        dloss[1] = 0.0
    el, eg, size = distill_exact(dloss, logits, ids, top, lse, labels, t, alpha)
    rel = distill_slack(logits, t)
    span = 40.0
    one = ops.distill_loss(logits, ids, top, lse, labels, t, alpha)
    check(one, el, rel * 2 * max(1.0, t * t) * (1 + el.abs()) + span * U)
    loss, dz = ops.distill_loss_grad(dloss, logits, ids, top, lse, labels, t, alpha)
    check(loss, el, rel * 2 * max(1.0, t * t) * (1 + el.abs()) + span * U)
    assert dz.dtype == logits.dtype
    # values below the smallest normal one of fp32 may be flushed to zero
    check(dz, eg, 2 * rel * size + 2.0 ** -126)
    leaf = logits.clone().requires_grad_(True)
    out = ops.distill_loss(leaf, ids, top, lse, labels, t, alpha)
    (again,) = torch.autograd.grad(out, leaf, dloss)
    assert torch.equal(again, dz)
    return loss, dz


DISTILLS = [  # rows, V, K, tail, labels, temperature, alpha
    (1, 1, 1, False, True, 1.0, 0.5), (3, 5, 2, True, True, 2.0, 0.5), (4, 8, 8, True, False, 1.0, 1.0), (4, 31, 7, True, True, 1.0, 0.25),
    (3, 257, 64, False, True, 4.0, 0.5), (3, 1000, 16, True, True, 1.5, 0.9), (2, 4097, 100, True, False, 2.0, 1.0),
    (2, 32000, 64, True, True, 2.0, 0.5), (2, 50257, 100, False, False, 1.0, 1.0), (2, 333, 400, True, True, 1.0, 0.0),
    (0, 64, 4, True, True, 1.0, 0.5), (3, 40, 0, True, True, 1.0, 0.5), (2, 128256, 256, True, True, 0.5, 0.5), (300, 130, 5, True, True, 1.0, 0.5),
    (300, 24000, 16, True, True, 1.0, 1.0), (300, 12000, 16, True, True, 1.0, 1.0),   # rows that take just under 48 KB
    (2, 500001, 64, True, True, 2.0, 0.5), (150, 32000, 64, True, True, 1.0, 0.5), (5, 70000, 1024, True, True, 4.0, 0.5),
]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,V,K,tail,labels,t,alpha", DISTILLS)
def test_distill(device, dtype, rows, V, K, tail, labels, t, alpha):
    if device == "cuda" and V * dtype.itemsize > 8 * (220 * 1024 - 24 * K):
        pytest.skip("rows of at most 8 * (220 KB - 24 bytes an entry)")
    args = distill_inputs(rows, V, K, device, dtype, tail, labels, t, torch.int64 if K % 2 else torch.int32)
    check_distill(device, *args, t, alpha)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("tail", [True, False])
def test_distill_edges(device, tail):
    """Rows without entries or labels, entries that are none, repeated ids, -inf on both sides, labels out of range."""
    logits, ids, top, lse, labels = distill_inputs(8, 77, 6, device, torch.float32, tail, True, 2.0, torch.int64)
    lowest = torch.finfo(torch.float32).min
    ids[0] = -1                                    # no entry
    ids[1, 2:] = 77                                # out of range from the third on
    ids[2, 3:5] = ids[2, 0]                        # an id three times
    top[3, 1] = -math.inf                          # an entry of probability zero
    top[4] = -math.inf                             # all of them
    ids[5, 1], logits[5, 70] = 70, -math.inf       # a masked logit where the teacher has nothing
    top[5, 1] = -math.inf
    logits[6, 60:] = -math.inf                     # masked vocabulary outside of the entries
    ids[6] = torch.arange(6, device=device)
    logits[7, 60:] = lowest
    ids[7] = torch.arange(6, device=device)
    labels[0], labels[1], labels[3] = -1, -100, 77
    labels[5:] = 3
    if tail:
        lse += 1.0                                 # the teacher keeps mass outside of its entries in every row
    loss, dz = check_distill(device, logits, ids, top, lse, labels, 2.0, 0.5)
    assert float(loss[0]) == 0.0 and not dz[0].any()
    assert not dz[6, 60:].any()


@pytest.mark.parametrize("device", DEVICES)
def test_distill_no_mass_left(device):
    """Entries that cover the vocabulary leave nothing outside: no division by it."""
    logits, _, _, _, labels = distill_inputs(3, 12, 4, device, torch.float32, False, True)
    teacher = rnd(3, 3, 12, device=device)
    ids = torch.arange(12, device=device).expand(3, 12).contiguous()
    lse = torch.logsumexp(teacher, -1) + torch.tensor([0.0, 1e-6, -1e-3], device=device)
    check_distill(device, logits, ids, teacher, lse, labels, 1.0, 0.75)


@pytest.mark.parametrize("device", DEVICES)
def test_distill_weightless_row(device):
    """A row of weight zero has no gradient even where its logits are NaN; the others are not touched by it."""
    logits, ids, top, lse, labels = distill_inputs(4, 300, 8, device)
    dloss = torch.tensor([1.0, 0.0, 2.0, 1.0], device=device)
    want = ops.distill_loss_grad(dloss, logits, ids, top, lse, labels, 1.0, 0.5)
    bad = logits.clone()
    bad[1, 5] = math.nan
    loss, dz = ops.distill_loss_grad(dloss, bad, ids, top, lse, labels, 1.0, 0.5)
    assert not dz[1].any() and torch.equal(dz, want[1]) and torch.isnan(loss[1])
    assert torch.equal(loss[[0, 2, 3]], want[0][[0, 2, 3]])


@pytest.mark.parametrize("device", DEVICES)
def test_distill_differences(device):
    """Against central differences of the loss in fp32: step 1e-2, truncation step^2 / 6 of a third derivative of at most
    alpha t^2 / t^3 + 1 = 2 per unit direction, rounding 2^-20 of the loss over the step."""
    logits, ids, top, lse, labels = distill_inputs(3, 50, 5, device)
    for tail in (lse, None):
        _, dz = ops.distill_loss_grad(torch.ones(3, device=device), logits, ids, top, tail, labels, 2.0, 0.6)
        step = rnd(31, 3, 50, device=device) * 0.2
        value = lambda z: ops.distill_loss(z, ids, top, tail, labels, 2.0, 0.6).double().sum().item()
        want = (value(logits + 1e-2 * step) - value(logits - 1e-2 * step)) / 2e-2
        assert abs((dz.double() * step.double()).sum().item() - want) < 1e-3


@pytest.mark.parametrize("device", DEVICES)
def test_distill_shapes_and_views(device):
    """Leading dimensions, strided logits (a slice of a padded vocabulary), unaligned views, teacher logits of another type."""
    logits, ids, top, lse, labels = distill_inputs(6, 300, 7, device, torch.bfloat16)
    want = ops.distill_loss_grad(torch.ones(6, device=device), logits, ids, top, lse, labels, 1.0, 0.5)
    padded = torch.full((6, 320), 9.0, dtype=torch.bfloat16, device=device)
    padded[:, :300] = logits
    flat = torch.zeros(6 * 300 + 1, dtype=torch.bfloat16, device=device)
    flat[1:] = logits.reshape(-1)
    for z in (padded[:, :300], flat[1:].view(6, 300), logits.view(2, 3, 300)):
        sh = z.shape[:-1]
        loss, dz = ops.distill_loss_grad(torch.ones(sh, device=device), z, ids.view(*sh, 7), top.float().view(*sh, 7), lse.view(sh),
                                         labels.view(sh), 1.0, 0.5)
        assert loss.shape == sh and dz.shape == z.shape and dz.is_contiguous()
        # the two may add up a row in another order: each is within 2 * distill_slack * (1 + loss) of the exact value (as in
        # check_distill), so they are within twice that of one another
        twice = 4 * distill_slack(logits, 1.0) * (1 + want[0].double().cpu())
        check(loss.reshape(-1), want[0], twice)
        assert (dz.reshape(6, 300).float() - want[1].float()).abs().max() < 1e-2
        check(ops.distill_loss(z, ids.view(*sh, 7), top.view(*sh, 7), lse.view(sh), labels.view(sh), 1.0, 0.5).reshape(-1), want[0], twice)


@pytest.mark.parametrize("device", DEVICES)
def test_distill_far_apart(device):
    """Logits far from the entries': sums that leave fp32's range relative to an entry, large offsets common to a row, small and
    large temperatures, a row of equal logits."""
    for t in (2.0, 0.25, 8.0):
        logits, ids, top, lse, labels = distill_inputs(6, 900, 4, device, torch.float32, True, True, t, torch.int64)
        ids[:, :] = torch.arange(4, device=device)
        logits[0, 500:] += 300.0                # the row's maximum is e^300 above the entries
        logits[1] += 10000.0
        logits[2] -= 5000.0
        logits[3] = 7.25
        logits[4, 4:] = -400.0                  # the entries hold everything
        ids[5], labels[5] = -1, 3
        logits[5, :] -= 200.0                   # no entries, a label far below zero
        check_distill(device, logits, ids, top, lse, labels, t, 0.5)


def test_distill_refusals():
    logits, ids, top, lse, labels = distill_inputs(4, 30, 5, "cpu")
    bad = [(logits, ids[:3], top, lse, labels, 1.0, 1.0), (logits, ids.float(), top, lse, labels, 1.0, 1.0),
           (logits, ids, top[:, :3], lse, labels, 1.0, 1.0), (logits, ids, top, lse.double(), labels, 1.0, 1.0),
           (logits, ids, top, lse[:2], labels, 1.0, 1.0), (logits, ids, top, lse, labels.int(), 1.0, 1.0),
           (logits, ids, top, lse, labels, 0.0, 1.0), (logits, ids, top, lse, labels, -1.0, 1.0),
           (logits, ids, top, lse, labels, 1.0, 1.5), (logits, ids, top, lse, labels, math.inf, 0.5)]
    for args in bad:
        with pytest.raises((ValueError, RuntimeError)):
            ops.distill_loss(*args)
    with pytest.raises((ValueError, RuntimeError)):
        ops.distill_loss_grad(torch.ones(3), logits, ids, top, lse, labels, 1.0, 1.0)


@pytest.mark.gpu
def test_distill_refusals_gpu():
    from jaxpp_b200.ops import native

    args = distill_inputs(2, 1100, 1025, "cuda")
    with pytest.raises(native.NativeError):
        ops.distill_loss(*args)                                       # more than 1024 entries
    args = distill_inputs(2, 30, 5, "cuda")
    for i, other in ((0, args[0].half()), (1, args[1].cpu()), (2, args[2].half())):
        with pytest.raises(native.NativeError):
            ops.distill_loss(*args[:i], other, *args[i + 1:])


# ---- order of the picks ---------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("tokens,k,experts,strangers", [
    (0, 2, 8, False), (1, 1, 1, False), (1, 2, 8, False), (33, 2, 3, True), (1000, 2, 8, False), (1024, 1, 64, False), (5000, 8, 64, True),
    (4097, 3, 33, False), (30000, 8, 256, True)])
def test_expert_order(device, tokens, k, experts, strangers):
    g = torch.Generator().manual_seed(tokens + experts)
    picks = torch.randint(0, experts, (tokens, k), generator=g)
    picks[picks == experts // 2] = 0                                   # an expert that nobody picks
    if strangers:
        picks[torch.rand(tokens, k, generator=g) < 0.2] = -1
        picks[torch.rand(tokens, k, generator=g) < 0.1] = experts + 2 ** 33
    dest, inv, offsets = moe.expert_order(picks.to(device), experts)
    flat = picks.reshape(-1).tolist()
    lists = [[] for _ in range(experts)]
    for i, e in enumerate(flat):
        if 0 <= e < experts:
            lists[e].append(i)
    order = [i for one in lists for i in one]
    want_inv = order + [-1] * (len(flat) - len(order))
    want_dest = [len(flat)] * len(flat)
    for place, i in enumerate(order):
        want_dest[i] = place
    want_off = [0]
    for one in lists:
        want_off.append(want_off[-1] + len(one))
    assert dest.tolist() == want_dest and inv.tolist() == want_inv and offsets.tolist() == want_off
    assert dest.dtype == torch.int64 and inv.dtype == torch.int32 and offsets.dtype == torch.int32


def test_expert_order_refusals():
    for picks, experts in ((torch.zeros(4, 2, dtype=torch.int32), 8), (torch.zeros(4, 2, dtype=torch.int64), 0),
                           (torch.zeros(4, 2, dtype=torch.int64), 257)):
        with pytest.raises((ValueError, RuntimeError)):
            moe.expert_order(picks, experts)


# ---- streams and graphs -----------------------------------------------------------------------------------------------------
def _calls():
    """(name, call on fresh operands): what a program would capture."""
    x, y, w_post, gate, w_pre = norm_inputs(48, 1024, 4, True, True, torch.bfloat16, "cuda")
    _, _, a, b = ops.residual_norm(x, y, w_post, gate, w_pre, 0.9, 1e-5)
    logits, ids, top, lse, labels = distill_inputs(60, 3001, 17, "cuda", torch.bfloat16, True, True, 2.0)
    picks = torch.randint(0, 8, (700, 2), generator=torch.Generator().manual_seed(1)).cuda()
    many = torch.randint(0, 64, (9000, 2), generator=torch.Generator().manual_seed(2)).cuda()
    offsets = moe.expert_order(picks, 8)[2]
    rows, w, dy = rnd(3, 1400, 256, dtype=torch.bfloat16, device="cuda"), rnd(4, 8, 192, 256, dtype=torch.bfloat16, device="cuda"), rnd(
        5, 1400, 192, dtype=torch.bfloat16, device="cuda")
    g = torch.ones(60, device="cuda")
    return {
        "residual_norm": (lambda: ops.residual_norm(x, y, w_post, gate, w_pre, 0.9, 1e-5), x),
        "residual_norm_bwd": (lambda: ops.residual_norm_bwd(y, x, x, y, w_post, gate, w_pre, a, b, 0.9), y),
        "distill_loss": (lambda: (ops.distill_loss(logits, ids, top, lse, labels, 2.0, 0.5),), logits),
        "distill_loss_grad": (lambda: ops.distill_loss_grad(g, logits, ids, top, lse, labels, 2.0, 0.5), logits),
        "expert_order": (lambda: moe.expert_order(picks, 8), picks),
        "expert_order, many": (lambda: moe.expert_order(many, 64), many),
        "linear_ragged": (lambda: (ops.linear_ragged(rows, w, offsets),), rows),
        "linear_ragged_dgrad": (lambda: (ops.linear_ragged_dgrad(dy, w, offsets),), dy),
        "linear_ragged_wgrad": (lambda: (ops.linear_ragged_wgrad(dy, rows, offsets),), rows),
    }


@pytest.mark.gpu
def test_captured_and_replayed_with_other_values():
    """Every op in a graph of its own, replayed after its input has changed, and two graphs replayed at once on two streams."""
    graphs = []
    for name, (call, first) in _calls().items():
        call()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call()
        graphs.append((name, call, first, graph, out))
    for name, call, first, graph, out in graphs:
        first.copy_(first.flip(0))
        want = [t.clone() for t in call()]
        graph.replay()
        torch.cuda.synchronize()
        for p, q in zip(out, want):
            assert torch.equal(p, q), name
    streams = [torch.cuda.Stream() for _ in range(3)]
    wants = [[t.clone() for t in call()] for _, call, _, _, _ in graphs]
    torch.cuda.synchronize()
    for round_ in range(3):
        for i, (_, _, _, graph, _) in enumerate(graphs):
            with torch.cuda.stream(streams[(i + round_) % 3]):
                graph.replay()
        torch.cuda.synchronize()
        for (name, _, _, _, out), want in zip(graphs, wants):
            assert all(torch.equal(p, q) for p, q in zip(out, want)), name


@pytest.mark.gpu
def test_several_streams_and_threads_at_once():
    """The same calls from three threads on streams of their own give what one call alone gives."""
    import threading

    calls = _calls()
    want = {name: [t.clone() for t in call()] for name, (call, _) in calls.items()}
    torch.cuda.synchronize()
    bad = []

    def run():
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(10):
                for name, (call, _) in calls.items():
                    got = call()
                    torch.cuda.current_stream().synchronize()
                    if not all(torch.equal(p, q) for p, q in zip(got, want[name])):
                        bad.append(name)

    threads = [threading.Thread(target=run) for _ in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


FIRST_CALLS = """
import torch
from jaxpp_b200.ops import core as ops
from jaxpp_b200.parallel import moe

x = torch.randn(64, 4096, device="cuda").bfloat16()
w, y = torch.randn(2, 512, 4096, device="cuda").bfloat16(), torch.ones(4096, device="cuda", dtype=torch.bfloat16)
offsets = torch.tensor([0, 30, 64], dtype=torch.int32, device="cuda")
ids, top = torch.randint(0, 4096, (64, 8), device="cuda"), torch.randn(64, 8, device="cuda")

def calls():
    return (*ops.residual_norm(x, x, y, None, y), ops.linear_ragged(x, w, offsets), ops.linear_ragged_wgrad(x[:, :512], x, offsets),
            ops.distill_loss(x, ids, top, None, None, 2.0, 1.0), *moe.expert_order(ids, 200))

torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = calls()
graph.replay()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(got, calls()))
"""


@pytest.mark.gpu
def test_first_calls_of_a_process_captured():
    """Nothing that a first call sets up (the status word, shared-memory limits, tensor maps) breaks a capture under way."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    run = subprocess.run([sys.executable, "-c", FIRST_CALLS], cwd=root, capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stderr[-2000:]
