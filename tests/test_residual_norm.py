"""Residual norm where the plain cases of ``test_step_operators`` do not reach: sizes far from one, sums over rows held to the
precision of fp32, and CTAs that have many rows, whole groups of them and rows behind one another in the ring."""
import math

import pytest
import torch

import jaxpp_b200 as jp  # noqa: F401  (registers the ops)
from jaxpp_b200.ops import core as ops

from tests.test_step_operators import U, check, norm_exact, norm_inputs, rnd

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


@pytest.fixture(autouse=True)
def status():
    yield
    if torch.cuda.is_available():
        from jaxpp_b200.ops import native

        if native.is_available():
            torch.cuda.synchronize()
            assert native.read_status() == 0, "a kernel reported a time-out or a bad argument"


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("pre", [True, False])
@pytest.mark.parametrize("size,eps", [(1e15, 1e-5), (1e13, 1e-5), (1e-13, 1e-36), (1e-16, 1e-36)])
def test_block_outputs_of_any_size(device, dtype, pre, size, eps):
    """The norm takes the size of y out: the gradients for y are those at size one, divided by it, and the others the same."""
    x, y, w_post, gate, w_pre = norm_inputs(6, 264, 3, True, pre, dtype, device)
    y = (y.float() * size).to(dtype)
    dr = (rnd(11, 6, 264) + 2 * y.float().cpu() / size).to(dtype).to(device)      # along y: the projection counts
    dh = rnd(12, 6, 264, dtype=dtype, device=device) if pre else None
    ins = [None if t is None else t.double().cpu().requires_grad_(True) for t in (x, y, w_post, gate, w_pre)]
    er, eh = norm_exact(*ins, 0.75, eps)
    total = (er * dr.double().cpu()).sum() + ((eh * dh.double().cpu()).sum() if pre else 0.0)
    want = torch.autograd.grad(total, [t for t in ins if t is not None])
    r, h, a, b = ops.residual_norm(x, y, w_post, gate, w_pre, 0.75, eps)
    got = ops.residual_norm_bwd(dr, dh, x, y, w_post, gate, w_pre, a, b, 0.75)
    got = [g for g, t in zip(got, ins) if t is not None]
    # as in test_residual_norm: the sizes of the terms, each with 32 + log2(d) roundings a few times over
    depth = 32 + math.log2(264)
    inv = 1.0 if not pre else 1 / er.detach().square().mean(-1, keepdim=True).add(eps).sqrt()
    terms = dr.double().cpu().abs() + (inv * (2 * dh.double().cpu().abs() + 4 * er.detach().abs() * inv) if pre else 0)
    rp = 1 / ins[1].detach().square().mean(-1, keepdim=True).add(eps).sqrt()
    top, gmax = terms.amax(-1, keepdim=True), float(gate.float().abs().max())
    check(got[0], want[0], 4 * depth * U * terms)
    check(got[1], want[1], 16 * depth * U * rp * gmax * top)
    for g, w in zip(got[2:], want[2:]):     # sums over six rows of products of two such terms
        check(g, w, 32 * depth * U * 6 * float(top.max()) * max(1.0, gmax))


# ---- many rows and gate rows to a CTA, sums held to fp32 -----------------------------------------------------------------------
SMS = 148
MANY = [  # rows, d, gate rows (0: one vector; None: no gate)
    (1200, 4096, 1200),     # a gate row with every row, four or eight of them to a CTA
    (620, 8192, 310),       # gate rows in the ring for two rows each; fp32 backward with a ring of one stage
    (1200, 8192, 300),      # gate rows loaded when they change, two or three to a CTA
    (900, 15000, 300),      # bf16 alone: rows that do not fill their threads, four pieces each, one stage, gates in the ring
    (900, 16384, 150),      # bf16 alone: one stage, gates loaded
    (5000, 1600, 2500), (9000, 520, 1500), (6000, 264, 6000),
    (1200, 5120, 0), (3000, 2048, None), (20000, 128, 0), (700, 7168, 7),
]
HAVE = {  # what there is: post-norm, gate, pre-norm, gradient of r, gradient of h
    "all": (True, True, True, True, True), "one norm": (True, True, False, True, False), "no post-norm": (False, True, True, True, True),
    "nothing over r": (True, True, True, False, True), "nothing over h": (True, True, True, True, False),
}


def terms_of(x, y, w_post, gate, w_pre, dr, dh, scale, eps):
    """Exact results and gradients in 64 bits, and for each the sum of the sizes of the terms that it is made of."""
    rows, d = x.shape
    ins = [None if t is None else t.double().requires_grad_(True) for t in (x, y, w_post, gate, w_pre)]
    r, h = norm_exact(*ins, scale, eps)
    total = sum((o * g.double()).sum() for o, g in ((r, dr), (h, dh)) if g is not None)
    live = [i for i, t in enumerate(ins) if t is not None]
    grads = dict(zip(live, torch.autograd.grad(total, [ins[i] for i in live], allow_unused=True)))
    r, h = r.detach(), None if h is None else h.detach()
    x, y, w_post, gate, w_pre = (None if t is None else t.detach().double() for t in (x, y, w_post, gate, w_pre))
    one = torch.ones((), dtype=torch.float64, device=x.device)
    rstd1 = one if w_post is None else (y.square().mean(-1, keepdim=True) + eps).rsqrt()
    w = one if w_post is None else w_post
    groups = 1 if gate is None else gate.numel() // d
    g = one if gate is None else gate.reshape(groups, d).repeat_interleave(rows // groups, 0)
    p = (y * rstd1).abs()
    r_size = (scale * x).abs() + (g * w).abs() * p
    dR = torch.zeros_like(x) if dr is None else dr.double().abs()
    sizes = {}
    if w_pre is not None:
        rstd2 = (r.square().mean(-1, keepdim=True) + eps).rsqrt()
        sizes["h"] = r_size * rstd2 * w_pre.abs()
        if dh is not None:
            u, hat = (dh.double() * w_pre).abs(), r_size * rstd2
            dR = dR + rstd2 * (u + hat * (u * hat).mean(-1, keepdim=True))
            sizes[4] = (dh.double().abs() * hat).sum(0)
    v = dR * (g * w).abs()
    sizes["r"], sizes[0] = r_size, abs(scale) * dR
    sizes[1] = v if w_post is None else rstd1 * (v + p * (v * p).mean(-1, keepdim=True))
    if w_post is not None:
        sizes[2] = (dR * g.abs() * p).sum(0)
    if gate is not None:
        sizes[3] = (dR * w.abs() * p).reshape(groups, rows // groups, d).sum(1).reshape(gate.shape)
    return r, h, grads, sizes


def near(got, want, slack):
    """``check`` of test_step_operators, where the tensors are."""
    half = torch.finfo(got.dtype).eps / 2
    assert got.shape == want.shape and not torch.isnan(got).any()
    off = (got.double() - want).abs() - (half * want.abs() * (1 + 2 ** -7) + slack)
    assert float(off.max()) <= 0, f"off by {float(off.max()):.3g} more than allowed at {int(off.argmax())}"


def many(rows, d, gates, have, dtype, device):
    post, with_gate, pre, has_dr, has_dh = HAVE[have]
    x, y, w_post, gate, w_pre = norm_inputs(rows, d, gates if with_gate else None, post, pre, dtype, device)
    # gradients along the outputs in part, so that the sums over rows are as large as their terms
    sign = 1.0 if gate is None else gate.float().reshape(-1, d).sign().repeat_interleave(rows // (gate.numel() // d), 0)
    dr = (rnd(11, rows, d).to(device) * 0.5 + 2 * y.float() * sign).to(dtype) if has_dr else None
    dh = (rnd(12, rows, d).to(device) * 0.5 + 0.3 * x.float()).to(dtype) if has_dh else None
    return x, y, w_post, gate, w_pre, dr, dh


def check_many(rows, d, gates, have, dtype, device):
    x, y, w_post, gate, w_pre, dr, dh = many(rows, d, gates, have, dtype, device)
    scale, eps = 0.75, 1e-5
    er, eh, grads, sizes = terms_of(x, y, w_post, gate, w_pre, dr, dh, scale, eps)
    r, h, a, b = ops.residual_norm(x, y, w_post, gate, w_pre, scale, eps)
    # Roundings: a sum of squares over a row is a tree of 16 + log2(d) at most, so that a reciprocal root has half as many and two;
    # a term of dR has two such roots, one more such sum (`depth`) and 16 of its own, a term of the others one root more.
    depth = 32 + math.log2(d)
    near(r, er, (depth / 2 + 8) * U * sizes["r"])
    if eh is not None:
        near(h, eh, (depth + 16) * U * sizes["h"])
    # Sums over rows: a CTA's rows one after the other, then the partial rows of the CTAs in eight sums or more of 64 at most.
    threads = -(-(d * x.element_size() // 16) // (4 if d * x.element_size() > 16384 else 2))
    ctas = min(rows, SMS * (512 // (-(-threads // 32) * 32))) if device == "cuda" else 1
    one_by_one = -(-rows // ctas) + 64 + 32 if device == "cuda" else 24 + math.log2(rows)      # (the CPU's sums are cascades)
    for sum_dtype in (torch.float32, None):
        back = ops.residual_norm_bwd(dr, dh, x, y, w_post, gate, w_pre, a, b, scale, sum_dtype)
        for i, t in enumerate((x, y, w_post, gate, w_pre)):
            if t is None:
                assert back[i].numel() == 0
                continue
            if i == 4 and dh is None:
                assert back[4].shape == t.shape and not back[4].any()
                continue
            assert back[i].dtype == (dtype if i < 2 or sum_dtype is None else sum_dtype)
            slack = (2 * depth + 16 + (depth / 2 + 8 if i else 0) + (one_by_one if i >= 2 else 0)) * U * sizes[i]
            near(back[i], grads[i], slack)
            if i in (2, 4) and back[i].dtype == torch.float32:
                # the bound tells fp32 sums from sums that were kept in, or went by way of, 16 bits, and from sums off by a hundredth
                assert ((grads[i].bfloat16().double() - grads[i]).abs() > slack).any() and (grads[i].abs() * 1e-2 > slack).any()
    again = ops.residual_norm_bwd(dr, dh, x, y, w_post, gate, w_pre, a, b, scale)
    assert all(torch.equal(p, q) for p, q in zip(again, back))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("have", sorted(HAVE))
@pytest.mark.parametrize("rows,d,gates", MANY)
def test_many_rows_to_a_cta(rows, d, gates, have, dtype):
    if d * dtype.itemsize > 32768:
        pytest.skip("rows of at most 32 KB")
    check_many(rows, d, gates, have, dtype, "cuda")


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("have", sorted(HAVE))
@pytest.mark.parametrize("rows,d,gates", [(40, 264, 0), (300, 1024, 4), (160, 2048, 40), (130, 1600, 0), (64, 72, None)])
def test_sums_over_rows_are_held_to_fp32(device, rows, d, gates, have, dtype):
    check_many(rows, d, gates, have, dtype, device)
