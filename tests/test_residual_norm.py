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
