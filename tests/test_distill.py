"""Distillation loss where the plain cases of ``test_step_operators`` do not reach: broken teachers, students that leave next to
nothing outside of the entries, and CTAs and clusters that have several rows each."""
import math

import pytest
import torch

import jaxpp_b200 as jp  # noqa: F401  (registers the ops)
from jaxpp_b200.ops import core as ops

from tests.test_step_operators import U, check, check_distill, distill_exact, distill_inputs, distill_slack, rnd

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
@pytest.mark.parametrize("tail", [True, False])
@pytest.mark.parametrize("V,K", [(90, 6), (300, 200), (70000, 5)])     # a CTA a row, several entries a thread, a cluster a row
def test_a_broken_teacher_shows(device, tail, V, K):
    """A NaN among a row's teacher values is a NaN loss and gradient of that row, and of no other one."""
    args = distill_inputs(7, V, K, device, torch.float32, tail, True, 2.0, torch.int64)
    dloss = 1 + rnd(4, 7, device=device).abs()
    dloss[5] = 0.0
    want = ops.distill_loss_grad(dloss, *args, 2.0, 0.5)
    logits, ids, top, lse, labels = args
    top = top.clone()
    top[0] = math.nan                    # nothing but NaN
    top[2, K - 1] = math.nan             # one entry
    top[5, 0] = math.nan                 # in a row of weight zero: no gradient all the same
    broken = [0, 2, 5]
    if tail:
        lse = lse.clone()
        lse[3] = math.nan
        broken.append(3)
    ids = ids.clone()
    top[6, 1], ids[6, 1] = math.nan, -1  # no entry: what it holds does not count
    want[0][6], want[1][6] = (t[0] for t in ops.distill_loss_grad(
        dloss[6:], logits[6:], ids[6:], torch.where(ids[6:] < 0, 0.0, top[6:]), None if lse is None else lse[6:], labels[6:], 2.0, 0.5))
    loss, dz = ops.distill_loss_grad(dloss, logits, ids, top, lse, labels, 2.0, 0.5)
    again = ops.distill_loss(logits, ids, top, lse, labels, 2.0, 0.5)
    for r in range(7):
        if r in broken:
            assert torch.isnan(loss[r]) and torch.isnan(again[r]), r
            assert torch.isnan(dz[r]).all() if r != 5 else not dz[r].any(), r
        else:
            assert torch.isfinite(loss[r]) and torch.isfinite(again[r]), r
            if r != 6:
                assert torch.equal(loss[r], want[0][r]) and torch.equal(dz[r], want[1][r]), r
    torch.testing.assert_close(loss[6], want[0][6], rtol=1e-5, atol=1e-5)     # (another number of rows may sum in another order)
    torch.testing.assert_close(dz[6], want[1][6], rtol=1e-5, atol=1e-5)


@pytest.mark.parametrize("device", DEVICES)
def test_terms_without_weight_are_left_out(device):
    """alpha 0 is the cross entropy alone and alpha 1 the divergence alone, whatever the other one's tensors hold."""
    logits, ids, top, lse, labels = distill_inputs(4, 60, 5, device)
    ones = torch.ones(4, device=device)
    logits[1, ids[1, 0]] = -math.inf                 # the divergence of this row is infinite
    labels[1], labels[2] = ids[1, 1], -1
    want = ops.distill_loss_grad(ones, logits, ids, top, lse, labels, 1.0, 0.0)
    got = ops.distill_loss_grad(ones, logits, ids, torch.full_like(top, math.nan), lse, labels, 2.0, 0.0)
    for p, q in zip(got, want):
        assert torch.isfinite(q).all()
        torch.testing.assert_close(p, q, rtol=1e-6, atol=1e-6)
    plain, _ = ops.cross_entropy(logits, labels.clamp(min=0))
    torch.testing.assert_close(got[0], torch.where(labels < 0, 0.0, plain), rtol=1e-6, atol=1e-6)
    logits[1] = logits[0]
    logits[3, labels[3]] = -math.inf                 # an infinite cross entropy
    ids[3] = (labels[3] + 1 + torch.arange(5, device=device)) % 60
    loss, dz = ops.distill_loss_grad(ones, logits, ids, top, None, labels, 1.0, 1.0)
    assert torch.isfinite(loss).all() and torch.isfinite(dz).all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [900, 70000])
@pytest.mark.parametrize("t,alpha", [(1.0, 0.5), (2.0, 0.5), (4.0, 1.0), (1.5, 0.75), (0.5, 0.5)])
def test_masks_of_the_lowest_value(device, dtype, V, t, alpha):
    """A vocabulary masked with the type's lowest value, whole parts of a row's cluster with nothing else among them, counts as
    one masked with -inf; a row of nothing else is a row of equal logits."""
    logits, ids, top, lse, labels = distill_inputs(5, V, 6, device, dtype, True, alpha < 1, t, torch.int64)
    ids[:] = torch.arange(6, device=device) + 11
    if labels is not None:
        labels[:] = torch.arange(9, 14, device=device)
    lowest = torch.finfo(dtype).min if t >= 1 else torch.finfo(dtype).min * t      # (no overflow by the temperature)
    logits[1, V // 2:] = lowest
    logits[2, 17:] = lowest
    logits[3, :] = lowest
    logits[4, :9], logits[4, V // 3:] = lowest, -math.inf
    loss, dz = check_distill(device, logits, ids, top, lse, labels, t, alpha)
    assert not dz[1, V // 2:].any() and not dz[2, 17:].any() and not dz[4, V // 3:].any()
    other = torch.where(logits == lowest, -math.inf, logits.float()).to(dtype)
    keep = [0, 1, 2, 4]
    for tail in (lse, None):
        got = ops.distill_loss_grad(torch.ones(5, device=device), logits, ids, top, tail, labels, t, alpha)
        want = ops.distill_loss_grad(torch.ones(5, device=device), other, ids, top, tail, labels, t, alpha)
        assert torch.equal(got[0][keep], want[0][keep]) and torch.equal(got[1][keep], want[1][keep])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V,t,alpha", [(900, 4.0, 1.0), (900, 1.0, 0.5), (900, 2.0, 0.5), (900, 1.5, 0.75), (70000, 4.0, 0.5), (70000, 1.0, 1.0)])
def test_students_that_leave_next_to_nothing(device, dtype, V, t, alpha):
    """The teacher keeps mass outside of the entries and the student almost none, with weights as a scaled loss has them: what is
    outside has a gradient of the size of the teacher's rest, however small the student's is.  Tolerances as in ``check_distill``;
    what is flushed to zero on the way is below the smallest normal number, times the weight."""
    gaps = [20.0, 26.0, 27.0, 28.0, 29.0, 45.0, 60.0, 78.0, 83.0, 91.0, 120.0]     # 2^-40 is 27.7 nats, 2^-126 is 87.3
    rows, K = len(gaps), 5
    logits, ids, top, lse, labels = distill_inputs(rows, V, K, device, torch.float32, True, alpha < 1, t, torch.int64)
    first = V // 2 - 2
    ids[:] = torch.arange(first, first + K, device=device)
    outside = torch.ones(V, dtype=torch.bool, device=device)
    outside[first:first + K] = False
    logits[:, first:first + K] = rnd(1, rows, K, device=device)
    tail = rnd(2, rows, V, device=device) * 0.5
    for r, gap in enumerate(gaps):
        # the outside as a whole lies `gap` below: its elements by the logarithm of their number more, but for the 120 (nothing
        # is left) and the 91, whose sum of elements below 2^-126 is above it
        down = gap if gap in (91.0, 120.0) else gap + math.log(V - K)
        if gap == 91.0 and V < 1000:
            down = 88.5
        logits[r, outside] = t * (tail[r, outside] * 0.5 - down)
    logits[5, 3:first // 2] = -800.0 * t
    logits = logits.to(dtype)
    lse = torch.logsumexp(top.float() / t, -1) + torch.linspace(0.01, 2.0, rows, device=device)      # q leaves 1 % to 86 %
    dloss = torch.tensor([1.0, -1024.0, 3.0e4, 1.0e6] * 3, device=device)[:rows]
    dloss[7:9] = 4096.0
    if labels is not None:
        labels[0], labels[5], labels[6], labels[8] = first, first + 1, 7, V - 1
    z = logits.double().cpu() / t
    left = torch.logsumexp(z[:, outside.cpu()], -1) - torch.logsumexp(z, -1)
    assert (left + 126 * math.log(2)).abs().min() > 0.2           # (on the border either answer would be right)
    el, eg, size = distill_exact(dloss, logits, ids, top, lse, labels, t, alpha)
    rel = distill_slack(logits, t)
    loss, dz = ops.distill_loss_grad(dloss, logits, ids, top, lse, labels, t, alpha)
    check(loss, el, rel * 2 * max(1.0, t * t) * (1 + el.abs()) + 200 * U)
    check(ops.distill_loss(logits, ids, top, lse, labels, t, alpha), el, rel * 2 * max(1.0, t * t) * (1 + el.abs()) + 200 * U)
    check(dz, eg, 2 * rel * size + 2.0 ** -126 * (1 + t * dloss.abs().double().cpu()[:, None]))


# ---- several rows to a CTA or a cluster ------------------------------------------------------------------------------------------
def exact_rows(dloss, logits, ids, top, lse, labels, t, alpha):
    """``distill_exact`` for all rows at once, where the tensors are."""
    z, V = logits.double(), logits.shape[-1]
    valid = (ids >= 0) & (ids < V) & (top != -math.inf)
    at = ids.long().masked_fill(~valid, 0)
    teacher = (top.double() / t).masked_fill(~valid, -math.inf)
    some = valid.any(-1)
    logp, logp1 = torch.log_softmax(z / t, -1), torch.log_softmax(z, -1)
    logq = teacher - (torch.logsumexp(teacher, -1) if lse is None else lse.double())[:, None]
    q = torch.where(valid, logq.exp(), 0.0)
    soft = torch.where(q > 0, q * (logq - logp.gather(-1, at)), 0.0).sum(-1)
    listed = torch.zeros_like(z).scatter_add(-1, at, valid.double()) > 0
    mass, ratio = q.sum(-1), torch.zeros_like(soft)
    if lse is not None:
        q_o, p_o = (1 - mass).clamp(min=0), logp.exp().masked_fill(listed, 0.0).sum(-1)
        rest = (q_o > 0) & (p_o >= 2.0 ** -126)
        ratio = torch.where(rest, q_o / p_o, 0.0)
        soft = soft + torch.where(rest, q_o * torch.where(rest, ratio, 1.0).log(), 0.0)
        mass = mass + torch.where(rest, q_o, 0.0)
    q_at = torch.zeros_like(z).scatter_add(-1, at, q)
    on = some[:, None].double() * alpha * t
    grad = on * (logp.exp() * (mass[:, None] - torch.where(listed, 0.0, ratio[:, None])) - q_at)
    size = on * (logp.exp() * (mass + ratio)[:, None] + q_at)
    loss = torch.where(some, alpha * t * t * soft, 0.0)
    if labels is not None:
        known = (labels >= 0) & (labels < V)
        y = labels.masked_fill(~known, 0)[:, None]
        loss = loss + torch.where(known, (alpha - 1) * logp1.gather(-1, y)[:, 0], 0.0)
        hit = torch.zeros_like(z).scatter(-1, y, 1.0)
        on = known[:, None].double() * (1 - alpha)
        grad, size = grad + on * (logp1.exp() - hit), size + on * ((logp1.exp() - hit).abs() + 2 * hit)
    w = dloss.double()[:, None]
    return loss, grad * w, size * w.abs()


def near(got, want, slack):
    """``check`` of test_step_operators, where the tensors are."""
    half = torch.finfo(got.dtype).eps / 2
    assert got.shape == want.shape and not torch.isnan(got).any()
    off = (got.double() - want).abs() - (half * want.abs() * (1 + 2 ** -7) + slack)
    assert float(off.max()) <= 0, f"off by {float(off.max()):.3g} more than allowed at {int(off.argmax())}"


def uneven(rows, V, K, device, dtype, tail, labels, t, ids_dtype):
    """Inputs whose rows differ in kind, so that what one leaves behind would show in the next: without entries, with repeated ones,
    without a label or one that is listed, weightless, with logits far apart."""
    logits, ids, top, lse, lab = distill_inputs(rows, V, K, device, dtype, tail, labels, t, ids_dtype)
    dloss = rnd(9, rows, device=device)
    kind = torch.arange(rows, device=device)
    ids[kind % 7 == 3] = -1
    if K > 2:
        ids[kind % 5 == 1, 2] = ids[kind % 5 == 1, 0]           # an id twice (where there are entries)
        ids[kind % 10 == 6, 1:] = ids[kind % 10 == 6, :1]       # and one K times
    if lab is not None:
        lab[kind % 4 == 2] = -1
        if K:
            lab[kind % 6 == 5] = ids[kind % 6 == 5, 0].long()
    if lse is not None:
        lse += 0.3
    dloss[kind % 11 == 4] = 0.0
    logits[kind % 13 == 12, V // 2:] += 120.0                   # far above the entries, where these lie below
    return dloss, logits, ids, top, lse, lab


SEVERAL = [  # rows, V, K, tail, labels, temperature, alpha
    (2000, 130, 5, True, True, 1.0, 0.5), (3000, 257, 200, True, True, 2.0, 0.5), (2000, 4097, 100, False, True, 4.0, 0.5),
    (900, 24000, 16, True, True, 1.5, 0.9), (1400, 12000, 300, True, False, 2.0, 1.0), (700, 50257, 100, False, False, 1.0, 1.0),
    (500, 50257, 600, True, True, 2.0, 0.5),     # one CTA of 256 threads to an SM
    (300, 70000, 64, True, True, 2.0, 0.5), (160, 70000, 64, True, True, 1.0, 0.5), (120, 128256, 300, True, True, 4.0, 0.5),
    (90, 200000, 40, False, True, 1.5, 0.5), (60, 420000, 20, True, True, 2.0, 0.5),
]


def check_several(device, dtype, rows, V, K, tail, labels, t, alpha):
    dloss, *args = uneven(rows, V, K, device, dtype, tail, labels, t, torch.int64 if K % 2 else torch.int32)
    el, eg, size = exact_rows(dloss, *args, t, alpha)
    rel = distill_slack(args[0], t)
    slack = rel * 2 * max(1.0, t * t) * (1 + el.abs()) + 40 * U
    near(ops.distill_loss(*args, t, alpha), el, slack)
    loss, dz = ops.distill_loss_grad(dloss, *args, t, alpha)
    near(loss, el, slack)
    near(dz, eg, 2 * rel * size + 2.0 ** -126)
    again = ops.distill_loss_grad(dloss, *args, t, alpha)
    assert torch.equal(loss, again[0]) and torch.equal(dz, again[1])
    return dloss, args, (el, eg, size)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,V,K,tail,labels,t,alpha", SEVERAL)
def test_several_rows_to_a_cta_or_cluster(dtype, rows, V, K, tail, labels, t, alpha):
    check_several("cuda", dtype, rows, V, K, tail, labels, t, alpha)


@pytest.mark.parametrize("tail,labels,t,alpha", [(True, True, 2.0, 0.5), (False, True, 1.0, 0.25), (True, False, 1.5, 1.0)])
def test_rows_of_every_kind(tail, labels, t, alpha):
    """The same rows on the CPU, and the two 64-bit forms against one another."""
    dloss, args, got = check_several("cpu", torch.float32, 60, 90, 7, tail, labels, t, alpha)
    for p, q in zip(got, distill_exact(dloss, *args, t, alpha)):
        torch.testing.assert_close(p, q, rtol=1e-9, atol=1e-12)


@pytest.mark.parametrize("device", DEVICES)
def test_temperatures(device):
    """Those at both ends of the range are right, those outside of it are refused: at 1e-10 an exponent has no digit left, at 1e25
    the square of the temperature is no number."""
    for t in (2.0 ** -14, 2.0 ** -7, 64.0, 2.0 ** 14):
        logits, ids, top, lse, labels = distill_inputs(5, 300, 6, device, torch.float32, True, True, t, torch.int64)
        lse += 0.5
        check_distill(device, logits, ids, top, lse, labels, t, 0.5)
        check_distill(device, logits, ids, top, None, labels, t, 0.5)
    for t in (0.0, 1e-10, 2.0 ** -15, 1e25, 20000.0, math.nan):
        with pytest.raises((ValueError, RuntimeError)):
            ops.distill_loss(logits, ids, top, lse, labels, t, 0.5)
        with pytest.raises((ValueError, RuntimeError)):
            ops.distill_loss_grad(torch.ones(5, device=device), logits, ids, top, lse, labels, t, 0.5)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("K", [0, 1, 64, 1024])
def test_the_largest_rows(dtype, K):
    """Rows of 8 times (220 KB less 24 bytes an entry) are taken, with any start of a row on its 16 bytes; longer ones are refused."""
    from jaxpp_b200.ops import native

    most = 8 * (220 * 1024 - 24 * K) // dtype.itemsize
    for V in (most, most - 1, most - 3):
        check_several("cuda", dtype, 3, V, K, K % 2 == 0, True, 2.0, 0.5)
    with pytest.raises(native.NativeError):
        ops.distill_loss(*distill_inputs(2, most + 1, K, "cuda", dtype), 1.0, 0.5)
