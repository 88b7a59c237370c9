"""Products grouped by ragged rows against plain 64-bit ones, on the CPU (reference) and the GPU (tcgen05 kernels).

Tolerances: half a step of the result's type and, for the fp32 accumulation of K products 16 at a time, K / 16 + 16 additions that
lose at most 2^-23 (a truncated step) of the sum of the products' sizes each."""
import pytest
import torch

from jaxpp_b200.ops import core as ops
from jaxpp_b200.ops import sink

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


@pytest.fixture(autouse=True)
def status():
    yield
    if torch.cuda.is_available():
        from jaxpp_b200.ops import native

        if native.is_available():
            torch.cuda.synchronize()
            assert native.read_status() == 0, "a kernel reported a time-out or a bad argument"


def rnd(seed, *shape, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(torch.bfloat16)


def bounds(sizes, head, tail):
    off = [head]
    for s in sizes:
        off.append(off[-1] + s)
    return off, off[-1] + tail


def near(got, want, sizes, k, what):
    """``sizes``: sum of the sizes of the products behind each value."""
    got = got.detach()
    half = torch.finfo(got.dtype).eps / 2
    slack = (k / 16 + 16) * 2.0 ** -23 * sizes + half * want.abs() * (1 + 2.0 ** -7)
    off = (got.double().cpu() - want).abs() - slack
    assert got.shape == want.shape and not torch.isnan(got).any(), what
    assert off.numel() == 0 or off.max() <= 0, f"{what}: {off.max().item():.3g} more than allowed"


def oracle(x, w, dy, off):
    T, (E, N, K) = x.shape[0], w.shape
    x, w, dy = x.double(), w.double(), dy.double()
    y, dx, dw = torch.zeros(T, N).double(), torch.zeros(T, K).double(), torch.zeros(E, N, K).double()
    sy, sx, sw = torch.zeros_like(y), torch.zeros_like(dx), torch.zeros_like(dw)
    for e in range(E):
        a, b = off[e], off[e + 1]
        y[a:b], sy[a:b] = x[a:b] @ w[e].t(), x[a:b].abs() @ w[e].abs().t()
        dx[a:b], sx[a:b] = dy[a:b] @ w[e], dy[a:b].abs() @ w[e].abs()
        dw[e], sw[e] = dy[a:b].t() @ x[a:b], dy[a:b].abs().t() @ x[a:b].abs()
    return (y, sy), (dx, sx), (dw, sw)


CASES = [  # group sizes, rows in front, rows behind, N, K
    ([1], 0, 0, 8, 8), ([0, 0, 3], 0, 0, 16, 24), ([1, 0, 2, 1], 1, 2, 136, 72), ([15, 16, 17, 0, 1], 0, 0, 64, 64),
    ([31, 33, 32, 0, 64], 3, 5, 200, 128), ([63, 64, 65], 0, 0, 264, 200), ([127, 128, 129, 1, 0], 2, 0, 384, 520),
    ([255, 256, 257], 0, 1, 512, 256), ([300, 0, 700, 24], 0, 0, 1032, 328), ([513, 40, 600, 2, 1000, 15, 0, 290], 7, 9, 768, 384),
    ([2000, 1], 0, 0, 2304, 192), ([0, 0], 4, 3, 40, 48), ([70] * 40, 0, 0, 128, 128), ([5] * 200, 0, 0, 72, 64), ([0] * 1000 + [3] * 24, 0, 0, 16, 16),
    ([1, 1], 0, 0, 2048, 4096), ([2600, 1500], 0, 100, 4096, 1024),
    ([1, 0, 3], 0, 1, 19208, 72), ([20, 20, 1], 2, 0, 9608, 40), ([0, 1, 2], 1, 2, 136, 4104), ([3, 0, 30, 1], 0, 0, 4352, 200),
    ([0, 0, 0], 2, 1, 64, 4096), ([40, 0, 90], 1, 0, 136, 2056), ([130, 300, 0], 0, 2, 2056, 64),
]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("sizes,head,tail,N,K", CASES)
def test_linear_ragged(device, sizes, head, tail, N, K):
    off, T = bounds(sizes, head, tail)
    x, w, dy = rnd(1, T, K), rnd(2, len(sizes), N, K, scale=0.1), rnd(3, T, N)
    (y, sy), (dx, sx), (dw, sw) = oracle(x, w, dy, off)
    # what rows of no group hold reaches nothing
    x[:head], x[T - tail:], dy[:head], dy[T - tail:] = [float("nan")] * 4
    offsets = torch.tensor(off, dtype=torch.int32, device=device)
    x, w, dy = x.to(device).requires_grad_(True), w.to(device).requires_grad_(True), dy.to(device)
    out = ops.linear_ragged(x, w, offsets)
    near(out, y, sy, K, "forward")
    assert not out.detach()[:head].any() and not out.detach()[T - tail:].any()
    gx, gw = torch.autograd.grad(out, (x, w), dy)
    near(gx, dx, sx, N, "input gradient")
    near(gw, dw, sw, T, "weight gradient")
    wide = ops.linear_ragged_wgrad(dy, x.detach(), offsets, torch.float32)
    assert wide.dtype == torch.float32
    near(wide, dw, sw, T, "weight gradient, fp32")
    acc = torch.ones(len(sizes), N, K, device=device)
    got = sink.accumulate(torch.ops.b200.linear_ragged_wgrad.default, acc, dy, x.detach(), offsets, torch.float32)
    assert got is acc
    near(acc, dw + 1, sw + 1, T, "accumulated weight gradient")


@pytest.mark.parametrize("device", DEVICES)
def test_groups_are_apart(device):
    """NaN and infinities of one group, in its rows or its weights, reach no other group."""
    sizes = [70, 0, 41, 130, 9]
    off, T = bounds(sizes, 0, 0)
    x, w, dy = rnd(1, T, 136), rnd(2, 5, 72, 136), rnd(3, T, 72)
    want = oracle(x, w, dy, off)
    a, b = off[2], off[3]
    x[a:b], dy[a:b], w[2], w[1] = float("nan"), float("inf"), float("inf"), float("nan")
    offsets = torch.tensor(off, dtype=torch.int32, device=device)
    x, w, dy = x.to(device), w.to(device), dy.to(device)
    others = [t for t in range(T) if not a <= t < b]
    for got, (exact, size), k in ((ops.linear_ragged(x, w, offsets), want[0], 136), (ops.linear_ragged_dgrad(dy, w, offsets), want[1], 72)):
        near(got.cpu()[others], exact[others], size[others], k, "rows")
    dw = ops.linear_ragged_wgrad(dy, x, offsets).cpu()
    for e in (0, 1, 3, 4):
        near(dw[e], want[2][0][e], want[2][1][e], T, "weights")


@pytest.mark.parametrize("device", DEVICES)
def test_offsets_out_of_order(device):
    """Offsets that decrease or leave the rows are taken as the nearest that do not: nothing outside is touched."""
    x, w, dy = rnd(1, 50, 64).to(device), rnd(2, 4, 72, 64).to(device), rnd(3, 50, 72).to(device)
    for given, taken in (([-5, 20, 10, 30, 99], [0, 20, 20, 30, 50]), ([60, 1, 2, 3, 4], [50] * 5), ([2, 2 ** 31 - 1, -2 ** 31, 7, 7], [2] + [50] * 4)):
        a, b = (torch.tensor(v, dtype=torch.int32, device=device) for v in (given, taken))
        assert torch.equal(ops.linear_ragged(x, w, a), ops.linear_ragged(x, w, b))
        assert torch.equal(ops.linear_ragged_dgrad(dy, w, a), ops.linear_ragged_dgrad(dy, w, b))
        assert torch.equal(ops.linear_ragged_wgrad(dy, x, a), ops.linear_ragged_wgrad(dy, x, b))


@pytest.mark.parametrize("device", DEVICES)
def test_no_rows_and_views(device):
    w = rnd(2, 3, 24, 40).to(device)
    zero = torch.zeros(4, dtype=torch.int32, device=device)
    assert ops.linear_ragged(torch.zeros(0, 40, dtype=torch.bfloat16, device=device), w, zero).shape == (0, 24)
    dw = ops.linear_ragged_wgrad(torch.zeros(0, 24, dtype=torch.bfloat16, device=device), torch.zeros(0, 40, dtype=torch.bfloat16, device=device), zero)
    assert dw.shape == (3, 24, 40) and not dw.any()
    off = torch.tensor([0, 9, 9, 20], dtype=torch.int32, device=device)
    big, flat = rnd(4, 20, 100).to(device), rnd(5, 20 * 40 + 1).to(device)
    for x in (big[:, 8:48], flat[1:].view(20, 40), rnd(6, 40, 20).to(device).t()):
        assert torch.equal(ops.linear_ragged(x, w, off), ops.linear_ragged(x.clone(memory_format=torch.contiguous_format), w, off))
    wt = rnd(7, 3, 40, 24).to(device).transpose(1, 2)
    x = flat[:800].view(20, 40)
    assert torch.equal(ops.linear_ragged(x, wt, off), ops.linear_ragged(x, wt.contiguous(), off))


def test_linear_ragged_refusals():
    x, w, off = rnd(1, 10, 16), rnd(2, 3, 8, 16), torch.tensor([0, 3, 5, 10], dtype=torch.int32)
    for args in ((x, w, off.long()), (x, w, off[:3]), (x[:, :8], w, off), (x.view(1, 10, 16), w, off), (x, w[0], off), (x, w, off.view(1, 4))):
        with pytest.raises((ValueError, RuntimeError, IndexError)):
            ops.linear_ragged(*args)
    with pytest.raises((ValueError, RuntimeError)):
        ops.linear_ragged_dgrad(x, w, off)
    with pytest.raises((ValueError, RuntimeError)):
        ops.linear_ragged_wgrad(x[:5], x, off)
    with pytest.raises((ValueError, RuntimeError)):
        ops.linear_ragged_wgrad(x, x, off[:1])


@pytest.mark.gpu
def test_linear_ragged_refusals_gpu():
    from jaxpp_b200.ops import native

    off = torch.tensor([0, 3, 5, 10], dtype=torch.int32, device="cuda")
    x, w = rnd(1, 10, 16).cuda(), rnd(2, 3, 8, 16).cuda()
    for args in ((x.float(), w.float(), off), (x[:, :12], w[:, :, :12], off), (x, w[:, :4], off), (x, w.cpu(), off)):
        with pytest.raises(native.NativeError):
            ops.linear_ragged(*args)
    with pytest.raises(native.NativeError):
        ops.linear_ragged(x, rnd(3, 1025, 8, 16).cuda(), torch.zeros(1026, dtype=torch.int32, device="cuda"))
    with pytest.raises((ValueError, RuntimeError)):
        ops.linear_ragged(x, w, off.cpu())


@pytest.mark.gpu
def test_parts_replayed_with_other_offsets():
    """A captured product whose reductions are cut decides how from the offsets of each replay."""
    E, N, K = 8, 1096, 4096
    w, x = rnd(1, E, N, K, scale=0.1).cuda(), rnd(2, 2, K).cuda()
    offsets = torch.zeros(E + 1, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.linear_ragged(x, w, offsets)
    for counts in ([1, 1], [2], [0] * 7 + [1], [0], [0, 0, 0, 1, 1]):
        off = bounds(counts + [0] * (E - len(counts)), 0, 0)[0]
        offsets.copy_(torch.tensor(off, dtype=torch.int32))
        x.copy_(rnd(sum(off), 2, K))
        graph.replay()
        (y, sy), _, _ = oracle(x.cpu(), w.cpu(), torch.zeros(2, N), off)
        near(got, y, sy, K, f"replayed with {counts}")
