"""Which kernels ragged products take (the host's rules, without a GPU, for 148 SMs), and the CTA pairs of the large ones with ragged
sizes: feature sizes that no tile and no 64-column block divides, groups without rows, rows of no group on both ends."""
import pytest
import torch

from jaxpp_b200.ops import core as ops
from jaxpp_b200.ops import native, sink

from tests.test_ragged import bounds, near, oracle, rnd

SMS = 148


@pytest.fixture(autouse=True)
def status():
    yield
    if torch.cuda.is_available() and native.is_available():
        torch.cuda.synchronize()
        assert native.read_status() == 0, "a kernel reported a time-out or a bad argument"


def forms(rows, groups, N, K):
    """Block rows and parts forward and of the input gradient, and the edge of the weight gradient's tiles."""
    lib = native.load()
    fwd, bwd = (lib.jpb_linear_ragged_form(rows, groups, N, K, i, SMS) for i in (0, 1))
    return (fwd % 1024, fwd // 1024), (bwd % 1024, bwd // 1024), lib.jpb_linear_ragged_wgrad_form(rows, groups, N, K, SMS)


def test_rules():
    assert forms(8192, 8, 28672, 4096) == ((256, 1), (256, 1), 256)         # the large products
    assert forms(2, 8, 28672, 4096)[:2] == ((32, 1), (32, 4))               # a token of two experts; 32 tiles of the input gradient
    assert forms(2000, 8, 2048, 512) == ((128, 1), (128, 1), 256)           # small ones
    assert forms(300, 4, 256, 4096)[0] == (128, 8)
    assert forms(40, 8, 512, 512)[2] == forms(4096, 2, 512, 512)[2] == 128  # few tiles
    assert forms(4096, 4, 1024, 1024)[2] == 256
    for rows in (1, 30, 700, 5000):                                         # reductions below 2048 are never cut
        assert forms(rows, 4, 1024, 2040)[0][1] == 1


PAIRS = [  # group sizes, rows in front, rows behind, N, K
    ([900, 0, 1300, 257, 1], 3, 5, 2312, 1864),       # neither N nor K in blocks of 64
    ([700, 33, 1200], 0, 0, 2304, 1800),
    ([2049, 0, 0, 515], 1, 0, 1800, 2304),
    ([1025, 700], 0, 0, 4104, 1288),                  # eight columns in the last tile: the pair's second CTA lies wholly behind
    ([300] * 8, 2, 2, 2000, 2072),
    ([0, 1700, 0], 40, 3, 2056, 2120),
]


def operands(sizes, head, tail, N, K):
    off, T = bounds(sizes, head, tail)
    assert forms(T, len(sizes), N, K) == ((256, 1), (256, 1), 256)
    x, w, dy = (t.cuda() for t in (rnd(1, T, K), rnd(2, len(sizes), N, K, scale=0.1), rnd(3, T, N)))
    exact = [tuple(t.cpu() for t in pair) for pair in oracle(x, w, dy, off)]
    return off, T, x, w, dy, exact


@pytest.mark.gpu
@pytest.mark.parametrize("sizes,head,tail,N,K", PAIRS)
def test_pairs(sizes, head, tail, N, K):
    off, T, x, w, dy, ((y, sy), (dx, sx), (dw, sw)) = operands(sizes, head, tail, N, K)
    x[:head], x[T - tail:], dy[:head], dy[T - tail:] = [float("nan")] * 4     # what rows of no group hold reaches nothing
    offsets = torch.tensor(off, dtype=torch.int32, device="cuda")
    out, gx = ops.linear_ragged(x, w, offsets), ops.linear_ragged_dgrad(dy, w, offsets)
    near(out, y, sy, K, "forward")
    near(gx, dx, sx, N, "input gradient")
    for t in (out, gx):
        assert not t[:head].any() and not t[T - tail:].any()
    near(ops.linear_ragged_wgrad(dy, x, offsets), dw, sw, T, "weight gradient")
    near(ops.linear_ragged_wgrad(dy, x, offsets, torch.float32), dw, sw, T, "weight gradient, fp32")
    acc = torch.ones(len(sizes), N, K, device="cuda")
    sink.accumulate(torch.ops.b200.linear_ragged_wgrad.default, acc, dy, x, offsets, torch.float32)
    near(acc, dw + 1, sw + 1, T, "accumulated weight gradient")


@pytest.mark.gpu
def test_groups_of_pairs_are_apart():
    """NaN and infinities of one group, in its rows or its weights, reach no other group."""
    sizes = [700, 0, 411, 1300, 9]
    off, T, x, w, dy, want = operands(sizes, 0, 0, 2312, 1864)
    a, b = off[2], off[3]
    x[a:b], dy[a:b], w[2], w[1] = float("nan"), float("inf"), float("inf"), float("nan")
    offsets = torch.tensor(off, dtype=torch.int32, device="cuda")
    others = [t for t in range(T) if not a <= t < b]
    for got, (exact, size), k in ((ops.linear_ragged(x, w, offsets), want[0], 1864), (ops.linear_ragged_dgrad(dy, w, offsets), want[1], 2312)):
        near(got.cpu()[others], exact[others], size[others], k, "rows")
    dw = ops.linear_ragged_wgrad(dy, x, offsets).cpu()
    assert not dw[1].any()
    for e in (0, 3, 4):
        near(dw[e], want[2][0][e], want[2][1][e], T, "weights")


@pytest.mark.gpu
def test_offsets_of_pairs_out_of_order():
    """Offsets that decrease or leave the rows are taken as the nearest that do not: nothing outside is touched."""
    _, _, x, w, dy, _ = operands([2500, 0, 0, 0], 0, 0, 2056, 1800)
    for given, taken in (([-5, 1200, 700, 1300, 9999], [0, 1200, 1200, 1300, 2500]), ([6000, 1, 2, 3, 4], [2500] * 5),
                         ([2, 2 ** 31 - 1, -2 ** 31, 7, 7], [2] + [2500] * 4)):
        a, b = (torch.tensor(v, dtype=torch.int32, device="cuda") for v in (given, taken))
        assert torch.equal(ops.linear_ragged(x, w, a), ops.linear_ragged(x, w, b))
        assert torch.equal(ops.linear_ragged_dgrad(dy, w, a), ops.linear_ragged_dgrad(dy, w, b))
        assert torch.equal(ops.linear_ragged_wgrad(dy, x, a), ops.linear_ragged_wgrad(dy, x, b))


@pytest.mark.gpu
@pytest.mark.parametrize("sizes,N,K", [([0] * 20 + [1400] + [2] * 40, 264, 200), ([3000] + [0] * 200, 1032, 328), ([1, 3900, 2], 136, 4104)])
def test_one_group_has_nearly_all(sizes, N, K):
    """Blocks go by the mean of the groups: a group far above it has many."""
    off, T = bounds(sizes, 0, 0)
    x, w, dy = (t.cuda() for t in (rnd(1, T, K), rnd(2, len(sizes), N, K, scale=0.1), rnd(3, T, N)))
    (y, sy), (dx, sx), (dw, sw) = [tuple(t.cpu() for t in pair) for pair in oracle(x, w, dy, off)]
    offsets = torch.tensor(off, dtype=torch.int32, device="cuda")
    near(ops.linear_ragged(x, w, offsets), y, sy, K, "forward")
    near(ops.linear_ragged_dgrad(dy, w, offsets), dx, sx, N, "input gradient")
    near(ops.linear_ragged_wgrad(dy, x, offsets), dw, sw, T, "weight gradient")


@pytest.mark.gpu
def test_products_repeat_bit_for_bit():
    """Every form gives the same bits on every call: no sum is taken in the order in which CTAs come."""
    for sizes, N, K in (([2600, 1500], 4096, 1024), ([900, 0, 1300, 257, 1], 2312, 1864), ([1, 1], 2048, 4096), ([40, 0, 90], 136, 2056),
                        ([70] * 40, 128, 128), ([513, 40, 600, 2, 1000, 15, 0, 290], 768, 384)):
        off, T = bounds(sizes, 0, 0)
        x, w, dy = (t.cuda() for t in (rnd(1, T, K), rnd(2, len(sizes), N, K, scale=0.1), rnd(3, T, N)))
        offsets = torch.tensor(off, dtype=torch.int32, device="cuda")
        call = lambda: (ops.linear_ragged(x, w, offsets), ops.linear_ragged_dgrad(dy, w, offsets), ops.linear_ragged_wgrad(dy, x, offsets),
                        ops.linear_ragged_wgrad(dy, x, offsets, torch.float32))
        first = call()
        for _ in range(20):
            assert all(torch.equal(p, q) for p, q in zip(call(), first)), (sizes, N, K)


def test_most_rows():
    """Row numbers have room for a step past the last one in 32 bits: more rows are refused, here and at the C entry (without memory for
    them: the entry looks at the sizes first)."""
    most = ops.MAX_RAGGED_ROWS - 1
    meta = lambda *shape: torch.empty(*shape, dtype=torch.bfloat16, device="meta")
    w, offsets = meta(2, 16, 8), torch.empty(3, dtype=torch.int32, device="meta")
    assert ops.linear_ragged(meta(most, 8), w, offsets).shape == (most, 16)
    assert ops.linear_ragged_wgrad(meta(most, 16), meta(most, 8), offsets).shape == (2, 16, 8)
    for call in (lambda n: ops.linear_ragged(meta(n, 8), w, offsets), lambda n: ops.linear_ragged_dgrad(meta(n, 16), w, offsets),
                 lambda n: ops.linear_ragged_wgrad(meta(n, 16), meta(n, 8), offsets)):
        for n in (most + 1, 2 ** 31 - 1, 2 ** 31):
            with pytest.raises(ValueError):
                call(n)
    lib = native.load()
    for n in (most + 1, 2 ** 31 - 1):
        assert lib.jpb_linear_ragged(None, None, None, None, n, 2, 16, 8, 0, None, None) == -2
        assert lib.jpb_linear_ragged_wgrad(None, None, None, None, n, 2, 16, 8, 0, 0, None) == -2
