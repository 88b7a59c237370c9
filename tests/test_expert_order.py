"""Order of the picks at the edges of its kernels' steps and sizes."""
import pytest
import torch

import jaxpp_b200 as jp  # noqa: F401  (registers the ops)
from jaxpp_b200.parallel import moe

CPU_PICKS = (1, 33, 2047, 2048, 2049)


def check(n, experts, kind, device):
    """Against a stable sort of the picks that name an expert."""
    g = torch.Generator().manual_seed(n + experts)
    picks = {"any": torch.randint(0, experts, (n,), generator=g), "strangers": torch.randint(-1, experts + 1, (n,), generator=g),
             "one expert": torch.full((n,), experts - 1), "none": torch.full((n,), -1)}[kind]
    dest, inv, offsets = (t.cpu() for t in moe.expert_order(picks.to(device), experts))
    known = (picks >= 0) & (picks < experts)
    order = torch.argsort(torch.where(known, picks, experts), stable=True)[: int(known.sum())]
    want_inv = torch.full((n,), -1, dtype=torch.int32)
    want_inv[: len(order)] = order.int()
    want_dest = torch.full((n,), n)
    want_dest[order] = torch.arange(len(order))
    counts = torch.tensor([int((picks == e).sum()) for e in range(experts)])
    assert torch.equal(inv, want_inv) and torch.equal(dest, want_dest)
    assert offsets.tolist() == [0] + counts.cumsum(0).tolist()


@pytest.mark.parametrize("kind", ["any", "strangers", "one expert", "none"])
@pytest.mark.parametrize("experts", [1, 32, 33, 256])
def test_order(experts, kind):
    for n in CPU_PICKS:
        check(n, experts, kind, "cpu")


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["any", "strangers", "one expert", "none"])
@pytest.mark.parametrize("experts", [1, 32, 33, 256])
def test_order_at_the_kernels_steps(experts, kind):
    """One launch up to 2048 picks, steps of 1024, runs of one step up to 131072 picks and of two from there on."""
    for n in (*CPU_PICKS, 1023, 1024, 1025, 4096, 131071, 131072, 131073, 262145):
        check(n, experts, kind, "cuda")


def test_most_picks():
    """As many as the documents say, and no more (without memory for them)."""
    dest, inv, offsets = moe.expert_order(torch.empty(2 ** 31 - 2 ** 24 - 1, dtype=torch.int64, device="meta"), 8)
    assert dest.shape == inv.shape == (2 ** 31 - 2 ** 24 - 1,) and offsets.shape == (9,)
    with pytest.raises(ValueError):
        moe.expert_order(torch.empty(2 ** 31 - 2 ** 24, dtype=torch.int64, device="meta"), 8)
