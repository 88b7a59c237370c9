"""Ops whose eager calls go past the dispatcher: whatever else may be under way sees them as it sees every other op."""
import pytest
import torch
import torch.fx as fx

import jaxpp_b200 as jp  # noqa: F401  (registers the ops)
from jaxpp_b200.ops import core as ops
from jaxpp_b200.parallel import moe


def rnd(seed, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


X, W = rnd(0, 6, 16), rnd(1, 16)
E, OFF = rnd(2, 3, 8, 16), torch.tensor([0, 2, 2, 6], dtype=torch.int32)
DY = rnd(3, 6, 8)
IDS, TOP, LSE, LAB = torch.arange(24).view(6, 4) % 16, rnd(4, 6, 4), rnd(5, 6).abs() + 3, torch.arange(6)
CALLS = {  # name: op, tensors, what follows them
    "residual_norm": (ops.residual_norm, (X, X, W, W, W), (0.9, 1e-5)),
    "residual_norm_bwd": (ops.residual_norm_bwd, (X, X, X, X, W, W, W, LSE, LSE), (0.9,)),
    "distill_loss": (ops.distill_loss, (X, IDS, TOP, LSE, LAB), (2.0, 0.5)),
    "distill_loss_grad": (ops.distill_loss_grad, (LSE, X, IDS, TOP, LSE, LAB), (2.0, 0.5)),
    "linear_ragged": (ops.linear_ragged, (X, E, OFF), ()),
    "linear_ragged_dgrad": (ops.linear_ragged_dgrad, (DY, E, OFF), ()),
    "linear_ragged_wgrad": (ops.linear_ragged_wgrad, (DY, X, OFF), ()),
    "expert_order": (moe.expert_order, (IDS,), (16,)),
}
NAMES = sorted(CALLS)


def flat(out):
    return list(out) if isinstance(out, (tuple, list)) else [out]


def same(a, b):
    return len(flat(a)) == len(flat(b)) and all(torch.equal(p, q) for p, q in zip(flat(a), flat(b)))


@pytest.mark.parametrize("name", NAMES)
def test_compiled_whole(name):
    op, tensors, rest = CALLS[name]
    torch._dynamo.reset()
    got = torch.compile(lambda *t: op(*t, *rest), backend="aot_eager", fullgraph=True)(*tensors)
    assert same(got, op(*tensors, *rest))


def test_compiled_with_gradients():
    torch._dynamo.reset()

    def loss(x, w, e):
        r, h, _, _ = ops.residual_norm(x, x, w, None, w, 1.0, 1e-5)
        return ops.distill_loss(ops.linear_ragged(h, e, OFF) + r[:, :8], IDS % 8, TOP, None, None, 1.0, 1.0).sum()

    grads = []
    for f in (loss, torch.compile(loss, backend="aot_eager", fullgraph=True)):
        leaves = [t.clone().requires_grad_(True) for t in (X, W, E)]
        grads.append(torch.autograd.grad(f(*leaves), leaves))
    assert same(*grads)


@pytest.mark.parametrize("name", NAMES)
def test_symbolically_traced(name):
    op, tensors, rest = CALLS[name]
    names = ["a", "b", "c", "d", "e", "f", "g", "h", "i"][: len(tensors)]
    scope = {"op": op, "rest": rest}
    exec(f"def f({', '.join(names)}): return op({', '.join(names)}, *rest)", scope)
    traced = fx.symbolic_trace(scope["f"])
    assert sum("b200" in str(n.target) for n in traced.graph.nodes if n.op == "call_function") == 1
    assert same(traced(*tensors), op(*tensors, *rest))


@pytest.mark.parametrize("name", NAMES)
def test_modes_and_profiles_see_it(name):
    op, tensors, rest = CALLS[name]
    seen = []

    class Function(torch.overrides.TorchFunctionMode):
        def __torch_function__(self, fn, types, args=(), kwargs=None):
            seen.append(str(fn))
            return fn(*args, **(kwargs or {}))

    class Dispatch(torch.utils._python_dispatch.TorchDispatchMode):
        def __torch_dispatch__(self, fn, types, args=(), kwargs=None):
            seen.append(str(fn))
            return fn(*args, **(kwargs or {}))

    for mode in (Function, Dispatch):
        seen.clear()
        with mode():
            op(*tensors, *rest)
        assert any(name in s for s in seen), mode
    with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CPU]) as prof:
        op(*tensors, *rest)
    assert any(name in e.key for e in prof.key_averages())


@pytest.mark.parametrize("name", NAMES)
def test_tensors_without_data(name):
    """Meta tensors give meta tensors of the results' shapes."""
    op, tensors, rest = CALLS[name]
    want = flat(op(*tensors, *rest))
    got = flat(op(*[t.to("meta") for t in tensors], *rest))
    assert [(t.shape, t.dtype, t.is_meta) for t in got] == [(t.shape, t.dtype, True) for t in want]


def test_transforms_and_keywords():
    op, (x, y, w, g, _), rest = CALLS["residual_norm"]
    f = lambda a: op(a, a, w, None, w, 1.0, 1e-5)[1]
    batch = torch.stack([x, 2 * x, 3 * x])
    torch.testing.assert_close(torch.vmap(f)(batch), torch.stack([f(b) for b in batch]))
    assert same(op(x, y, w, g, w, scale=0.9, eps=1e-5), op(x, y, w, g, w, 0.9, 1e-5))


@pytest.mark.parametrize("name", NAMES)
def test_plain_calls_go_past_the_dispatcher(name):
    """What the detour is for: nothing under way, no gradient to record."""
    op, tensors, rest = CALLS[name]
    target = op if hasattr(op, "packet") else moe._expert_order
    real, calls = target._impl, []
    target._impl = lambda *a: calls.append(1) or real(*a)
    try:
        op(*tensors, *rest)
    finally:
        target._impl = real
    assert calls
