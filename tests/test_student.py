"""The operators of a step together: a student with sandwich norms and dropless experts, trained against a teacher's top logits."""
import dataclasses

import pytest
import torch
from torch.utils import _pytree as pytree

import jaxpp_b200 as jp
from jaxpp_b200.models import lm_trainer as lt
from jaxpp_b200.models import transformer as tf
from jaxpp_b200.ops import core as ops
from jaxpp_b200.parallel import moe

from tests.helpers import assert_trees_equal, local


def mesh(pp, kind="cpu"):
    return jp.MpmdMesh.create({"mpmd": pp, "data": 1, "model": 1}, kind=kind, multi_process=False)


def batch(cfg, n_mb, mb, k, tail, device="cpu", seed=3):
    g = torch.Generator().manual_seed(seed)
    tokens = torch.randint(0, cfg.vocab, (n_mb, mb, cfg.seq), generator=g)
    labels = torch.randint(0, cfg.vocab, (n_mb, mb, cfg.seq), generator=g)
    logits = torch.randn(n_mb, mb, cfg.seq, cfg.vocab, generator=g) * 2
    top, ids = logits.topk(k, -1)
    ids = ids.to(torch.int32)
    ids[:, :, :3], labels[:, :, :3] = -1, -1        # prompt tokens carry neither
    teacher = [ids, top.to(cfg.dtype)] + ([torch.logsumexp(logits / 2.0, -1)] if tail else [])
    return [t.to(device) for t in (tokens, labels, *teacher)]


STUDENT = dict(vocab=100, d_model=32, n_layers=4, n_heads=2, n_kv_heads=1, ffn=48, seq=16, dtype=torch.float32, sandwich_norm=True,
               residual_scale=0.9, residual_gate=0.5)
HYPER = lt.Hyper(lr=1e-2, inplace_update=False, distill_alpha=0.7, distill_temperature=2.0)


@pytest.mark.parametrize("family,schedule,pp,stage_layers,recompute,tail", [
    ("llama", jp.Std1F1B(2), 2, None, False, True), ("llama", jp.ZeroBubble(2), 2, (2.5, 1.5), False, False),
    ("mixtral", jp.DualPipeV(4, 2), 2, None, False, True), ("mixtral", jp.Std1F1B(2), 2, (1.5, 2.5), True, True),
])
def test_student_pipelined_matches_unpipelined(family, schedule, pp, stage_layers, recompute, tail):
    extra = dict(n_experts=4, top_k=2, dropless=True) if family == "mixtral" else {}
    cfg = tf.ModelConfig(family, n_stages=schedule.num_stages, stage_layers=stage_layers, recompute=recompute, **STUDENT, **extra)
    step = lt.make_train_step(cfg, schedule, HYPER)
    state = lt.init_state(cfg, schedule, "cpu")
    data = batch(cfg, 4, 2, 5, tail)
    ref = step(state, *data)
    got = jp.mpmd_jit_with_loop(step, mesh(pp))(state, *data)
    assert_trees_equal(ref, got, exact=True)
    new = ref[0]["params"]["layers"]["001"]
    for key in ("attn_post_norm", "ffn_post_norm", "attn_gate", "ffn_gate") + (("router", "e_up", "e_down") if extra else ("w_up",)):
        assert not torch.equal(new[key], state["params"]["layers"]["001"][key]), key


def test_step_takes_a_teacher_exactly_when_it_distills():
    cfg = tf.ModelConfig("llama", n_stages=1, **STUDENT)
    sched = jp.Std1F1B(1)
    state = lt.init_state(cfg, sched, "cpu")
    data = batch(cfg, 1, 1, 4, False)
    for hyper, args in ((HYPER, data[:2]), (dataclasses.replace(HYPER, distill_alpha=None), data)):
        with pytest.raises(ValueError):
            lt.make_train_step(cfg, sched, hyper)(state, *args)


def test_configurations_that_do_not_go_together():
    for kw in (dict(family="gpt2", sandwich_norm=True), dict(family="llama", dropless=True), dict(family="llama", residual_gate=1.0),
               dict(family="mixtral", n_experts=4, ep=2, dropless=True)):
        args = {**{k: v for k, v in STUDENT.items() if k not in ("sandwich_norm", "residual_scale", "residual_gate")}, **kw}
        with pytest.raises(ValueError):
            tf.ModelConfig(**args)


def test_dropless_experts_match_slots_with_room_for_all():
    """With room for every pick the capacity form drops nothing: same sums of the same products, a token's picks in the same order.
    (Padding rows change the blocking of a CPU product, hence fp32 tolerances: 2^-20 of sums of a few unit terms.)"""
    torch.manual_seed(0)
    T, d, F, E, k = 37, 24, 40, 5, 2
    p = {"router": torch.randn(E, d) * 0.3, "w_up": torch.randn(E, 2 * F, d) * 0.2, "w_down": torch.randn(E, d, F) * 0.2}
    x = torch.randn(T, d)
    outs = []
    with mesh(1):
        for f in (lambda x_, q: moe.moe_ffn(x_, q, E, k, float(E), 1, "data"), lambda x_, q: moe.moe_ffn_dropless(x_, q, E, k)):
            leaves = {n: t.clone().requires_grad_(True) for n, t in p.items()}
            xl = x.clone().requires_grad_(True)
            y, aux = f(xl, leaves)
            g = torch.autograd.grad((y * torch.cos(torch.arange(d))).sum() + aux, [xl, *leaves.values()])
            outs.append((y, aux, *g))
    for a, b in zip(*outs):
        torch.testing.assert_close(a, b, rtol=1e-5, atol=1e-5)


def test_plain_residual_norm_is_the_sum_of_two_ops():
    """Without a post-norm and gates at scale one the op is the residual addition and the next RMSNorm."""
    g = torch.Generator().manual_seed(0)
    x, y, w = torch.randn(5, 32, generator=g), torch.randn(5, 32, generator=g), torch.randn(32, generator=g)
    r, h, _, _ = ops.residual_norm(x, y, None, None, w, 1.0, 1e-5)
    assert torch.equal(r, x + y)
    torch.testing.assert_close(h, ops.rmsnorm(x + y, w, 1e-5)[0], rtol=1e-6, atol=1e-6)


# ---- on the GPU -------------------------------------------------------------------------------------------------------------
GPU = dict(vocab=1000, d_model=256, n_layers=2, n_heads=4, n_kv_heads=2, ffn=320, seq=65, sandwich_norm=True, residual_scale=0.9,
           residual_gate=0.7, dtype=torch.bfloat16, n_experts=8, top_k=2, dropless=True)


def one_step(device, dtype, stages=1, jit=False, recompute=False, steps=1, **over):
    sched = jp.Std1F1B(1) if stages == 1 else jp.Interleaved1F1B(stages, 1)
    cfg = tf.ModelConfig("mixtral", n_stages=stages, recompute=recompute, **{**GPU, "dtype": dtype, **over})
    state = lt.init_state(dataclasses.replace(cfg, dtype=torch.bfloat16), sched, "cpu")    # the same weights whatever the type
    state = pytree.tree_map(lambda t: t.to(device), state)
    if dtype is torch.float32:
        state["params"] = pytree.tree_map(lambda t: t.float(), state["params"])
    step = lt.make_train_step(cfg, sched, dataclasses.replace(HYPER, lr=1e-3))
    if jit:
        step = jp.mpmd_jit_with_loop(step, mesh(1, device))
    losses = []
    for i in range(steps):
        state, ls = step(state, *batch(dataclasses.replace(cfg, dtype=torch.bfloat16), 2, 3, 12, True, device, seed=7 + i % 2))
        losses.append(local(ls).float().cpu())
    return state, torch.stack(losses)


@pytest.mark.gpu
@pytest.mark.parametrize("recompute", [False, True])
def test_student_step_on_the_gpu(recompute):
    """A compiled bf16 step against the same step in fp32 on the CPU.  An activation rounded to bf16 is off by 2^-9 of its size
    on average and a block rounds about ten times (a norm undoes nothing of that): the loss, a mean of 400 tokens, and the first
    moments (0.1 of the gradients), as a whole, are held to 16 and 32 such roundings, 2^-5 and 2^-4.  Every token goes to all
    three experts: which experts a rounded router picks out of more is no matter of rounding."""
    ref, ref_loss = one_step("cpu", torch.float32, n_experts=3, top_k=3)
    got, loss = one_step("cuda", torch.bfloat16, stages=2, jit=True, recompute=recompute, n_experts=3, top_k=3)
    assert (loss - ref_loss).abs().max() <= 2.0 ** -5 * ref_loss.abs().max()
    flat = lambda s: torch.cat([local(t).double().cpu().reshape(-1) for t in pytree.tree_leaves(s["m"], is_leaf=lambda t: isinstance(t, jp.MpmdArray))])
    a, b = flat(ref), flat(got)
    assert float((a - b).norm()) <= 2.0 ** -4 * float(a.norm())
    from jaxpp_b200.ops import native

    torch.cuda.synchronize()
    assert native.read_status() == 0


@pytest.mark.gpu
def test_student_steps_replayed():
    """Several steps through the compiled program (recorded and replayed as graphs where it is launch-bound) and eagerly: the
    forward kernels are the same and take the same values, so that the first losses are equal bit for bit; later ones see
    parameter sums that the compiled step keeps in fp32 and the eager one rounds (2^-9 of an update of 1e-3)."""
    _, eager = one_step("cuda", torch.bfloat16, steps=6)
    _, jitted = one_step("cuda", torch.bfloat16, jit=True, steps=6)
    assert torch.equal(eager[0], jitted[0])
    assert (eager - jitted).abs().max() <= 2.0 ** -6 * eager.abs().max()
    _, again = one_step("cuda", torch.bfloat16, jit=True, steps=6)
    assert torch.equal(again, jitted)
