"""Worker for ``test_student_multiprocess``: a student with sandwich norms and gates, trained against a teacher's top logits, sharded
over pipeline ranks and a tensor-parallel axis, against the un-sharded single-process step."""
import os
import sys

import torch
import torch.distributed as dist
from torch.utils import _pytree as pytree

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))

import jaxpp_b200 as jp  # noqa: E402
from jaxpp_b200.launch import distributed_main  # noqa: E402
from jaxpp_b200.models import lm_trainer as lt  # noqa: E402
from jaxpp_b200.models import transformer as tf  # noqa: E402


def main(pp, tp, schedule, tail):
    mesh = jp.MpmdMesh.create({"mpmd": pp, "data": 1, "model": tp}, kind="cpu", multi_process=True)
    base = dict(vocab=250, d_model=64, n_layers=4, n_heads=4, n_kv_heads=2, ffn=128, seq=32, dtype=torch.float32, sandwich_norm=True,
                residual_scale=0.9, residual_gate=0.5)
    cfg1, cfgt = (tf.ModelConfig("llama", n_stages=schedule.num_stages, tp=n, **base) for n in (1, tp))
    hyper = lt.Hyper(lr=1e-2, inplace_update=False, distill_alpha=0.7, distill_temperature=2.0)
    g = torch.Generator().manual_seed(5)
    tokens, labels = (torch.randint(0, 250, (4, 2, 32), generator=g) for _ in range(2))
    teacher = torch.randn(4, 2, 32, 250, generator=g) * 2
    top, ids = teacher.topk(6, -1)
    batch = [tokens, labels, ids, top] + ([torch.logsumexp(teacher / 2.0, -1)] if tail else [])
    state1 = lt.init_state(cfg1, schedule, "cpu")
    ref_state, ref_losses = lt.make_train_step(cfg1, schedule, hyper)(state1, *batch)
    me_pp, me_tp, owners = mesh.my_mpmd_axis_index, mesh.axis_index("model"), lt.owner_ranks(cfgt, schedule)

    def local_view(tree):
        mine = lambda v, group: v if owners[group] == me_pp else jp.ShapeDtypeStruct(tuple(v.shape), v.dtype)
        out = {"step": tree["step"]}
        for key in ("params", "master", "m", "v"):
            part = tf.shard_params_for_tp(cfg1, tree[key], tp, me_tp)
            out[key] = {k: mine(v, "embed" if k == "embed" else "head") for k, v in part.items() if k != "layers"}
            out[key]["layers"] = {n: {k: mine(v, int(n)) for k, v in layer.items()} for n, layer in part["layers"].items()}
        return out

    got, losses = jp.mpmd_jit_with_loop(lt.make_train_step(cfgt, schedule, hyper), mesh)(local_view(state1), *batch)
    want = local_view(ref_state)
    compared = set()
    for (path, x), y in zip(pytree.tree_flatten_with_path(want["m"], is_leaf=lambda x: isinstance(x, jp.ShapeDtypeStruct))[0],
                            pytree.tree_leaves(got["m"], is_leaf=lambda x: isinstance(x, jp.MpmdArray)), strict=True):
        t = y.local_tensor()
        assert (t is None) == isinstance(x, jp.ShapeDtypeStruct)
        if t is not None:      # the first moments are a tenth of the gradients: sums of a few hundred fp32 terms in another order
            torch.testing.assert_close(t, x, rtol=2e-3, atol=1e-6 * float(x.abs().max()) + 1e-8)
            compared.add(str(path[-1]))
    assert all(any(k in c for c in compared) for k in ("attn_post_norm", "ffn_post_norm", "attn_gate", "ffn_gate")), compared
    mean = losses.local_tensor()
    if mean is not None:       # every tensor-parallel rank has the mean loss of its own tokens
        mean = mean.clone()
        dist.all_reduce(mean, group=mesh.axis_group("model"))
        torch.testing.assert_close(mean / tp, ref_losses, rtol=1e-5, atol=1e-6)


if __name__ == "__main__":
    distributed_main({"tp2": lambda: main(1, 2, jp.Std1F1B(1), True), "pp2_tp2": lambda: main(2, 2, jp.Interleaved1F1B(4, 2), False)}[sys.argv[1]])
