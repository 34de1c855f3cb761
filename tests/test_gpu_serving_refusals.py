"""Calls of the serving wrappers on the GPU that are refused, and what they say."""
import pytest
import torch

from nativebit_amd import ops

pytestmark = pytest.mark.gpu


def test_plan_into_memory_of_its_inputs(dev):
    """Outputs over inputs, or over one another, in whole or in part."""
    def i32(*a):
        return torch.tensor(a, dtype=torch.int32, device=dev)
    R, n = 3, 6
    table = torch.full((R, 4), -1, dtype=torch.int32, device=dev)
    lens, new, free, state = i32(0, 0, 0), i32(1, 2, 3), torch.arange(20, dtype=torch.int32, device=dev), i32(20, 0)
    whole = torch.zeros(100, dtype=torch.int32, device=dev)
    chunks = ops.kv_plan_chunks(n, R)

    def out(**kw):
        a = dict(slots=whole[:n], positions=whole[n:2 * n], chunks=whole[2 * n:2 * n + 4 * chunks].view(-1, 4),
                 lens=whole[50:53], state=whole[53:55])
        return ops.KVPlan(**{**a, **kw})
    want = ops.kv_plan(table.clone(), lens, new, free, state, n)
    got = ops.kv_plan(table, lens, new, free, state, n, out=out())     # side by side
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    table.fill_(-1)
    both = torch.zeros(12, dtype=torch.int32, device=dev)
    for bad, kw in ((out(lens=lens), {}), (out(state=state), {}), (out(slots=free[3:9]), {}),
                    (out(positions=table.view(-1)[6:12]), {}), (out(positions=whole[:n]), {}),
                    (out(lens=whole[52:55]), {}), (out(state=whole[49:51]), {}), (out(lens=new), {}),
                    (out(lens=both[2:5]), {"new": both[:3]}), (out(lens=both[:3]), {"lens": both[2:5]})):
        args = {"lens": lens, "new": new, **kw}
        with pytest.raises(ValueError, match="overlaps"):
            ops.kv_plan(table, args["lens"], args["new"], free, state, n, out=bad)
    assert (table == -1).all() and (both == 0).all()
    # inputs may share memory
    ops.kv_plan(table, new, new, free, state, n, out=out())


def test_attention_names_the_argument(dev):
    """A plan of the wrong size beside a table whose rows lie apart (which is
    taken)."""
    k = torch.zeros(3, 1, 64, 16, dtype=torch.int8, device=dev)
    v, s = k.view(3, 1, 16, 64), torch.zeros(3, 1, device=dev)
    wide = torch.full((2, 5), -1, dtype=torch.int32, device=dev)
    z = torch.zeros(2, dtype=torch.int32, device=dev)
    plan = ops.KVPlan(z, z, torch.zeros(2, 4, dtype=torch.int32, device=dev), z, z)
    q = torch.zeros(2, 16, device=dev)
    assert ops.kv8_attention(q, plan, wide[:, :2], k, v, s, s).shape == (2, 16)
    for bad, name in ((plan._replace(chunks=z), "plan.chunks"), (plan._replace(lens=z[:1]), "plan.lens")):
        with pytest.raises(ValueError, match=name):
            ops.kv8_attention(q, bad, wide[:, :2], k, v, s, s)
