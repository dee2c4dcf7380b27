"""GPU: a sequence whose rows do not fit its cache is left as it was, whether its position is one number for all
sequences or a device array, split or not."""
import pytest
import torch

from tests.test_gpu_tree import Problem
from tests.test_gpu_window import compare, make

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


@pytest.mark.parametrize("kernel", ["mma", "tc"])
@pytest.mark.parametrize("splits", ["1", "4"])
def test_window_rows_past_the_cache_at_one_position(ctx, monkeypatch, kernel, splits):
    import kvmem_b200 as K
    monkeypatch.setenv("KVM_ATTEND", kernel)
    monkeypatch.setenv("KVM_ATTEND_SPLITS", splits)
    cap, base, rows = 900, 897, [4, 2]
    q, k, v = make(31, 2, 4, 8, 2, 128, cap, torch.float16)
    out = torch.full_like(q, 3.0).to(DEV)
    lse = torch.full((2, 4, 8), 5.0, device=DEV)
    ctx.window_attention(q.to(DEV), k.to(DEV), v.to(DEV), base=base, window=700, sinks=5, out=out, lse=lse,
                         rows=torch.tensor(rows, dtype=torch.int32, device=DEV))
    assert ctx.status() == K._abi.ERR_LENGTH
    assert (out[0] == 3).all() and (lse[0] == 5).all()
    assert (out[1, 2:] == 3).all() and (lse[1, 2:] == 5).all()
    compare(q[1:], k[1:], v[1:], out[1:], lse[1:], [base], 700, 5, rows=[2])


@pytest.mark.parametrize("kernel", ["mma", "tc"])
@pytest.mark.parametrize("splits", ["1", "4"])
def test_tree_nodes_past_the_tail_at_one_length(ctx, monkeypatch, kernel, splits):
    import kvmem_b200 as K
    monkeypatch.setenv("KVM_ATTEND", kernel)
    monkeypatch.setenv("KVM_ATTEND_SPLITS", splits)
    p = Problem(ctx, 32, 2, 6, 8, 2, 128, 64, 12, 5, [700, 300], [9, 9], torch.bfloat16)
    # The tail views hold 14 tokens: 9 recent ones and 5 nodes.
    p.tail, p.tail_d = [x[:, :14] for x in p.tail], [x[:, :14] for x in p.tail_d]
    out = torch.full((2, 6, 8, 128), 3.0, dtype=torch.bfloat16, device=DEV)
    lse = torch.full((2, 6, 8), 5.0, device=DEV)
    p.call(out=out, lse=lse, recent=9, rows=torch.tensor([6, 5], dtype=torch.int32, device=DEV))
    assert ctx.status() == K._abi.ERR_LENGTH
    assert (out[0] == 3).all() and (lse[0] == 5).all()
    assert (out[1, 5:] == 3).all() and (lse[1, 5:] == 5).all()
    p.verify(out, lse, rows=[0, 5])


@pytest.mark.parametrize("kernel", ["mma", "tc"])
@pytest.mark.parametrize("splits", ["1", "4"])
@pytest.mark.parametrize("bad", [5, -1])
def test_more_rows_than_the_batch_has(ctx, monkeypatch, kernel, splits, bad):
    import kvmem_b200 as K
    monkeypatch.setenv("KVM_ATTEND", kernel)
    monkeypatch.setenv("KVM_ATTEND_SPLITS", splits)
    rows = torch.tensor([bad, 3], dtype=torch.int32, device=DEV)
    q, k, v = make(33, 2, 4, 8, 2, 128, 900, torch.float16)
    out, lse = torch.full_like(q, 3.0).to(DEV), torch.full((2, 4, 8), 5.0, device=DEV)
    ctx.window_attention(q.to(DEV), k.to(DEV), v.to(DEV), base=800, window=700, sinks=5, out=out, lse=lse, rows=rows)
    assert ctx.status() == K._abi.ERR_LENGTH
    assert (out[0] == 3).all() and (lse[0] == 5).all() and (out[1, 3:] == 3).all() and (lse[1, 3:] == 5).all()
    compare(q[1:], k[1:], v[1:], out[1:], lse[1:], [800], 700, 5, rows=[3])

    p = Problem(ctx, 34, 2, 4, 8, 2, 128, 64, 12, 5, [700, 300], [9, 9], torch.float16)
    out, lse = torch.full((2, 4, 8, 128), 3.0, dtype=torch.float16, device=DEV), torch.full((2, 4, 8), 5.0, device=DEV)
    p.call(out=out, lse=lse, rows=rows)
    assert ctx.status() == K._abi.ERR_LENGTH
    assert (out[0] == 3).all() and (lse[0] == 5).all() and (out[1, 3:] == 3).all() and (lse[1, 3:] == 5).all()
    p.verify(out, lse, rows=[0, 3])
