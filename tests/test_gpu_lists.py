"""GPU: page lists of no columns, lists in wider tables, and trees of no words."""
import numpy as np
import pytest
import torch

from tests import util as U
from tests.test_gpu_pages import Mirror
from tests.test_gpu_tree import Problem

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


@pytest.mark.parametrize("kernel", ["mma", "tc"])
@pytest.mark.parametrize("kinds", [None, (U.Q8_0, U.Q4_0)])
@pytest.mark.parametrize("seqs", [1, 2])
def test_a_list_without_columns_names_no_page(ctx, monkeypatch, kernel, kinds, seqs):
    import kvmem_b200 as K
    monkeypatch.setenv("KVM_ATTEND", kernel)
    p = Problem(ctx, 61, seqs, 3, 8, 2, 128, 64, 6, 4, [300] * seqs, [7] * seqs, torch.float16, kinds=kinds)
    none = torch.empty((seqs, 0), dtype=torch.int32, device=DEV)
    n = torch.zeros(seqs, dtype=torch.int32, device=DEV)
    out, lse = p.call(sel_ids=none, sel_n=n)
    ctx.check_status()
    p.verify(out, lse, lists=[[]] * seqs)
    out, lse = p.call(sel_ids=none, sel_n=n + 1)  # a count past it is reported
    assert ctx.status() == K._abi.ERR_INVALID_ARGUMENT
    p.verify(out, lse, lists=[[]] * seqs)


def test_freeing_a_list_without_columns_drops_nothing(ctx):
    import kvmem_b200 as K
    m = Mirror(ctx, 62, 3, 9, 4, 64)
    none = torch.empty((2, 0), dtype=torch.int32, device=DEV)
    n = torch.zeros(2, dtype=torch.int32, device=DEV)
    m.pool.free([0, 2], none, n)
    ctx.check_status()
    m.verify()
    m.pool.free([0, 2], none, n + 1)
    assert ctx.status() == K._abi.ERR_INVALID_ARGUMENT
    m.verify()


@pytest.mark.parametrize("shape", [(3, 0), (1, 3, 0)])
def test_a_tree_without_words_is_refused(ctx, shape):
    import kvmem_b200 as K
    p = Problem(ctx, 63, 1, 3, 4, 1, 64, 32, 4, 2, [64], [0], torch.float16)
    with pytest.raises(K.KvmError) as e:
        p.call(tree=torch.empty(shape, dtype=torch.int32, device=DEV))
    assert e.value.code == K._abi.ERR_INVALID_ARGUMENT
    ctx.check_status()


@pytest.mark.parametrize("kernel", ["mma", "tc"])
@pytest.mark.parametrize("kinds", [None, (U.Q8_0, U.Q4_0)])
def test_a_count_past_the_columns_of_a_wider_table_is_reported(ctx, monkeypatch, kernel, kinds):
    """Lists that are the first columns of wider rows: a count reaches to the columns given, not into what lies behind."""
    import kvmem_b200 as K
    monkeypatch.setenv("KVM_ATTEND", kernel)
    p = Problem(ctx, 64, 2, 3, 8, 2, 128, 64, 12, 5, [700, 700], [7, 3], torch.float16, kinds=kinds)
    wide = torch.zeros((2, 16), dtype=torch.int32, device=DEV)
    mine = [p.lists[i][:2] for i in range(2)]
    assert all(len(x) == 2 for x in mine)
    wide[:, :2] = torch.from_numpy(np.stack(mine).astype(np.int32))
    wide[:, 2:] = wide[:, :1]  # resident pages, which must not be read
    view = wide[:, :2]
    two = torch.full((2,), 2, dtype=torch.int32, device=DEV)
    out, lse = p.call(sel_ids=view, sel_n=two)
    ctx.check_status()
    p.verify(out, lse, lists=mine)
    out, lse = p.call(sel_ids=view, sel_n=two + 3)
    assert ctx.status() == K._abi.ERR_INVALID_ARGUMENT
    p.verify(out, lse, lists=mine)
