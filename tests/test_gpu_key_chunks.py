"""GPU: how many key chunks a tree call takes: a short page list beside a large tail view is not split for its table."""
import pytest
import torch

from tests import util as U
from tests.test_gpu_tree import Problem

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


def widen(p, capacity):
    """The tail as the first tokens of a cache of `capacity`."""
    big = [torch.zeros(x.shape[0], capacity, *x.shape[2:], dtype=x.dtype, device=DEV) for x in p.tail_d]
    for b, x in zip(big, p.tail_d):
        b[:, :x.shape[1]] = x
    p.tail_d = big


@pytest.mark.parametrize("kinds", [None, (U.Q8_0, U.Q8_0)])
@pytest.mark.parametrize("bound", [0, 1024])
def test_a_short_list_beside_a_large_tail_view_is_one_chunk(monkeypatch, kinds, bound):
    import kvmem_b200 as K
    monkeypatch.setenv("KVM_ATTEND", "tc")
    monkeypatch.setenv("KVM_ATTEND_SPLITS", "1")
    c = K.RecallContext(0)
    keep = torch.empty(max(bound, 1), dtype=torch.uint8, device=DEV)
    if bound:
        c.bind_workspace(keep)
    p = Problem(c, 71, 1, 5, 4, 1, 64, 16, 30, 12, [470], [40], torch.float16, kinds=kinds)
    widen(p, 131072)
    before = c.launches
    out, lse = p.call()
    assert c.launches - before == 1
    c.check_status()
    p.verify(out, lse)
    p.pool.close()
    c.close()


def test_a_list_of_more_boxes_than_the_table_holds_is_split(ctx, monkeypatch):
    """640 pages of 16 tokens: 80 key tiles of 8 boxes, where one chunk's table takes 64 tiles."""
    monkeypatch.setenv("KVM_ATTEND", "tc")
    monkeypatch.setenv("KVM_ATTEND_SPLITS", "1")
    p = Problem(ctx, 72, 1, 5, 4, 1, 64, 16, 700, 640, [11200], [40], torch.float16)
    widen(p, 5000)
    p.pool.plan(torch.arange(640, dtype=torch.int32, device=DEV)[None], torch.tensor([640], dtype=torch.int32, device=DEV))
    p.slot_of, p.page_of = p.pool.read()
    full = [p.page_of[0][p.page_of[0] >= 0]]
    assert len(full[0]) == 640
    before = ctx.launches
    out, lse = p.call(lists=full)
    assert ctx.launches - before == 2
    ctx.check_status()
    p.verify(out, lse, lists=full)
