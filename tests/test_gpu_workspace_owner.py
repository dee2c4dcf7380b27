"""GPU: the page statistics that the first half of a sharded score leaves in the workspace are not taken for page
masses once another call has written there."""
import numpy as np
import pytest
import torch

from tests import util as U
from tests.test_gpu_window import compare, make

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


class Halves:
    """A sharded score of one rank (the whole history), in its two halves."""

    def __init__(self, bound=True):
        import kvmem_b200 as K
        from kvmem_b200.shard import ShardCompute, ShardGeometry
        rng = np.random.default_rng(41)
        self.dims = L, H, G, D, B, P = 2, 8, 2, 64, 32, 21
        self.ctx = K.RecallContext(0)
        self.keep = torch.empty(1 << 21, dtype=torch.uint8, device=DEV)
        if bound:
            self.ctx.bind_workspace(self.keep)
        self.comp = ShardCompute(self.ctx)
        self.geo = ShardGeometry(layers=L, rows=1, q_heads=H, kv_heads=G, groups=1, total_pages=P, page0=0, local_pages=P)
        self.qd = torch.from_numpy(U.make_q(rng, U.F32, L, 1, H, D).reshape(-1).copy()).to(DEV).view(torch.float32).view(L, 1, H, D)
        self.kd = torch.from_numpy(U.make_k(rng, U.F16, L, P * B, G, D).reshape(-1).copy()).to(DEV)
        self.desc = K.RecallContext.make_desc(layers=L, q_heads=H, kv_heads=G, head_dim=D, tokens=P * B - 3, page_tokens=B)
        self.q = K.RecallContext.make_query(self.qd, 1)
        self.k = K.RecallContext.make_kcache(self.kd, U.F16, kv_heads=G, head_dim=D, capacity_tokens=P * B)
        other = K.RecallContext(0)
        self.want = other.score_pages(self.desc, self.q, self.k, want_rows=False)[1].view(L, P).clone()
        other.close()

    def first(self):
        stats = self.comp.partial(self.desc, self.q, self.k, self.geo)
        self.stats = self.comp.merge_stats(stats[None], 1, self.geo)

    def second(self):
        return self.comp.finish(self.desc, self.geo, self.stats)

    def right(self, mass):
        torch.testing.assert_close(mass, self.want, rtol=1e-5, atol=1e-9)


def window(ctx):
    q, k, v = make(42, 1, 2, 8, 2, 128, 900, torch.float16)
    out, lse = ctx.window_attention(q.to(DEV), k.to(DEV), v.to(DEV), base=890, window=800, sinks=4, want_lse=True)
    ctx.check_status()
    compare(q, k, v, out, lse, [890], 800, 4)


def test_split_attention_between_the_halves_is_reported(monkeypatch):
    import kvmem_b200 as K
    monkeypatch.setenv("KVM_ATTEND_SPLITS", "4")
    h = Halves()
    h.first()
    window(h.ctx)
    with pytest.raises(K.KvmError) as e:
        h.second()
    assert e.value.code == K._abi.ERR_STALE
    h.first()  # from the start again
    h.right(h.second())
    h.right(h.second())  # the statistics stay for a second reading
    h.ctx.close()


def test_another_score_between_the_halves_is_reported():
    import kvmem_b200 as K
    h = Halves()
    h.first()
    h.ctx.score_pages(h.desc, h.q, h.k, want_rows=False)
    with pytest.raises(K.KvmError) as e:
        h.second()
    assert e.value.code == K._abi.ERR_STALE
    h.ctx.close()


def test_another_workspace_between_the_halves_is_reported():
    import kvmem_b200 as K
    h = Halves()
    h.first()
    other = torch.zeros(1 << 21, dtype=torch.uint8, device=DEV)
    h.ctx.bind_workspace(other)
    with pytest.raises(K.KvmError) as e:
        h.second()
    assert e.value.code == K._abi.ERR_STALE
    h.ctx.close()


@pytest.mark.parametrize("bound,splits", [(True, "1"), (False, "4")])
def test_attention_that_writes_elsewhere_is_fine_between_the_halves(monkeypatch, bound, splits):
    """Not split, or with the context's own scratch."""
    monkeypatch.setenv("KVM_ATTEND_SPLITS", splits)
    h = Halves(bound)
    h.first()
    window(h.ctx)
    h.right(h.second())
    h.ctx.close()
