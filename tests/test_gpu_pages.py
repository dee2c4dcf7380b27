"""GPU: forking, copying, freeing and compacting the pages of a residency pool, against the same rules in numpy (all
integers and bytes: equal), and a run of them with selection, stage-in and attention as a branching lane uses them."""
import math

import numpy as np
import pytest
import torch

from tests.attend_util import attend64, check, tree_words

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


class Mirror:
    """A pool and its numpy mirror: tables and bytes."""

    def __init__(self, ctx, seed, rows, pages, slots, k_bytes, v_bytes=0, pad=0):
        import kvmem_b200 as K
        self.rng = np.random.default_rng(seed)
        self.pool = K.ResidencyPool(ctx, rows, pages, slots)
        self.cache, self.host = [], []
        for n in [k_bytes] + ([v_bytes] if v_bytes else []):
            h = self.rng.integers(0, 256, (rows, slots, n + pad), dtype=np.uint8)
            d = torch.from_numpy(h).to(DEV)
            self.host.append(h[:, :, :n].copy())
            self.cache.append(d[:, :, :n])
        self.layout = K.cache_layout(*self.cache)
        sets = [[np.sort(self.rng.permutation(pages)[:int(self.rng.integers(0, min(slots, pages) + 1))]) for _ in range(rows)]
                for _ in range(2)]
        for sel in sets:
            ids = np.zeros((rows, slots), np.int32)
            for r, x in enumerate(sel):
                ids[r, :len(x)] = x
            self.pool.plan(torch.from_numpy(ids).to(DEV),
                           torch.tensor([len(x) for x in sel], dtype=torch.int32, device=DEV))
        self.slot_of, self.page_of = [x.copy() for x in self.pool.read()]

    def verify(self):
        torch.cuda.synchronize()
        slot_of, page_of = self.pool.read()
        assert np.array_equal(slot_of, self.slot_of) and np.array_equal(page_of, self.page_of)
        for d, h in zip(self.cache, self.host):
            assert np.array_equal(d.cpu().numpy(), h)

    # the rules
    def fork(self, src, dst, end):
        for s, d in zip(src, dst):
            keep = (self.page_of[s] >= 0) & (self.page_of[s] < end)
            self.slot_of[d] = np.where(np.arange(self.slot_of.shape[1]) < end, self.slot_of[s], -1)
            self.page_of[d] = np.where(keep, self.page_of[s], -1)
            for h in self.host:
                h[d, keep] = h[s, keep]

    def free(self, rows, lists):
        for r, ids in zip(rows, lists):
            for p in ids:
                if 0 <= p < self.slot_of.shape[1] and self.slot_of[r, p] >= 0:
                    self.page_of[r, self.slot_of[r, p]] = -1
                    self.slot_of[r, p] = -1

    def compact(self, rows):
        used = []
        for r in rows:
            c = int((self.page_of[r] >= 0).sum())
            used.append(c)
            holes = [s for s in range(c) if self.page_of[r, s] < 0]
            movers = [s for s in range(c, len(self.page_of[r])) if self.page_of[r, s] >= 0]
            for s, d in zip(movers, holes):
                p = self.page_of[r, s]
                self.page_of[r, s], self.page_of[r, d], self.slot_of[r, p] = -1, p, d
                for h in self.host:
                    h[r, d] = h[r, s]
        return used

    def copy(self, items):
        """Returns whether (a source was absent, a slot was)."""
        absent = full = False
        before = self.slot_of.copy(), [h.copy() for h in self.host]
        for sr, sp, dr, dp in items:
            s = before[0][sr, sp]
            if s < 0:
                absent = True
                continue
            d = self.slot_of[dr, dp]
            if d < 0:
                free = np.flatnonzero(self.page_of[dr] < 0)
                if not len(free):
                    full = True
                    continue
                d = free[0]
                self.slot_of[dr, dp], self.page_of[dr, d] = d, dp
            for h, b in zip(self.host, before[1]):
                h[dr, d] = b[sr, s]
        return absent, full


SHAPES = [
    # rows, pages, slots, K bytes, V bytes, padding between slots
    (4, 9, 5, 16, 32, 0),
    (6, 300, 40, 278528 // 16, 147456 // 16, 0),
    (5, 50, 300, 16384, 0, 0),          # more slots than threads of a plan, one plane
    (3, 20, 7, 16384 * 3 + 48, 16, 16),  # ragged chunks, padded slots
    (4, 12, 6, 1001, 34, 0),            # sizes and addresses that no 16-byte copy takes
    (3, 8, 4, 100, 100, 4),
]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("ctas", [0, 1, 7])
def test_fork(ctx, shape, ctas):
    m = Mirror(ctx, 1, *shape)
    rows, pages = shape[0], shape[1]
    m.pool.fork(m.layout, [0], [2], page_end=pages // 2, ctas=ctas)
    m.fork([0], [2], pages // 2)
    m.verify()
    src, dst = ([1, 1], [0, 2]) if rows == 3 else ([2, 1, 2], [0, 3, rows - 1])
    if rows == 4:
        src, dst = [2, 2], [0, 3]
    m.pool.fork(m.layout, src, dst, ctas=ctas)
    m.fork(src, dst, pages)
    m.verify()
    m.pool.fork(m.layout, [dst[0]], [src[0]], page_end=0)
    m.fork([dst[0]], [src[0]], 0)
    m.verify()
    ctx.check_status()


@pytest.mark.parametrize("shape", SHAPES)
def test_free_and_compact(ctx, shape):
    m = Mirror(ctx, 2, *shape)
    rows, pages, slots = shape[:3]
    for turn in range(3):
        some = list(m.rng.permutation(rows)[:max(1, rows - turn)])
        width = 1 + slots // 2
        ids = m.rng.integers(0, pages, (len(some), width)).astype(np.int32)  # repeated and absent pages too
        counts = m.rng.integers(0, width + 1, len(some)).astype(np.int32)
        m.pool.free(some, torch.from_numpy(ids).to(DEV), torch.from_numpy(counts).to(DEV))
        m.free(some, [x[:n] for x, n in zip(ids, counts)])
        m.verify()
        used = torch.full((rows,), -7, dtype=torch.int32, device=DEV)
        m.pool.compact(m.layout, some, used=used)
        want = m.compact(some)
        m.verify()
        assert used.tolist() == want + [-7] * (rows - len(some))
    m.pool.compact(m.layout)
    m.compact(range(rows))
    m.verify()
    ctx.check_status()


@pytest.mark.parametrize("shape", SHAPES)
def test_copy(ctx, shape):
    import kvmem_b200 as K
    m = Mirror(ctx, 3, *shape)
    rows, pages = shape[:2]
    for n in (1, 5, 60):
        items, taken, sources = [], set(), set()
        for _ in range(n):
            s, d = (int(m.rng.integers(rows)), int(m.rng.integers(pages))), (int(m.rng.integers(rows)), int(m.rng.integers(pages)))
            if d not in taken and d not in sources and s not in taken and s != d:
                taken.add(d)
                sources.add(s)
                items.append(s + d)
        m.pool.copy_pages(m.layout, items)
        absent, full = m.copy(items)
        code = ctx.status()
        assert code in ([0] if not absent and not full else [K._abi.ERR_STALE] * absent + [K._abi.ERR_BUDGET_EXCEEDED] * full)
        m.verify()


def test_more_items_and_rows_than_a_launch_takes(ctx):
    m = Mirror(ctx, 4, 1500, 6, 3, 64, 32)
    full = int((m.page_of[:100] >= 0).sum(1).argmax())
    assert (m.page_of[full] >= 0).all()
    src, dst = [full] * 1400, list(range(100, 1500))
    m.pool.fork(m.layout, src, dst)
    m.fork(src, dst, 6)
    m.verify()
    m.pool.free(range(100, 1500), torch.full((1400, 1), int(m.page_of[full, 1]), dtype=torch.int32, device=DEV),
                torch.ones(1400, dtype=torch.int32, device=DEV))
    m.free(range(100, 1500), [[int(m.page_of[full, 1])]] * 1400)
    items = [(full, p, r, (p + 1) % 6) for r in range(100, 600) for p in range(6) if m.slot_of[full, p] >= 0]
    assert len(items) > 1024
    items = torch.tensor(items, dtype=torch.int32)[torch.from_numpy(m.rng.permutation(len(items)))].contiguous()
    m.pool.copy_pages(m.layout, items)
    m.copy([tuple(x) for x in items.tolist()])
    ctx.status()
    m.verify()
    ids = torch.from_numpy(m.rng.integers(0, 6, (1500, 2)).astype(np.int32))
    m.pool.free(range(1500), ids.to(DEV), torch.full((1500,), 2, dtype=torch.int32, device=DEV))
    m.free(range(1500), ids.numpy())
    m.pool.compact(m.layout)
    m.compact(range(1500))
    m.verify()
    ctx.check_status()


def test_restore_lists_of_changed_rows_are_dropped(ctx):
    """After a compaction a second stage-in must not write to the slots of the old plan."""
    import kvmem_b200 as K
    m = Mirror(ctx, 5, 2, 8, 4, 64)
    host = torch.zeros(2, 8, 64, dtype=torch.uint8).pin_memory()
    L = K.stage_layout([dict(host_base=host.data_ptr(), host_row_stride=512, host_page_stride=64,
                             dev_base=m.cache[0].data_ptr(), dev_row_stride=256, dev_slot_stride=64, bytes=64)])
    sel = torch.tensor([[1, 5, 7], [0, 2, 6]], dtype=torch.int32, device=DEV)
    n = torch.tensor([3, 3], dtype=torch.int32, device=DEV)
    m.pool.plan(sel, n, force_reload=True)
    m.pool.stage_in(L)
    m.slot_of, m.page_of = [x.copy() for x in m.pool.read()]
    m.host[0] = m.cache[0].cpu().numpy().copy()
    m.pool.free([0, 1], torch.tensor([[1], [0]], dtype=torch.int32, device=DEV), torch.tensor([1, 1], dtype=torch.int32, device=DEV))
    m.free([0, 1], [[1], [0]])
    m.pool.compact(m.layout)
    m.compact([0, 1])
    host.fill_(99)
    m.pool.stage_in(L)
    m.verify()


def test_captured_branch(ctx):
    """Fork, free and compact in one graph, replayed after the source row has changed."""
    m = Mirror(ctx, 6, 4, 30, 12, 4096, 1024)
    ids = torch.tensor([[0, 3, 6, 9, 12], [1, 4, 7, 10, 13]], dtype=torch.int32, device=DEV)
    counts = torch.tensor([5, 4], dtype=torch.int32, device=DEV)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        m.pool.fork(m.layout, [0, 1], [2, 3], page_end=25)
        m.pool.free([2, 3], ids, counts)
        m.pool.compact(m.layout, [2, 3])
    for _ in range(3):
        g.replay()
        m.fork([0, 1], [2, 3], 25)
        m.free([2, 3], [ids[0].tolist(), ids[1, :4].tolist()])
        m.compact([2, 3])
        m.verify()
        sel = torch.from_numpy(np.sort(m.rng.permutation(30)[:9])[None].repeat(4, 0).astype(np.int32)).to(DEV)
        m.pool.plan(sel.contiguous(), torch.tensor([9, 8, 7, 6], dtype=torch.int32, device=DEV))
        torch.cuda.synchronize()
        m.slot_of, m.page_of = [x.copy() for x in m.pool.read()]
    ctx.check_status()


def test_tables_alias_the_pool(ctx):
    m = Mirror(ctx, 7, 3, 10, 4, 64)
    a, b = m.pool.tables()
    assert a.shape == (3, 10) and np.array_equal(a.cpu().numpy(), m.slot_of) and np.array_equal(b.cpu().numpy(), m.page_of)
    m.pool.fork(m.layout, [0], [1])
    m.fork([0], [1], 10)
    assert np.array_equal(a.cpu().numpy(), m.slot_of)


def test_refusals(ctx):
    import kvmem_b200 as K
    A = K._abi
    m = Mirror(ctx, 8, 4, 10, 4, 64)

    def code(f, *a, **kw):
        with pytest.raises(K.KvmError) as e:
            f(*a, **kw)
        return e.value.code

    pool, L = m.pool, m.layout
    assert code(pool.fork, L, [0], [4]) == A.ERR_INVALID_ARGUMENT
    assert code(pool.fork, L, [4], [0]) == A.ERR_INVALID_ARGUMENT
    assert code(pool.fork, L, [0, 1], [2, 2]) == A.ERR_INVALID_ARGUMENT
    assert code(pool.fork, L, [0, 1], [1, 2]) == A.ERR_INVALID_ARGUMENT
    assert code(pool.fork, L, [1], [1]) == A.ERR_INVALID_ARGUMENT
    assert code(pool.copy_pages, L, [(0, 0, 1, 1), (0, 1, 1, 1)]) == A.ERR_INVALID_ARGUMENT
    assert code(pool.copy_pages, L, [(0, 0, 1, 1), (1, 1, 2, 2)]) == A.ERR_INVALID_ARGUMENT
    assert code(pool.copy_pages, L, [(0, 10, 1, 1)]) == A.ERR_INVALID_ARGUMENT
    assert code(pool.copy_pages, L, [(0, 0, 5, 1)]) == A.ERR_INVALID_ARGUMENT
    assert code(pool.compact, L, [0, 0]) == A.ERR_INVALID_ARGUMENT
    assert code(pool.compact, L, [7]) == A.ERR_INVALID_ARGUMENT
    one = torch.zeros((2, 1), dtype=torch.int32, device=DEV)
    assert code(pool.free, [0, 0], one, one[:, 0].contiguous()) == A.ERR_INVALID_ARGUMENT
    assert code(pool.free, [9], one, one[:, 0].contiguous()) == A.ERR_INVALID_ARGUMENT
    bad = K.cache_layout(m.cache[0])
    bad.dev_slot_stride[0] = 32
    assert code(pool.fork, bad, [0], [1]) == A.ERR_INVALID_ARGUMENT
    t = K.Transfer(pool, torch.zeros((4, 1), dtype=torch.int32, device=DEV), torch.zeros(4, dtype=torch.int32, device=DEV))
    for f in (lambda: pool.fork(L, [0], [1]), lambda: pool.compact(L), lambda: pool.copy_pages(L, [(0, 0, 1, 1)]),
              lambda: pool.free([0], one, one[:, 0].contiguous())):
        assert code(f) == A.ERR_PENDING
    t.abort()
    t.close()
    m.verify()
    # out of range on the device: left out and reported
    pool.free([0], torch.tensor([[10, -1]], dtype=torch.int32, device=DEV), torch.tensor([2], dtype=torch.int32, device=DEV))
    assert ctx.status() == A.ERR_INVALID_ARGUMENT
    pool.free([0], torch.tensor([[m.page_of[0].max()]], dtype=torch.int32, device=DEV), torch.tensor([3], dtype=torch.int32, device=DEV))
    assert ctx.status() == A.ERR_INVALID_ARGUMENT
    m.free([0], [[m.page_of[0].max()]])
    m.verify()


def test_a_lane_recalls_branches_drafts_and_goes_on(ctx):
    """Selection by scores, plan and stage-in from pinned records; a fork; attention of a drafted tree on both rows; the
    branch drops pages, compacts, takes one page from the other row; attention again; window attention over the same
    tail as a dense cache."""
    import kvmem_b200 as K
    rng = np.random.default_rng(9)
    gen = torch.Generator().manual_seed(9)
    hq, hkv, dim, page, pages, slots, N, recent = 8, 2, 128, 32, 24, 8, 11, 20
    tokens = pages * page - 13
    rec = [torch.randn(pages, page, hkv, dim, generator=gen).half().pin_memory() for _ in range(2)]
    cache = [torch.zeros(2, slots, page, hkv, dim, dtype=torch.float16, device=DEV) for _ in range(2)]
    size = page * hkv * dim * 2
    L = K.stage_layout([dict(host_base=r.data_ptr(), host_row_stride=0, host_page_stride=size, dev_base=c.data_ptr(),
                             dev_row_stride=slots * size, dev_slot_stride=size, bytes=size) for r, c in zip(rec, cache)])
    pool = K.ResidencyPool(ctx, 2, pages, slots)
    scores = torch.rand(2, pages, generator=gen).to(DEV)
    ids, n = ctx.select_topk(scores, [0, pages - 1], 7)
    n[1] = 0  # the second row starts empty
    pool.plan(ids, n)
    pool.stage_in(L)
    pool.fork(L, [0], [1])
    q = torch.randn(1, N, hq, dim, generator=gen).half()
    tail = [torch.randn(1, recent + N, hkv, dim, generator=gen).half() for _ in range(2)]
    see = np.zeros((N, N), bool)
    for i in range(N):
        if i:
            see[i] = see[int(rng.integers(0, i))]
        see[i, i] = True
    args = dict(layout=L, page_tokens=page, tokens=tokens, recent=recent, tree=tree_words(see).to(DEV), want_lse=True)
    qd, td = q.to(DEV), [t.to(DEV) for t in tail]

    def verify(out, lse, listed):
        planes = [torch.cat([r[p, :max(0, min(page, tokens - p * page))] for p in listed] + [t[0]]) for r, t in zip(rec, tail)]
        held = planes[0].shape[0] - N
        vis = torch.cat([torch.ones(N, held, dtype=torch.bool), torch.from_numpy(see)], 1)
        check(out[0], lse[0], attend64(q[0], planes[0], planes[1], vis, 1 / math.sqrt(dim)), torch.float16, held + N,
              float(planes[1].abs().max()))

    listed = ids[0, :int(n[0])].tolist()
    a = pool.tree_attention(qd, *td, sel_ids=ids[:1], sel_n=n[:1], **args)
    b = pool.tree_attention(qd, *td, row0=1, **args)
    ctx.check_status()
    verify(*a, listed)
    verify(*b, listed)
    drop = listed[1:4]
    pool.free([1], torch.tensor([drop], dtype=torch.int32, device=DEV), torch.tensor([3], dtype=torch.int32, device=DEV))
    used = torch.zeros(1, dtype=torch.int32, device=DEV)
    pool.compact(L, [1], used=used)
    pool.copy_pages(L, [(0, drop[0], 1, drop[0])])
    left = [p for p in listed if p not in drop[1:]]
    b = pool.tree_attention(qd, *td, row0=1, **args)
    ctx.check_status()
    verify(*b, left)
    assert int(used) == len(listed) - 3 and (pool.read()[1][1] >= 0).sum() == len(left)
    # The tail alone, as a chain in a dense cache with a window as long as it: the two entry points agree with each other.
    chain = K.tree_mask(list(range(-1, N - 1))).to(DEV)
    none = torch.zeros(1, dtype=torch.int32, device=DEV)
    x, xl = pool.tree_attention(qd, *td, sel_ids=ids[:1], sel_n=none, **{**args, "tree": chain})
    y, yl = ctx.window_attention(qd, *td, base=recent, window=1000, want_lse=True)
    ctx.check_status()
    assert torch.equal(x, y) and torch.equal(xl, yl)
