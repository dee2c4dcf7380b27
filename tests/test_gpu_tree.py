"""GPU: kvm_tree_attention (a tree of drafted tokens over the pages of a residency pool) against attention in 64 bits.

Bounds: tests/attend_util.py."""
import math

import numpy as np
import pytest
import torch

from tests import util as U
from tests.attend_util import attend64, check, tree_words

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
NAN = float("nan")


def random_tree(rng, n):
    see = np.zeros((n, n), bool)
    for i in range(n):
        p = -1 if i == 0 else int(rng.integers(-1, i))
        if p >= 0:
            see[i] = see[p]
        see[i, i] = True
    return see


class Problem:
    """Pool rows row0, row0 + step, ...; their pages in permuted slots; a list of pages per sequence."""

    def __init__(self, ctx, seed, seqs, nodes, hq, hkv, dim, page, pages, slots, tokens, recent, dtype, kinds=None,
                 row0=0, step=1, garbage=False):
        import kvmem_b200 as K
        rng = np.random.default_rng(seed)
        g = torch.Generator().manual_seed(seed)
        self.dim, self.page, self.dtype, self.seqs, self.nodes = dim, page, dtype, seqs, nodes
        self.tokens, self.recent = tokens, recent
        rows = row0 + (seqs - 1) * step + 1
        self.kinds = kinds
        shape = (rows, slots, page, hkv)
        if kinds:
            enc = [U.make_quant_rows(rng, t, int(np.prod(shape)), dim).reshape(shape + (-1,)) for t in kinds]
            self.vals = [torch.from_numpy(U.decode_rows_f32(e, t, dim)) for e, t in zip(enc, kinds)]
            self.cache = [torch.from_numpy(e).to(DEV) for e in enc]
        else:
            self.vals = [torch.randn(*shape, dim, generator=g).to(dtype) for _ in range(2)]
            self.vals[0] = (self.vals[0].float() * torch.empty(dim).uniform_(0.5, 2, generator=g)).to(dtype)
            self.cache = [x.to(DEV) for x in self.vals]
        self.layout = K.cache_layout(*self.cache)
        self.pool = K.ResidencyPool(ctx, rows, pages, slots)
        self.row0, self.step = row0, step
        # Two selections: slots end up permuted.
        first = [np.sort(rng.permutation(pages)[:slots]) for _ in range(rows)]
        self.lists = [np.sort(rng.permutation(pages)[:int(rng.integers(1, slots + 1))]) for _ in range(rows)]
        for i in range(seqs):  # the last page of the history is listed: it may be partly filled
            n_pages = -(-tokens[i] // page)
            if 0 < n_pages <= pages and n_pages - 1 not in self.lists[row0 + i * step]:
                x = self.lists[row0 + i * step]
                x[-1] = n_pages - 1
                self.lists[row0 + i * step] = np.unique(x)
        for sel in (first, self.lists):
            ids = np.zeros((rows, slots), np.int32)
            for r, x in enumerate(sel):
                ids[r, :len(x)] = x
            self.pool.plan(torch.from_numpy(ids).to(DEV),
                           torch.tensor([len(x) for x in sel], dtype=torch.int32, device=DEV))
        self.slot_of, self.page_of = self.pool.read()
        if garbage and not kinds:  # unused slots and the unfilled end of pages hold NaN and infinities
            for r in range(rows):
                for s in range(slots):
                    p = self.page_of[r, s]
                    t = tokens[(r - row0) // step] if r >= row0 and (r - row0) % step == 0 else 0
                    held = 0 if p < 0 else max(0, min(page, t - int(p) * page))
                    self.cache[0][r, s, held:] = NAN
                    self.cache[1][r, s, held:] = float("inf")
        cap = max(recent) + nodes + 3
        self.q = (torch.randn(seqs, nodes, hq, dim, generator=g) + 0.2).to(dtype)
        self.tail = [torch.randn(seqs, cap, hkv, dim, generator=g).to(dtype) for _ in range(2)]
        self.tail_d = [x.to(DEV).clone() for x in self.tail]
        if garbage:
            for i in range(seqs):
                for x, bad in zip(self.tail_d, (float("inf"), NAN)):
                    x[i, recent[i] + nodes:] = bad
        self.see = np.stack([random_tree(rng, nodes) for _ in range(seqs)])

    def lists_d(self, lists=None):
        mine = lists or [self.lists[self.row0 + i * self.step] for i in range(self.seqs)]
        width = max(1, max(len(x) for x in mine))
        ids = np.full((len(mine), width), 0x7fffffff, np.int32)
        for r, x in enumerate(mine):
            ids[r, :len(x)] = x
        return torch.from_numpy(ids).to(DEV), torch.tensor([len(x) for x in mine], dtype=torch.int32, device=DEV)

    def call(self, lists="own", tree="own", **kw):
        a = dict(layout=self.layout, page_tokens=self.page, row0=self.row0, row_step=self.step, want_lse=True,
                 tokens=torch.tensor(self.tokens, dtype=torch.int64, device=DEV),
                 recent=torch.tensor(self.recent, dtype=torch.int32, device=DEV))
        if lists is not None:
            a["sel_ids"], a["sel_n"] = self.lists_d(None if lists == "own" else lists)
        if tree is not None:
            a["tree"] = tree_words(self.see).to(DEV) if isinstance(tree, str) else tree
        if self.kinds:
            a["k_type"], a["v_type"] = self.kinds
        a.update(kw)
        return self.pool.tree_attention(self.q.to(DEV), *self.tail_d, **a)

    def verify(self, out, lse, lists="own", see=None, rows=None, scale=None, decoded=None):
        see = self.see if see is None else see
        for i in range(self.seqs):
            r = self.row0 + i * self.step
            pages = self.lists[r] if lists == "own" else (self.page_of[r][self.page_of[r] >= 0] if lists is None else lists[i])
            n = self.nodes if rows is None else rows[i]
            if n == 0:
                continue
            planes = []
            for val, tail in zip(self.vals, self.tail):
                parts = [val[r, self.slot_of[r, p], :max(0, min(self.page, self.tokens[i] - int(p) * self.page))].double()
                         for p in pages if self.slot_of[r, p] >= 0]
                planes.append(torch.cat(parts + [tail[i, :self.recent[i] + n].double()]))
            held = planes[0].shape[0] - n
            vis = torch.cat([torch.ones(n, held, dtype=torch.bool), torch.from_numpy(see[i][:n, :n].copy())], 1)
            exp = attend64(self.q[i, :n], planes[0], planes[1], vis, scale or 1 / math.sqrt(self.dim),
                           decoded=bool(self.kinds) if decoded is None else decoded)
            vmax = float(planes[1].abs().max()) if planes[1].numel() else 0.0
            check(out[i, :n], None if lse is None else lse[i, :n], exp, self.dtype, held + n, vmax)


CASES = [
    # seqs, nodes, hq, hkv, dim, page, pages, slots, tokens, recent, dtype
    (1, 1, 24, 4, 256, 256, 9, 5, [2200], [100], torch.float16),
    (1, 1, 1, 1, 64, 16, 3, 1, [1], [0], torch.bfloat16),            # one token of history, one page
    (3, 1, 4, 1, 128, 64, 20, 7, [1280, 700, 65], [0, 63, 5], torch.float16),
    (2, 16, 24, 4, 256, 128, 6, 4, [768, 513], [7, 90], torch.bfloat16),
    (2, 5, 40, 8, 128, 48, 30, 11, [1440, 1000], [47, 0], torch.bfloat16),  # 48 divides no tile
    (1, 33, 12, 2, 64, 16, 40, 25, [601], [3], torch.float16),       # two words of tree
    (1, 64, 8, 8, 64, 32, 12, 12, [300], [31], torch.float16),       # every slot used
    (2, 60, 5, 1, 128, 128, 8, 5, [1000, 1], [66, 2], torch.bfloat16),
    (1, 3, 7, 1, 256, 1, 200, 130, [200], [0], torch.float16),       # pages of one token
    (1, 2, 2, 1, 64, 1000, 3, 2, [2500], [0], torch.float16),        # pages that are no multiple of a tile
    (1, 4, 4, 2, 128, 64, 4, 3, [0], [0], torch.float16),            # no history: the tree alone
]


@pytest.mark.parametrize("case", CASES)
@pytest.mark.parametrize("splits", ["", "1", "4"])
@pytest.mark.parametrize("kernel", ["", "mma", "tc"])
def test_tree(ctx, monkeypatch, case, splits, kernel):
    if kernel == "tc" and case[5] % 16:
        pytest.skip("the tcgen05 kernel takes pages of a multiple of 16 tokens")
    monkeypatch.setenv("KVM_ATTEND", kernel)
    if splits:
        monkeypatch.setenv("KVM_ATTEND_SPLITS", splits)
    p = Problem(ctx, 11, *case, garbage=True)
    out, lse = p.call()
    ctx.check_status()
    p.verify(out, lse)


@pytest.mark.parametrize("kinds", [(U.Q8_0, U.Q4_0), (U.Q8_0, U.Q8_0), (U.Q4_0, U.Q8_0), (U.Q4_0, U.Q4_0)])
@pytest.mark.parametrize("case", [
    (1, 1, 24, 4, 256, 256, 9, 5, [2200], [100], torch.float16),
    (2, 16, 24, 4, 256, 128, 6, 4, [768, 513], [7, 90], torch.bfloat16),
    (2, 5, 16, 8, 128, 48, 30, 11, [1440, 1000], [47, 0], torch.float16),
    (1, 33, 12, 3, 64, 16, 40, 25, [601], [3], torch.bfloat16),      # rows of 68 and 36 bytes
])
@pytest.mark.parametrize("splits", ["", "1", "3"])
@pytest.mark.parametrize("kernel", ["mma", "tc"])
def test_quantised_pages(ctx, monkeypatch, kinds, case, splits, kernel):
    if kernel == "tc" and case[5] % 16:
        pytest.skip("the tcgen05 kernel takes pages of a multiple of 16 tokens")
    monkeypatch.setenv("KVM_ATTEND", kernel)
    if splits:
        monkeypatch.setenv("KVM_ATTEND_SPLITS", splits)
    p = Problem(ctx, 12, *case, kinds=kinds)
    out, lse = p.call()
    ctx.check_status()
    p.verify(out, lse, decoded=kernel == "tc")


def test_quantised_holes_and_poisoned_nodes(ctx, monkeypatch):
    """All resident pages with free slots between them over many tiles, garbage behind the tail, NaN in a drafted node."""
    monkeypatch.setenv("KVM_ATTEND", "tc")
    monkeypatch.setenv("KVM_ATTEND_SPLITS", "1")
    p = Problem(ctx, 26, 1, 9, 16, 2, 128, 32, 90, 70, [89 * 32 + 3], [50], torch.bfloat16, kinds=(U.Q8_0, U.Q4_0), garbage=True)
    out, lse = p.call(lists=None)
    ctx.check_status()
    p.verify(out, lse, lists=None, decoded=True)
    j = 4
    for x in p.tail_d:
        x[0, 50 + j, :, ::7] = NAN
    out, lse = p.call(lists=None)
    for i in range(9):
        assert torch.isfinite(out[0, i]).all().item() == (not p.see[0][i, j])


@pytest.mark.parametrize("scale", [2.0 ** -60, 2.0 ** -20, 3.0e4, 2.0 ** 60])
def test_quantised_pages_take_queries_of_any_size(ctx, scale):
    """bf16 queries far outside fp16's range; the logit scale keeps the logits where they were."""
    p = Problem(ctx, 27, 1, 4, 8, 2, 128, 64, 12, 6, [700], [0], torch.bfloat16, kinds=(U.Q8_0, U.Q8_0))
    p.q = (p.q.float() * scale).to(torch.bfloat16)
    p.tail_d[0].zero_(), p.tail[0].zero_()
    out, lse = p.call(scale=0.09 / scale)
    ctx.check_status()
    p.verify(out, lse, scale=0.09 / scale, decoded=True)


@pytest.mark.parametrize("kinds", [None, (U.Q8_0, U.Q4_0)])
def test_every_resident_page_and_a_chain(ctx, kinds):
    """No list: all resident pages of the row; no tree: node i sees the nodes up to i. Rows 1, 3, 5 of the pool."""
    p = Problem(ctx, 13, 3, 7, 8, 2, 128, 32, 40, 20, [1280, 800, 100], [5, 0, 31], torch.float16, kinds=kinds, row0=1,
                step=2)
    out, lse = p.call(lists=None, tree=None)
    ctx.check_status()
    p.verify(out, lse, lists=None, see=np.tril(np.ones((3, 7, 7), bool)))


def test_one_tree_for_all_and_scalars(ctx):
    p = Problem(ctx, 14, 2, 9, 8, 2, 64, 64, 20, 6, [1000, 1000], [12, 12], torch.bfloat16)
    out, _ = p.call(tree=tree_words(p.see[0]).to(DEV), tokens=1000, recent=12, scale=0.3, want_lse=False)
    ctx.check_status()
    p.verify(out, None, see=np.stack([p.see[0], p.see[0]]), scale=0.3)


def test_rows_that_see_nothing(ctx):
    """No pages, no recent tokens, a mask without the node itself: 0 and -inf."""
    p = Problem(ctx, 15, 2, 4, 4, 1, 128, 64, 5, 3, [320, 320], [0, 0], torch.float16)
    p.see[0, 2] = False
    p.see[1, :] = False
    out, lse = p.call(lists=[[], []])
    ctx.check_status()
    p.verify(out, lse, lists=[[], []])
    assert (out[1] == 0).all() and torch.isinf(lse[1]).all() and (out[0, 2] == 0).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("kernel", ["mma", "tc"])
def test_a_poisoned_node_stays_with_those_that_see_it(ctx, monkeypatch, dtype, kernel):
    monkeypatch.setenv("KVM_ATTEND", kernel)
    p = Problem(ctx, 16, 1, 40, 6, 2, 64, 32, 10, 4, [300], [9], dtype)
    j = 17
    for x in p.tail_d + p.tail:
        x[0, 9 + j, :, ::5] = NAN
    out, lse = p.call()
    ctx.check_status()
    sees = p.see[0][:, j]
    for i in range(40):
        assert torch.isfinite(out[0, i]).all().item() == (not sees[i])
    keep = np.flatnonzero(~sees)
    p.tail[0][0, 9 + j] = p.tail[1][0, 9 + j] = 0
    r = p.row0
    planes = [torch.cat([v[r, p.slot_of[r, x], :max(0, min(32, 300 - int(x) * 32))].double() for x in p.lists[r]] +
                        [t[0, :49].double()]) for v, t in zip(p.vals, p.tail)]
    vis = torch.cat([torch.ones(40, planes[0].shape[0] - 40, dtype=torch.bool), torch.from_numpy(p.see[0])], 1)
    exp = attend64(p.q[0, keep], planes[0], planes[1], vis[keep], 0.125)
    check(out[0, torch.from_numpy(keep).to(DEV)], lse[0, torch.from_numpy(keep).to(DEV)], exp, dtype, planes[0].shape[0],
          float(planes[1].abs().max()))


def test_padded_batch_is_left_as_it_was(ctx):
    p = Problem(ctx, 17, 3, 6, 8, 2, 128, 64, 12, 5, [700, 300, 64], [3, 0, 9], torch.float16)
    rows = [2, 0, 6]
    out = torch.full((3, 6, 8, 128), 7.0, dtype=torch.float16, device=DEV)
    lse = torch.full((3, 6, 8), 5.0, device=DEV)
    for splits in (None, "3"):
        with pytest.MonkeyPatch.context() as m:
            if splits:
                m.setenv("KVM_ATTEND_SPLITS", splits)
            p.call(out=out, lse=lse, rows=torch.tensor(rows, dtype=torch.int32, device=DEV))
        ctx.check_status()
        p.verify(out, lse, rows=rows)
        for i in range(3):
            assert (out[i, rows[i]:] == 7).all() and (lse[i, rows[i]:] == 5).all()


def test_listed_twice_counts_twice(ctx):
    p = Problem(ctx, 18, 1, 1, 4, 1, 64, 16, 9, 5, [140], [0], torch.float16)
    x = int(p.lists[0][0])
    twice = [[x, x]]
    out, lse = p.call(lists=twice)
    ctx.check_status()
    p.verify(out, lse, lists=twice)


def test_bad_pages_are_left_out_and_reported(ctx):
    import kvmem_b200 as K
    A = K._abi
    p = Problem(ctx, 19, 1, 2, 4, 1, 64, 16, 30, 6, [480], [1], torch.float16)
    gone = int(np.flatnonzero(p.slot_of[0] < 0)[0])
    good = p.lists[0].tolist()
    out, lse = p.call(lists=[good + [gone]])
    assert ctx.status() == A.ERR_STALE
    p.verify(out, lse)
    out, lse = p.call(lists=[[30] + good + [-1]])
    assert ctx.status() == A.ERR_INVALID_ARGUMENT
    p.verify(out, lse)
    ids, n = p.lists_d()
    out, lse = p.call(sel_ids=ids, sel_n=n + 5)  # a count past the list's row
    assert ctx.status() == A.ERR_INVALID_ARGUMENT
    p.verify(out, lse)
    out = torch.full((1, 2, 4, 64), 3.0, dtype=torch.float16, device=DEV)
    p.call(out=out, recent=torch.tensor([1000], dtype=torch.int32, device=DEV))
    assert ctx.status() == A.ERR_LENGTH and (out == 3).all()


def test_a_v_scale_out_of_range_is_reported(ctx):
    import kvmem_b200 as K
    p = Problem(ctx, 20, 1, 1, 4, 1, 64, 16, 4, 3, [64], [0], torch.float16, kinds=(U.Q8_0, U.Q8_0))
    s = int(p.slot_of[0, p.lists[0][0]])
    p.cache[1][0, s, 0, 0, :2] = torch.tensor([0xFF, 0x7B], dtype=torch.uint8)  # 65504
    p.call()
    assert ctx.status() == K._abi.ERR_NONFINITE


@pytest.mark.parametrize("plane", [0, 1])
@pytest.mark.parametrize("value,err", [(65280.0, False), (65536.0, True), (-1e5, True), (float("inf"), False)])
def test_a_bf16_tail_beside_quantised_pages_keeps_to_the_range_of_fp16(ctx, plane, value, err):
    """65280 is bf16's last value below 65504; infinities are passed on as they are."""
    import kvmem_b200 as K
    p = Problem(ctx, 22, 1, 3, 4, 1, 128, 16, 4, 3, [64], [5], torch.bfloat16, kinds=(U.Q8_0, U.Q4_0))
    p.tail_d[plane][0, 2, 0, 7] = value
    p.call()
    assert ctx.status() == (K._abi.ERR_NONFINITE if err else 0)


@pytest.mark.parametrize("scale,err", [(511.0, False), (512.0, True)])
def test_a_k_scale_out_of_range_is_reported(ctx, scale, err):
    import kvmem_b200 as K
    p = Problem(ctx, 23, 1, 2, 4, 1, 64, 32, 4, 3, [128], [0], torch.bfloat16, kinds=(U.Q4_0, U.Q4_0))
    s = int(p.slot_of[0, p.lists[0][0]])
    p.cache[0][0, s, 0, 0, :2] = torch.tensor([scale], dtype=torch.float16).view(torch.uint8)
    p.call()
    assert ctx.status() == (K._abi.ERR_NONFINITE if err else 0)


def test_long_list_with_table_refills(ctx, monkeypatch):
    """Pages of 2 tokens, 1,500 of them: more entries than the kernel holds at a time."""
    monkeypatch.setenv("KVM_ATTEND_SPLITS", "1")
    p = Problem(ctx, 21, 1, 2, 4, 2, 64, 2, 1600, 1500, [3199], [5], torch.float16)
    p2 = [np.flatnonzero(p.slot_of[0] >= 0)]
    out, lse = p.call(lists=p2)
    ctx.check_status()
    p.verify(out, lse, lists=p2)


@pytest.mark.parametrize("dim,page,dtype", [(64, 16, torch.float16), (128, 64, torch.bfloat16), (256, 128, torch.float16)])
@pytest.mark.parametrize("kernel", ["mma", "tc"])
def test_many_tiles_in_one_chunk_with_holes(ctx, monkeypatch, dim, page, dtype, kernel):
    """Twenty and more key tiles in one chunk, some of them partly filled or absent in the middle, garbage in all that
    is not visible."""
    monkeypatch.setenv("KVM_ATTEND", kernel)
    monkeypatch.setenv("KVM_ATTEND_SPLITS", "1")
    slots = 2816 // page
    p = Problem(ctx, 25, 1, 5, 8, 2, dim, page, slots + 9, slots, [(slots + 8) * page + 3], [70], dtype, garbage=True)
    # all resident pages in slot order (free slots are holes), then a list with pages past the history in the middle
    out, lse = p.call(lists=None)
    ctx.check_status()
    p.verify(out, lse, lists=None)
    half = (slots // 2) * page + 5
    p.tokens = [half]
    for r, s in zip(*np.nonzero(p.page_of >= 0)):
        held = max(0, min(page, half - int(p.page_of[r, s]) * page))
        p.cache[0][r, s, held:], p.cache[1][r, s, held:] = NAN, float("inf")
    pages = p.lists[0][np.argsort(p.lists[0] % 3, kind="stable")]
    out, lse = p.call(lists=[pages])
    ctx.check_status()
    p.verify(out, lse, lists=[pages])


def test_per_head_rows_equal_a_shared_selection(ctx):
    """Pool rows per KV head (kv_heads = 1, one sequence per head), with q, tail and out as strided views."""
    import kvmem_b200 as K
    hkv, g, dim, page, slots = 4, 3, 128, 32, 5
    p = Problem(ctx, 22, hkv, 2, g, 1, dim, page, 9, slots, [280] * hkv, [4] * hkv, torch.float16)
    out, lse = p.call()
    ctx.check_status()
    p.verify(out, lse)
    # the same numbers through [1][nodes][hkv * g][dim] views
    q = p.q.to(DEV).permute(1, 0, 2, 3).reshape(2, hkv * g, dim)
    o = torch.empty_like(q)
    tails = [x.permute(1, 0, 2, 3).reshape(x.shape[1], hkv, dim) for x in p.tail_d]
    view = lambda x, heads: x.view(x.shape[0], hkv, heads, dim).permute(1, 0, 2, 3)  # noqa: E731
    ids, n = p.lists_d()
    p.pool.tree_attention(view(q, g), view(tails[0], 1), view(tails[1], 1), layout=p.layout, page_tokens=page, tokens=280,
                          recent=4, sel_ids=ids, sel_n=n, tree=tree_words(p.see).to(DEV), out=view(o, g))
    ctx.check_status()
    assert torch.equal(view(o, g), out)


def test_graph_replay_follows_the_selection(ctx):
    p = Problem(ctx, 23, 1, 3, 8, 2, 128, 64, 40, 12, [2500], [9], torch.bfloat16)
    ids, n = p.lists_d([p.lists[0].tolist()])
    full = torch.zeros((1, 12), dtype=torch.int32, device=DEV)
    full[:, :ids.shape[1]] = ids
    out, lse = p.call(sel_ids=full, sel_n=n)
    q = p.q.to(DEV)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        p.pool.tree_attention(q, *p.tail_d, layout=p.layout, page_tokens=64, tokens=2500, recent=9, sel_ids=full,
                              sel_n=n, out=out, lse=lse)
    for drop in (0, 1, len(p.lists[0]) - 1):
        left = p.lists[0][drop:]
        full.zero_()
        full[0, :len(left)] = torch.from_numpy(left.astype(np.int32))
        n.fill_(len(left))
        g.replay()
        torch.cuda.synchronize()
        p.verify(out, lse, lists=[left], see=np.tril(np.ones((1, 3, 3), bool)))
    ctx.check_status()


def test_refusals(ctx):
    import kvmem_b200 as K
    A = K._abi
    p = Problem(ctx, 24, 2, 3, 4, 2, 64, 16, 10, 4, [100, 90], [2, 2], torch.float16)

    def code(**kw):
        with pytest.raises(K.KvmError) as e:
            p.call(**kw)
        return e.value.code

    assert code(page_tokens=0) == A.ERR_INVALID_ARGUMENT
    assert code(page_tokens=17) == A.ERR_INVALID_ARGUMENT           # a page larger than its slot
    assert code(row0=1) == A.ERR_INVALID_ARGUMENT                   # rows 1, 2 of 2
    assert code(row_step=2) == A.ERR_INVALID_ARGUMENT
    assert code(k_type=A.Q5_0, v_type=A.Q5_0) == A.ERR_UNSUPPORTED
    assert code(k_type=A.BF16) == A.ERR_UNSUPPORTED
    assert code(recent=8) == A.ERR_LENGTH                           # 8 + 3 nodes in a tail of 8
    assert code(scale=-0.5) == A.ERR_INVALID_ARGUMENT
    assert code(layout=K.cache_layout(p.cache[0])) == A.ERR_INVALID_ARGUMENT
    assert code(tree=torch.zeros(2, 1, dtype=torch.int32, device=DEV)) == A.ERR_INVALID_ARGUMENT
    sel, n = p.lists_d()
    t = K.Transfer(p.pool, sel, n)
    assert code() == A.ERR_PENDING
    t.abort()
    t.close()
    ctx.check_status()


def test_a_long_list_of_small_pages_with_a_small_bound_workspace():
    """More page boxes than one key chunk of the tcgen05 kernel holds, and no room for a second chunk's rows."""
    import kvmem_b200 as K
    c = K.RecallContext(0)
    c.bind_workspace(torch.empty(1024, dtype=torch.uint8, device=DEV))
    p = Problem(c, 27, 1, 20, 2, 2, 64, 16, 700, 640, [11200], [5], torch.bfloat16)
    p2 = [np.flatnonzero(p.slot_of[0] >= 0)]
    out, lse = p.call(lists=p2)
    c.check_status()
    p.verify(out, lse, lists=p2)


def test_lists_of_another_type_and_negative_rows_are_refused(ctx):
    import kvmem_b200 as K
    p = Problem(ctx, 26, 2, 3, 4, 2, 64, 16, 10, 4, [100, 90], [2, 2], torch.float16)
    sel, n = p.lists_d()
    for kw in (dict(sel_ids=sel.float(), sel_n=n), dict(row0=-1), dict(row_step=1 << 32), dict(page_tokens=-16),
               dict(tree=torch.zeros(3, 1, device=DEV))):
        with pytest.raises(K.KvmError) as e:
            p.call(**kw)
        assert e.value.code == K._abi.ERR_INVALID_ARGUMENT, kw
    ctx.check_status()
