"""GPU: caches of more than 4 GiB per plane, read and copied at their far end."""
import math

import numpy as np
import pytest
import torch

from tests import util as U
from tests.attend_util import attend64, check
from tests.test_gpu_window import make

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
GIB4 = 1 << 32


@pytest.mark.parametrize("kernel,width", [("mma", 1), ("tc", 1), ("tc", 40)])
@pytest.mark.parametrize("layout", ["tokens", "heads"])
def test_window_at_the_end_of_a_large_cache(ctx, monkeypatch, kernel, width, layout):
    monkeypatch.setenv("KVM_ATTEND", kernel)
    hq, hkv, dim, cap, tail, sinks, window = 16, 8, 128, 2_200_000, 900, 5, 700
    q, k, v = make(91, 1, width, hq, hkv, dim, sinks + tail, torch.float16)
    shape = (1, cap, hkv, dim) if layout == "tokens" else (1, hkv, cap, dim)
    big = [torch.empty(shape, dtype=torch.float16, device=DEV) for _ in range(2)]
    assert big[0].numel() * 2 > GIB4
    if layout == "heads":
        big = [x.transpose(1, 2) for x in big]
    for b, x in zip(big, (k, v)):
        b[:, :sinks], b[:, cap - tail:] = x[:, :sinks].to(DEV), x[:, sinks:].to(DEV)
    out, lse = ctx.window_attention(q.to(DEV), *big, base=cap - width, window=window, sinks=sinks, want_lse=True)
    ctx.check_status()
    p = sinks + tail - width + torch.arange(width)[:, None]  # positions among the tokens that are there
    t = torch.arange(sinks + tail)[None]
    see = (t <= p) & ((t < sinks) | (p - t < window))
    exp = attend64(q[0], k[0], v[0], see, 1 / math.sqrt(dim))
    check(out[0], lse[0], exp, torch.float16, window + sinks, float(v.abs().max()))


@pytest.mark.parametrize("kernel", ["mma", "tc"])
@pytest.mark.parametrize("kinds", [None, (U.Q8_0, U.Q8_0)])
def test_tree_over_the_last_slots_of_a_large_pool(ctx, monkeypatch, kernel, kinds):
    import kvmem_b200 as K
    monkeypatch.setenv("KVM_ATTEND", kernel)
    rows, hq, hkv, dim, page, last, nodes, recent = 3, 16, 8, 256, 256, 5, 3, 20
    slots = 3000 if kinds else 1500
    rb = U.row_bytes(U.Q8_0, dim) if kinds else dim * 2
    cache = [torch.empty((rows, slots, page, hkv, rb), dtype=torch.uint8, device=DEV) for _ in range(2)]
    assert cache[0].numel() > GIB4
    rng = np.random.default_rng(92)
    gen = torch.Generator().manual_seed(92)
    n = last * page * hkv
    if kinds:
        enc = [U.make_quant_rows(rng, U.Q8_0, n, dim) for _ in range(2)]
        vals = [torch.from_numpy(U.decode_rows_f32(e, U.Q8_0, dim)) for e in enc]
        enc = [torch.from_numpy(e) for e in enc]
    else:
        vals = [torch.randn(n, dim, generator=gen).half() for _ in range(2)]
        enc = [v.view(torch.uint8) for v in vals]
    for c, e in zip(cache, enc):
        c[rows - 1, slots - last:] = e.reshape(last, page, hkv, rb).to(DEV)
    pool = K.ResidencyPool(ctx, rows, slots, slots)
    full = torch.arange(slots, dtype=torch.int32, device=DEV).expand(rows, slots).contiguous()
    pool.plan(full, torch.full((rows,), slots, dtype=torch.int32, device=DEV))
    slot_of, _ = pool.read()
    assert (slot_of[rows - 1] == np.arange(slots)).all()
    q = torch.randn(1, nodes, hq, dim, generator=gen).half()
    tail = [torch.randn(1, recent + nodes, hkv, dim, generator=gen).half() for _ in range(2)]
    ids = torch.arange(slots - last, slots, dtype=torch.int32, device=DEV)[None]
    types = dict(k_type=U.Q8_0, v_type=U.Q8_0) if kinds else {}
    out, lse = pool.tree_attention(q.to(DEV), *[x.to(DEV) for x in tail], layout=K.cache_layout(*cache), page_tokens=page,
                                   tokens=slots * page - 7, recent=recent, sel_ids=ids, row0=rows - 1,
                                   sel_n=torch.tensor([last], dtype=torch.int32, device=DEV), want_lse=True, **types)
    ctx.check_status()
    planes = [torch.cat([v.reshape(last * page, hkv, dim)[:last * page - 7].double(), t[0].double()]) for v, t in zip(vals, tail)]
    held = planes[0].shape[0] - nodes
    see = torch.cat([torch.ones(nodes, held, dtype=torch.bool), torch.ones(nodes, nodes).tril().bool()], 1)
    exp = attend64(q[0], planes[0], planes[1], see, 1 / math.sqrt(dim), decoded=bool(kinds) and kernel == "tc")
    check(out[0], lse[0], exp, torch.float16, held + nodes, float(planes[1].abs().max()))


@pytest.mark.parametrize("size", [1 << 20, (1 << 20) + 4])
def test_pages_at_the_end_of_a_large_pool(ctx, size):
    """Copied between rows, forked and compacted; 16-byte copies and plain ones."""
    import kvmem_b200 as K
    rows, slots = 3, 1400
    cache = torch.empty((rows, slots, size), dtype=torch.uint8, device=DEV)
    assert cache.numel() > GIB4
    pool = K.ResidencyPool(ctx, rows, 2 * slots, slots)
    L = K.cache_layout(cache)
    full = torch.arange(slots, dtype=torch.int32, device=DEV).expand(rows, slots).contiguous()
    pool.plan(full, torch.tensor([0, slots, slots], dtype=torch.int32, device=DEV))
    cache[1:, slots - 3:] = torch.randint(0, 256, (2, 3, size), dtype=torch.uint8, device=DEV)
    want = cache[1:, slots - 3:].clone()
    pool.copy_pages(L, [(1, slots - 1, 2, slots - 2), (1, slots - 2, 0, 7)])
    want[1, 1] = want[0, 2]
    assert torch.equal(cache[1:, slots - 3:], want) and torch.equal(cache[0, 0], want[0, 1])
    pool.fork(L, [2], [0])
    assert torch.equal(cache[0, slots - 3:], want[1])
    drop = torch.arange(0, slots - 2, dtype=torch.int32, device=DEV)[None].contiguous()
    pool.free([0], drop, torch.tensor([slots - 2], dtype=torch.int32, device=DEV))
    pool.compact(L, [0])
    assert torch.equal(cache[0, :2], want[1, 1:])
    slot_of, page_of = pool.read()
    assert page_of[0, 0] == slots - 2 and page_of[0, 1] == slots - 1 and (page_of[0, 2:] < 0).all()
    ctx.check_status()
