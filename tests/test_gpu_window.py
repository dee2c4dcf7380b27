"""GPU: kvm_window_attention (sliding window with sinks over a dense cache) against attention in 64 bits.

Bounds: tests/attend_util.py."""
import math

import pytest
import torch

from tests.attend_util import attend64, check

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
NAN = float("nan")


def make(seed, seqs, width, hq, hkv, dim, cap, dtype):
    g = torch.Generator().manual_seed(seed)
    q = torch.randn(seqs, width, hq, dim, generator=g) + 0.3
    k = torch.randn(seqs, cap, hkv, dim, generator=g) * torch.empty(dim).uniform_(0.5, 2, generator=g)
    v = torch.randn(seqs, cap, hkv, dim, generator=g)
    return [x.to(dtype) for x in (q, k, v)]


def visible(base, width, cap, window, sinks):
    p = base + torch.arange(width)[:, None]
    t = torch.arange(cap)[None]
    return (t <= p) & ((t < sinks) | (p - t < window))


def compare(q, k, v, out, lse, bases, window, sinks, rows=None, scale=None):
    dim = q.shape[3]
    for b in range(q.shape[0]):
        n = q.shape[1] if rows is None else rows[b]
        if n == 0:
            continue
        see = visible(bases[b], n, k.shape[1], window, sinks)
        exp = attend64(q[b, :n], k[b], v[b], see, scale or 1 / math.sqrt(dim))
        seen = see.any(0)
        vmax = float(v[b][seen].abs().max()) if seen.any() else 0.0
        check(out[b, :n], None if lse is None else lse[b, :n], exp, q.dtype, int(see.sum(1).max()), vmax)


CASES = [
    # seqs, width, hq, hkv, dim, bases, window, sinks, dtype
    (1, 1, 4, 1, 128, [0], 1, 0, torch.float16),              # one key
    (1, 1, 24, 4, 256, [700], 255, 4, torch.bfloat16),
    (3, 1, 40, 8, 128, [0, 63, 1000], 128, 65, torch.float16),  # ragged positions, sinks past a tile
    (2, 1, 7, 1, 256, [300, 511], 64, 0, torch.float16),        # no sinks, window of one tile
    (1, 2, 12, 2, 64, [129], 100, 3, torch.bfloat16),
    (2, 3, 16, 1, 128, [200, 77], 1000, 1, torch.float16),      # window past the start, 48 packed rows
    (1, 137, 6, 2, 64, [1003], 511, 3, torch.float16),
    (1, 100, 8, 8, 64, [0], 33, 0, torch.bfloat16),             # one head per KV head
    (1, 65, 24, 4, 256, [500], 70, 300, torch.float16),         # more sinks than window
    (1, 40, 4, 2, 128, [10], 0, 5, torch.float16),              # window 0: sinks only
    (1, 5, 4, 2, 128, [3], 0, 0, torch.bfloat16),               # nothing visible
    (1, 200, 2, 1, 128, [0], 10 ** 9, 0, torch.float16),        # plain causal attention
    (1, 70, 5, 1, 64, [900], 1, 64, torch.bfloat16),            # itself and the sinks
    (1, 33, 6, 1, 256, [2900], 2700, 130, torch.bfloat16),      # two dozen tiles
    (1, 300, 4, 1, 128, [2500], 2400, 1, torch.float16),
    (2, 129, 1, 1, 64, [3000, 1700], 2990, 0, torch.float16),
]


@pytest.mark.parametrize("case", CASES)
@pytest.mark.parametrize("splits", ["", "1", "3"])
@pytest.mark.parametrize("kernel", ["", "mma", "tc"])
def test_window(ctx, monkeypatch, case, splits, kernel):
    monkeypatch.setenv("KVM_ATTEND", kernel)
    seqs, width, hq, hkv, dim, bases, window, sinks, dtype = case
    if splits:
        monkeypatch.setenv("KVM_ATTEND_SPLITS", splits)
    q, k, v = make(1, seqs, width, hq, hkv, dim, max(bases) + width + 9, dtype)
    base = bases[0] if seqs == 1 else torch.tensor(bases, dtype=torch.int64, device=DEV)
    out, lse = ctx.window_attention(q.to(DEV), k.to(DEV), v.to(DEV), base=base, window=window, sinks=sinks, want_lse=True)
    ctx.check_status()
    compare(q, k, v, out, lse, bases, window, sinks)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim,hq,hkv,width", [(64, 12, 2, 19), (128, 16, 4, 1), (128, 8, 2, 40), (256, 6, 1, 3), (256, 24, 4, 30)])
@pytest.mark.parametrize("kernel", ["mma", "tc"])
def test_masked_garbage_does_not_reach_rows(ctx, monkeypatch, dtype, dim, hq, hkv, width, kernel):
    """NaN and infinities in keys that no row sees, and in keys that only some rows of a tile see."""
    monkeypatch.setenv("KVM_ATTEND", kernel)
    base, window, sinks, cap = 150, 40, 2, 260
    q, k, v = make(2, 1, width, hq, hkv, dim, cap, dtype)
    see = visible(base, width, cap, window, sinks)
    dead = ~see.any(0)
    k[0, dead], v[0, dead] = NAN, float("inf")
    some = see.any(0) & ~see.all(0)
    poisoned = [int(some.nonzero()[0]), int(some.nonzero()[-1])] if some.any() else []
    for t in poisoned:
        v[0, t, :, ::3], k[0, t, :, 1] = NAN, float("inf")
    out, lse = ctx.window_attention(q.to(DEV), k.to(DEV), v.to(DEV), base=base, window=window, sinks=sinks, want_lse=True)
    ctx.check_status()
    clean = ~see[:, poisoned].any(1) if poisoned else torch.ones(width, dtype=torch.bool)
    assert clean.any()
    kc, vc = k.clone(), v.clone()
    kc[0, dead], vc[0, dead] = 0, 0
    for t in poisoned:
        kc[0, t], vc[0, t] = 0, 0
    rows = clean.nonzero()[:, 0]
    exp = attend64(q[0, rows], kc[0], vc[0], see[rows], 1 / math.sqrt(dim))
    check(out[0, rows.to(DEV)], lse[0, rows.to(DEV)], exp, dtype, window + sinks, float(vc[0].abs().max()))
    # A row that sees the poisoned key says so, as the formula does.
    for t in poisoned:
        for i in see[:, t].nonzero()[:, 0].tolist():
            assert not torch.isfinite(out[0, i]).all()


def test_strides_rows_and_streams(ctx):
    """Head-major cache, heads before rows in q and out, unused rows left as they were, another stream, a given scale."""
    seqs, width, hq, hkv, dim, cap = 3, 6, 8, 2, 128, 400
    bases, rows = [20, 390, 7], [6, 0, 3]
    q, k, v = make(3, seqs, width, hq, hkv, dim, cap, torch.float16)
    qd = q.to(DEV).transpose(1, 2).contiguous().transpose(1, 2)
    kd = k.to(DEV).transpose(1, 2).contiguous().transpose(1, 2)
    vd = torch.zeros(seqs, cap, hkv, dim + 8, dtype=torch.float16, device=DEV)[..., :dim].copy_(v.to(DEV))
    out = torch.full((seqs, hq, width, dim), 7.0, dtype=torch.float16, device=DEV).transpose(1, 2)
    lse = torch.full((seqs, width, hq), 5.0, device=DEV)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    o, _ = ctx.window_attention(qd, kd, vd, base=torch.tensor(bases, device=DEV), window=50, sinks=3, scale=0.2, out=out,
                                lse=lse, rows=torch.tensor(rows, dtype=torch.int32, device=DEV), stream=s)
    s.synchronize()
    ctx.check_status(stream=s)
    assert o is out
    compare(q, k, v, out, lse, bases, 50, 3, rows=rows, scale=0.2)
    for b in range(seqs):
        assert (out[b, rows[b]:] == 7).all() and (lse[b, rows[b]:] == 5).all()


@pytest.mark.parametrize("splits", ["1", "4"])
def test_sequence_past_its_cache_is_left_out(ctx, monkeypatch, splits):
    import kvmem_b200 as K
    monkeypatch.setenv("KVM_ATTEND_SPLITS", splits)
    q, k, v = make(4, 2, 2, 4, 1, 64, 300, torch.float16)
    out = torch.full_like(q, 3.0).to(DEV)
    base = torch.tensor([299, 100], device=DEV)  # 299 + 2 rows > 300 tokens
    ctx.window_attention(q.to(DEV), k.to(DEV), v.to(DEV), base=base, window=64, sinks=1, out=out)
    assert ctx.status() == K._abi.ERR_LENGTH
    assert (out[0] == 3).all()
    compare(q[1:], k[1:], v[1:], out[1:], None, [100], 64, 1)


def test_graph_replay_follows_the_device_positions(ctx):
    q, k, v = make(5, 2, 1, 8, 2, 128, 2000, torch.bfloat16)
    qd, kd, vd = q.to(DEV), k.to(DEV), v.to(DEV)
    base = torch.tensor([5, 1500], device=DEV)
    out = torch.empty_like(qd)
    ctx.window_attention(qd, kd, vd, base=base, window=700, sinks=4, out=out)  # takes the scratch
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ctx.window_attention(qd, kd, vd, base=base, window=700, sinks=4, out=out)
    # A larger eager call grows the scratch; the captured one keeps its own.
    big = make(6, 8, 1, 40, 8, 128, 3000, torch.float16)
    ctx.window_attention(*[x.to(DEV) for x in big], base=2999, window=3000)
    for bases in ([5, 1500], [1999, 0], [700, 701]):
        base.copy_(torch.tensor(bases))
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        compare(q, k, v, out, None, bases, 700, 4)
    ctx.check_status()


def test_bound_workspace_bounds_the_chunks():
    import kvmem_b200 as K
    c = K.RecallContext(0)
    c.bind_workspace(torch.empty(40000, dtype=torch.uint8, device=DEV)[:39936])
    q, k, v = make(7, 1, 1, 8, 2, 128, 3000, torch.float16)
    out, lse = c.window_attention(q.to(DEV), k.to(DEV), v.to(DEV), base=2999, window=3000, want_lse=True)
    c.check_status()
    compare(q, k, v, out, lse, [2999], 3000, 0)
    c.close()


def test_results_do_not_change_between_runs(ctx):
    q, k, v = [x.to(DEV) for x in make(8, 2, 9, 8, 2, 128, 3000, torch.float16)]
    a, la = ctx.window_attention(q, k, v, base=2900, window=2000, sinks=64, want_lse=True)
    for _ in range(3):
        b, lb = ctx.window_attention(q, k, v, base=2900, window=2000, sinks=64, want_lse=True)
        assert torch.equal(a, b) and torch.equal(la, lb)


def test_refusals(ctx):
    import kvmem_b200 as K
    A = K._abi
    q, k, v = [x.to(DEV) for x in make(9, 1, 2, 4, 2, 64, 50, torch.float16)]

    def code(**kw):
        args = dict(q=q, k=k, v=v, base=10, window=8, sinks=0)
        args.update(kw)
        with pytest.raises(K.KvmError) as e:
            ctx.window_attention(args.pop("q"), args.pop("k"), args.pop("v"), **args)
        return e.value.code

    assert code(base=49) == A.ERR_LENGTH
    assert code(base=-1) == A.ERR_INVALID_ARGUMENT
    assert code(scale=-1.0) == A.ERR_INVALID_ARGUMENT
    assert code(scale=NAN) == A.ERR_INVALID_ARGUMENT
    assert code(k=k.bfloat16()) == A.ERR_INVALID_ARGUMENT
    assert code(q=q.float()) == A.ERR_INVALID_ARGUMENT
    assert code(q=q[:, :, :3]) == A.ERR_INVALID_ARGUMENT          # 3 query heads on 2 KV heads
    assert code(q=q.cpu()) == A.ERR_INVALID_ARGUMENT
    assert code(base=torch.tensor([1.0], device=DEV)) == A.ERR_INVALID_ARGUMENT
    d32 = [x[..., :32].contiguous() for x in (q, k, v)]
    assert code(q=d32[0], k=d32[1], v=d32[2]) == A.ERR_UNSUPPORTED
    odd = torch.empty(q.numel() + 1, dtype=q.dtype, device=DEV)[1:].view(q.shape)
    assert code(q=odd) == A.ERR_UNSUPPORTED                       # 2-byte aligned
    out, _ = ctx.window_attention(q[:, :0], k, v, base=0, window=8)
    assert out.shape[1] == 0
    ctx.check_status()


@pytest.mark.parametrize("bad", [dict(window=-1), dict(sinks=-1), dict(window=-(1 << 40))])
def test_negative_arguments_are_refused_as_the_librarys_errors(ctx, bad):
    import kvmem_b200 as K
    q, k, v = [x.to(DEV) for x in make(9, 1, 2, 4, 2, 64, 50, torch.float16)]
    with pytest.raises(K.KvmError) as e:
        ctx.window_attention(q, k, v, **{**dict(base=10, window=8, sinks=0), **bad})
    assert e.value.code == K._abi.ERR_INVALID_ARGUMENT
