"""GPU: quantised pages: garbage in what no row sees, the precision that the decoded form states, captured split calls.

Bounds of the decoded form (the tcgen05 kernel), for o = sum_t p_t v_t with A = sum_t p_t |v_t|, whatever the output's type:
the output's rounding u |o|; P and V rounded to fp16, 2^-11 A each (a bf16 tail's are finer); the second product summed in
32 bits by steps of 16, (T / 16 + 8) 2^-22 A; logits off by delta = ((D / 16 + 8) 2^-22 + 2^-11) max_t S_t with S_t = scale
sum_d |q_d k_td| (K rounded to fp16), twice delta A; P below fp16's smallest normal number 2^-25 each: T 2^-25 max|v|. Code times
scale is a multiple of 2^-24 and so exact below fp16's smallest normal number."""
import math

import numpy as np
import pytest
import torch

from tests import util as U
from tests.attend_util import UNIT, attend64
from tests.test_gpu_tree import Problem

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


def poison(p, seed=0):
    """Free slots, and the tokens of a page past the history, hold random codes under scales that are NaN or infinite."""
    rng = np.random.default_rng(seed)
    rows, slots = p.page_of.shape
    for r in range(rows):
        t = p.tokens[(r - p.row0) // p.step] if r >= p.row0 and (r - p.row0) % p.step == 0 else 0
        for s in range(slots):
            page = int(p.page_of[r, s])
            held = 0 if page < 0 else max(0, min(p.page, t - page * p.page))
            for plane, kind in zip(p.cache, p.kinds):
                bad = plane[r, s, held:]
                if not bad.numel():
                    continue
                junk = rng.integers(0, 256, tuple(bad.shape), dtype=np.uint8)
                block = 34 if kind == U.Q8_0 else 18
                scales = rng.choice(np.array([0x7E00, 0x7C00, 0xFC00, 0x7BFF], np.uint16), junk.shape[:-1] + (junk.shape[-1] // block,))
                junk = junk.reshape(junk.shape[:-1] + (-1, block))
                junk[..., 0], junk[..., 1] = scales & 255, scales >> 8
                bad.copy_(torch.from_numpy(junk.reshape(tuple(bad.shape))))


def planes_of(p, i, pages):
    r = p.row0 + i * p.step
    return [torch.cat([val[r, p.slot_of[r, x], :max(0, min(p.page, p.tokens[i] - int(x) * p.page))].double() for x in pages] +
                      [tail[i, :p.recent[i] + p.nodes].double()]) for val, tail in zip(p.vals, p.tail)]


def check_decoded(p, out, lse):
    for i in range(p.seqs):
        k, v = planes_of(p, i, p.lists[p.row0 + i * p.step])
        t = k.shape[0]
        see = torch.cat([torch.ones(p.nodes, t - p.nodes, dtype=torch.bool), torch.from_numpy(p.see[i])], 1)
        o, l64, size, delta = attend64(p.q[i], k, v, see, 1 / math.sqrt(p.dim))
        step = (p.dim / 16 + 8) * 2.0 ** -22
        delta = delta * (1 + 2.0 ** -11 / step)
        acc = (t / 16 + 8) * 2.0 ** -22
        tol = 1.1 * (UNIT[p.dtype] * o.abs() + (2.0 ** -10 + acc + 2 * delta[..., None]) * size) + t * 2.0 ** -25 * float(v.abs().max())
        worst = float(((out[i].double().cpu() - o).abs() / tol).max())
        assert worst <= 1.0, f"error {worst:.3g} of its bound"
        assert ((lse[i].double().cpu() - l64).abs() <= 1.1 * delta + 2.0 ** -20 + l64.abs() * 2.0 ** -22).all()


KINDS = [(U.Q8_0, U.Q4_0), (U.Q8_0, U.Q8_0), (U.Q4_0, U.Q8_0), (U.Q4_0, U.Q4_0)]


@pytest.mark.parametrize("kinds", KINDS)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("case", [
    # seqs, nodes, hq, hkv, dim, page, pages, slots, tokens, recent
    (1, 1, 24, 4, 256, 256, 9, 5, [2200], [100]),
    (2, 16, 24, 4, 256, 128, 6, 4, [768, 513], [7, 90]),
    (2, 5, 16, 8, 128, 48, 30, 11, [1440, 1000], [47, 0]),
    (1, 33, 12, 3, 64, 16, 40, 25, [601], [3]),
])
def test_the_decoded_form_is_as_precise_as_it_says(ctx, monkeypatch, kinds, dtype, case):
    monkeypatch.setenv("KVM_ATTEND", "tc")
    p = Problem(ctx, 81, *case, dtype, kinds=kinds)
    out, lse = p.call()
    ctx.check_status()
    check_decoded(p, out, lse)


@pytest.mark.parametrize("kinds", KINDS[:3])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("kernel,page", [("mma", 64), ("mma", 24), ("tc", 64), ("tc", 48), ("tc", 256)])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_garbage_that_no_row_sees(ctx, monkeypatch, kinds, dtype, kernel, page, dim):
    monkeypatch.setenv("KVM_ATTEND", kernel)
    p = Problem(ctx, 82, 2, 5, 8, 2, dim, page, 9, 6, [8 * page + 5, 6 * page + page // 2 + 1], [19, 0], dtype, kinds=kinds, garbage=True)
    poison(p)
    for lists in ("own", None):  # the listed pages; every resident one, with free slots between them
        out, lse = p.call(lists=lists)
        ctx.check_status()
        p.verify(out, lse, lists=lists, decoded=kernel == "tc")


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_a_captured_split_call_follows_its_arrays(ctx, monkeypatch, dtype, dim):
    monkeypatch.setenv("KVM_ATTEND_SPLITS", "3")
    p = Problem(ctx, 83, 2, 4, 12, 2, dim, 64, 30, 14, [1500, 900], [33, 250], dtype, kinds=(U.Q8_0, U.Q4_0))
    width = 14
    ids = torch.zeros((2, width), dtype=torch.int32, device=DEV)
    n = torch.zeros(2, dtype=torch.int32, device=DEV)
    tokens = torch.tensor(p.tokens, dtype=torch.int64, device=DEV)
    recent = torch.tensor(p.recent, dtype=torch.int32, device=DEV)
    q, out, lse = p.q.to(DEV), torch.empty_like(p.q, device=DEV), torch.empty(2, 4, 12, device=DEV)
    call = lambda: p.call(sel_ids=ids, sel_n=n, tokens=tokens, recent=recent, tree=None, out=out, lse=lse)  # noqa: E731
    call()  # takes the scratch
    torch.cuda.synchronize()
    args = dict(layout=p.layout, page_tokens=64, tokens=tokens, recent=recent, sel_ids=ids, sel_n=n, k_type=U.Q8_0, v_type=U.Q4_0,
                out=out, lse=lse)
    g = torch.cuda.CUDAGraph()
    before = ctx.launches
    with torch.cuda.graph(g):
        p.pool.tree_attention(q, *p.tail_d, **args)
    assert ctx.launches - before == 2
    chain = np.tril(np.ones((2, 4, 4), bool))
    first = list(p.tokens), list(p.recent)
    for step in range(3):
        lists = [p.lists[i][step:] for i in range(2)]
        p.tokens, p.recent = [x - 65 * step for x in first[0]], [x - 11 * step for x in first[1]]
        ids.zero_()
        for i, x in enumerate(lists):
            ids[i, :len(x)] = torch.from_numpy(x.astype(np.int32)).to(DEV)
        n.copy_(torch.tensor([len(x) for x in lists], dtype=torch.int32))
        tokens.copy_(torch.tensor(p.tokens))
        recent.copy_(torch.tensor(p.recent, dtype=torch.int32))
        out.fill_(7.0)
        g.replay()
        torch.cuda.synchronize()
        p.verify(out, lse, lists=lists, see=chain, decoded=True)
    ctx.check_status()
