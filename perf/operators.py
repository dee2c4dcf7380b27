"""Cases, inputs and plain forms of the attention and page operators over the paged K/V cache.

Three groups, each named by a case's "op":

* ``tree``    attention of a tree of drafted tokens (one node: plain decode) over the pages that a residency pool
              holds, plus the row's tail (recent committed tokens, then the drafted ones);
* ``window``  attention with a sliding window and a few first tokens that stay visible, over a dense cache;
* ``fork``, ``branch``, ``copy``  pages of the pool: forking rows, a whole branch (fork, free, compact), copying pages
              between rows.

``own`` chooses between the framework's entry points and the plain forms below (elementary torch operations in 32
bits, rounded once at the end).
"""
import math

import numpy as np
import torch

own = False

DEV = "cuda"
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
BLOCK_BYTES = {"q8_0": 34, "q4_0": 18}
PLANES = {"f16": ("f16", "f16"), "bf16": ("bf16", "bf16"), "k8v4": ("q8_0", "q4_0"), "k8v8": ("q8_0", "q8_0")}


def listed():
    return [
        # One decode token, pages chosen per KV head (each head is a pool row of its own): 4 query heads per row.
        dict(name="tree decode, per-head pages", op="tree", rows=8, nodes=1, q_heads=4, kv_heads=1, dim=128,
             page=64, pages=256, listed=18, recent=37, dtype="f16", cache="f16", lse=False),
        # One decode token of the 27B-class shape over the 32 recalled pages and the two kept ones.
        dict(name="tree decode, recalled pages", op="tree", rows=1, nodes=1, q_heads=24, kv_heads=4, dim=256,
             page=256, pages=512, listed=34, recent=201, dtype="f16", cache="f16", lse=True),
        # 16 drafted tokens over a quantised history (q8_0 keys, q4_0 values), 64 recalled pages and two kept ones.
        dict(name="tree of 16, k8v4 pages", op="tree", rows=1, nodes=16, q_heads=24, kv_heads=4, dim=256, page=256,
             pages=1024, listed=66, recent=90, dtype="bf16", cache="k8v4", lse=False),
        # 8 lanes, each with a wide tree: the contraction outweighs the reading.
        dict(name="tree of 60, 8 lanes", op="tree", rows=8, nodes=60, q_heads=40, kv_heads=8, dim=128, page=128,
             pages=512, listed=26, recent=77, dtype="bf16", cache="bf16", lse=True),
        # One decode token of one conversation inside a short window.
        dict(name="window decode, one lane", op="window", seqs=1, width=1, q_heads=24, kv_heads=4, dim=256, base=36864,
             window=1023, sinks=4, dtype="bf16", lse=False),
        # One decode token of 8 lanes, ragged positions, a long window.
        dict(name="window decode, 8 lanes", op="window", seqs=8, width=1, q_heads=40, kv_heads=8, dim=128, base=65000,
             window=4096, sinks=128, dtype="f16", lse=True),
        # A 1,024-row prompt chunk far into a conversation.
        dict(name="window prompt chunk", op="window", seqs=1, width=1024, q_heads=24, kv_heads=4, dim=256, base=36864,
             window=4096, sinks=256, dtype="bf16", lse=True),
        # A whole prompt from its first token, odd length, narrow window.
        dict(name="window whole prompt", op="window", seqs=1, width=16381, q_heads=32, kv_heads=8, dim=128, base=0,
             window=1000, sinks=64, dtype="f16", lse=False),
        # A lane of a small model forked once: 4 layers, 18 resident pages each.
        dict(name="fork, 4 layers", op="fork", layers=4, lanes=2, pages=256, slots=18, resident=18, page_end=256,
             k_bytes=131072, v_bytes=131072),
        # One lane of the 27B-class shape forked into three branches (16 of its layers).
        dict(name="fork, 3 branches", op="fork", layers=16, lanes=4, pages=512, slots=34, resident=34, page_end=500,
             k_bytes=524288, v_bytes=524288),
        # A branch of a quantised lane: fork, drop the pages it will not use, close the holes.
        dict(name="branch, k8v4", op="branch", layers=16, lanes=2, pages=1024, slots=66, resident=63, page_end=1024,
             freed=31, k_bytes=278528, v_bytes=147456),
        # Pages that another lane holds already are copied on the device instead of staged from the host.
        dict(name="copy, pages between lanes", op="copy", layers=12, lanes=8, pages=512, slots=40, resident=24, items=333,
             k_bytes=262144, v_bytes=262144),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    heads = [(32, 8, 128), (24, 4, 256), (40, 8, 128), (8, 8, 64), (12, 2, 64), (16, 1, 128), (7, 1, 256)]
    op = rng.choice(["tree", "tree", "window", "window", "fork", "branch", "copy"])
    if op == "tree":
        hq, hkv, dim = rng.choice(heads)
        page = rng.choice([16, 32, 48, 64, 128, 256])
        cache = rng.choice(["f16", "bf16", "k8v4", "k8v8"])
        c = dict(op=op, rows=_log(rng, 1, 8), nodes=_log(rng, 1, 64), q_heads=hq, kv_heads=hkv, dim=dim, page=page,
                 listed=max(1, _log(rng, 64, 16384) // page), recent=rng.randrange(0, page),
                 dtype=cache if cache in DTYPES else rng.choice(["f16", "bf16"]), cache=cache, lse=rng.random() < 0.5)
        c["pages"] = c["listed"] + rng.randrange(1, 300)
        bound = work(dict(listed()[3], recent=0))
        while work(c)["bytes"] > bound["bytes"] or work(c)["flops"] > bound["flops"]:
            c["rows"], c["nodes"], c["listed"] = max(1, c["rows"] - 1), max(1, c["nodes"] * 3 // 4), max(1, c["listed"] * 3 // 4)
        return c
    if op == "window":
        hq, hkv, dim = rng.choice(heads)
        decode = rng.random() < 0.5
        c = dict(op=op, seqs=_log(rng, 1, 12) if decode else rng.choice([1, 1, 2, 3]),
                 width=rng.choice([1, 1, 2, 3, 5]) if decode else _log(rng, 17, 8192), q_heads=hq, kv_heads=hkv, dim=dim,
                 base=rng.choice([0, _log(rng, 1, 65536)]), window=_log(rng, 1, 8192),
                 sinks=rng.choice([0, 1, 4, _log(rng, 1, 512)]), dtype=rng.choice(["f16", "bf16"]), lse=rng.random() < 0.5)
        bound = work(listed()[7])
        while work(c)["bytes"] > bound["bytes"] or work(c)["flops"] > bound["flops"]:
            c["width"], c["window"] = max(1, c["width"] * 3 // 4), max(1, c["window"] * 3 // 4)
        return c
    slots = _log(rng, 3, 70)
    c = dict(op=op, layers=_log(rng, 1, 16), lanes=rng.choice([2, 2, 3, 4]), pages=slots + _log(rng, 1, 1000), slots=slots,
             k_bytes=16 * _log(rng, 128, 32768), v_bytes=16 * _log(rng, 128, 32768))
    c["resident"] = rng.randrange(max(1, slots // 2), slots + 1)
    if op == "copy":
        c["resident"] = max(1, slots // 2)
        c["items"] = _log(rng, 1, max(1, c["layers"] * (c["lanes"] - 1) * c["resident"] // 2))
    else:
        c["page_end"] = rng.choice([c["pages"], max(1, c["pages"] * 3 // 4)])
    if op == "branch":
        c["lanes"], c["freed"] = 2, rng.randrange(0, c["resident"] + 1)
    bound = work(listed()[9])["bytes"]
    while work(c)["bytes"] > bound:
        c["k_bytes"], c["v_bytes"] = 16 * (c["k_bytes"] // 24), 16 * (c["v_bytes"] // 24)
    return c


# ------------------------------------------------------------------ inputs


def _row_bytes(kind, dim):
    return 2 * dim if kind in DTYPES else dim // 32 * BLOCK_BYTES[kind]


def _plan(slot_of, page_of, sel):
    """A selection's residency, the pool's rule: pages that left free their slots, new pages (ascending) take the free
    slots (ascending)."""
    for r, want in enumerate(sel):
        keep = set(int(p) for p in want)
        for s in range(page_of.shape[1]):
            p = page_of[r, s]
            if p >= 0 and p not in keep:
                page_of[r, s], slot_of[r, p] = -1, -1
        new = sorted(p for p in keep if slot_of[r, p] < 0)
        for p, s in zip(new, np.flatnonzero(page_of[r] < 0)):
            page_of[r, s], slot_of[r, p] = p, s


def _tables(rng, rows, pages, slots, last):
    """Residency after two selections (the second one is `last`, a list of ascending page lists)."""
    slot_of, page_of = np.full((rows, pages), -1, np.int32), np.full((rows, slots), -1, np.int32)
    first = [np.sort(rng.permutation(pages)[:min(len(x), pages)]) for x in last]
    _plan(slot_of, page_of, first)
    _plan(slot_of, page_of, last)
    return first, slot_of, page_of


def _pool(state, first, last, pages, slots):
    """The framework's handle with the same residency."""
    import kvmem_b200 as K
    state["ctx"] = K.RecallContext(0)
    pool = K.ResidencyPool(state["ctx"], len(last), pages, slots)
    width = max(len(x) for x in last)
    for sel in (first, last):
        ids = np.zeros((len(sel), width), np.int32)
        for r, x in enumerate(sel):
            ids[r, :len(x)] = x
        pool.plan(torch.from_numpy(ids).to(DEV), torch.tensor([len(x) for x in sel], dtype=torch.int32, device=DEV))
    state["pool"] = pool
    state["layout"] = K.cache_layout(state["k"], state["v"])
    state["slot_of"], state["page_of"] = pool.tables()


def _quantised(g, kind, shape, dim):
    """GGUF blocks of 32: codes round(40 N(0, 1)) with scales U(0.005, 0.03), or 4-bit codes with scales U(0.02, 0.1)."""
    nb = dim // 32
    if kind == "q8_0":
        d = torch.empty(*shape, nb, 1, device=DEV).uniform_(0.005, 0.03, generator=g)
        codes = (torch.randn(*shape, nb, 32, device=DEV, generator=g) * 40).round().clamp(-127, 127).to(torch.int8)
    else:
        d = torch.empty(*shape, nb, 1, device=DEV).uniform_(0.02, 0.1, generator=g)
        codes = torch.randint(0, 256, (*shape, nb, 16), device=DEV, generator=g, dtype=torch.uint8)
    return torch.cat([d.half().view(torch.uint8).view(*shape, nb, 2), codes.view(torch.uint8)], -1).reshape(*shape, -1)


def _keys(g, shape, dim, dtype, towards):
    """Keys with uneven channels; every 16th token or so leans towards the queries' mean direction, as recalled ones do."""
    k = torch.randn(*shape, dim, device=DEV, generator=g) * torch.empty(dim, device=DEV).uniform_(0.5, 2, generator=g)
    near = (torch.rand(*shape, 1, device=DEV, generator=g) < 0.06).float() * 0.8
    return (k * (1 - near) + near * towards).to(dtype)


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    rng = np.random.default_rng(seed)
    if case["op"] == "tree":
        return _prepare_tree(case, g, rng)
    if case["op"] == "window":
        return _prepare_window(case, g)
    return _prepare_pages(case, g, rng)


def _prepare_tree(c, g, rng):
    R, N, Hq, Hkv, D, page, dt = c["rows"], c["nodes"], c["q_heads"], c["kv_heads"], c["dim"], c["page"], DTYPES[c["dtype"]]
    slots, pages, tail = c["listed"], c["pages"], c["recent"] + N
    s = dict(case=c)
    mean = torch.randn(R, Hkv, D, device=DEV, generator=g)
    s["q"] = (torch.randn(R, N, Hkv, Hq // Hkv, D, device=DEV, generator=g) + 0.5 * mean[:, None, :, None]).view(R, N, Hq, D).to(dt)
    planes = []
    for kind in PLANES[c["cache"]]:
        shape = (R, slots, page, Hkv)
        if kind in DTYPES:
            planes.append(_keys(g, shape, D, dt, mean[:, None, None]) if not planes else
                          torch.randn(*shape, D, device=DEV, generator=g).to(dt))
        else:
            planes.append(_quantised(g, kind, shape, D))
    s["k"], s["v"] = planes
    s["tail_k"] = _keys(g, (R, tail, Hkv), D, dt, mean[:, None])
    s["tail_v"] = torch.randn(R, tail, Hkv, D, device=DEV, generator=g).to(dt)
    # Histories of different lengths whose last page is partly filled; page 0 and the last page are always listed.
    tokens = np.array([(pages - int(x)) * page - int(y) for x, y in zip(rng.integers(0, max(1, pages - slots), R), rng.integers(0, page, R))])
    last = []
    for r in range(R):
        n_pages = -(-int(tokens[r]) // page)
        keep = [0, n_pages - 1][:slots]
        rest = rng.permutation(np.arange(1, n_pages - 1))[:slots - len(keep)]
        last.append(np.sort(np.concatenate([keep, rest]).astype(np.int64)))
    first, slot_of, page_of = _tables(rng, R, pages, slots, last)
    ids = np.zeros((R, slots), np.int32)
    for r, x in enumerate(last):
        ids[r, :len(x)] = x
    s["ids"], s["n"] = torch.from_numpy(ids).to(DEV), torch.tensor([len(x) for x in last], dtype=torch.int32, device=DEV)
    s["tokens"] = torch.from_numpy(tokens).to(DEV)
    # A tree per row: each node hangs on an earlier one.
    parents = np.array([[-1 if i == 0 else int(rng.integers(-1, i)) for i in range(N)] for _ in range(R)])
    see = np.zeros((R, N, N), bool)
    for i in range(N):
        for r in range(R):
            if parents[r, i] >= 0:
                see[r, i] = see[r, parents[r, i]]
            see[r, i, i] = True
    words = -(-N // 32)
    bits = np.zeros((R, N, words * 32), np.uint8)
    bits[:, :, :N] = see
    s["tree"] = torch.from_numpy(np.packbits(bits, axis=-1, bitorder="little").view(np.int32).reshape(R, N, words)).to(DEV)
    if own:
        _pool(s, first, last, pages, slots)
    else:
        s["slot_of"] = torch.from_numpy(slot_of).to(DEV)
    return s


def _prepare_window(c, g):
    B, W, Hq, Hkv, D, dt = c["seqs"], c["width"], c["q_heads"], c["kv_heads"], c["dim"], DTYPES[c["dtype"]]
    cap = c["base"] + W
    mean = torch.randn(B, Hkv, D, device=DEV, generator=g)
    q = torch.randn(B, W, Hkv, Hq // Hkv, D, device=DEV, generator=g) + 0.5 * mean[:, None, :, None]
    s = dict(case=c, q=q.view(B, W, Hq, D).to(dt), k=_keys(g, (B, cap, Hkv), D, dt, mean[:, None]),
             v=torch.randn(B, cap, Hkv, D, device=DEV, generator=g).to(dt))
    # Lanes stand at different positions, up to an eighth behind the longest.
    back = torch.randint(0, c["base"] // 8 + 1, (B,), device=DEV, generator=g)
    back[0] = 0
    s["base"] = c["base"] - back
    if own:
        import kvmem_b200 as K
        s["ctx"] = K.RecallContext(0)
    return s


def _prepare_pages(c, g, rng):
    L, lanes, slots, pages = c["layers"], c["lanes"], c["slots"], c["pages"]
    rows = L * lanes
    s = dict(case=c)
    for name in ("k", "v"):
        s[name] = torch.randint(-32768, 32767, (rows, slots, c[name + "_bytes"] // 2), dtype=torch.int16, device=DEV, generator=g)
    # Row of (layer, lane) = layer * lanes + lane. Lane 0 holds a full working set; for copies every lane holds some.
    last = [np.sort(rng.permutation(pages)[:c["resident"]]) for _ in range(rows)]
    first, slot_of, page_of = _tables(rng, rows, pages, slots, last)
    s["src"] = [l * lanes for l in range(L) for _ in range(1, lanes)]
    s["dst"] = [l * lanes + b for l in range(L) for b in range(1, lanes)]
    if c["op"] == "copy":
        pairs = [(l, b, p) for l in range(L) for b in range(1, lanes) for p in last[l * lanes]]
        pick = [pairs[i] for i in rng.permutation(len(pairs))]
        # As many new pages per row as it has room for.
        room, items = {}, []
        for l, b, p in pick:
            r = l * lanes + b
            new = slot_of[r, p] < 0
            if len(items) < c["items"] and (not new or room.get(r, slots - c["resident"]) > 0):
                room[r] = room.get(r, slots - c["resident"]) - int(new)
                items.append((l * lanes, int(p), r, int(p)))
        s["items"] = torch.tensor(items, dtype=torch.int32).reshape(-1, 4)
    if c["op"] == "branch":
        ids = np.zeros((L, max(1, c["freed"])), np.int32)
        for l in range(L):
            ids[l, :c["freed"]] = rng.permutation(last[l * lanes])[:c["freed"]]
        s["ids"] = torch.from_numpy(ids).to(DEV)
        s["n"] = torch.full((L,), c["freed"], dtype=torch.int32, device=DEV)
    if own:
        _pool(s, first, last, pages, slots)
    else:
        s["slot_of"], s["page_of"] = torch.from_numpy(slot_of).to(DEV), torch.from_numpy(page_of).to(DEV)
        s["src_d"], s["dst_d"] = torch.tensor(s["src"], device=DEV), torch.tensor(s["dst"], device=DEV)
        if "items" in s:
            s["items_d"] = s["items"].to(DEV).long()
    return s


# ------------------------------------------------------------------ one pass


def run(state):
    return RUN[state["case"]["op"]](state)


def _softmax(s, see, v, eq):
    """Softmax over the last axis of s where `see`, and its product with v; rows that see nothing give 0 and -inf."""
    s = s.masked_fill(~see, -math.inf)
    m = s.amax(-1, keepdim=True)
    m = torch.where(torch.isinf(m) & (m < 0), torch.zeros_like(m), m)
    p = torch.exp(s - m)
    total = p.sum(-1, keepdim=True)
    lse = (m + torch.log(total)).squeeze(-1)
    p = torch.where(total > 0, p / total, torch.zeros_like(p))
    return torch.einsum(eq, p, v), lse


def _values(x, kind, dim):
    """f32 values of cache rows."""
    if kind in DTYPES:
        return x.float()
    b = x.view(*x.shape[:-1], dim // 32, BLOCK_BYTES[kind])
    d = b[..., :2].contiguous().view(torch.float16).float()
    codes = b[..., 2:]
    if kind == "q8_0":
        codes = codes.contiguous().view(torch.int8).float()
    else:
        codes = torch.cat([codes & 15, codes >> 4], -1).float() - 8
    return (d * codes).reshape(*x.shape[:-1], dim)


def _run_tree(s):
    c = s["case"]
    if own:
        import kvmem_b200 as K
        kinds = {"f16": K.F16, "bf16": K.BF16, "q8_0": K.Q8_0, "q4_0": K.Q4_0}
        kk, vk = PLANES[c["cache"]]
        out, lse = s["pool"].tree_attention(s["q"], s["tail_k"], s["tail_v"], layout=s["layout"], page_tokens=c["page"],
                                            tokens=s["tokens"], recent=c["recent"], sel_ids=s["ids"], sel_n=s["n"],
                                            tree=s["tree"], k_type=kinds[kk], v_type=kinds[vk], want_lse=c["lse"])
        return (out, lse) if c["lse"] else out
    R, N, Hq, Hkv, D, page = c["rows"], c["nodes"], c["q_heads"], c["kv_heads"], c["dim"], c["page"]
    row = torch.arange(R, device=DEV)[:, None]
    slot = s["slot_of"].gather(1, s["ids"].long()).long().clamp_min(0)
    kk, vk = PLANES[c["cache"]]
    k = torch.cat([_values(s["k"][row, slot], kk, D).view(R, -1, Hkv, D), s["tail_k"].float()], 1)
    v = torch.cat([_values(s["v"][row, slot], vk, D).view(R, -1, Hkv, D), s["tail_v"].float()], 1)
    at = s["ids"].long()[:, :, None] * page + torch.arange(page, device=DEV)
    there = (at < s["tokens"][:, None, None]) & (torch.arange(c["listed"], device=DEV)[None, :, None] < s["n"][:, None, None])
    bits = (s["tree"][..., None] >> torch.arange(32, device=DEV, dtype=torch.int32)) & 1
    see = torch.cat([there.view(R, 1, -1).expand(R, N, -1), torch.ones(R, N, c["recent"], dtype=torch.bool, device=DEV),
                     bits.reshape(R, N, -1)[..., :N] > 0], -1)
    q = s["q"].float().view(R, N, Hkv, Hq // Hkv, D)
    scores = torch.einsum("rnhgd,rthd->rnhgt", q, k) / math.sqrt(D)
    out, lse = _softmax(scores, see[:, :, None, None], v, "rnhgt,rthd->rnhgd")
    out = out.reshape(R, N, Hq, D).to(s["q"].dtype)
    return (out, lse.reshape(R, N, Hq)) if c["lse"] else out


def _run_window(s):
    c = s["case"]
    if own:
        out, lse = s["ctx"].window_attention(s["q"], s["k"], s["v"], base=s["base"], window=c["window"], sinks=c["sinks"],
                                             want_lse=c["lse"])
        return (out, lse) if c["lse"] else out
    B, W, Hq, Hkv, D, window, sinks = (c[x] for x in ("seqs", "width", "q_heads", "kv_heads", "dim", "window", "sinks"))
    # Rows in blocks; each block's keys are its sinks and its own stretch of the cache.
    rows = min(W, 256)
    blocks = -(-W // rows)
    i = torch.arange(blocks * rows, device=DEV).view(blocks, rows)
    at = s["base"][:, None, None] + i                                                           # [B, blocks, rows]
    reach = min(window, c["base"] + W) + rows - 1
    near = at[:, :, :1] + (rows - 1) - torch.arange(reach, device=DEV)                           # [B, blocks, reach]
    few = min(sinks, c["base"] + W)
    key = torch.cat([torch.arange(few, device=DEV).expand(B, blocks, few), near], -1)            # [B, blocks, keys]
    a, t = at[..., None], key[:, :, None]
    first = torch.arange(few + reach, device=DEV) < few
    see = (t <= a) & (first | ((t >= few) & (a - t < window)))
    pick = key.clamp(0, s["k"].shape[1] - 1)
    b = torch.arange(B, device=DEV)[:, None, None]
    q = torch.nn.functional.pad(s["q"].float(), (0, 0, 0, 0, 0, blocks * rows - W)).view(B, blocks, rows, Hkv, Hq // Hkv, D)
    scores = torch.einsum("bcrhgd,bcthd->bchgrt", q, s["k"][b, pick].float()) / math.sqrt(D)
    out, lse = _softmax(scores, see[:, :, None, None], s["v"][b, pick].float(), "bchgrt,bcthd->bcrhgd")
    out = out.reshape(B, blocks * rows, Hq, D)[:, :W].to(s["q"].dtype)
    lse = lse.permute(0, 1, 4, 2, 3).reshape(B, blocks * rows, Hq)[:, :W]
    return (out, lse) if c["lse"] else out


def _fork(s, page_end):
    src, dst = s["src_d"], s["dst_d"]
    slot_of, page_of = s["slot_of"][src], s["page_of"][src]
    s["slot_of"][dst] = torch.where(torch.arange(slot_of.shape[1], device=DEV) < page_end, slot_of, -1)
    s["page_of"][dst] = torch.where(page_of < page_end, page_of, -1)
    moved = ((page_of >= 0) & (page_of < page_end))[:, :, None]
    s["k"][dst] = torch.where(moved, s["k"][src], s["k"][dst])
    s["v"][dst] = torch.where(moved, s["v"][src], s["v"][dst])


def _pages_out(s):
    return s["k"], s["v"], s["slot_of"], s["page_of"]


def _run_fork(s):
    c = s["case"]
    if own:
        s["pool"].fork(s["layout"], s["src"], s["dst"], page_end=c["page_end"])
    else:
        _fork(s, c["page_end"])
    return _pages_out(s)


def _run_branch(s):
    c = s["case"]
    if own:
        s["pool"].fork(s["layout"], s["src"], s["dst"], page_end=c["page_end"])
        s["pool"].free(s["dst"], s["ids"], s["n"])
        s["pool"].compact(s["layout"], s["dst"])
        return _pages_out(s)
    _fork(s, c["page_end"])
    dst = s["dst_d"]
    slot_of, page_of = s["slot_of"][dst], s["page_of"][dst]
    gone = torch.zeros_like(slot_of)
    listed_ = torch.arange(s["ids"].shape[1], device=DEV)[None] < s["n"][:, None]
    gone.scatter_add_(1, s["ids"].long(), listed_.int())
    slot_of = torch.where(gone > 0, -1, slot_of)
    page_of = torch.where((page_of >= 0) & (gone.gather(1, page_of.long().clamp_min(0)) > 0), -1, page_of)
    # The k-th resident slot behind the count goes to the k-th free slot before it.
    held, slot = page_of >= 0, torch.arange(page_of.shape[1], device=DEV).expand_as(page_of)
    count = held.sum(1, keepdim=True)
    hole, mover = ~held & (slot < count), held & (slot >= count)
    order = torch.argsort((~mover).int(), dim=1, stable=True)
    source = torch.where(hole, order.gather(1, (hole.cumsum(1) - 1).clamp_min(0)), slot)
    row = torch.arange(dst.numel(), device=DEV)[:, None]
    page_of = torch.where(mover, -1, page_of.gather(1, source))
    spread = torch.full((slot_of.shape[0], slot_of.shape[1] + 1), -1, dtype=torch.int32, device=DEV)
    spread.scatter_(1, torch.where(page_of >= 0, page_of, slot_of.shape[1]).long(), slot.int())
    s["slot_of"][dst], s["page_of"][dst] = spread[:, :-1], page_of
    s["k"][dst], s["v"][dst] = s["k"][dst][row, source], s["v"][dst][row, source]
    return _pages_out(s)


def _run_copy(s):
    if own:
        s["pool"].copy_pages(s["layout"], s["items"])
        return _pages_out(s)
    src_row, src_page, row, page = s["items_d"].unbind(1)
    src_slot, slot = s["slot_of"][src_row, src_page].long(), s["slot_of"][row, page].long()
    # New pages take their row's free slots in the order of the items.
    new = slot < 0
    mine = torch.nn.functional.one_hot(row, s["slot_of"].shape[0]) * new[:, None]
    rank = (mine.cumsum(0) * mine).sum(1) - 1
    free = torch.argsort((s["page_of"] >= 0).int(), dim=1, stable=True)
    slot = torch.where(new, free[row, rank.clamp_min(0)], slot)
    s["slot_of"][row, page], s["page_of"][row, slot] = slot.int(), page.int()
    s["k"][row, slot], s["v"][row, slot] = s["k"][src_row, src_slot], s["v"][src_row, src_slot]
    return _pages_out(s)


RUN = {"tree": _run_tree, "window": _run_window, "fork": _run_fork, "branch": _run_branch, "copy": _run_copy}


# ------------------------------------------------------------------ least work


def work(case):
    c = case
    if c["op"] == "tree":
        R, N, Hq, Hkv, D = c["rows"], c["nodes"], c["q_heads"], c["kv_heads"], c["dim"]
        kk, vk = PLANES[c["cache"]]
        held = c["listed"] * c["page"]
        read = R * Hkv * (held * (_row_bytes(kk, D) + _row_bytes(vk, D)) + (c["recent"] + N) * 4 * D)
        return {"bytes": read + R * N * Hq * (4 * D + (4 if c["lse"] else 0)),
                "flops": 4 * R * N * Hq * D * (held + c["recent"] + (N + 1) // 2)}
    if c["op"] == "window":
        B, W, Hq, Hkv, D = c["seqs"], c["width"], c["q_heads"], c["kv_heads"], c["dim"]
        pos = c["base"] + np.arange(W, dtype=np.int64)
        near = np.minimum(c["window"], pos + 1)
        far = np.minimum(c["sinks"], np.maximum(0, pos + 1 - near))
        keys = min(int(near[0]) + W - 1, c["base"] + W)
        keys += min(c["sinks"], max(0, c["base"] + W - keys))
        return {"bytes": B * (Hkv * keys * 4 * D + W * Hq * (4 * D + (4 if c["lse"] else 0))),
                "flops": 4 * B * Hq * D * int((near + far).sum())}
    size = c["k_bytes"] + c["v_bytes"]
    if c["op"] == "copy":
        return {"bytes": 2 * c["items"] * size, "flops": 0}
    held = c["layers"] * max(1, c["resident"] * min(c["page_end"], c["pages"]) // c["pages"])
    move = held * size * c["lanes"]
    if c["op"] == "branch":
        left = c["resident"] - c["freed"]
        # Of the pages left, those in slots behind the count move (spread evenly over the slots).
        move += 2 * c["layers"] * size * (left * (c["resident"] - left) // max(1, c["resident"]))
    return {"bytes": move, "flops": 0}


# ------------------------------------------------------------------ the definition in 64 bits


def exact(case, seed):
    """out and lse from the definition, row by row and head by head, in 64 bits. Pages are bytes: they have no such value."""
    c = case
    if c["op"] not in ("tree", "window"):
        return None
    global own
    was, own = own, False
    s = prepare(c, seed)
    own = was
    q = s["q"].double()
    group = c["q_heads"] // c["kv_heads"]
    out = torch.zeros(q.shape, dtype=torch.float64, device=DEV)
    lse = torch.full(q.shape[:-1], -math.inf, dtype=torch.float64, device=DEV)
    for r in range(q.shape[0]):
        if c["op"] == "tree":
            keys, values, seen = _tree_row(s, r)
        else:
            keys, values = s["k"][r].double(), s["v"][r].double()
        for lo in range(0, q.shape[1], 512):
            hi = min(q.shape[1], lo + 512)
            if c["op"] == "tree":
                k, v, see = keys, values, seen[lo:hi]
            else:
                pos = s["base"][r] + torch.arange(lo, hi, device=DEV)
                t = torch.arange(keys.shape[0], device=DEV)
                see = (t[None] <= pos[:, None]) & ((t[None] < c["sinks"]) | (pos[:, None] - t[None] < c["window"]))
                some = see.any(0).nonzero()[:, 0]
                k, v, see = keys[some], values[some], see[:, some]
            for h in range(c["q_heads"]):
                z = q[r, lo:hi, h] @ k[:, h // group].T * c["dim"] ** -0.5
                z[~see] = -math.inf
                lse[r, lo:hi, h] = torch.logsumexp(z, 1)
                part = torch.exp(z - lse[r, lo:hi, h, None]) @ v[:, h // group]
                out[r, lo:hi, h] = torch.where(see.any(1)[:, None], part, 0.0)
    return (out, lse) if c["lse"] else out


def _tree_row(s, r):
    """(K, V, visible) of one row, page by page."""
    c = s["case"]
    planes = []
    for name, kind in zip("kv", PLANES[c["cache"]]):
        parts = []
        for i in range(int(s["n"][r])):
            p = int(s["ids"][r, i])
            n = max(0, min(c["page"], int(s["tokens"][r]) - p * c["page"]))
            x = s[name][r, int(s["slot_of"][r, p])][:n]
            if kind == "q8_0":
                blocks = x.reshape(n, c["kv_heads"], -1, 34)
                x = blocks[..., :2].contiguous().view(torch.float16).double() * blocks[..., 2:].contiguous().view(torch.int8).double()
            elif kind == "q4_0":
                blocks = x.reshape(n, c["kv_heads"], -1, 18)
                low, high = (blocks[..., 2:] % 16).double(), (blocks[..., 2:] // 16).double()
                x = blocks[..., :2].contiguous().view(torch.float16).double() * (torch.cat([low, high], -1) - 8)
            parts.append(x.double().reshape(n, c["kv_heads"], c["dim"]))
        planes.append(torch.cat(parts + [s["tail_" + name][r].double()]))
    N, held = c["nodes"], planes[0].shape[0] - c["nodes"]
    see = torch.ones(N, held + N, dtype=torch.bool, device=DEV)
    words = s["tree"][r].cpu().numpy().view(np.uint32)
    for i in range(N):
        for j in range(N):
            see[i, held + j] = bool(words[i, j // 32] >> np.uint32(j % 32) & 1)
    return planes[0], planes[1], see
