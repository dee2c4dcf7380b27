"""Host-side API over the C ABI (``include/kvm_recall.h``).

Two layers:

* ``RecallContext`` / ``ResidencyPool`` — direct wrappers of the C entry
  points, taking device tensors (torch is used only to own device memory and
  streams) and returning device tensors;
* ``AttentionCuda``, ``PageSoftmaxCuda`` and ``pick_scored_blocks`` — mirrors
  of the reference's interfaces for this path, with the same argument meaning
  and error behaviour, so callers and tests read like the reference's own:
  ``llama_kvmem_attention_cuda::score`` (src/adapter/llama-kvmem-attention-cuda.h:9-18),
  ``kvmem::PageSoftmaxCuda`` (kvmem/include/kvmem/page_softmax_cuda.hpp:10-31) and
  ``KvMemStore::pick_scored_blocks`` (kvmem/src/host/kvmem_store.cpp:418-451).
"""
from __future__ import annotations

import contextlib
import ctypes as C
import struct
from dataclasses import dataclass
from typing import Optional, Sequence

import torch

from . import _abi as A

_ATTN_TYPES = {torch.float16: A.F16, torch.bfloat16: A.BF16}
_TORCH_QTYPE = {torch.float32: A.F32, torch.float16: A.F16, torch.bfloat16: A.BF16}


def _stream_ptr(stream) -> int:
    if stream is None:
        stream = torch.cuda.current_stream()
    return stream.cuda_stream


def _stream_on(device: int, stream) -> int:
    """The given stream, else the current stream of `device` (whichever device is current)."""
    return (stream if stream is not None else torch.cuda.current_stream(device)).cuda_stream


def _bad(where: str, what: str, code: int = A.ERR_INVALID_ARGUMENT) -> A.KvmError:
    return A.KvmError(code, f"{where}: {what}")


def _pack(where: str, form: struct.Struct, *values) -> bytes:
    try:
        return form.pack(*values)
    except struct.error as e:  # negative, or past 32 bits
        raise _bad(where, f"an argument is out of range ({e})") from None


def _u32s(where: str, values) -> None:
    """ctypes takes integers modulo 2^32; here they are refused."""
    if len(values) and (min(values) < 0 or max(values) > 0xFFFFFFFF):
        raise _bad(where, "an argument is out of range")


def _on_device(device: int, where: str, *tensors) -> None:
    for t in tensors:
        if t is not None and t.get_device() != device:
            raise _bad(where, f"a tensor is on {t.device}, the context on cuda:{device}")


def _seq_arg(x, device: int, n: int, where: str, dtype):
    """(scalar, device address) of a per-sequence argument: an int, or a tensor [n] of `dtype` on the device."""
    if isinstance(x, torch.Tensor):
        if x.dtype is not dtype or x.get_device() != device or x.dim() != 1 or len(x) < n or not x.is_contiguous():
            raise _bad(where, f"a per-sequence tensor is contiguous {dtype} [{n}] on cuda:{device}")
        return 0, x.data_ptr()
    if x < 0:
        raise _bad(where, "negative argument")
    return int(x), 0


# The attention calls' C structures, packed in one go (native alignment, as ctypes lays them out; a ctypes.Structure of
# as many fields takes several times as long to fill, and a decode step makes this call once per layer).
_ROWS = struct.Struct("@PQQQ")
_KCACHE = struct.Struct("@PiIQQQQ")
_WINDOW = struct.Struct("@3Ii4IQPPfI")
_TREE = struct.Struct("@3I3i6IQ5P2IPQfI")
assert [x.size for x in (_ROWS, _KCACHE, _WINDOW, _TREE)] == [C.sizeof(x) for x in (A.Rows, A.KCache, A.WindowDesc, A.TreeDesc)]


def _view4(t: torch.Tensor, shape, where: str):
    """(address, byte strides of sequence, row and head) of a 16-bit [sequence][row][head][dim] tensor (dim contiguous).
    The stride of a dimension of one element says nothing: it is taken as one row."""
    a, b, c, d = t.stride()
    n0, n1, n2, dim = shape
    if d != 1 and dim != 1:
        raise _bad(where, "the last dimension must be contiguous", A.ERR_UNSUPPORTED)
    return t.data_ptr(), 2 * (a if n0 > 1 else dim), 2 * (b if n1 > 1 else dim), 2 * (c if n2 > 1 else dim)


def _attention_args(where: str, device: int, q, k, v, out, lse, want_lse, stream):
    """Checks of an attention call and its tensors as C structures: (out, lse, its address, type, q shape, KV heads,
    q, k, v, out). Outputs that are not given are allocated for the stream of the call."""
    dtype = q.dtype
    t = _ATTN_TYPES.get(dtype)
    qs, ks = q.shape, k.shape
    if t is None or len(qs) != 4 or len(ks) != 4:
        raise _bad(where, "q, k, v are 4-D, q fp16 or bf16")
    if k.dtype is not dtype or v.dtype is not dtype or v.shape != ks or ks[0] != qs[0] or ks[3] != qs[3]:
        raise _bad(where, "k and v do not match q")
    if q.get_device() != device or k.get_device() != device or v.get_device() != device:
        raise _bad(where, f"q, k and v are on cuda:{device}")
    if out is None or (want_lse and lse is None):
        with torch.cuda.stream(stream) if stream is not None else contextlib.nullcontext():
            if out is None:
                out = q.new_empty(qs)
            if lse is None and want_lse:
                lse = q.new_empty(qs[:3], dtype=torch.float32)
    if out.shape != qs or out.dtype is not dtype or out.get_device() != device:
        raise _bad(where, "out does not match q")
    if lse is not None and (lse.shape != qs[:3] or lse.dtype is not torch.float32 or not lse.is_contiguous() or
                            lse.get_device() != device):
        raise _bad(where, "lse is contiguous float32 [seqs][rows][q_heads]")
    kp, k0, k1, k2 = _view4(k, ks, where)
    vp, v0, v1, v2 = _view4(v, ks, where)
    return (out, lse, None if lse is None else lse.data_ptr(), t, qs, ks[2], _ROWS.pack(*_view4(q, qs, where)),
            _KCACHE.pack(kp, t, 0, k0, k1, k2, ks[1]), _KCACHE.pack(vp, t, 0, v0, v1, v2, ks[1]),
            _ROWS.pack(*_view4(out, qs, where)))


class _DeviceTable:
    """Device memory of the library as __cuda_array_interface__ (int32)."""

    def __init__(self, ptr: int, shape: tuple, owner):
        self.owner = owner
        self.__cuda_array_interface__ = {"data": (ptr, False), "shape": shape, "typestr": "<i4", "version": 3}


def row_bytes(ktype: int, dim: int) -> int:
    return int(A.load().kvm_row_bytes(ktype, dim))


class RecallContext:
    """One kvm_ctx: device, status word, scoring workspace, stage-in stream."""

    def __init__(self, device: int = 0):
        self.lib = A.load()
        self.device = device
        h = C.c_void_p()
        A.check(self.lib.kvm_ctx_create(device, C.byref(h)), "kvm_ctx_create")
        self.h = h
        self._workspace: Optional[torch.Tensor] = None

    def close(self) -> None:
        if getattr(self, "h", None):
            self.lib.kvm_ctx_destroy(self.h)
            self.h = self._workspace = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    # -- status / workspace ------------------------------------------------
    def status(self, stream=None) -> int:
        return int(self.lib.kvm_ctx_status(self.h, _stream_ptr(stream)))

    def check_status(self, where: str = "device", stream=None) -> None:
        A.check(self.status(stream), where)

    @property
    def launches(self) -> int:
        return int(self.lib.kvm_ctx_launches(self.h))

    def bind_workspace(self, tensor: torch.Tensor) -> None:
        """The context's scratch from now on; held until another one is bound or the context is closed."""
        A.check(self.lib.kvm_ctx_bind_workspace(self.h, tensor.data_ptr(), tensor.numel() * tensor.element_size()),
                "kvm_ctx_bind_workspace")
        self._workspace = tensor

    def device_bytes(self) -> int:
        return int(self.lib.kvm_ctx_device_bytes(self.h))

    # -- descriptors -------------------------------------------------------
    @staticmethod
    def make_desc(*, layers, q_heads, kv_heads, head_dim, tokens, page_tokens, groups=1, scale=0.0, softcap=0.0,
                  mask: Optional[torch.Tensor] = None, mask_row_stride: int = 0) -> A.ScoreDesc:
        d = A.ScoreDesc()
        d.layers, d.q_heads, d.kv_heads, d.head_dim = layers, q_heads, kv_heads, head_dim
        d.tokens, d.page_tokens, d.groups = tokens, page_tokens, groups
        d.scale, d.softcap = scale, softcap
        if mask is not None:
            d.mask = mask.data_ptr()
            d.mask_type = _TORCH_QTYPE[mask.dtype]
            d.mask_row_stride = mask_row_stride or mask.stride(0) * mask.element_size()
        return d

    @staticmethod
    def make_query(q: torch.Tensor, rows: int, *, strides=None, data_ptr: Optional[int] = None,
                   row_ids: Optional[Sequence[int]] = None, row_count: int = 0) -> A.Query:
        """q dense [layers][rows][heads][dim] unless strides=(layer, row, head) bytes.
        row_ids: score only these rows of the tensor (the reference's sampled `rows`);
        `rows` is then len(row_ids) and row_count the rows the tensor holds."""
        qq = A.Query()
        qq.data = data_ptr if data_ptr is not None else q.data_ptr()
        qq.type = _TORCH_QTYPE[q.dtype]
        qq.rows = rows
        es = q.element_size()
        if strides is None:
            L, R, H, D = q.shape
            strides = (R * H * D * es, H * D * es, D * es)
        qq.layer_stride, qq.row_stride, qq.head_stride = strides
        if row_ids is not None:
            ids = (C.c_uint32 * max(1, len(row_ids)))(*row_ids)
            qq.row_ids = C.cast(ids, C.POINTER(C.c_uint32))
            qq._ids = ids  # keeps the host list alive with the descriptor
            qq.rows = len(row_ids)
            qq.row_count = row_count or (q.shape[1] if q.dim() == 4 else 0)
        return qq

    @staticmethod
    def make_kcache(k: torch.Tensor, ktype: int, *, kv_heads: int, head_dim: int, capacity_tokens: int,
                    layer_stride: Optional[int] = None, data_ptr: Optional[int] = None) -> A.KCache:
        """k: device bytes holding [layers][capacity_tokens][kv_heads] rows of ktype."""
        kc = A.KCache()
        kc.data = data_ptr if data_ptr is not None else k.data_ptr()
        kc.type = ktype
        rb = row_bytes(ktype, head_dim)
        kc.head_stride = rb
        kc.token_stride = rb * kv_heads
        kc.layer_stride = layer_stride if layer_stride is not None else rb * kv_heads * capacity_tokens
        kc.capacity_tokens = capacity_tokens
        return kc

    # -- entry points ------------------------------------------------------
    def score_pages(self, desc: A.ScoreDesc, q: A.Query, k: A.KCache, *, want_rows=True, want_mean=True,
                    out_rows: Optional[torch.Tensor] = None, out_mean: Optional[torch.Tensor] = None, stream=None):
        pages = -(-desc.tokens // desc.page_tokens)
        dev = torch.device("cuda", self.device)
        if want_rows and out_rows is None:
            out_rows = torch.empty((desc.layers, desc.groups, q.rows, pages), dtype=torch.float32, device=dev)
        if want_mean and out_mean is None:
            out_mean = torch.empty((desc.layers, desc.groups, pages), dtype=torch.float32, device=dev)
        rc = self.lib.kvm_score_pages(self.h, C.byref(desc), C.byref(q), C.byref(k),
                                      out_rows.data_ptr() if out_rows is not None else None,
                                      out_mean.data_ptr() if out_mean is not None else None, _stream_ptr(stream))
        A.check(rc, "kvm_score_pages")
        return out_rows, out_mean

    def prefill_attention(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, base: int,
                          sample_rows: Sequence[int] = (), page_tokens: int = 64, pages: Optional[int] = None,
                          scale: float = 0.0, out: Optional[torch.Tensor] = None,
                          page_lse: Optional[torch.Tensor] = None, stream=None):
        """Causal prompt attention with the page LSE of the sampled rows captured in the same pass
        (kvm_prefill_attention; the engine's causal_softmax_attention_with_page_lse).

        q: [width][q_heads][head_dim] fp16 / bf16 prompt rows at positions base .. base + width - 1;
        k, v: [capacity][kv_heads][head_dim] cache views holding keys 0 .. base + width - 1.
        Returns (out [width][q_heads][head_dim], page_lse [samples][q_heads][pages] or None)."""
        assert q.dim() == 3 and k.dim() == 3 and v.dim() == 3 and q.dtype == k.dtype == v.dtype
        width, hq, dim = q.shape
        cap, hkv, _ = k.shape
        t = _TORCH_QTYPE[q.dtype]
        d = A.PrefillDesc()
        d.q_heads, d.kv_heads, d.head_dim, d.type = hq, hkv, dim, t
        d.base, d.width, d.scale = base, width, scale
        rows = list(sample_rows)
        d.samples = len(rows)
        d.page_tokens = page_tokens
        d.pages = pages if pages is not None else -(-(base + width) // page_tokens)
        ids = (C.c_uint32 * max(1, len(rows)))(*rows)
        d.sample_rows = C.cast(ids, C.POINTER(C.c_uint32))
        if out is None:
            out = torch.empty_like(q)
        if rows and page_lse is None:
            page_lse = torch.empty((len(rows), hq, d.pages), dtype=torch.float32, device=q.device)
        es = q.element_size()

        def view(x: torch.Tensor) -> A.KCache:
            kc = A.KCache()
            kc.data, kc.type = x.data_ptr(), t
            kc.token_stride, kc.head_stride = x.stride(0) * es, x.stride(1) * es
            kc.layer_stride, kc.capacity_tokens = 0, x.shape[0]
            return kc

        kc, vc = view(k), view(v)
        rc = self.lib.kvm_prefill_attention(self.h, C.byref(d), q.data_ptr(), q.stride(0) * es, q.stride(1) * es,
                                            C.byref(kc), C.byref(vc), out.data_ptr(), out.stride(0) * es,
                                            out.stride(1) * es, page_lse.data_ptr() if rows else None,
                                            _stream_ptr(stream))
        A.check(rc, "kvm_prefill_attention")
        return out, (page_lse if rows else None)

    def window_attention(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, base, window: int, sinks: int = 0,
                         rows: Optional[torch.Tensor] = None, scale: float = 0.0, out: Optional[torch.Tensor] = None,
                         lse: Optional[torch.Tensor] = None, want_lse: bool = False, stream=None):
        """Attention with a sliding window and `sinks` first tokens that stay visible (kvm_window_attention).

        q: [seqs][width][q_heads][head_dim] (or [width][q_heads][head_dim]) fp16 / bf16, row i at position
        base + i; k, v: [seqs][capacity][kv_heads][head_dim] (or without seqs) views of the cache, any strides that
        are multiples of 16 bytes. base: int, or int64 tensor [seqs] on the device; rows: int32 tensor [seqs], the
        rows used per sequence (the others keep what `out` and `lse` hold).
        Returns (out like q, lse [seqs][width][q_heads] f32 or None)."""
        w, dev = "kvm_window_attention", self.device
        flat = q.dim() == 3
        if flat:
            q, k, v = q.unsqueeze(0), k.unsqueeze(0), v.unsqueeze(0)
            out = None if out is None else out.unsqueeze(0)
            lse = None if lse is None else lse.unsqueeze(0)
        out, lse, lse_p, t, (B, W, Hq, D), hkv, qq, kk, vv, oo = _attention_args(w, dev, q, k, v, out, lse, want_lse, stream)
        base, seq_base = _seq_arg(base, dev, B, w, torch.int64)
        seq_rows = 0 if rows is None else _seq_arg(rows, dev, B, w, torch.int32)[1]
        d = _pack(w, _WINDOW, Hq, hkv, D, t, B, W, min(window, 0xFFFFFFFF), min(sinks, 0xFFFFFFFF), base, seq_base,
                  seq_rows, scale, 0)
        rc = self.lib.kvm_window_attention(self.h, d, qq, kk, vv, oo, lse_p, _stream_on(dev, stream))
        if rc:
            A.check(rc, w)
        if flat:
            return out[0], (None if lse is None else lse[0])
        return out, lse

    def page_mass_from_lse(self, desc: A.ScoreDesc, rows: int, lse: torch.Tensor, *, want_rows=True,
                           want_mean=True, stream=None):
        """Whole-history page LSE [layers][rows][q_heads][pages] -> (mass_rows, mass_mean) as score_pages."""
        pages = -(-desc.tokens // desc.page_tokens)
        dev = lse.device
        out_rows = torch.empty((desc.layers, desc.groups, rows, pages), dtype=torch.float32, device=dev) \
            if want_rows else None
        out_mean = torch.empty((desc.layers, desc.groups, pages), dtype=torch.float32, device=dev) \
            if want_mean else None
        rc = self.lib.kvm_page_mass_from_lse(self.h, C.byref(desc), rows, lse.data_ptr(),
                                             out_rows.data_ptr() if out_rows is not None else None,
                                             out_mean.data_ptr() if out_mean is not None else None,
                                             _stream_ptr(stream))
        A.check(rc, "kvm_page_mass_from_lse")
        return out_rows, out_mean

    def select_topk(self, scores: torch.Tensor, keep: Sequence[int], budget: int, *, signed: bool = False,
                    out_ids: Optional[torch.Tensor] = None, out_n: Optional[torch.Tensor] = None, stream=None):
        """scores [nrows][pages] f32 on the device -> (ids [nrows][min(budget,pages)], n [nrows])."""
        assert scores.dtype == torch.float32 and scores.dim() == 2
        nrows, pages = scores.shape
        width = min(budget, pages)
        if out_ids is None:
            out_ids = torch.zeros((nrows, width), dtype=torch.int32, device=scores.device)
        if out_n is None:
            out_n = torch.zeros((nrows,), dtype=torch.int32, device=scores.device)
        kp = (C.c_uint32 * max(1, len(keep)))(*keep)
        rc = self.lib.kvm_select_topk(self.h, scores.data_ptr(), nrows, pages, scores.stride(0), kp, len(keep),
                                      budget, int(signed), out_ids.data_ptr(), out_n.data_ptr(), out_ids.stride(0),
                                      _stream_ptr(stream))
        A.check(rc, "kvm_select_topk")
        return out_ids, out_n

    def select_topk_media(self, scores: torch.Tensor, keep: Sequence[int], budget: int, *, block_tokens: int,
                          media_ranges: Sequence[tuple], signed: bool = False, stream=None):
        """select_topk with media groups (KvMemStore::pick_scored_blocks with the store's
        media ranges, token [begin, end) pairs; pages of block_tokens tokens)."""
        assert scores.dtype == torch.float32 and scores.dim() == 2
        nrows, pages = scores.shape
        width = min(budget, pages)
        out_ids = torch.zeros((nrows, width), dtype=torch.int32, device=scores.device)
        out_n = torch.zeros((nrows,), dtype=torch.int32, device=scores.device)
        kp = (C.c_uint32 * max(1, len(keep)))(*keep)
        flat = [int(x) for r in media_ranges for x in r]
        rg = (C.c_uint32 * max(1, len(flat)))(*flat)
        rc = self.lib.kvm_select_topk_media(self.h, scores.data_ptr(), nrows, pages, scores.stride(0), kp, len(keep),
                                            budget, int(signed), block_tokens, rg, len(media_ranges),
                                            out_ids.data_ptr(), out_n.data_ptr(), out_ids.stride(0),
                                            _stream_ptr(stream))
        A.check(rc, "kvm_select_topk_media")
        return out_ids, out_n

    def restore_k(self, ktype: int, items: Sequence[tuple], *, n_head: int, head_dim: int, n_rot: int = 0,
                  theta: Optional[Sequence[float]] = None, nrot: int = 0, stream=None) -> None:
        """items: (src_ptr, dst_ptr, tokens, pos0) -> kvm_restore_k (raw-K restore transform)."""
        arr = (A.RestoreItem * max(1, len(items)))()
        for i, (src, dst, tokens, pos0) in enumerate(items):
            arr[i].src, arr[i].dst, arr[i].tokens, arr[i].pos0 = src, dst, tokens, pos0
        th = (C.c_float * max(1, n_rot // 2))(*(list(theta or [])[: n_rot // 2]))
        rc = self.lib.kvm_restore_k(self.h, ktype, arr, len(items), n_head, head_dim, n_rot, th, nrot,
                                    _stream_ptr(stream))
        A.check(rc, "kvm_restore_k")

    @staticmethod
    def make_graph(graph: dict):
        """kvm_graph from dict(block, accepted, completed, rows=[(source, samples, [(target, mass), ...])],
        spans=None | [(begin, end, end_known)]); returns (struct, keepalive)."""
        rows = graph.get("rows", [])
        edges = [e for r in rows for e in r[2]]
        spans = graph.get("spans")
        ra = (A.GraphRow * max(1, len(rows)))()
        ea = (A.GraphEdge * max(1, len(edges)))()
        sa = (A.GraphSpan * max(1, len(spans or [])))()
        off = 0
        for i, (src, samples, es) in enumerate(rows):
            ra[i].source, ra[i].samples, ra[i].edge_begin, ra[i].edge_count = src, samples, off, len(es)
            off += len(es)
        for i, (tgt, mass) in enumerate(edges):
            ea[i].target, ea[i].mass = tgt, mass
        for i, (b, e, known) in enumerate(spans or []):
            sa[i].begin, sa[i].end, sa[i].end_known = b, e, int(bool(known))
        g = A.Graph()
        g.block_tokens, g.has_messages = graph["block"], int(spans is not None)
        g.accepted_through, g.completed_through = graph["accepted"], graph["completed"]
        g.rows, g.nrows, g.edges, g.nedges = ra, len(rows), ea, len(edges)
        g.spans, g.nspans = sa, len(spans or [])
        return g, (ra, ea, sa)

    def propagate_scores(self, raw: torch.Tensor, starts: Sequence[int], transport_mask: Sequence[int],
                         accepted: int, graph: dict, *, alpha: float = 0.2, cross: float = 0.25,
                         out: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
        """raw [n] f32 on the device -> propagated scores [n] f32 (kvm_propagate_scores)."""
        n = raw.numel()
        if out is None:
            out = torch.empty_like(raw)
        st = (C.c_uint64 * max(1, n))(*starts)
        tm = (C.c_uint8 * max(1, n))(*[1 if x else 0 for x in transport_mask])
        g, keep = self.make_graph(graph)
        rc = self.lib.kvm_propagate_scores(self.h, raw.data_ptr(), n, st, tm, accepted, C.byref(g), alpha, cross,
                                           out.data_ptr(), _stream_ptr(stream))
        A.check(rc, "kvm_propagate_scores")
        return out

    def lrfu_preview(self, scores: torch.Tensor, prev: Optional[torch.Tensor], *, lam: float = 0.5,
                     fraction: float = 0.9, out: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
        """scores [n] f32, prev [n_prev] f32 (committed history, device) -> candidate [n] f32."""
        n = scores.numel()
        if out is None:
            out = torch.empty_like(scores)
        n_prev = 0 if prev is None else prev.numel()
        rc = self.lib.kvm_lrfu_preview(self.h, scores.data_ptr(), n, prev.data_ptr() if n_prev else None, n_prev,
                                       lam, fraction, out.data_ptr(), _stream_ptr(stream))
        A.check(rc, "kvm_lrfu_preview")
        return out

    def meank_add(self, k: A.KCache, sums: torch.Tensor, counts: torch.Tensor, *, tok0: int, n: int,
                  page_tokens: int, kv_heads: int, head_dim: int, stream=None) -> None:
        """Adds tokens [tok0, tok0 + n) of every layer of `k` into the per-page sums
        [L][P][Hkv*D] f32 and their count into counts [P] (int32 tensor, read as u32)."""
        L, P, E = sums.shape
        if E != kv_heads * head_dim or counts.numel() < P:
            raise A.KvmError(A.ERR_INVALID_ARGUMENT, "meank_add: table shape")
        rc = self.lib.kvm_meank_add(self.h, C.byref(k), L, kv_heads, head_dim, tok0, n, page_tokens,
                                    sums.data_ptr(), P, counts.data_ptr(), _stream_ptr(stream))
        A.check(rc, "kvm_meank_add")

    def meank_score(self, sums: torch.Tensor, counts: torch.Tensor, q: torch.Tensor, layer_rows: Sequence[int],
                    score_mask: Sequence[int], *, q_heads: int, kv_heads: int, head_dim: int, aggregation: int = 0,
                    scale: float = 0.0, out: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
        """sums [L][P][Hkv*D] f32, counts [P] u32 (int32 tensor), q [L][R][Hq*D] f32 -> out [P] f32."""
        L, P, _ = sums.shape
        R = q.shape[1]
        if out is None:
            out = torch.empty((P,), dtype=torch.float32, device=sums.device)
        lr = (C.c_uint32 * L)(*layer_rows)
        sm = (C.c_uint8 * P)(*[1 if x else 0 for x in score_mask])
        rc = self.lib.kvm_meank_score(self.h, sums.data_ptr(), counts.data_ptr(), q.data_ptr(), lr, L, R, q_heads,
                                      kv_heads, head_dim, P, sm, aggregation, scale, out.data_ptr(),
                                      _stream_ptr(stream))
        A.check(rc, "kvm_meank_score")
        return out

    def layerwise_accumulate(self, tile: torch.Tensor, score_mask: torch.Tensor, accum: torch.Tensor, *,
                             halves: int = 1, keep_halves: bool = False, stream=None) -> None:
        """kvm_layerwise_accumulate: tile f32 [pages * halves], score_mask u8 [pages],
        accum f64 [pages * (2 if keep_halves else 1)] (all device)."""
        pages = score_mask.numel()
        A.check(self.lib.kvm_layerwise_accumulate(self.h, tile.data_ptr(), pages, halves, int(keep_halves),
                                                  score_mask.data_ptr(), accum.data_ptr(), _stream_ptr(stream)),
                "kvm_layerwise_accumulate")

    def layerwise_finish(self, accum: torch.Tensor, pages: int, *, keep_halves: bool = False,
                         out: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
        """kvm_layerwise_finish -> scores f32 [pages] (device)."""
        if out is None:
            out = torch.empty((pages,), dtype=torch.float32, device=accum.device)
        A.check(self.lib.kvm_layerwise_finish(self.h, accum.data_ptr(), pages, int(keep_halves), out.data_ptr(),
                                              _stream_ptr(stream)), "kvm_layerwise_finish")
        return out

    def stagein_copies(self, ops: Sequence[tuple], ctas: int = 0, stream=None) -> None:
        arr = (A.Copy * max(1, len(ops)))()
        for i, (src, dst, nbytes) in enumerate(ops):
            arr[i].src, arr[i].dst, arr[i].bytes = src, dst, nbytes
        A.check(self.lib.kvm_stagein_copies(self.h, arr, len(ops), ctas, _stream_ptr(stream)), "kvm_stagein_copies")

    def wait(self, timeout_s: float = 30.0, stream=None) -> None:
        A.check(self.lib.kvm_stagein_wait(self.h, _stream_ptr(stream), int(timeout_s * 1e6)), "kvm_stagein_wait")

    def recall_step(self, desc: A.ScoreDesc, q: A.Query, k: A.KCache, keep: Sequence[int], budget: int, *,
                    mass_mean: torch.Tensor, sel_ids: torch.Tensor, sel_n: torch.Tensor,
                    pool: Optional["ResidencyPool"] = None, layout: Optional[A.StageLayout] = None,
                    chunks: int = 0, stage_ctas: int = 0, force_reload: bool = False, first_layers: int = 0,
                    stream=None) -> None:
        st = A.StepDesc()
        st.score = C.pointer(desc)
        st.q = C.pointer(q)
        st.k = C.pointer(k)
        kp = (C.c_uint32 * max(1, len(keep)))(*keep)
        st.keep = C.cast(kp, C.POINTER(C.c_uint32))
        st.nkeep, st.budget, st.chunks, st.stage_ctas = len(keep), budget, chunks, stage_ctas
        st.force_reload = int(force_reload)
        st.first_layers = first_layers
        rc = self.lib.kvm_recall_step(self.h, C.byref(st), pool.h if pool is not None else None,
                                      C.byref(layout) if layout is not None else None, mass_mean.data_ptr(),
                                      sel_ids.data_ptr(), sel_n.data_ptr(), _stream_ptr(stream))
        A.check(rc, "kvm_recall_step")


class ResidencyPool:
    """Device residency table (kvm_pool) for `rows` selections over `pages` pages and `slots` slots."""

    def __init__(self, ctx: RecallContext, rows: int, pages: int, slots: int):
        self.ctx, self.rows, self.pages, self.slots = ctx, rows, pages, slots
        h = C.c_void_p()
        A.check(ctx.lib.kvm_pool_create(ctx.h, rows, pages, slots, C.byref(h)), "kvm_pool_create")
        self.h = h

    def close(self) -> None:
        if getattr(self, "h", None):
            self.ctx.lib.kvm_pool_destroy(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def reset(self, stream=None) -> None:
        A.check(self.ctx.lib.kvm_pool_reset(self.h, _stream_ptr(stream)), "kvm_pool_reset")

    def plan(self, sel_ids: torch.Tensor, sel_n: torch.Tensor, *, force_reload=False, stream=None):
        n_restore = torch.zeros((self.rows,), dtype=torch.int32, device=sel_ids.device)
        n_evict = torch.zeros((self.rows,), dtype=torch.int32, device=sel_ids.device)
        rc = self.ctx.lib.kvm_plan_residency(self.ctx.h, self.h, sel_ids.data_ptr(), sel_n.data_ptr(),
                                             sel_ids.stride(0), int(force_reload), n_restore.data_ptr(),
                                             n_evict.data_ptr(), _stream_ptr(stream))
        A.check(rc, "kvm_plan_residency")
        return n_restore, n_evict

    def stage_in(self, layout: A.StageLayout, ctas: int = 0, stream=None) -> None:
        A.check(self.ctx.lib.kvm_stagein_pool(self.ctx.h, self.h, C.byref(layout), ctas, _stream_ptr(stream)),
                "kvm_stagein_pool")

    def stage_in_range(self, layout: A.StageLayout, page0: int, page_count: int, ctas: int = 0,
                       stream=None) -> None:
        """kvm_shard_stagein: the planned restores of pages [page0, page0 + page_count) from
        this rank's records (layout.host_base starts at page0) into layout.dev_base, which
        may be a peer mapping of the decode GPU's cache (ipc_open)."""
        A.check(self.ctx.lib.kvm_shard_stagein(self.ctx.h, self.h, C.byref(layout), page0, page_count, ctas,
                                               _stream_ptr(stream)), "kvm_shard_stagein")

    def read(self, stream=None):
        import numpy as np
        slot_of = np.empty((self.rows, self.pages), np.int32)
        page_of = np.empty((self.rows, self.slots), np.int32)
        rc = self.ctx.lib.kvm_pool_read(self.h, slot_of.ctypes.data, page_of.ctypes.data, _stream_ptr(stream))
        A.check(rc, "kvm_pool_read")
        return slot_of, page_of


    # -- attention over the resident pages ---------------------------------
    def tree_attention(self, q: torch.Tensor, tail_k: torch.Tensor, tail_v: torch.Tensor, *, layout: A.StageLayout,
                       page_tokens: int, tokens, recent=0, sel_ids: Optional[torch.Tensor] = None,
                       sel_n: Optional[torch.Tensor] = None, tree: Optional[torch.Tensor] = None,
                       rows: Optional[torch.Tensor] = None, row0: int = 0, row_step: int = 1,
                       k_type: Optional[int] = None, v_type: Optional[int] = None, scale: float = 0.0,
                       out: Optional[torch.Tensor] = None, lse: Optional[torch.Tensor] = None, want_lse: bool = False,
                       stream=None):
        """Attention of drafted tokens (one per sequence: plain decode) over this pool's pages and each sequence's
        tail (kvm_tree_attention).

        q: [seqs][nodes][q_heads][head_dim] fp16 / bf16; tail_k, tail_v: [seqs][>= recent + nodes][kv_heads][head_dim]
        of the same type, the recent committed tokens and then the drafted ones. Sequence i reads pool row row0 +
        i * row_step: the pages listed in sel_ids [seqs][.] / sel_n [seqs] (select_topk's outputs), or every resident
        page. tokens: history length, int or int64 tensor [seqs]; recent: int or int32 tensor [seqs]; tree: int32
        tensor [nodes][words] or [seqs][nodes][words] (tree_mask), None for a chain; rows: int32 tensor [seqs], nodes
        used. k_type / v_type: type of the pages (default: q's). Returns (out like q, lse [seqs][nodes][q_heads])."""
        w, dev = "kvm_tree_attention", self.ctx.device
        out, lse, lse_p, t, (R, N, Hq, D), hkv, qq, kk, vv, oo = _attention_args(w, dev, q, tail_k, tail_v, out, lse, want_lse,
                                                                                 stream)
        tokens, seq_tokens = _seq_arg(tokens, dev, R, w, torch.int64)
        recent, seq_recent = _seq_arg(recent, dev, R, w, torch.int32)
        ids = ns = stride = width = words = tree_p = tree_stride = 0
        if sel_ids is not None:
            n0, width = sel_ids.shape if sel_ids.dim() == 2 else (0, 0)
            stride = sel_ids.stride(0) if n0 > 1 and width else width
            if sel_n is None or n0 < R or sel_ids.dtype is not torch.int32 or stride < width or \
                    (width > 1 and sel_ids.stride(1) != 1) or sel_ids.get_device() != dev:
                raise _bad(w, "sel_ids is int32 [seqs][.] on the device, with sel_n [seqs]")
            ns = _seq_arg(sel_n, dev, R, w, torch.int32)[1]
            ids = sel_ids.data_ptr() or ns  # (a table without columns has no address, and 0 means every resident page)
        if tree is not None:
            shape = tree.shape
            if tree.dtype is not torch.int32 or not tree.is_contiguous() or tree.get_device() != dev or \
                    shape[:-1] not in ((N,), (R, N)) or shape[-1] * 32 < N:
                raise _bad(w, "tree is contiguous int32 [nodes][words] or [seqs][nodes][words] on the device")
            words = shape[-1]
            tree_p, tree_stride = tree.data_ptr(), (N * words if len(shape) == 3 else 0)
        seq_rows = 0 if rows is None else _seq_arg(rows, dev, R, w, torch.int32)[1]
        d = _pack(w, _TREE, Hq, hkv, D, t, t if k_type is None else k_type, t if v_type is None else v_type, R, N, row0,
                  row_step, page_tokens, recent, tokens, seq_tokens, seq_recent, seq_rows, ids, ns, stride, words, tree_p,
                  tree_stride, scale, width)
        rc = self.ctx.lib.kvm_tree_attention(self.ctx.h, self.h, d, layout, qq, kk, vv, oo, lse_p, _stream_on(dev, stream))
        if rc:
            A.check(rc, w)
        return out, lse

    # -- pages --------------------------------------------------------------
    def tables(self):
        """(slot_of [rows][pages], page_of [rows][slots]) int32 tensors that alias the pool's device tables: for
        reading, while the pool lives."""
        a, b = C.c_void_p(), C.c_void_p()
        A.check(self.ctx.lib.kvm_pool_tables(self.h, C.byref(a), C.byref(b)), "kvm_pool_tables")
        dev = torch.device("cuda", self.ctx.device)
        return (torch.as_tensor(_DeviceTable(a.value, (self.rows, self.pages), self), device=dev),
                torch.as_tensor(_DeviceTable(b.value, (self.rows, self.slots), self), device=dev))

    def fork(self, layout: A.StageLayout, src_rows: Sequence[int], dst_rows: Sequence[int], *,
             page_end: Optional[int] = None, ctas: int = 0, stream=None) -> None:
        """Row dst_rows[i] becomes a copy of row src_rows[i]: its resident pages below page_end (default: all), in
        the same slots (kvm_pool_fork)."""
        n = len(dst_rows)
        if len(src_rows) != n:
            raise A.KvmError(A.ERR_INVALID_ARGUMENT, "kvm_pool_fork: as many sources as destinations")
        page_end = self.pages if page_end is None else page_end
        for x in (src_rows, dst_rows, (page_end, ctas)):
            _u32s("kvm_pool_fork", x)
        src, dst = (C.c_uint32 * max(1, n))(*src_rows), (C.c_uint32 * max(1, n))(*dst_rows)
        A.check(self.ctx.lib.kvm_pool_fork(self.ctx.h, self.h, C.byref(layout), src, dst, n, page_end, ctas,
                                           _stream_on(self.ctx.device, stream)), "kvm_pool_fork")

    def copy_pages(self, layout: A.StageLayout, items, *, ctas: int = 0, stream=None) -> None:
        """items: (src_row, src_page, dst_row, dst_page) tuples, or a contiguous int32 CPU tensor [n][4]
        (kvm_pool_copy)."""
        _u32s("kvm_pool_copy", (ctas,))
        if isinstance(items, torch.Tensor):
            if items.device.type != "cpu" or items.dtype != torch.int32 or items.dim() != 2 or items.shape[1] != 4 or \
                    not items.is_contiguous():
                raise A.KvmError(A.ERR_INVALID_ARGUMENT, "kvm_pool_copy: items is a contiguous int32 CPU tensor [n][4]")
            n, ptr = items.shape[0], items.data_ptr()
        else:
            for x in items:
                _u32s("kvm_pool_copy", x)
            arr = (A.PageCopy * max(1, len(items)))(*[A.PageCopy(*x) for x in items])
            n, ptr = len(items), C.cast(arr, C.c_void_p)
        A.check(self.ctx.lib.kvm_pool_copy(self.ctx.h, self.h, C.byref(layout), ptr, n, ctas,
                                           _stream_on(self.ctx.device, stream)), "kvm_pool_copy")

    def free(self, rows: Sequence[int], ids: torch.Tensor, counts: torch.Tensor, *, stream=None) -> None:
        """Drops the pages ids[i][: counts[i]] (int32, device) of row rows[i] (kvm_pool_free)."""
        n = len(rows)
        w = "kvm_pool_free"
        _u32s(w, rows)
        _on_device(self.ctx.device, w, ids)
        if ids.dim() != 2 or ids.shape[0] < n or ids.dtype is not torch.int32 or not ids.is_contiguous():
            raise A.KvmError(A.ERR_INVALID_ARGUMENT, f"{w}: ids is contiguous int32 [rows][.]")
        arr = (C.c_uint32 * max(1, n))(*rows)
        n_ids = _seq_arg(counts, self.ctx.device, n, w, torch.int32)[1]
        # (a table without columns has no address)
        A.check(self.ctx.lib.kvm_pool_free(self.ctx.h, self.h, arr, n, ids.data_ptr() or n_ids, n_ids, ids.shape[1],
                                           _stream_on(self.ctx.device, stream)), w)

    def compact(self, layout: A.StageLayout, rows: Optional[Sequence[int]] = None, *, used: Optional[torch.Tensor] = None,
                ctas: int = 0, stream=None) -> None:
        """Brings the resident pages of `rows` (default: all) into their first slots (kvm_pool_compact); used: int32
        tensor [rows], receives the number of resident pages."""
        rows = range(self.rows) if rows is None else rows
        n = len(rows)
        w = "kvm_pool_compact"
        _u32s(w, rows)
        _u32s(w, (ctas,))
        arr = (C.c_uint32 * max(1, n))(*rows)
        ptr = None if used is None else _seq_arg(used, self.ctx.device, n, w, torch.int32)[1]
        A.check(self.ctx.lib.kvm_pool_compact(self.ctx.h, self.h, C.byref(layout), arr, n, ptr, ctas,
                                              _stream_on(self.ctx.device, stream)), w)


class Transfer:
    """A working-set transfer over a ResidencyPool (kvm_transfer): the GPU side of
    kvmem::MemoryTransfer (kvmem/include/kvmem/memory_contract.hpp:171-185). The
    plan goes into a shadow of the pool's tables; start_spill / poll / start_restore /
    publish / abort keep the reference's names and order; failures raise KvmError
    (the reference's MemoryError codes)."""

    def __init__(self, pool: "ResidencyPool", sel_ids: torch.Tensor, sel_n: torch.Tensor, *,
                 force_reload: bool = False, stream=None):
        self.pool, self.lib = pool, pool.ctx.lib
        h = C.c_void_p()
        rc = self.lib.kvm_transfer_prepare(pool.ctx.h, pool.h, sel_ids.data_ptr(), sel_n.data_ptr(),
                                           sel_ids.stride(0), int(force_reload), _stream_ptr(stream), C.byref(h))
        A.check(rc, "kvm_transfer_prepare")
        self.h = h

    def start_spill(self, layout: Optional[A.StageLayout] = None, stale: Optional[torch.Tensor] = None,
                    ctas: int = 0, stream=None) -> None:
        rc = self.lib.kvm_transfer_start_spill(self.h, C.byref(layout) if layout is not None else None,
                                               stale.data_ptr() if stale is not None else None, ctas,
                                               _stream_ptr(stream))
        A.check(rc, "kvm_transfer_start_spill")

    def poll(self) -> str:
        """'Complete' or 'Pending' (TransferStatus); a failed step raises."""
        rc = self.lib.kvm_transfer_poll(self.h)
        if rc == A.ERR_PENDING:
            return "Pending"
        A.check(rc, "kvm_transfer_poll")
        return "Complete"

    def wait(self, timeout_s: float = 30.0) -> None:
        import time
        t0 = time.time()
        while self.poll() == "Pending":
            if time.time() - t0 > timeout_s:
                raise A.KvmError(A.ERR_TIMEOUT, "kvm_transfer_poll")
            time.sleep(0.0005)

    def start_restore(self, layout: A.StageLayout, ctas: int = 0, stream=None) -> None:
        A.check(self.lib.kvm_transfer_start_restore(self.h, C.byref(layout), ctas, _stream_ptr(stream)),
                "kvm_transfer_start_restore")

    def publish(self, stream=None) -> None:
        A.check(self.lib.kvm_transfer_publish(self.h, _stream_ptr(stream)), "kvm_transfer_publish")

    def abort(self, timeout_s: float = 30.0) -> bool:
        """Drains, then drops the transfer; True when the previous view is preserved."""
        kept = C.c_int(0)
        A.check(self.lib.kvm_transfer_abort(self.h, int(timeout_s * 1e6), C.byref(kept)), "kvm_transfer_abort")
        return bool(kept.value)

    def close(self) -> None:
        if getattr(self, "h", None):
            self.lib.kvm_transfer_destroy(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class StageOut:
    """Double-buffered stage-out (kvm_stageout): device regions gathered into
    two pinned host slots in turn. Method names follow the reference's
    kvmem_stageout_* functions (src/adapter/llama-kvmem-stagein.h:50-55);
    failures raise KvmError instead of returning false / -1."""

    SLAB = 32 << 20  # the reference's slot size
    GATHER_MAX = 8192

    def __init__(self, device: int = 0, slot_bytes: int = SLAB, max_items: int = GATHER_MAX):
        self.lib = A.load()
        self.slot_bytes = slot_bytes
        h = C.c_void_p()
        A.check(self.lib.kvm_stageout_create(device, slot_bytes, max_items, C.byref(h)), "kvm_stageout_create")
        self.h = h

    def close(self) -> None:
        if getattr(self, "h", None):
            self.lib.kvm_stageout_destroy(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def enqueue(self, dev_ptr: int, nbytes: int) -> Optional[int]:
        """Queue a device region; its slot offset, or None when the batch is full."""
        off = C.c_uint64()
        rc = self.lib.kvm_stageout_enqueue(self.h, dev_ptr, nbytes, C.byref(off))
        if rc == A.ERR_LENGTH:
            return None
        A.check(rc, "kvm_stageout_enqueue")
        return off.value

    def used(self) -> int:
        return int(self.lib.kvm_stageout_used(self.h))

    def submit(self, ctas: int = 0, stream=None) -> int:
        slot = C.c_int(-1)
        A.check(self.lib.kvm_stageout_submit(self.h, ctas, _stream_ptr(stream), C.byref(slot)), "kvm_stageout_submit")
        return slot.value

    def wait(self, slot: int, timeout_s: float = 30.0) -> None:
        A.check(self.lib.kvm_stageout_wait(self.h, slot, int(timeout_s * 1e6)), "kvm_stageout_wait")

    def slot_view(self, slot: int, offset: int, nbytes: int):
        """numpy uint8 view of bytes [offset, offset + nbytes) of a slot (no copy)."""
        import numpy as np
        base = self.lib.kvm_stageout_slot_base(self.h, slot)
        if not base or offset + nbytes > self.slot_bytes:
            raise ValueError("slot range")
        buf = (C.c_uint8 * nbytes).from_address(base + offset)
        return np.frombuffer(buf, dtype=np.uint8)

    def clear(self) -> None:
        A.check(self.lib.kvm_stageout_clear(self.h), "kvm_stageout_clear")


def tree_mask(parents: Sequence[int]) -> torch.Tensor:
    """The visibility words int32 [nodes][words] (CPU) of a tree of drafted tokens given by parents, -1 for a root
    (kvm_tree_mask)."""
    n = len(parents)
    words = max(1, -(-n // 32))
    out = torch.zeros((n, words), dtype=torch.int32)
    arr = (C.c_int32 * max(1, n))(*parents)
    A.check(A.load().kvm_tree_mask(arr, n, words, out.data_ptr()), "kvm_tree_mask")
    return out


def cache_layout(*planes: torch.Tensor) -> A.StageLayout:
    """Layout of a paged cache alone (no host records): one or two device tensors [rows][slots][...] whose slots are
    contiguous."""
    out = []
    for t in planes:
        if t.dim() < 3 or not t[0, 0].is_contiguous():
            raise A.KvmError(A.ERR_INVALID_ARGUMENT, "cache_layout: [rows][slots][...] with contiguous slots")
        es = t.element_size()
        out.append(dict(host_base=None, host_row_stride=0, host_page_stride=0, dev_base=t.data_ptr(),
                        dev_row_stride=t.stride(0) * es, dev_slot_stride=t.stride(1) * es, bytes=t[0, 0].numel() * es))
    return stage_layout(out)


def ipc_export(t: torch.Tensor) -> bytes:
    """Opaque handle (kvm_ipc_export) naming a device tensor's memory for another process."""
    buf = (C.c_uint8 * A.IPC_HANDLE_BYTES)()
    A.check(A.load().kvm_ipc_export(t.data_ptr(), buf), "kvm_ipc_export")
    return bytes(buf)


def ipc_open(device: int, handle: bytes) -> int:
    """Maps another process's device memory on `device` (peer access enabled); returns the address."""
    buf = (C.c_uint8 * A.IPC_HANDLE_BYTES).from_buffer_copy(handle)
    ptr = C.c_void_p()
    A.check(A.load().kvm_ipc_open(device, buf, C.byref(ptr)), "kvm_ipc_open")
    return int(ptr.value)


def ipc_close(device: int, ptr: int) -> None:
    A.check(A.load().kvm_ipc_close(device, ptr), "kvm_ipc_close")


def stage_layout(planes: Sequence[dict]) -> A.StageLayout:
    """planes: up to two dicts with host_base, host_row_stride, host_page_stride,
    dev_base, dev_row_stride, dev_slot_stride, bytes."""
    L = A.StageLayout()
    L.planes = len(planes)
    for j, p in enumerate(planes):
        L.host_base[j] = p["host_base"]
        L.host_row_stride[j] = p["host_row_stride"]
        L.host_page_stride[j] = p["host_page_stride"]
        L.dev_base[j] = p["dev_base"]
        L.dev_row_stride[j] = p["dev_row_stride"]
        L.dev_slot_stride[j] = p["dev_slot_stride"]
        L.bytes[j] = p["bytes"]
    return L


# ----------------------------------------------------------------------------
# Mirrors of the reference interfaces for this path.
# ----------------------------------------------------------------------------

@dataclass
class TensorView:
    """The parts of a ggml tensor the reference scorer reads: `data` (device
    tensor owning the bytes), element / block `type`, ne[0..2] and byte strides
    nb[1..2] (ggml order: ne0 = head_dim, ne1 = rows or tokens, ne2 = heads)."""
    data: torch.Tensor
    type: int
    ne: tuple
    nb: tuple


class AttentionCuda:
    """Mirror of llama_kvmem_attention_cuda (src/adapter/llama-kvmem-attention-cuda.h:9-18).

    score(q, k, mask, scale, softcap, block, rows) returns masses[len(rows)][pages]
    (mean over all query heads of the page-softmax mass), or None when the
    inputs are outside what the kernel handles (the reference's `false`,
    after which the caller builds its fallback graph). CUDA failures raise.
    """

    def __init__(self, device: int = 0):
        self.ctx = RecallContext(device)

    def score(self, q: TensorView, k: TensorView, mask: Optional[TensorView], scale: float, softcap: float,
              block: int, rows: Sequence[int]):
        D, _, Hq = q.ne[0], q.ne[1], q.ne[2]
        T, Hkv = k.ne[1], k.ne[2]
        if q.type not in (A.F32, A.F16, A.BF16) or D > 256 or D % 32:
            return None
        pages = -(-T // block)
        desc = RecallContext.make_desc(layers=1, q_heads=Hq, kv_heads=Hkv, head_dim=D, tokens=T, page_tokens=block,
                                       groups=1, scale=scale, softcap=softcap)
        kc = A.KCache()
        kc.data, kc.type = k.data.data_ptr(), k.type
        kc.layer_stride, kc.token_stride, kc.head_stride = 0, k.nb[1], k.nb[2]
        kc.capacity_tokens = T
        if not rows:
            return []
        # Every sampled row in one call (one pass over K), as the reference's batch.
        qq = A.Query()
        qq.data = q.data.data_ptr()
        qq.type = q.type
        qq.layer_stride, qq.row_stride, qq.head_stride = 0, q.nb[1], q.nb[2]
        ids = (C.c_uint32 * len(rows))(*rows)
        qq.row_ids = C.cast(ids, C.POINTER(C.c_uint32))
        qq.rows, qq.row_count = len(rows), q.ne[1]
        if mask is not None:
            desc.mask = mask.data.data_ptr()
            desc.mask_type = mask.type
            desc.mask_row_stride = mask.nb[1]
        try:
            out_rows, _ = self.ctx.score_pages(desc, qq, kc, want_mean=False)
        except A.KvmError as e:
            if e.code == A.ERR_UNSUPPORTED:
                return None
            raise
        self.ctx.check_status("llama_kvmem_attention_cuda::score")
        return out_rows.view(len(rows), pages).tolist()


class PageSoftmaxCuda:
    """Mirror of kvmem::PageSoftmaxCuda (kvmem/include/kvmem/page_softmax_cuda.hpp:10-31)
    over device-resident per-page K sums.

    score(sums, counts, q, layer_rows, frame, aggregation) -> list of doubles
    over frame pages; frame is the dict form of QueryScoreFrame (score_mask
    selects the softmax domain). Geometry errors raise ValueError
    (std::invalid_argument), a non-finite / FP16-overflowing operand raises
    ValueError, CUDA failures raise RuntimeError.
    """

    def __init__(self, device: int = 0, workspace: Optional[torch.Tensor] = None):
        self.ctx = RecallContext(device)
        if workspace is not None:
            if workspace.data_ptr() % 256:
                raise ValueError("page softmax borrowed workspace is missing, unaligned or too small")
            self.ctx.bind_workspace(workspace)

    def score(self, sums: torch.Tensor, counts: torch.Tensor, q: torch.Tensor, layer_rows: Sequence[int],
              frame: dict, aggregation: int = 0, *, q_heads: int, kv_heads: int, head_dim: int,
              scale: float = 0.0) -> list:
        try:
            out = self.ctx.meank_score(sums, counts, q, layer_rows, frame["score_mask"], q_heads=q_heads,
                                       kv_heads=kv_heads, head_dim=head_dim, aggregation=aggregation, scale=scale)
        except A.KvmError as e:
            if e.code in (A.ERR_INVALID_ARGUMENT, A.ERR_NONFINITE):
                raise ValueError(str(e)) from e
            if e.code == A.ERR_LENGTH:
                raise OverflowError(str(e)) from e
            raise
        return [float(x) for x in out.cpu().double()]

    def device_bytes(self) -> int:
        return self.ctx.device_bytes()


def pick_scored_blocks(ctx: RecallContext, scores: torch.Tensor, mandatory: Sequence[int], budget: int,
                       signed_scores: bool = False) -> list:
    """Mirror of KvMemStore::pick_scored_blocks with candidates = every page of
    the (device f32) score row and no media groups. Raises ValueError for an
    invalid candidate or mandatory page (std::invalid_argument) and
    RuntimeError when mandatory pages exceed the budget (std::runtime_error)."""
    try:
        ids, n = ctx.select_topk(scores.view(1, -1), mandatory, budget, signed=signed_scores)
        ctx.check_status("pick_scored_blocks")
    except A.KvmError as e:
        if e.code in (A.ERR_INVALID_ARGUMENT, A.ERR_NONFINITE):
            raise ValueError(str(e)) from e
        raise RuntimeError(str(e)) from e
    return ids[0, : int(n[0])].tolist()
