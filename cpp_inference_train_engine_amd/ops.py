"""Operator interface over the C ABI for the paged, ragged MLA decode path.

Mirrors the three subsystems of the path:
  (a) ``build_metadata``   -> ``mla_build_metadata``   (GPU ragged-batch metadata)
  (b) ``append_latent``    -> ``mla_append_latent``    (paged latent/rope append)
  (c) ``decode_attention`` -> ``mla_decode_attention`` (absorbed split-K decode)
and, beside them,
  (d) ``append_latent_q8``, ``read_latent_q8`` -> the 8-bit latent cache
  (e) ``plan_attention``, ``latent_attention`` -> attention of any rows of a batch over a 16-bit or
      8-bit cache, prefixes that sessions share computed once
All tensors are torch CUDA (HIP) tensors; calls are stream-ordered on the
current torch stream unless ``stream`` is given.
"""
from __future__ import annotations

from contextlib import nullcontext
from dataclasses import dataclass, field

from . import (CACHE_16BIT, CACHE_Q8, DECODE_FUSED_MERGE, DTYPE_BF16, DTYPE_F16, INFO_INTS, MAX_WORK,
               PLACE_MAX_SESSIONS, PLAN_INFO_INTS, WORK_DESC_INTS, WORK_PAGES, check, lib, ptr, stream_handle)


def _torch():
    import torch
    return torch


@dataclass
class RaggedBatch:
    """Device metadata of one continuous-batching step (all int32 tensors)."""

    B: int
    page_size: int
    max_pages: int
    num_pool_pages: int
    max_work: int
    max_rows: int
    cu_seqlens_q: object
    cu_seqlens_k: object
    page_table: object
    slot_mapping: object
    num_splits: object
    cu_splits: object
    work_session: object
    work_split: object
    work_desc: object
    work_pages: object
    info: object
    placed: bool = False  # XCD-placed for this device (decode merges inside its launch)
    host_info: list = field(default_factory=list)

    def read_info(self, stream=None):
        """Synchronise and return [W, split, total_q, total_k, n_xcd placed for, 0, 0, 0];
        raises on a bad batch."""
        import numpy as np
        h = np.zeros(INFO_INTS, np.int32)
        check(lib().mla_read_metadata_info(stream_handle(stream), ptr(self.info), h.ctypes.data))
        self.host_info = h.tolist()
        return self.host_info


def xcd_count() -> int:
    """XCDs of the current device when it keeps the workgroups w with one residue w % n on one
    XCD (the premise of XCD placement), else 0.  The first call per device runs a probe
    kernel."""
    return int(lib().mla_xcd_placement_supported())


def placed_work_slots(ctx_len, q_len, page_size: int, split_pages: int, n_xcd: int) -> int:
    """Work-list slots of an XCD-placed build (host arrays of the batch's lengths): n_xcd
    times the largest item count of one XCD, as mla_build_metadata deals the sessions
    (by pages read, largest first, in rounds of n_xcd: XCDs 0..n-1, then n-1..0, ..)."""
    import numpy as np
    ctx = np.asarray(ctx_len, np.int64)
    q = np.asarray(q_len, np.int64)
    pages = np.where(q > 0, -(-(ctx + q) // page_size), 0)
    items = -(-pages // split_pages)
    order = np.lexsort((np.arange(len(pages)), -pages))
    r = np.arange(len(pages))
    xcd = np.where((r // n_xcd) % 2 == 0, r % n_xcd, n_xcd - 1 - r % n_xcd)
    cnt = np.bincount(xcd, weights=items[order], minlength=n_xcd)
    return int(n_xcd * cnt.max()) if len(pages) else 0


def build_metadata(ctx_len, q_len, cu_pages, page_ids, page_size: int, max_pages: int,
                   num_pool_pages: int, split_pages: int = 0, target_blocks: int = 1024,
                   max_work: int | None = None, max_rows: int | None = None,
                   placement: bool = False, placement_xcds: int | None = None,
                   stream=None) -> RaggedBatch:
    """(a) Build cu_seqlens, padded page tables, slot mapping and the block-to-session
    map on the GPU (one launch, two for a large
    page table).  Inputs are device int32 tensors.  ``placement``: lay
    the work list out so that each session's items run on one XCD (B <= 256; max_work
    must hold ``placed_work_slots``); decode attention over it then merges the split
    partials inside its launch.  ``placement_xcds``: the placed layout for that many XCDs
    instead of this device's (mla_build_metadata_placed; no fused merge over it unless
    the count is the device's)."""
    torch = _torch()
    dev = ctx_len.device
    B = int(ctx_len.numel())
    if max_rows is None:
        max_rows = max(1, 4 * B)
    if max_work is None:
        max_work = max(1, min(MAX_WORK, target_blocks + 2 * B))
    i32 = dict(dtype=torch.int32, device=dev)
    rb = RaggedBatch(
        B=B, page_size=page_size, max_pages=max_pages, num_pool_pages=num_pool_pages,
        max_work=max_work, max_rows=max_rows,
        cu_seqlens_q=torch.empty(B + 1, **i32), cu_seqlens_k=torch.empty(B + 1, **i32),
        page_table=torch.empty(max(1, B * max_pages), **i32),
        slot_mapping=torch.empty(max_rows, **i32), num_splits=torch.empty(max(B, 1), **i32),
        cu_splits=torch.empty(B + 1, **i32), work_session=torch.empty(max_work, **i32),
        work_split=torch.empty(max_work, **i32),
        work_desc=torch.empty(max_work * WORK_DESC_INTS, **i32),
        work_pages=torch.empty(max_work * WORK_PAGES, **i32),
        info=torch.empty(INFO_INTS, **i32),
        placed=bool(placement) or (placement_xcds is not None and placement_xcds == xcd_count()))
    if placement_xcds is not None:
        fn, place = lib().mla_build_metadata_placed, int(placement_xcds)
    else:
        fn, place = lib().mla_build_metadata, int(bool(placement))
    check(fn(
        stream_handle(stream), B, ptr(ctx_len), ptr(q_len), ptr(cu_pages), ptr(page_ids),
        page_size, max_pages, num_pool_pages, split_pages, target_blocks, max_work, max_rows,
        place, ptr(rb.cu_seqlens_q), ptr(rb.cu_seqlens_k), ptr(rb.page_table),
        ptr(rb.slot_mapping), ptr(rb.num_splits), ptr(rb.cu_splits), ptr(rb.work_session),
        ptr(rb.work_split), ptr(rb.work_desc), ptr(rb.work_pages), ptr(rb.info)))
    return rb


class PagedLatentCache:
    """Device page pool: [layers, pages, page_size * (kv_rank + rope_dim)] 16-bit words.
    Each page record is latent [page_size][kv_rank] followed by rope [page_size][rope_dim]."""

    def __init__(self, n_layers: int, num_pages: int, page_size: int, kv_rank: int,
                 rope_dim: int, dtype: int = DTYPE_F16, device="cuda", storage=None):
        torch = _torch()
        self.n_layers, self.num_pages, self.page_size = n_layers, num_pages, page_size
        self.kv_rank, self.rope_dim, self.dtype = kv_rank, rope_dim, dtype
        tdt = _dtype_of(dtype)
        rec = page_size * (kv_rank + rope_dim)
        if storage is None:
            storage = torch.zeros((n_layers, num_pages, rec), dtype=tdt, device=device)
        assert storage.shape == (n_layers, num_pages, rec) and storage.dtype == tdt
        self.pages = storage

    def layer(self, l: int):
        return self.pages[l]

    @property
    def record_words(self) -> int:
        return self.page_size * (self.kv_rank + self.rope_dim)


def append_latent(cache: PagedLatentCache, layer: int, ckv, krope, slot_mapping,
                  stream=None) -> None:
    """(b) Round ckv [T x kv_rank] / krope [T x rope_dim] (fp32) to the cache dtype and
    write row t to flat slot slot_mapping[t] of ``layer``'s page pool."""
    T = int(ckv.shape[0])
    assert ckv.is_contiguous() and krope.is_contiguous()
    check(lib().mla_append_latent(stream_handle(stream), T, cache.kv_rank, cache.rope_dim,
                                  cache.page_size, cache.dtype, ptr(ckv), ptr(krope),
                                  ptr(slot_mapping), cache.num_pages, ptr(cache.layer(layer))))


def decode_workspace_bytes(max_work: int, max_sessions: int, n_heads: int, kv_rank: int) -> int:
    return int(lib().mla_decode_workspace_bytes(max_work, max_sessions, n_heads, kv_rank))


def decode_workspace(max_work: int, max_sessions: int, n_heads: int, kv_rank: int,
                     device="cuda"):
    """Decode workspace (head block of merge counters and status word, split partials),
    zeroed."""
    torch = _torch()
    n = max(decode_workspace_bytes(max_work, max_sessions, n_heads, kv_rank), 4)
    return torch.zeros(n, dtype=torch.uint8, device=device)


def decode_status(workspace, clear: bool = False, stream=None) -> int:
    """Synchronise and return the decode status word of ``workspace`` (OR of
    DECODE_STATUS_XCD / DECODE_STATUS_UNPLACED raised by fused calls since it was last
    cleared; 0 when every fused merge's premises held).  ``clear`` also zeroes the head."""
    import numpy as np
    h = np.zeros(1, np.int32)
    check(lib().mla_decode_status(stream_handle(stream), ptr(workspace), int(workspace.numel()),
                                  int(bool(clear)), h.ctypes.data))
    return int(h[0])


def _decode_call(fn, batch: RaggedBatch, pages, q_latent, q_rope, scale, kv_rank, rope_dim,
                 dtype, out, lse, workspace, flags, stream, fused=None):
    torch = _torch()
    rows, H = int(q_latent.shape[0]), int(q_latent.shape[1])
    if out is None:
        out = torch.zeros((rows, H, kv_rank), dtype=torch.float32, device=q_latent.device)
    if workspace is None:
        workspace = decode_workspace(batch.max_work, batch.B, H, kv_rank, q_latent.device)
    if fused is None:
        fused = batch.placed
    if fused and not batch.placed:
        raise ValueError("fused decode needs metadata placed for this device's XCDs "
                         "(build_metadata(..., placement=True))")
    if fused:
        flags |= DECODE_FUSED_MERGE
    check(getattr(lib(), fn)(
        stream_handle(stream), batch.B, H, kv_rank, rope_dim, batch.page_size, dtype,
        float(scale), ptr(batch.cu_seqlens_q), ptr(batch.page_table), batch.max_pages,
        batch.num_pool_pages, ptr(pages), ptr(q_latent), ptr(q_rope), ptr(batch.num_splits),
        ptr(batch.cu_splits), ptr(batch.work_desc), ptr(batch.work_pages), ptr(batch.info),
        batch.max_work, ptr(out), ptr(lse), ptr(workspace), int(workspace.numel()), flags))
    return out


def decode_attention(batch: RaggedBatch, pages, q_latent, q_rope, scale: float, *,
                     kv_rank: int, rope_dim: int, dtype: int = DTYPE_F16, out=None, lse=None,
                     workspace=None, flags: int = 0, stream=None, fused: bool | None = None):
    """(c) Absorbed MLA decode attention for every session with one query row.
    q_latent [rows, H, kv_rank], q_rope [rows, H, rope_dim] in the cache dtype;
    returns out [rows, H, kv_rank] fp32 (and fills lse [rows, H] if given).  ``fused``
    (default: whether the metadata is XCD-placed) merges the splits inside the decode
    launch; it needs placed metadata."""
    return _decode_call("mla_decode_attention", batch, pages, q_latent, q_rope, scale, kv_rank,
                        rope_dim, dtype, out, lse, workspace, flags, stream, fused)


def decode_partials(batch: RaggedBatch, pages, q_latent, q_rope, scale: float, *,
                    kv_rank: int, rope_dim: int, dtype: int = DTYPE_F16, out=None, lse=None,
                    workspace=None, flags: int = 0, stream=None, fused: bool = False):
    """First launch of decode_attention: final rows of one-item sessions, split partials
    of the others in ``workspace`` (pass the same workspace to ``decode_merge``); with
    ``fused`` (placed metadata) also the rows of split sessions."""
    return _decode_call("mla_decode_partials", batch, pages, q_latent, q_rope, scale, kv_rank,
                        rope_dim, dtype, out, lse, workspace, flags, stream, fused)


def decode_merge(batch: RaggedBatch, n_heads: int, kv_rank: int, out, workspace, lse=None,
                 stream=None):
    """Second launch of decode_attention: log-sum-exp merge of the split partials."""
    check(lib().mla_decode_merge(
        stream_handle(stream), batch.B, n_heads, kv_rank, ptr(batch.cu_seqlens_q),
        ptr(batch.num_splits), ptr(batch.cu_splits), ptr(batch.info), batch.max_work, ptr(out),
        ptr(lse), ptr(workspace), int(workspace.numel())))
    return out


def prefill_attention(batch: RaggedBatch, pages, q_latent, q_rope, scale: float, *,
                      kv_rank: int, rope_dim: int, max_q_len: int, dtype: int = DTYPE_F16,
                      out=None, lse=None, flags: int = 0, stream=None):
    """(c) Absorbed MLA chunked-prefill attention for every session with q_len > 1: query
    row i of a session attends causally to its keys [0, ctx + i].  The chunk's latent
    rows must already be in ``pages``.  q_latent [rows, H, kv_rank], q_rope
    [rows, H, rope_dim] in the cache dtype; returns out [rows, H, kv_rank] fp32 (rows of
    sessions with q_len <= 1 are left as they were)."""
    torch = _torch()
    rows, H = int(q_latent.shape[0]), int(q_latent.shape[1])
    if out is None:
        out = torch.zeros((rows, H, kv_rank), dtype=torch.float32, device=q_latent.device)
    check(lib().mla_prefill_attention(
        stream_handle(stream), batch.B, H, kv_rank, rope_dim, batch.page_size, dtype,
        float(scale), ptr(batch.cu_seqlens_q), ptr(batch.cu_seqlens_k), ptr(batch.page_table),
        batch.max_pages, batch.num_pool_pages, ptr(pages), ptr(q_latent), ptr(q_rope),
        ptr(batch.info), int(max_q_len), ptr(out), ptr(lse), flags))
    return out


# ------------------------------------------------- 8-bit cache, planned attention ----
def _dtype_of(code: int):
    """torch's type of a cache's words."""
    torch = _torch()
    if code != DTYPE_F16 and code != DTYPE_BF16:
        raise ValueError(f"dtype: {code!r}, wanted DTYPE_F16 or DTYPE_BF16 (a cache holds 16-bit words)")
    return torch.float16 if code == DTYPE_F16 else torch.bfloat16


_current_device = None


def _gpu() -> int:
    """Index of the current GPU (0.05 us; torch.cuda.current_device 0.2)."""
    global _current_device
    if _current_device is None:
        torch = _torch()
        torch.cuda.current_device()  # initialises the device
        _current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)
    return _current_device()


def _check(what: str, t, shape, dtype, gpu: int) -> int:
    """Address of a contiguous tensor of this shape and type on GPU ``gpu``, or ValueError: the
    kernels see addresses only."""
    if t.dtype is not dtype or t.shape != shape or not t.is_contiguous():
        raise ValueError(f"{what}: wanted a contiguous {dtype} tensor of shape {tuple(shape)}, got "
                         f"{t.dtype} {tuple(t.shape)}")
    if t.get_device() != gpu:
        raise ValueError(f"{what}: wanted on the current GPU, is on {t.device}")
    return t.data_ptr()


def _check_list(what: str, t, gpu: int) -> int:
    """The same of a one-dimensional int32 tensor of any length."""
    return _check(what, t, (t.numel(),), _torch().int32, gpu)


def _allocating_on(stream):
    """Tensors that a call makes belong to the stream it works on: their fill comes before the
    call's kernels, and their memory is not given to another stream's work while those run."""
    return nullcontext() if stream is None else _torch().cuda.stream(stream)


class QuantizedLatentCache:
    """Device page pool of the 8-bit latent cache: uint8 [layers, pages, record bytes], a record
    as mla_hip.h lays it out (e4m3 latents with a power-of-two scale for each 32 columns, rope
    keys in 16 bits of ``dtype``)."""

    def __init__(self, n_layers: int, num_pages: int, page_size: int, kv_rank: int,
                 rope_dim: int, dtype: int = DTYPE_F16, device="cuda", storage=None):
        torch = _torch()
        self.n_layers, self.num_pages, self.page_size = n_layers, num_pages, page_size
        self.kv_rank, self.rope_dim, self.dtype = kv_rank, rope_dim, dtype
        _dtype_of(dtype)
        rec = int(lib().mla_q8_page_bytes(page_size, kv_rank, rope_dim))
        if rec == 0:
            raise ValueError("8-bit latent cache: page_size must be a multiple of 16 up to 65,536, "
                             "kv_rank of 32 up to 512, rope_dim of 8 up to 64")
        if storage is None:
            storage = torch.zeros((n_layers, num_pages, rec), dtype=torch.uint8, device=device)
        if (tuple(storage.shape) != (n_layers, num_pages, rec) or storage.dtype != torch.uint8 or
                not storage.is_contiguous()):
            raise ValueError(f"8-bit latent cache: storage must be a contiguous uint8 tensor of "
                             f"shape {(n_layers, num_pages, rec)}")
        self._pages = storage
        self._place = storage.get_device(), storage.data_ptr(), n_layers and storage.stride(0)

    @property
    def pages(self):
        return self._pages

    def layer(self, l: int):
        return self.pages[l]

    @property
    def record_bytes(self) -> int:
        return int(self.pages.shape[2])

    def _layer_address(self, l: int, gpu: int) -> int:
        device, first, size = self._place
        if device != gpu:
            raise ValueError(f"cache: wanted on the current GPU, is on {self.pages.device}")
        if not -self.n_layers <= l < self.n_layers:
            raise IndexError(f"layer {l} of {self.n_layers}")
        return first + l % self.n_layers * size


def append_latent_q8(cache: QuantizedLatentCache, layer: int, ckv, krope, slot_mapping,
                     stream=None) -> None:
    """(d) Quantise ckv [T x kv_rank] (fp32) to 8 bits, round krope [T x rope_dim] (fp32) to the
    cache's 16-bit dtype, and write row t to flat slot slot_mapping[t] of ``layer``'s pool.  Slots
    outside the pool are skipped; the others are distinct."""
    f32, gpu, T = _torch().float32, _gpu(), int(ckv.shape[0])
    x = _check("ckv", ckv, (T, cache.kv_rank), f32, gpu)
    k = _check("krope", krope, (T, cache.rope_dim), f32, gpu)
    slots = _check_list("slot_mapping", slot_mapping, gpu)
    if slot_mapping.numel() < T:
        raise ValueError(f"slot_mapping: {slot_mapping.numel()} slots for {T} rows")
    check(lib().mla_append_latent_q8(stream_handle(stream), T, cache.kv_rank, cache.rope_dim,
                                     cache.page_size, cache.dtype, x, k, slots, cache.num_pages,
                                     cache._layer_address(layer, gpu)))


def read_latent_q8(cache: QuantizedLatentCache, layer: int, slot_mapping, ckv=None, krope=None,
                   stream=None):
    """(d) The tokens at flat slots slot_mapping[T] of ``layer``'s pool as 16-bit rows of the
    cache's dtype: (ckv [T x kv_rank], krope [T x rope_dim]), exact.  Rows whose slot lies outside
    the pool are left as they were (zero in tensors that this call makes)."""
    gpu, T, dt = _gpu(), int(slot_mapping.shape[0]), _dtype_of(cache.dtype)
    slots = _check_list("slot_mapping", slot_mapping, gpu)
    if ckv is None or krope is None:
        with _allocating_on(stream):
            if ckv is None:
                ckv = _torch().zeros((T, cache.kv_rank), dtype=dt, device=cache.pages.device)
            if krope is None:
                krope = _torch().zeros((T, cache.rope_dim), dtype=dt, device=cache.pages.device)
    x = _check("ckv", ckv, (T, cache.kv_rank), dt, gpu)
    k = _check("krope", krope, (T, cache.rope_dim), dt, gpu)
    check(lib().mla_read_latent_q8(stream_handle(stream), T, cache.kv_rank, cache.rope_dim,
                                   cache.page_size, cache.dtype, slots, cache.num_pages,
                                   cache._layer_address(layer, gpu), x, k))
    return ckv, krope


@dataclass
class SharedPrefixes:
    """Prefixes that groups of consecutive sessions share (device int32 tensors): group g is the
    sessions [cu_groups[g], cu_groups[g+1]), its prefix prefix_len[g] tokens on the pages
    page_ids[cu_pages[g]:cu_pages[g+1]]."""

    cu_groups: object
    prefix_len: object
    cu_pages: object
    page_ids: object

    @property
    def n_groups(self) -> int:
        return int(self.prefix_len.shape[0])


class AttentionPlan:
    """What ``plan_attention`` built, for ``latent_attention`` calls over the same batch.  It keeps
    the tensors and sizes that it was made of: setting a field of the batch or of the prefixes
    later changes nothing for its calls."""

    def __init__(self, batch: RaggedBatch, n_heads: int, kv_rank: int, rows: int, max_q_len: int,
                 prefixes: SharedPrefixes | None, words):
        self.batch, self.n_heads, self.kv_rank = batch, n_heads, kv_rank
        self.rows, self.max_q_len, self.prefixes = rows, max_q_len, prefixes
        self.words = words  # the plan itself (device int32)
        self.n_groups = prefixes.n_groups if prefixes is not None else 0
        self.info = None    # host copy of its info once read_info has been called
        # the arguments of a call that are the plan's: sizes, and addresses with their tensors
        self._B, self._page_size = batch.B, batch.page_size
        self._max_pages, self._pool_pages = batch.max_pages, batch.num_pool_pages
        lists = (prefixes.cu_pages, prefixes.page_ids) if self.n_groups else (None, None)
        self._tensors = (batch.page_table, *lists, words)
        self._device, self._gpu = words.device, words.get_device()
        self._table = ptr(batch.page_table)
        self._shared = (ptr(lists[0]), ptr(lists[1]))
        self._words = (ptr(words), 4 * words.numel())
        self._records = {}

    def record_words(self, rope_dim: int, q8: bool) -> int:
        """Bytes of an 8-bit page record, or 16-bit words of a 16-bit one."""
        n = self._records.get((rope_dim, q8))
        if n is None:
            page = self._page_size
            n = (int(lib().mla_q8_page_bytes(page, self.kv_rank, rope_dim)) if q8 else
                 page * (self.kv_rank + rope_dim))
            self._records[rope_dim, q8] = n
        return n

    def read_info(self, stream=None):
        """Synchronise and return [jobs, 0, jobs of 16 rows, jobs of 128 rows, partial rows, query
        rows, ..]; raises when the batch or the prefixes are invalid.  Calls after it launch no
        more workgroups than the plan has jobs, unless the plan was made in a captured graph: each
        replay builds that one anew, and its jobs change (before the first one it holds nothing)."""
        import numpy as np
        h = np.zeros(PLAN_INFO_INTS, np.int32)
        check(lib().mla_read_plan_info(stream_handle(stream), self._words[0], h.ctypes.data))
        if not self._captured:
            self.info, self._own_info = h.copy(), h  # (calls read the second)
            self._info = h.ctypes.data
        return h.tolist()

    _info = None
    _captured = False  # made in a captured graph


def plan_attention(batch: RaggedBatch, n_heads: int, kv_rank: int, *, rows: int | None = None,
                   max_q_len: int | None = None, prefixes: SharedPrefixes | None = None,
                   stream=None) -> AttentionPlan:
    """(e) Plan the attention of a batch (one launch): which workgroup takes which query rows over
    which keys.  ``rows``: query rows of the calls (default the batch's max_rows); ``max_q_len``:
    at least every session's q_len (default ``rows``; a tighter bound makes a smaller plan, and
    calls without ``read_info`` launch fewer workgroups).  The plan serves every layer's
    ``latent_attention``."""
    torch, gpu = _torch(), _gpu()
    rows = batch.max_rows if rows is None else rows
    max_q_len = max(rows, 1) if max_q_len is None else max_q_len
    groups, shared = 0, (None, None, None, None)
    if prefixes is not None:
        x = prefixes
        groups = x.n_groups
        shared = (_check("cu_groups", x.cu_groups, (groups + 1,), torch.int32, gpu),
                  _check("prefix_len", x.prefix_len, (groups,), torch.int32, gpu),
                  _check("cu_pages", x.cu_pages, (groups + 1,), torch.int32, gpu),
                  _check_list("page_ids", x.page_ids, gpu))
    n = int(lib().mla_attention_plan_bytes(batch.B, rows, n_heads, kv_rank, max_q_len, groups))
    if n == 0:
        raise ValueError(f"plan_attention: no plan for B={batch.B}, rows={rows}, n_heads={n_heads}, "
                         f"kv_rank={kv_rank}, max_q_len={max_q_len}, groups={groups}")
    info = _check_list("batch", batch.info, gpu)
    with _allocating_on(stream):
        words = torch.empty(n // 4, dtype=torch.int32, device=batch.info.device)
        captured = words.is_cuda and torch.cuda.is_current_stream_capturing()
    check(lib().mla_plan_attention(
        stream_handle(stream), batch.B, rows, n_heads, kv_rank, batch.page_size, max_q_len,
        ptr(batch.cu_seqlens_q), ptr(batch.cu_seqlens_k), info, groups, *shared,
        prefixes.page_ids.numel() if groups else 0, batch.num_pool_pages, ptr(words), n))
    plan = AttentionPlan(batch, n_heads, kv_rank, rows, max_q_len, prefixes, words)
    plan._captured = captured
    return plan


def attention_workspace(plan: AttentionPlan):
    """Workspace of ``latent_attention`` calls with this plan (or one of the same sizes).  Calls
    that share one are ordered on one stream."""
    torch = _torch()
    n = int(lib().mla_attention_workspace_bytes(plan._B, plan.rows, plan.n_heads, plan.kv_rank,
                                                plan.max_q_len, plan.n_groups))
    return torch.empty(max(n, 16), dtype=torch.uint8, device=plan._device)


def latent_attention(plan: AttentionPlan, pages, q_latent, q_rope, scale: float, *,
                     rope_dim: int, dtype: int = DTYPE_F16, q8: bool = False, out=None, lse=None,
                     workspace=None, stream=None):
    """(e) Attention of every query row of the plan's batch over its cache and its group's prefix:
    ``pages`` is a layer of a PagedLatentCache or, with ``q8``, of a QuantizedLatentCache.
    q_latent [rows, H, kv_rank] and q_rope [rows, H, rope_dim] in ``dtype``; returns out
    [rows, H, kv_rank] in ``dtype`` (and fills lse [rows, H], fp32, if given).  Rows past the
    batch's are left as they were, and over a failed plan (``AttentionPlan.read_info`` raises) all
    of them: zero in a tensor that the call makes."""
    torch, gpu = _torch(), _gpu()
    rows, H, kv = plan.rows, plan.n_heads, plan.kv_rank
    dt = torch.float16 if dtype == DTYPE_F16 else torch.bfloat16
    if out is None or workspace is None:
        with _allocating_on(stream):
            if out is None:
                out = torch.zeros((rows, H, kv), dtype=dt, device=q_latent.device)
            if workspace is None:
                workspace = attention_workspace(plan)
    args = (
        stream_handle(stream), plan._B, rows, H, kv, rope_dim, plan._page_size, plan.max_q_len, dtype,
        CACHE_Q8 if q8 else CACHE_16BIT, scale, plan._table, plan._max_pages, plan._pool_pages,
        _check("pages", pages, (plan._pool_pages, plan.record_words(rope_dim, q8)),
               torch.uint8 if q8 else dt, gpu),
        _check("q_latent", q_latent, (rows, H, kv), dt, gpu),
        _check("q_rope", q_rope, (rows, H, rope_dim), dt, gpu),
        plan.n_groups, *plan._shared, *plan._words, plan._info,
        _check("out", out, (rows, H, kv), dt, gpu),
        None if lse is None else _check("lse", lse, (rows, H), torch.float32, gpu),
        _check("workspace", workspace, (workspace.numel(),), torch.uint8, gpu), workspace.numel())
    if plan._gpu != gpu:
        raise ValueError(f"plan: wanted on the current GPU, is on {plan._device}")
    check(lib().mla_latent_attention(*args))
    return out


__all__ = ["RaggedBatch", "build_metadata", "PagedLatentCache", "append_latent",
           "decode_workspace_bytes", "decode_workspace", "decode_status", "decode_attention",
           "decode_partials", "decode_merge", "prefill_attention", "QuantizedLatentCache",
           "append_latent_q8", "read_latent_q8", "SharedPrefixes", "AttentionPlan",
           "plan_attention", "attention_workspace", "latent_attention", "DTYPE_F16",
           "DTYPE_BF16"]


# ---------------------------------------------------------------- page layout ----
def page_tiled(page_size: int, kv_rank: int, rope_dim: int) -> bool:
    """Page records are tiled in MFMA-operand order for these shapes (see mla_hip.h)."""
    return page_size % 16 == 0 and kv_rank % 32 == 0 and rope_dim % 8 == 0


def latent_word(slot, r, page_size: int, kv_rank: int, rope_dim: int):
    """Word index of latent column r of token `slot` inside a page record (numpy-friendly)."""
    if not page_tiled(page_size, kv_rank, rope_dim):
        return slot * kv_rank + r
    t, n, j, g, e = slot // 16, slot % 16, r // 32, (r % 32) // 8, r % 8
    return ((t * (kv_rank // 32) + j) * 4 + g) * 128 + n * 8 + e


def rope_word(slot, c, page_size: int, kv_rank: int, rope_dim: int):
    """Word index of rope column c of token `slot` inside a page record."""
    base = page_size * kv_rank
    if not page_tiled(page_size, kv_rank, rope_dim):
        return base + slot * rope_dim + c
    t, n = slot // 16, slot % 16
    return base + (t * (rope_dim // 8) + c // 8) * 128 + n * 8 + c % 8
