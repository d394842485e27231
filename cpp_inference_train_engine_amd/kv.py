"""Operators of the paged key-value cache, over the C ABI: for layers whose heads have keys and
values of their own or share them in groups, with the metadata, pages and slots of the latent path.

  ``append_kv``           -> ``mla_append_kv``: new tokens' keys, rotated by their positions, and
                             values into the pages, the step's queries rotated beside them
  ``plan_kv_attention``,
  ``kv_attention``        -> attention of any rows of a batch (decode rows, drafted tokens, prompt
                             chunks) over its cache, in full or through a sliding window with sinks
All tensors are torch CUDA (HIP) tensors; calls are stream-ordered on the current torch stream
unless ``stream`` is given.
"""
from __future__ import annotations

from . import (DTYPE_BF16, DTYPE_F16, DTYPE_F32, PLAN_INFO_INTS, check, lib, ptr, stream_handle)
from .ops import RaggedBatch, _allocating_on, _check, _check_list, _dtype_of, _gpu, _torch

_row_codes = _int32 = None


def _row_code(dtype) -> int | None:
    """MLA_DTYPE_* of appended rows."""
    global _row_codes, _int32
    if _row_codes is None:
        torch = _torch()
        _int32 = torch.int32
        _row_codes = {torch.float16: DTYPE_F16, torch.bfloat16: DTYPE_BF16, torch.float32: DTYPE_F32}
    return _row_codes.get(dtype)


_INT_MAX = 2 ** 31 - 1


def _ints_of_c(**sizes) -> None:
    """A C int takes the low 32 bits of whatever it is given."""
    for name, n in sizes.items():
        if not -_INT_MAX <= n <= _INT_MAX:
            raise ValueError(f"{name}: {n} does not fit 32 bits")


class PagedKVCache:
    """Device page pool of keys and values: 16-bit [layers, pages, record words], a record keys
    [n_kv_heads][page_size][head_dim], then values [n_kv_heads][page_size][v_dim]."""

    def __init__(self, n_layers: int, num_pages: int, page_size: int, n_kv_heads: int, head_dim: int,
                 v_dim: int | None = None, dtype: int = DTYPE_F16, device="cuda", storage=None):
        torch = _torch()
        v_dim = head_dim if v_dim is None else v_dim
        self.n_layers, self.num_pages, self.page_size = n_layers, num_pages, page_size
        self.n_kv_heads, self.head_dim, self.v_dim, self.dtype = n_kv_heads, head_dim, v_dim, dtype
        _ints_of_c(num_pages=num_pages, page_size=page_size, n_kv_heads=n_kv_heads, head_dim=head_dim,
                   v_dim=v_dim)
        words = int(lib().mla_kv_page_words(n_kv_heads, head_dim, v_dim, page_size))
        if words == 0:
            raise ValueError("key-value cache: page_size must be a multiple of 16 up to 65,536, "
                             "head_dim and v_dim multiples of 16 up to 256, n_kv_heads positive")
        tdt = _dtype_of(dtype)
        if storage is None:
            storage = torch.zeros((n_layers, num_pages, words), dtype=tdt, device=device)
        if (tuple(storage.shape) != (n_layers, num_pages, words) or storage.dtype != tdt or
                not storage.is_contiguous()):
            raise ValueError(f"key-value cache: storage must be a contiguous {tdt} tensor of shape "
                             f"{(n_layers, num_pages, words)}")
        self._pages, self._dtype = storage, tdt
        self._place = storage.get_device(), storage.data_ptr(), 2 * num_pages * words
        self._shape = n_kv_heads, head_dim, v_dim, page_size
        self._key_words = n_kv_heads * page_size * head_dim

    @property
    def pages(self):
        return self._pages

    @property
    def record_words(self) -> int:
        return int(self._pages.shape[2])

    def layer(self, l: int):
        return self._pages[l]

    def keys(self, l: int):
        """A layer's keys [pages, n_kv_heads, page_size, head_dim], a view."""
        return self._pages[l][:, :self._key_words].view(self.num_pages, self.n_kv_heads,
                                                        self.page_size, self.head_dim)

    def values(self, l: int):
        """A layer's values [pages, n_kv_heads, page_size, v_dim], a view."""
        return self._pages[l][:, self._key_words:].view(self.num_pages, self.n_kv_heads,
                                                        self.page_size, self.v_dim)

    def _layer_address(self, l: int, gpu: int) -> int:
        device, first, size = self._place
        if device != gpu:
            raise ValueError(f"cache: wanted on the current GPU, is on {self._pages.device}")
        if not -self.n_layers <= l < self.n_layers:
            raise IndexError(f"layer {l} of {self.n_layers}")
        return first + l % self.n_layers * size


class Rotation:
    """How positions turn the columns of a head: pair i by position * frequencies[i] radians.
    ``frequencies``: one per pair, a device float64 tensor (kept) or numbers.  The pairs' columns are
    start + (2i, 2i + 1), with ``adjacent`` False start + (i, pairs + i); ``start`` is even."""

    def __init__(self, frequencies, start: int = 0, adjacent: bool = True, device="cuda"):
        torch = _torch()
        if not isinstance(frequencies, torch.Tensor):
            frequencies = torch.tensor(list(frequencies), dtype=torch.float64, device=device)
        if (frequencies.dtype != torch.float64 or frequencies.dim() != 1 or
                not frequencies.is_contiguous()):
            raise ValueError("rotation: frequencies must be a contiguous float64 tensor of one "
                             "dimension")
        self.frequencies, self.start, self.adjacent = frequencies, int(start), bool(adjacent)
        _ints_of_c(start=self.start, pairs=frequencies.numel())
        self._place = frequencies.get_device()
        self._args = ptr(frequencies), frequencies.numel(), self.start, int(self.adjacent)

    @classmethod
    def of_theta(cls, pairs: int, theta: float = 10000.0, start: int = 0, adjacent: bool = True,
                 device="cuda") -> "Rotation":
        """Frequencies theta^(-i / pairs)."""
        return cls([theta ** (-i / pairs) for i in range(pairs)], start, adjacent, device)


_NO_ROTATION = (None, 0, 0, 1)


def _ints(what: str, t, T: int, gpu: int) -> int:
    """Address of T integers, one for each row."""
    if t.dtype is not _int32 or t.dim() != 1 or not t.is_contiguous():
        raise ValueError(f"{what}: wanted a contiguous int32 tensor of one dimension, got {t.dtype} "
                         f"{tuple(t.shape)}")
    if t.shape[0] < T:
        raise ValueError(f"{what}: {t.shape[0]} for {T} rows")
    if t.get_device() != gpu:
        raise ValueError(f"{what}: wanted on the current GPU, is on {t.device}")
    return t.data_ptr()


def _rows(what: str, t, heads: int, dim: int, T: int, dtype, gpu: int):
    """Address and strides of rows [T, heads, dim] whose columns lie one behind the other."""
    if t.dtype is not dtype or t.shape != (T, heads, dim):
        raise ValueError(f"{what}: wanted {dtype} of shape {(T, heads, dim)}, got {t.dtype} "
                         f"{tuple(t.shape)}")
    row, head, column = t.stride()
    if column != 1:
        raise ValueError(f"{what}: columns must lie one behind the other, their stride is {column}")
    if t.get_device() != gpu:
        raise ValueError(f"{what}: wanted on the current GPU, is on {t.device}")
    return t.data_ptr(), row, head


def append_kv(cache: PagedKVCache, layer: int, k, v, slot_mapping, *, rotation: Rotation | None = None,
              positions=None, q=None, q_out=None, stream=None):
    """Rotate k [T, n_kv_heads, head_dim] by ``positions`` [T], round it and v [T, n_kv_heads, v_dim]
    to the cache's type and write row t to flat slot slot_mapping[t] of ``layer``'s pool.  Slots
    outside the pool are skipped; the others are distinct.  With q [T, H, head_dim] its rows are
    rotated the same way and returned, in ``q_out`` or a new tensor [T, H, head_dim] of the cache's
    type (rows of skipped slots, too), which shares no memory with q, k, v or the cache.  k, v and
    q are fp32 or 16-bit rows of one type; slices of one projection's rows are taken as they are.
    Without ``rotation`` nothing is turned."""
    gpu, T, rows = _gpu(), k.shape[0], k.dtype
    heads, dim, v_dim, page = cache._shape
    code = _row_code(rows)
    if T > _INT_MAX:
        raise ValueError(f"k: {T} rows do not fit 32 bits")
    if code is None:
        raise ValueError(f"k: wanted float32, float16 or bfloat16 rows, got {rows}")
    ka = _rows("k", k, heads, dim, T, rows, gpu)
    va = _rows("v", v, heads, v_dim, T, rows, gpu)
    qa, H, out = (None, 0, 0), heads, None
    if q is not None:
        H = q.shape[1]
        if H > _INT_MAX:
            raise ValueError(f"q: {H} heads do not fit 32 bits")
        qa = _rows("q", q, H, dim, T, rows, gpu)
        if q_out is None:
            with _allocating_on(stream):
                q_out = _torch().empty((T, H, dim), dtype=cache._dtype, device=q.device)
        out = _check("q_out", q_out, (T, H, dim), cache._dtype, gpu)
    slots = _ints("slot_mapping", slot_mapping, T, gpu)
    at, turn = None, _NO_ROTATION
    if rotation is not None:
        if positions is None:
            raise ValueError("positions: a rotation needs them")
        at = _ints("positions", positions, T, gpu)
        if rotation._place != gpu:
            raise ValueError(f"rotation: wanted on the current GPU, is on {rotation.frequencies.device}")
        turn = rotation._args
    check(lib().mla_append_kv(stream_handle(stream), T, H, heads, dim, v_dim, page, cache.dtype, code,
                              *ka, *va, *qa, at, *turn, slots, cache.num_pages,
                              cache._layer_address(layer, gpu), out))
    return q_out if q is not None else None


class KVAttentionPlan:
    """What ``plan_kv_attention`` built, for ``kv_attention`` calls over the same batch.  It keeps the
    tensors and sizes that it was made of: setting a field of the batch later changes nothing for
    its calls."""

    def __init__(self, batch: RaggedBatch, cache: PagedKVCache, n_heads: int, rows: int,
                 max_q_len: int, window: int | None, sinks: int, words):
        self.batch, self.n_heads, self.rows = batch, n_heads, rows
        self.max_q_len, self.window, self.sinks = max_q_len, window, sinks
        self.words = words  # the plan itself (device int32)
        self.info = None    # host copy of its info once read_info has been called
        heads, dim, v_dim, page = cache._shape
        self._cache_shape, self._dtype_code, self._dtype = cache._shape, cache.dtype, cache._dtype
        self._sizes = batch.B, rows, n_heads, heads, dim, v_dim, page, max_q_len, window or 0, sinks
        self._table = ptr(batch.page_table), batch.max_pages
        self._pool_pages = batch.num_pool_pages
        self._q_shape, self._out_shape = (rows, n_heads, dim), (rows, n_heads, v_dim)
        self._tensors = batch.page_table, words
        self._device, self._gpu = words.device, words.get_device()
        self._words = ptr(words), 4 * words.numel()
        self._workspace_bytes = int(lib().mla_kv_workspace_bytes(*self._sizes))

    def read_info(self, stream=None):
        """Synchronise and return [jobs, 0, jobs of few rows, jobs of many, partial rows, query rows,
        ..]; raises when the batch is invalid.  Calls after it launch no more workgroups than the
        plan has jobs, unless the plan was made in a captured graph: each replay builds that one
        anew, and its jobs change (before the first one it holds nothing:
        calls with it come behind a replay)."""
        import numpy as np
        h = np.zeros(PLAN_INFO_INTS, np.int32)
        check(lib().mla_read_kv_plan_info(stream_handle(stream), self._words[0], h.ctypes.data))
        if not self._captured:
            self.info, self._own_info = h.copy(), h  # (calls read the second)
            self._info = h.ctypes.data
        return h.tolist()

    _info = None
    _captured = False  # made in a captured graph


def plan_kv_attention(batch: RaggedBatch, cache: PagedKVCache, n_heads: int, *,
                      rows: int | None = None, max_q_len: int | None = None,
                      window: int | None = None, sinks: int = 0, stream=None) -> KVAttentionPlan:
    """Plan the attention of a batch over caches of this shape (one launch): which workgroup takes
    which query rows over which keys.  ``rows``: query rows of the calls (default the batch's
    max_rows); ``max_q_len``: at least every session's q_len (default ``rows``; a tighter bound makes
    a smaller plan and workspace).  ``window``: a row sees the last ``window`` keys up to its own and
    the first ``sinks`` ones; None: all keys up to its own.  The plan serves every such layer's
    ``kv_attention``."""
    torch, gpu = _torch(), _gpu()
    rows = batch.max_rows if rows is None else rows
    max_q_len = max(rows, 1) if max_q_len is None else max_q_len
    _ints_of_c(n_heads=n_heads, rows=rows, max_q_len=max_q_len, window=window or 0, sinks=sinks)
    if window is not None and window < 1:
        raise ValueError(f"window: {window}, wanted at least 1 (None: no window)")
    if batch.page_size != cache.page_size or batch.num_pool_pages > cache.num_pages:
        raise ValueError(f"cache: pages of {cache.page_size} tokens, {cache.num_pages} of them; the "
                         f"batch has {batch.page_size} and {batch.num_pool_pages}")
    sizes = batch.B, rows, n_heads, *cache._shape, max_q_len, window or 0, sinks
    n = int(lib().mla_kv_plan_bytes(*sizes))
    if n == 0:
        raise ValueError(f"plan_kv_attention: {lib().mla_last_error().decode(errors='replace')}")
    info = _check_list("batch", batch.info, gpu)
    with _allocating_on(stream):
        words = torch.empty(n // 4, dtype=torch.int32, device=batch.info.device)
        captured = words.is_cuda and torch.cuda.is_current_stream_capturing()
    check(lib().mla_plan_kv_attention(stream_handle(stream), *sizes, ptr(batch.cu_seqlens_q),
                                      ptr(batch.cu_seqlens_k), info, ptr(words), n))
    plan = KVAttentionPlan(batch, cache, n_heads, rows, max_q_len, window, sinks, words)
    plan._captured = captured
    return plan


def kv_attention_workspace(plan: KVAttentionPlan):
    """Workspace of ``kv_attention`` calls with this plan (or one of the same sizes).  Calls that
    share one are ordered on one stream."""
    return _torch().empty(max(plan._workspace_bytes, 16), dtype=_torch().uint8, device=plan._device)


def kv_attention(plan: KVAttentionPlan, cache: PagedKVCache, layer: int, q, scale: float, *, out=None,
                 lse=None, workspace=None, stream=None):
    """Attention of every query row of the plan's batch over its session's keys and values in
    ``layer`` of ``cache``: q [rows, H, head_dim] in the cache's type; returns out [rows, H, v_dim] in
    it (and fills lse [rows, H], fp32, if given).  ``out`` may be q itself where v_dim is head_dim, and
    shares no memory with q or the cache otherwise.  Rows past the batch's are left as they were, and
    over a failed plan (``KVAttentionPlan.read_info`` raises) all of them: zero in a tensor that the
    call makes."""
    torch, gpu = _torch(), _gpu()
    if cache._shape != plan._cache_shape or cache.dtype != plan._dtype_code:
        raise ValueError(f"cache: the plan is for (n_kv_heads, head_dim, v_dim, page_size) "
                         f"{plan._cache_shape} in {plan._dtype}, this one has {cache._shape} in "
                         f"{cache._dtype}")
    if cache.num_pages < plan._pool_pages:
        raise ValueError(f"cache: {cache.num_pages} pages, the batch's ids go up to "
                         f"{plan._pool_pages}")
    if plan._gpu != gpu:
        raise ValueError(f"plan: wanted on the current GPU, is on {plan._device}")
    if out is None or workspace is None:
        with _allocating_on(stream):
            if out is None:
                out = torch.zeros(plan._out_shape, dtype=plan._dtype, device=q.device)
            if workspace is None:
                workspace = kv_attention_workspace(plan)
    check(lib().mla_kv_attention(
        stream_handle(stream), *plan._sizes, plan._dtype_code, scale, *plan._table, plan._pool_pages,
        cache._layer_address(layer, gpu), _check("q", q, plan._q_shape, plan._dtype, gpu),
        *plan._words, plan._info, _check("out", out, plan._out_shape, plan._dtype, gpu),
        None if lse is None else _check("lse", lse, plan._q_shape[:2], torch.float32, gpu),
        _check("workspace", workspace, (workspace.numel(),), torch.uint8, gpu), workspace.numel()))
    return out


__all__ = ["PagedKVCache", "Rotation", "append_kv", "KVAttentionPlan", "plan_kv_attention",
           "kv_attention_workspace", "kv_attention"]
