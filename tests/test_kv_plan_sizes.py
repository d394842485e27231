"""A plan of the key-value cache's attention given to a call of other sizes, through the C entry point
(the Python one takes its sizes from the plan): the call is refused or writes nothing."""
import ctypes

import pytest
import torch

from kv_reference import Batch, near, say

NAMES = ("B", "rows", "H", "KH", "D", "DV", "page", "max_q_len", "window", "sinks")
# Two sets of sizes whose 32-bit hash, one multiplication for each size, is the same (0x1e4e6d61).
ALIKE = ((64, 512, 32, 8, 128, 128, 64, 12, 131072, 0), (64, 512, 32, 8, 128, 128, 64, 268, 234240, 0))


def make(gpu, sizes):
    """A batch for the sizes, its plan in a buffer large enough for any of this file's, and a call."""
    B, rows, H, KH, D, DV, page = sizes[:7]
    c = Batch(H, KH, D, DV, page, 1, [(40 + 5 * b, 1 + b % 3) for b in range(B)], seed=2)
    batch, cache, q = c.device(gpu)
    L, p = gpu.lib(), gpu.ptr
    need = max(L.mla_kv_plan_bytes(*s) for s in (sizes, *ALIKE))
    words = torch.zeros(need // 4 + 2 ** 20, dtype=torch.int32, device="cuda")
    n = 4 * words.numel()
    gpu.check(L.mla_plan_kv_attention(None, *sizes, p(batch.cu_seqlens_q), p(batch.cu_seqlens_k),
                                      p(batch.info), p(words), n))
    info = (ctypes.c_int32 * 8)()
    gpu.check(L.mla_read_kv_plan_info(None, p(words), info))
    wide = torch.zeros((2 * rows, 2 * H, 256), dtype=torch.bfloat16, device="cuda")
    wide.view(-1)[:q.numel()] = q.view(-1)
    out = torch.full_like(wide, 7)
    ws = torch.empty(2 ** 29, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()

    def call(s, host):
        st = L.mla_kv_attention(None, *s, 1, c.scale, p(batch.page_table), batch.max_pages,
                                batch.num_pool_pages * page // s[6], p(cache.pages), p(wide), p(words), n,
                                ctypes.addressof(info) if host else None, p(out), None, p(ws), ws.numel())
        torch.cuda.synchronize()
        return st

    return c, out, call


@pytest.mark.gpu
@pytest.mark.parametrize("first", [0, 1])
def test_sizes_that_hash_alike(gpu, first):
    say(f"sizes that hash alike {first}")
    c, out, call = make(gpu, ALIKE[first])
    assert call(ALIKE[1 - first], False) == 0 and (out == 7).all()
    assert call(ALIKE[1 - first], True) == 1 and (out == 7).all()
    for host in (False, True):
        out.fill_(7)
        assert call(ALIKE[first], host) == 0
        want, _, off, _ = c.expect()
        near(out.view(-1)[:c.rows * 32 * 128].view(c.rows, 32, 128), want, off, "out")
        assert (out.view(-1)[c.rows * 32 * 128:] == 7).all()


@pytest.mark.gpu
@pytest.mark.parametrize("window,sinks", [(0, 0), (30, 2)])
def test_each_size(gpu, window, sinks):
    say(f"each size {window}")
    sizes = (6, 13, 8, 4, 64, 48, 64, 3, window, sinks)
    c, out, call = make(gpu, sizes)
    for i, other in enumerate((7, 14, 16, 2, 48, 64, 128, 4, 31, 1)):
        s = list(sizes)
        s[i] = other
        if s[9] and not s[8]:
            s[8] = 30
        say(f"{NAMES[i]} {s}")
        assert call(s, False) == 0 and (out == 7).all()
        assert call(s, True) == 1 and (out == 7).all()
    assert call(sizes, True) == 0
    want, _, off, _ = c.expect(window or None, sinks)
    n = c.rows * 8 * 48
    near(out.view(-1)[:n].view(c.rows, 8, 48), want, off, "out")
    assert (out.view(-1)[n:] == 7).all()
