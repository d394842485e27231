"""Argument checks of the key-value cache's C entry points, which touch no device (CPU)."""
import ctypes

import pytest


@pytest.fixture(scope="module")
def L():
    import cpp_inference_train_engine_amd as mla
    return mla.lib()


def buffers():
    buf = ctypes.create_string_buffer(1 << 12)
    a = ctypes.addressof(buf)
    return buf, a - a % 256 + 256


def test_page_words(L):
    assert L.mla_kv_page_words(8, 128, 128, 64) == 8 * 64 * 256
    assert L.mla_kv_page_words(3, 80, 16, 48) == 3 * 48 * 96
    for shape in ((8, 128, 128, 24), (8, 72, 128, 64), (8, 128, 272, 64), (0, 64, 64, 64), (8, 64, 64, 0),
                  (8, 64, 64, 65552), (70000, 256, 256, 65536)):
        assert L.mla_kv_page_words(*shape) == 0


def test_append_arguments(L):
    keep, a = buffers()

    def call(T=1, H=8, KH=8, D=64, DV=64, page=64, dtype=0, row=0, k=a, v=a, q=None, at=a, f=a, pairs=8,
             start=0, adjacent=1, slots=a, pool=1, pages=a, q_out=None):
        return L.mla_append_kv(None, T, H, KH, D, DV, page, dtype, row, k, 512, 64, v, 512, 64, q, 512, 64, at,
                               f, pairs, start, adjacent, slots, pool, pages, q_out)
    assert call(T=0) == 0
    for kw in (dict(T=-1), dict(H=0), dict(KH=0), dict(D=0), dict(dtype=2), dict(row=3), dict(adjacent=2),
               dict(pool=-1), dict(pairs=-1), dict(pairs=33), dict(start=-2), dict(start=1), dict(start=50),
               dict(pairs=2 ** 30, start=2), dict(start=2 ** 31 - 2), dict(k=None), dict(v=None), dict(slots=None),
               dict(pages=None), dict(at=None), dict(f=None), dict(q=a), dict(pages=a + 2),
               dict(q=a, q_out=a + 8), dict(q=a, q_out=a), dict(q=a, q_out=a + 16),
               dict(q=a + 512, q_out=a)):
        assert call(**kw) == 1, kw
        assert b"mla_append_kv" in L.mla_last_error()
    for kw in (dict(D=40), dict(DV=264), dict(page=8), dict(page=65552)):
        assert call(**kw) == 3, kw


def test_plan_and_call_arguments(L):
    keep, a = buffers()
    sizes = dict(B=2, rows=4, H=8, KH=4, D=64, DV=64, page=64, max_q=3, window=0, sinks=0)
    bad = [dict(B=-1), dict(rows=-1), dict(H=0), dict(H=6), dict(KH=0), dict(max_q=0), dict(window=-1),
           dict(window=4, sinks=-1), dict(sinks=1), dict(rows=2 ** 28), dict(B=2 ** 23)]
    assert L.mla_kv_plan_bytes(*sizes.values()) > 0 and L.mla_kv_workspace_bytes(*sizes.values()) > 0
    for kw in bad + [dict(D=40), dict(DV=300), dict(page=20)]:
        s = {**sizes, **kw}.values()
        assert L.mla_kv_plan_bytes(*s) == 0 and L.mla_kv_workspace_bytes(*s) == 0
        assert L.mla_plan_kv_attention(None, *s, a, a, a, a, 1 << 40) in (1, 3)
        assert L.mla_kv_attention(None, *s, 0, 0.1, a, 4, 4, a, a, a, 1 << 40, None, a, None, a, 1 << 40) in (1, 3)
    s = sizes.values()
    need = L.mla_kv_plan_bytes(*s)
    assert L.mla_plan_kv_attention(None, *s, a, a, a, a, need - 1) == 1
    assert L.mla_plan_kv_attention(None, *s, a, a, a, a + 4, need) == 1
    for i in range(4):
        p = [a] * 4
        p[i] = None
        assert L.mla_plan_kv_attention(None, *s, *p, need) == 1
    assert L.mla_read_kv_plan_info(None, None, a) == 1 and L.mla_read_kv_plan_info(None, a, None) == 1

    def call(dtype=0, scale=0.1, table=a, max_pages=4, pool=4, pages=a, q=a, plan=a, plan_bytes=need, info=None,
             out=a, ws=a, ws_bytes=1 << 40):
        return L.mla_kv_attention(None, *s, dtype, scale, table, max_pages, pool, pages, q, plan, plan_bytes, info,
                                  out, None, ws, ws_bytes)
    zeros = ctypes.create_string_buffer(64)  # (an info of no plan)
    for kw in (dict(dtype=2), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("inf")),
               dict(scale=float("nan")), dict(max_pages=-1), dict(pool=-1), dict(table=None), dict(pages=None),
               dict(q=None), dict(plan=None), dict(out=None), dict(ws=None), dict(pages=a + 2), dict(q=a + 4),
               dict(out=a + 8), dict(ws=a + 4), dict(plan=a + 4), dict(plan_bytes=need - 1), dict(ws_bytes=16),
               dict(info=ctypes.addressof(zeros))):
        assert call(**kw) == 1, kw
    # no session can have a key: nothing to do, nothing launched
    assert call(max_pages=0) == 0 and call(pool=0) == 0


def test_largest_sizes(L):
    """Sizes whose counts would pass 32 bits are refused."""
    keep, a = buffers()
    append = lambda heads: L.mla_append_kv(None, 0, heads, 1, 256, 256, 64, 0, 0, a, 512, 64, a, 512, 64, None, 512,
                                           64, a, a, 8, 0, 1, a, 1, a, None)
    assert append(2 ** 23 - 4) == 0 and append(2 ** 23) == 3 and append(2 ** 31 - 1) == 3
    # 2^22 sessions of 256 rows: jobs of 512 threads at width 256, of 256 below it
    sizes = lambda width: (2 ** 22, 2 ** 30, 1, 1, width, width, 64, 256, 0, 0)
    assert L.mla_kv_plan_bytes(*sizes(128)) > 0 and L.mla_kv_plan_bytes(*sizes(256)) == 0
    assert b"too large" in L.mla_last_error()
