"""Outputs of the key-value cache's C entry points that lie over what the call reads (CPU: a call that is
let through fails at its launch, with MLA_ERR_GPU)."""
import ctypes

import pytest
import torch

INVALID, OK = 1, (0, 5)


@pytest.fixture(scope="module")
def L():
    if torch.cuda.is_available():
        pytest.skip("addresses of host memory, which no GPU may see")
    import cpp_inference_train_engine_amd as mla
    return mla.lib()


@pytest.fixture(scope="module")
def at():
    buf = ctypes.create_string_buffer(1 << 16)
    a = ctypes.addressof(buf)
    yield a - a % 256 + 256
    del buf


def test_append(L, at):
    """3 tokens of 4 heads on kv 2 x 16, values 32 wide, fp32 rows: q_out has 384 bytes, k's rows of 128
    bytes are 256 apart, v's of 256 are 512 apart, a page has 16 tokens of 2 x 48 16-bit words."""
    k, v, q, pages = at + 8192, at + 16384, at + 24576, at + 32768

    def call(q_out, k=k, v=v, k_head=16, T=3, fn=L.mla_append_kv):
        return fn(None, T, 4, 2, 16, 32, 16, 0, 2, k, 64, k_head, v, 128, 32, q, 64, 16, None, None, 0, 0, 1, at, 2,
                  pages, q_out)
    size = 3 * 4 * 16 * 2
    for base, behind in ((k, 2 * 256 + 128), (v, 2 * 512 + 256), (q, 2 * 256 + 256), (pages, 2 * 16 * 2 * 48 * 2)):
        assert call(base - size) in OK and call(base + behind) in OK, hex(base - at)
        for d in (16 - size, 0, 16, behind - 16):
            assert call(base + d) == INVALID, (hex(base - at), d)
            assert b"q_out overlaps" in L.mla_last_error()
    # heads one before the other: k's rows begin 64 bytes earlier
    assert call(k - 64 - size, k_head=-16) in OK and call(k - 64 - size + 16, k_head=-16) == INVALID
    assert call(k, T=0) == 0


def test_append_without_queries(L, at):
    assert L.mla_append_kv(None, 3, 4, 2, 16, 32, 16, 0, 2, at + 8192, 64, 16, at + 16384, 128, 32, None, 0, 0, None,
                           None, 0, 0, 1, at, 2, at + 32768, at + 8192) in OK


@pytest.mark.gpu
def test_append_over_its_own_rows(gpu):
    """q_out in the memory of k's, v's or q's rows or of the cache is refused, behind them it is taken."""
    cache = gpu.PagedKVCache(1, 2, 16, 2, 32, dtype=0)
    x = torch.randn((3, (4 + 2 + 2) * 32 + 4 * 32), device="cuda").half()
    q, k, v = (x[:, a:a + 32 * n].unflatten(1, (n, 32)) for a, n in ((0, 4), (128, 2), (192, 2)))
    slots = torch.arange(3, dtype=torch.int32, device="cuda")
    call = lambda k, v, q, out: gpu.append_kv(cache, 0, k, v, slots, q=q, q_out=out)
    apart = [t.contiguous() for t in (k, v, q)]
    room = x.view(-1)[:3 * 128].view(3, 4, 32)  # (over the first rows of x)
    for rows in ((k, apart[1], apart[2]), (apart[0], v, apart[2]), (apart[0], apart[1], q)):
        with pytest.raises(gpu.MlaError, match="overlaps"):
            call(*rows, room)
    with pytest.raises(gpu.MlaError, match="overlaps the pages"):
        call(*apart, cache.pages.view(-1)[:3 * 128].view(3, 4, 32))
    assert torch.equal(call(*apart, room), apart[2])
    assert torch.equal(cache.keys(0)[0, :, :3].transpose(0, 1), apart[0])


SIZES = (2, 4, 8, 4, 64, 64, 64, 3, 0, 0)  # 4 rows of 8 heads of 64: q and out 4,096 bytes, lse 128


def test_attention(L):
    ws_bytes = L.mla_kv_workspace_bytes(*SIZES)
    pool = 2 * 2 * L.mla_kv_page_words(4, 64, 64, 64)
    buf = ctypes.create_string_buffer(ws_bytes + pool + (1 << 16))
    a = ctypes.addressof(buf)
    a += 256 - a % 256
    plan, q, out, lse, pages, ws = a, a + 4096, a + 16384, a + 24576, a + 32768, a + 32768 + pool

    def call(q=q, out=out, lse=lse, pages=pages, ws=ws, sizes=SIZES):
        return L.mla_kv_attention(None, *sizes, 0, 0.1, plan, 4, 2, pages, q, plan, 1 << 40, None, out, lse, ws,
                                  ws_bytes)
    assert call() in OK and call(lse=None) in OK and call(out=q + 4096) in OK and call(out=q - 4096) in OK
    assert call(out=q) in OK  # (out may be q itself)
    for kw in (dict(out=q + 16), dict(out=q - 4080), dict(lse=q + 4092), dict(lse=q), dict(ws=q), dict(out=pages),
               dict(out=pages + pool - 16), dict(lse=pages - 124), dict(ws=pages), dict(ws=pages + pool - 256),
               dict(lse=out), dict(lse=out + 4092), dict(out=ws), dict(lse=ws + 256), dict(out=ws - 4080)):
        assert call(**kw) == INVALID, kw
        assert b"apart" in L.mla_last_error()
    # values of another width than the keys: a row of out lies over another row of q
    other = (2, 4, 8, 4, 64, 48, 64, 3, 0, 0)
    assert call(out=q, sizes=other) == INVALID and call(sizes=other) in OK


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("H,KH,D,page", [(8, 8, 64, 64), (32, 8, 128, 64), (4, 2, 80, 16), (4, 4, 256, 32)])
def test_attention_in_place_of_its_queries(gpu, H, KH, D, page, dtype):
    """out=q gives the rows that another tensor gets: decode rows, drafts, chunks, cut or not."""
    from kv_reference import Batch, say
    say(f"in place {H} {KH} {D} {dtype}")
    c = Batch(H, KH, D, D, page, dtype, [(700, 1), (30, 4), (100, 290), (0, 33), (20000, 3), (9000, 1)], seed=3)
    batch, cache, q = c.device(gpu)
    for window in (None, 100):
        plan = gpu.plan_kv_attention(batch, cache, H, rows=c.rows, max_q_len=290, window=window)
        want = gpu.kv_attention(plan, cache, 0, q, c.scale)
        x = q.clone()
        assert gpu.kv_attention(plan, cache, 0, x, c.scale, out=x) is x
        assert torch.equal(x, want)
        wide = torch.zeros((c.rows + 1, H, D), dtype=q.dtype, device="cuda")
        wide[1:] = q
        with pytest.raises(gpu.MlaError, match="apart"):
            gpu.kv_attention(plan, cache, 0, wide[1:], c.scale, out=wide[:-1])
