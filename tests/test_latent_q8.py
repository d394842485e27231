"""The 8-bit latent cache: append and read-back against the definition, bit for bit."""
import ctypes

import numpy as np
import pytest

import latent_reference as ref
from cpp_inference_train_engine_amd.workloads import to_bits

SHAPES = [  # kv, rope, page: both record forms (an even and an odd number of 32-column blocks)
    (32, 8, 16), (64, 0, 32), (96, 24, 48), (128, 16, 64), (160, 40, 16), (512, 64, 64)]


def _rows(rng, n, kv, dtype):
    """Blocks of every kind: ordinary, tiny, huge, zero, one large value among small ones, maxima
    at and just past a power-of-two limit, infinities, NaN, halves between two e4m3 values."""
    x = rng.standard_normal((n, kv)).astype(np.float32)
    b = x.reshape(n, kv // 32, 32)
    kinds = rng.integers(0, 10, (n, kv // 32))
    lo, hi = ref.K_RANGE[dtype]
    with np.errstate(over="ignore"):
        b[kinds == 1] *= np.float32(2.0 ** (lo - 6))
        b[kinds == 2] *= np.float32(2.0 ** min(hi + 6, 100))
    b[kinds == 3] = 0
    one = kinds == 4
    b[one] *= np.float32(1e-3)
    b[one, 5] = 300
    at = kinds == 5
    b[at] = np.clip(b[at], -1, 1)
    b[at, 7] = 448 * 2.0 ** -3
    past = kinds == 6
    b[past] = np.clip(b[past], -1, 1)
    b[past, 9] = np.nextafter(np.float32(448 * 2.0 ** -3), np.float32(1e9))
    odd = kinds == 7
    b[odd, 3], b[odd, 17], b[odd, 31] = np.inf, -np.inf, np.nan
    half = kinds == 8  # 448 sets k = 0: multiples of half a step of each binade
    b[half] = rng.integers(-31, 32, (int(half.sum()), 32)) / 16 * 2.0 ** rng.integers(
        -9, 8, (int(half.sum()), 32))
    b[half, 0] = 448
    b[kinds == 9] = np.float32(3e38) * np.sign(b[kinds == 9])
    return x


def test_the_reference_quantiser_rounds_to_the_nearest():
    """Of the oracle itself: no e4m3 value of the block's scale is nearer, and every stored value
    is one of the 16-bit type."""
    rng = np.random.default_rng(0)
    for dtype in (0, 1):
        x = _rows(rng, 200, 64, dtype)
        byte, k = ref.quantise(x, dtype)
        v = ref.e4m3_values()[byte].reshape(200, 2, 32) * 2.0 ** k[..., None]
        b = x.astype(np.float64).reshape(200, 2, 32)
        fine = np.isfinite(b)
        assert np.isnan(v[~fine]).all() and np.isfinite(v[fine]).all()
        grid = ref.e4m3_values()[:127][None] * 2.0 ** k.reshape(-1, 1)  # [blocks, 127]
        near = np.abs(np.abs(b).reshape(-1, 32, 1) - grid[:, None]).min(2).reshape(200, 2, 32)
        assert (np.abs(np.abs(v) - np.abs(b))[fine] == near[fine]).all()
        with np.errstate(over="ignore"):
            bits = to_bits(v.astype(np.float32), dtype).reshape(v.shape)
        assert (ref.from_bits(bits, dtype)[fine] == v[fine]).all()


def test_refusals_of_the_8_bit_cache():
    import cpp_inference_train_engine_amd as mla
    L = mla.lib()
    buf = ctypes.create_string_buffer(4096)
    a = ctypes.addressof(buf)
    a += -a % 256
    assert L.mla_q8_page_bytes(64, 128, 16) == 64 * 164
    assert L.mla_q8_page_bytes(64, 512, 64) == 64 * 656
    for shape in ((60, 128, 16), (64, 120, 16), (64, 128, 12), (64, 544, 16), (64, 128, 72),
                  (0, 128, 16), (64, 0, 16)):
        assert L.mla_q8_page_bytes(*shape) == 0
    ok = (None, 4, 128, 16, 64, 0, a, a, a, 10, a)

    def append(**kw):
        names = ("stream", "T", "kv", "rope", "page", "dtype", "ckv", "krope", "slots", "pool", "pages")
        v = dict(zip(names, ok), **kw)
        return L.mla_append_latent_q8(*[v[n] for n in names])

    def read(**kw):
        names = ("stream", "T", "kv", "rope", "page", "dtype", "slots", "pool", "pages", "ckv", "krope")
        v = dict(zip(names, (None, 4, 128, 16, 64, 0, a, 10, a, a, a)), **kw)
        return L.mla_read_latent_q8(*[v[n] for n in names])

    for f in (append, read):
        assert f(T=-1) == 1 and f(dtype=2) == 1 and f(pool=-1) == 1 and f(page=0) == 1
        assert f(kv=100) == 3 and f(kv=544) == 3 and f(rope=4) == 3 and f(page=40) == 3
        assert f(slots=None) == 1 and f(ckv=None) == 1 and f(krope=None) == 1 and f(pages=None) == 1
        assert f(pages=a + 8) == 1 and b"16 bytes" in L.mla_last_error()
        assert f(T=0, slots=None, ckv=None, pages=None) == 0  # nothing to do
    assert read(ckv=a + 2) == 1 and read(krope=a + 8) == 1


def test_python_wrappers_refuse_wrong_tensors(monkeypatch):
    import torch
    import cpp_inference_train_engine_amd as mla
    monkeypatch.setattr(mla.ops, "_gpu", lambda: 0)
    with pytest.raises(ValueError, match="multiple of 16"):
        mla.QuantizedLatentCache(1, 2, 60, 128, 16, device="cpu")
    with pytest.raises(ValueError, match="storage"):
        mla.QuantizedLatentCache(1, 2, 64, 128, 16, storage=torch.zeros((1, 2, 5), dtype=torch.uint8))
    c = mla.QuantizedLatentCache(1, 2, 64, 128, 16, device="cpu")
    assert c.record_bytes == 64 * 164
    x, r = torch.zeros((3, 128)), torch.zeros((3, 16))
    s = torch.zeros(3, dtype=torch.int32)
    for bad, what in (((x[:, :64], r, s), "ckv"), ((x.half(), r, s), "ckv"),
                      ((torch.zeros((128, 3)).T, r, s), "ckv"), ((x, r, s), "GPU")):
        with pytest.raises(ValueError, match=what):
            mla.append_latent_q8(c, 0, *bad)
    with pytest.raises(ValueError, match="slot_mapping"):
        mla.read_latent_q8(c, 0, s.long())
    with pytest.raises(ValueError, match="GPU"):
        mla.read_latent_q8(c, 0, s)


def _say(*a):
    print(*a, flush=True)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("kv,rope,page", SHAPES)
def test_append_and_read_back(gpu, kv, rope, page, dtype):
    """Every byte of the pool, and every bit of the rows read back, for sizes from one row on;
    slots outside the pool are skipped by both, and what no row names stays."""
    import torch
    dev = lambda x: torch.from_numpy(np.ascontiguousarray(x)).cuda()
    rng = np.random.default_rng(kv + rope + dtype)
    P = 9
    tdt = torch.float16 if dtype == 0 else torch.bfloat16
    for T in (1, 3, 17, 100):
        _say(f"append_q8 kv={kv} rope={rope} page={page} dtype={dtype} T={T}")
        x, key = _rows(rng, T, kv, dtype), rng.standard_normal((T, rope)).astype(np.float32)
        slots = rng.permutation(P * page)[:T].astype(np.int32)
        if T >= 17:
            slots[[2, 9, 11]] = [-1, P * page, 2 ** 31 - 1]
            if rope:
                key[0, 0], key[1, 1], key[3, 2] = np.inf, np.nan, 1e30
        cache = gpu.QuantizedLatentCache(2, P, page, kv, rope, dtype=dtype)
        start = rng.integers(0, 256, cache.pages.shape, dtype=np.uint8)
        cache.pages.copy_(dev(start))
        gpu.append_latent_q8(cache, 1, dev(x), dev(key), dev(slots))
        got = cache.pages.cpu().numpy()
        byte, k = ref.quantise(x, dtype)
        want = start.copy()
        with np.errstate(over="ignore"):
            ref.q8_store(want[1], page, kv, rope, slots, byte, to_bits(key, dtype).reshape(T, rope), k)
        if rope:  # a NaN's bits are the conversion's own
            at = ref.q8_order(page, kv, rope)[1][slots[1] % page, 1] if T >= 17 else None
            if at is not None:
                p = slots[1] // page
                bits = int(got[1][p, at]) | int(got[1][p, at + 1]) << 8
                assert np.isnan(ref.from_bits(bits, dtype))
                want[1][p, at:at + 2] = got[1][p, at:at + 2]
        assert np.array_equal(got, want)

        lat, keys = ref.q8_rows(got[1], page, kv, rope, dtype)
        inside = (slots >= 0) & (slots < P * page)
        twice = np.concatenate([slots, slots[:1]])  # a slot may be read twice
        fill = 7.0
        a = torch.full((T + 1, kv), fill, dtype=tdt, device="cuda")
        b = torch.full((T + 1, rope), fill, dtype=tdt, device="cuda")
        gpu.read_latent_q8(cache, 1, dev(twice), ckv=a, krope=b)
        inside = np.concatenate([inside, inside[:1]])
        safe = np.where(inside, twice, 0)
        np.testing.assert_array_equal(a.double().cpu().numpy(),
                                      np.where(inside[:, None], lat[safe], fill))
        np.testing.assert_array_equal(b.double().cpu().numpy(),
                                      np.where(inside[:, None], keys[safe], fill))
        made, _ = gpu.read_latent_q8(cache, 1, dev(slots))
        np.testing.assert_array_equal(made.double().cpu().numpy(),
                                      np.where(inside[:T, None], lat[safe[:T]], 0.0))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [0, 1])
def test_every_value_at_every_scale_reads_back_exactly(gpu, dtype):
    import torch
    lo, hi = ref.K_RANGE[dtype]
    n = (hi - lo + 1) * 8  # 8 slots of 32 columns: the 256 bytes
    page, P = 64, -(-n // 64)
    pool = np.zeros((P, 64 * 33), np.uint8)
    byte = np.tile(np.arange(256, dtype=np.uint8).reshape(8, 32), (hi - lo + 1, 1))
    k = np.repeat(np.arange(lo, hi + 1), 8)[:, None]
    ref.q8_store(pool, page, 32, 0, range(n), byte, np.zeros((n, 0), np.uint16), k)
    _say(f"read_q8, all values at all scales, dtype={dtype}")
    cache = gpu.QuantizedLatentCache(1, P, page, 32, 0, dtype=dtype,
                                     storage=torch.from_numpy(pool[None]).cuda())
    rows, none = gpu.read_latent_q8(cache, 0, torch.arange(n, dtype=torch.int32, device="cuda"))
    assert none.shape == (n, 0)
    np.testing.assert_array_equal(rows.double().cpu().numpy(),
                                  ref.e4m3_values()[byte] * 2.0 ** k)


@pytest.mark.gpu
def test_append_of_unaligned_rows_on_a_side_stream(gpu):
    """fp32 rows at any multiple of 4 bytes, on a stream of the caller's."""
    import torch
    rng = np.random.default_rng(5)
    flat = torch.from_numpy(rng.standard_normal(1 + 40 * 144).astype(np.float32)).cuda()
    x, key = flat[1:1 + 40 * 128].view(40, 128), flat[1 + 40 * 128:].view(40, 16)
    slots = torch.arange(40, dtype=torch.int32, device="cuda")
    a, b = (gpu.QuantizedLatentCache(1, 1, 64, 128, 16) for _ in range(2))
    _say("append_q8, unaligned rows, side stream")
    gpu.append_latent_q8(a, 0, x.clone(), key.clone(), slots)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        gpu.append_latent_q8(b, 0, x, key, slots)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(a.pages, b.pages)


@pytest.mark.gpu
def test_python_wrappers_refuse_wrong_tensors_on_the_gpu(gpu):
    import torch
    c = gpu.QuantizedLatentCache(1, 2, 64, 128, 16)
    x, r = torch.zeros((3, 128), device="cuda"), torch.zeros((3, 16), device="cuda")
    s = torch.zeros(3, dtype=torch.int32, device="cuda")
    for bad, what in (((x, r[:2], s), "krope"), ((x, r, s.long()), "slot_mapping"),
                      ((x, r, s[:2]), "slots for"), ((x, r.cpu(), s), "GPU")):
        with pytest.raises(ValueError, match=what):
            gpu.append_latent_q8(c, 0, *bad)
    for kw in (dict(ckv=x), dict(krope=r), dict(ckv=x[:2].half())):
        with pytest.raises(ValueError, match="krope" if "krope" in kw else "ckv"):
            gpu.read_latent_q8(c, 0, s, **kw)
