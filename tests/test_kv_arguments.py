"""What the Python wrappers of the key-value cache refuse before a kernel is called (CPU)."""
import pytest


@pytest.fixture(scope="module")
def mla():
    import cpp_inference_train_engine_amd as mla
    return mla


@pytest.mark.parametrize("dtype", [2, -1, 3])
def test_caches_hold_16_bit_words(mla, dtype):
    """DTYPE_F32 (2) is a type of appended rows."""
    assert mla.DTYPE_F32 == 2
    for make in (lambda: mla.PagedKVCache(1, 4, 64, 4, 64, dtype=dtype, device="cpu"),
                 lambda: mla.PagedLatentCache(1, 4, 64, 128, 16, dtype=dtype, device="cpu"),
                 lambda: mla.QuantizedLatentCache(1, 4, 64, 128, 16, dtype=dtype, device="cpu")):
        with pytest.raises(ValueError, match="dtype"):
            make()
    for dtype in (mla.DTYPE_F16, mla.DTYPE_BF16):
        assert mla.PagedKVCache(1, 4, 64, 4, 64, dtype=dtype, device="cpu").pages.element_size() == 2


WIDE = 2 ** 32 + 5  # a C int takes 5 of it


def test_sizes_past_32_bits(mla):
    import torch
    for shape in ((1, 4, WIDE + 59, 4, 64), (1, 4, 64, WIDE, 64), (1, 4, 64, 4, WIDE + 59),
                  (1, 4, 64, 4, 64, WIDE + 59)):
        with pytest.raises(ValueError, match="32 bits"):
            mla.PagedKVCache(*shape, device="cpu", storage=torch.zeros(1, dtype=torch.float16))
    for start in (2 ** 32, -2 ** 32, 2 ** 31):
        with pytest.raises(ValueError, match="32 bits"):
            mla.Rotation([1.0], start=start, device="cpu")


@pytest.mark.gpu
def test_sizes_of_calls_past_32_bits(gpu):
    import torch
    from kv_reference import Batch
    c = Batch(8, 4, 64, 48, 64, 0, [(100, 1), (20, 3)], seed=18)
    batch, cache, q = c.device(gpu)
    for kw in (dict(window=WIDE), dict(window=2 ** 32), dict(window=2 ** 31), dict(window=9, sinks=WIDE),
               dict(window=9, sinks=2 ** 32), dict(max_q_len=WIDE), dict(rows=WIDE), dict(n_heads=2 ** 32 + 8)):
        with pytest.raises(ValueError, match="32 bits"):
            gpu.plan_kv_attention(batch, cache, **{"n_heads": 8, "rows": 4, "max_q_len": 3, **kw})
    # the largest window and as many sinks see what no window does
    want = gpu.kv_attention(gpu.plan_kv_attention(batch, cache, 8, rows=4, max_q_len=3), cache, 0, q, 0.1)
    for sinks in (0, 2 ** 31 - 1):
        plan = gpu.plan_kv_attention(batch, cache, 8, rows=4, max_q_len=3, window=2 ** 31 - 1, sinks=sinks)
        assert torch.equal(gpu.kv_attention(plan, cache, 0, q, 0.1), want)
    # rows that are one row many times: more heads than an int holds
    slots = torch.zeros(1, dtype=torch.int32, device="cuda")
    k, v = torch.zeros((1, 4, 64), device="cuda"), torch.zeros((1, 4, 48), device="cuda")
    many = torch.zeros((1, 1, 64), device="cuda").expand(1, 2 ** 32 + 1, 64)
    with pytest.raises(ValueError, match="32 bits"):
        gpu.append_kv(cache, 0, k, v, slots, q=many, q_out=torch.zeros(1, device="cuda"))


@pytest.mark.gpu
def test_a_plans_info_is_its_own(gpu):
    """What a user does with ``plan.info`` changes nothing for the plan's calls."""
    import gc
    import torch
    from kv_reference import Batch
    c = Batch(8, 4, 64, 64, 64, 0, [(9000, 1), (20, 100)], seed=18)
    batch, cache, q = c.device(gpu)
    plan = gpu.plan_kv_attention(batch, cache, 8, rows=c.rows, max_q_len=100)
    want = gpu.kv_attention(plan, cache, 0, q, 0.1)
    read = plan.read_info()
    assert plan.info.tolist() == read
    for change in ("zero", "none"):
        if change == "zero":
            plan.info[:] = 0
        else:
            plan.info = None
            gc.collect()
        assert torch.equal(gpu.kv_attention(plan, cache, 0, q, 0.1), want), change
