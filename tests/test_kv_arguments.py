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
