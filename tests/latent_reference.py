"""Definitions in 64 bits that the tests of the 8-bit latent cache and of planned attention compare
with: the quantiser, the page records, the attention."""
import numpy as np

K_RANGE = {0: (-15, 7), 1: (-117, 119)}  # of a block's scale 2^k, by dtype (0 fp16, 1 bf16)
HALF_STEP = {0: 2.0 ** -11, 1: 2.0 ** -8}


def from_bits(bits, dtype):
    bits = np.asarray(bits, np.uint16)
    if dtype == 0:
        return np.ascontiguousarray(bits).view(np.float16).astype(np.float64)
    return (bits.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


def e4m3_values():
    """The value of every e4m3 byte."""
    b = np.arange(256)
    power, frac = b // 8 % 16, b % 8
    v = np.where(power == 0, frac / 8 * 2.0 ** -6, (1 + frac / 8) * 2.0 ** (power - 7.0))
    v[b % 128 == 127] = np.nan
    return np.where(b >= 128, -v, v)


def quantise(x, dtype):
    """(bytes [n, kv], k [n, kv / 32]) of fp32 rows; a non-finite value is the byte 0x7f."""
    lo, hi = K_RANGE[dtype]
    b = np.asarray(x, np.float32).astype(np.float64).reshape(len(x), -1, 32)
    fine = np.isfinite(b)
    amax = np.where(fine, np.abs(b), 0).max(2)
    k = np.full(amax.shape, lo)
    for n in range(lo, hi):  # the smallest power of two that holds the block
        k = np.where(amax > 448 * 2.0 ** n, n + 1, k)
    y = np.clip(np.where(fine, b, 0) / 2.0 ** k[..., None], -448, 448)
    sizes = e4m3_values()[:127]  # ascending, 0 .. 448; nearest, ties to the even byte
    at = np.searchsorted(sizes, np.abs(y))
    below, above = np.maximum(at - 1, 0), np.minimum(at, 126)
    down, up = np.abs(y) - sizes[below], sizes[above] - np.abs(y)
    byte = np.where((up < down) | ((up == down) & (above % 2 == 0)), above, below)
    byte = np.where(np.signbit(b), byte + 128, byte)
    byte = np.where(fine, byte, 127)
    return byte.reshape(len(x), -1).astype(np.uint8), k


def latent_byte(slot, r, kv):
    t, n, j, g, e = slot // 16, slot % 16, r // 32, r % 32 // 8, r % 8
    odd = (kv // 32) % 2 == 1 and j == kv // 32 - 1
    return t * 16 * kv + (j * 512 + (16 * g + n) * 8 + e if odd else
                          j // 2 * 1024 + (16 * g + n) * 16 + j % 2 * 8 + e)


def rope_byte(slot, c, page, kv, rope):
    return page * kv + 2 * ((slot // 16 * (rope // 8) + c // 8) * 128 + slot % 16 * 8 + c % 8)


def scale_byte(slot, j, page, kv, rope):
    return page * (kv + 2 * rope) + slot * (kv // 32) + j


_ORDER = {}


def q8_order(page, kv, rope):
    """Byte offsets [page, kv], [page, rope] and [page, kv / 32] of a record's tokens."""
    key = (page, kv, rope)
    if key not in _ORDER:
        _ORDER[key] = (
            np.array([[latent_byte(s, r, kv) for r in range(kv)] for s in range(page)]),
            np.array([[rope_byte(s, c, page, kv, rope) for c in range(rope)]
                      for s in range(page)], int).reshape(page, rope),
            np.array([[scale_byte(s, j, page, kv, rope) for j in range(kv // 32)]
                      for s in range(page)]))
    return _ORDER[key]


def q8_store(pool, page, kv, rope, slots, byte, key_bits, k):
    """Write rows into pool [pages, record] (uint8) at flat slots; slots outside are skipped."""
    lat, key, sc = q8_order(page, kv, rope)
    for t, s in enumerate(slots):
        if 0 <= s < len(pool) * page:
            rec, o = pool[s // page], s % page
            rec[lat[o]] = byte[t]
            rec[key[o]] = key_bits[t] & 255
            rec[key[o] + 1] = key_bits[t] >> 8
            rec[sc[o]] = k[t] + 127


def q8_rows(pool, page, kv, rope, dtype):
    """Every token row of a pool: latents [slots, kv] and rope keys [slots, rope] in 64 bits."""
    lat, key, sc = q8_order(page, kv, rope)
    v = e4m3_values()[pool[:, lat]].reshape(-1, kv // 32, 32)
    with np.errstate(over="ignore"):
        v = v * 2.0 ** (pool[:, sc].astype(np.float64).reshape(-1, kv // 32, 1) - 127)
    bits = pool[:, key].astype(np.uint16) | pool[:, key + 1].astype(np.uint16) << 8
    return v.reshape(-1, kv), from_bits(bits.reshape(len(pool) * page, rope), dtype)


def rows16(pool, page, kv, rope, dtype):
    """The same of a 16-bit pool [pages, words] (uint16)."""
    from cpp_inference_train_engine_amd.ops import latent_word, rope_word
    s = np.arange(page)[:, None]
    lat = latent_word(s, np.arange(kv)[None], page, kv, rope)
    key = rope_word(s, np.arange(rope)[None], page, kv, rope)
    return (from_bits(pool[:, lat].reshape(-1, kv), dtype),
            from_bits(pool[:, key].reshape(len(pool) * page, rope), dtype))


def attention(q_latent, q_rope, latent, key, visible, scale):
    """One session in 64 bits: q [rows, H, .], keys [n, .], visible [rows, n] -> (out, lse, mass):
    mass = sum of the weights times |latent|, what roundings of the weights are relative to.  A row
    that sees nothing is 0 with lse -inf; a row that sees a NaN latent is NaN."""
    s = (np.einsum("rhk,nk->rhn", q_latent, np.nan_to_num(latent, nan=0.0)) +
         np.einsum("rhk,nk->rhn", q_rope, np.nan_to_num(key, nan=0.0))) * scale
    bad = np.isnan(latent).any(1) | np.isnan(key).any(1)
    s = np.where(visible[:, None], s, -np.inf)
    top = s.max(2, keepdims=True) if s.shape[2] else np.full(s.shape[:2] + (1,), -np.inf)
    e = np.exp(s - np.where(np.isfinite(top), top, 0))
    l = e.sum(2, keepdims=True)
    w = e / np.where(l > 0, l, 1)
    clean = np.nan_to_num(latent, nan=0.0)
    out, mass = w @ clean, w @ np.abs(clean)
    with np.errstate(divide="ignore"):
        lse = (top + np.log(l))[..., 0]
    hit = (visible & bad[None]).any(1)
    out[hit], lse[hit] = np.nan, np.nan
    return out, lse, mass
