"""The softmax weights of planned attention where they meet the latents: a weighted mean of equal
latents is the latent, whatever the weights are."""
import numpy as np
import pytest

import latent_reference as ref
from cpp_inference_train_engine_amd.workloads import to_bits
from test_latent_attention import FORMATS, _say, call, device, expect, make, put16


def equal_latents(H, kv, rope, page, dtype, q8, sessions, groups, seed):
    """A batch whose cached latents are all one row (exact in 8 bits too) and whose scores have two
    values.  Every 32nd key has score d and the others 0, d log2 units apart, so that next to the
    reference maximum the others weigh 2^5 (1 + 0.98 h), h half a step of the 16-bit type: rounded
    to that type all of them lose 0.98 h.  Returns the case, the latent, and the score's scale."""
    c = make(H, kv, rope, page, dtype, q8, sessions, groups, seed=seed)
    rng = np.random.default_rng(seed)
    row = ((8 + rng.integers(0, 8, kv)) / 8 * rng.choice([-1, 1], kv)).astype(np.float32)
    lists = list(zip(c.prefix_pages, c.prefix)) + list(zip(c.own_pages, c.ctx + c.q))
    for pages, n in lists:
        slots = c.flat(pages, int(n))
        key = np.zeros((len(slots), rope), np.float32)
        key[::32, 0] = 1
        x, kb = np.tile(row, (len(slots), 1)), to_bits(key, dtype).reshape(len(slots), rope)
        if q8:
            byte, k = ref.quantise(x, dtype)
            ref.q8_store(c.pool, page, kv, rope, slots, byte, kb, k)
        else:
            put16(c, slots, to_bits(x, dtype), kb)
    c.ql[:] = 0
    one = np.zeros(c.qr.shape, np.float32)
    one[..., 0] = 1
    c.qr[:] = to_bits(one, dtype).reshape(c.qr.shape)
    d = 1 - np.log2(1 + 0.98 * ref.HALF_STEP[dtype])
    return c, row, float(d * np.log(2))


SHAPES = [(8, 128, 16, 64), (128, 128, 16, 64), (128, 512, 64, 64), (16, 512, 64, 64), (16, 64, 16, 32),
          (128, 96, 8, 16), (8, 256, 32, 32), (128, 224, 8, 128), (8, 384, 16, 16), (128, 288, 64, 64)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,q8", FORMATS)
@pytest.mark.parametrize("H,kv,rope,page", SHAPES)
def test_a_mean_of_equal_latents_is_the_latent(gpu, H, kv, rope, page, dtype, q8):
    """The row before its rounding is the latent but for the sums in 32 bits, and weights that are
    off by 2^-17 each at most where they are carried in parts: within 1e-5 of it, and half a step
    of the type is 2^-12 of a value at least.  So its rounding gives the latent, bit for bit.  The
    score's two values are exact, ln of the mass carries 1e-5 for 32-bit sums and exponentials."""
    import torch
    sessions, groups = [(700, 1), (31, 4), (0, 1), (0, 40), (130, 1), (1500, 1)], [(3, 300), (1, 33)]
    c, row, scale = equal_latents(H, kv, rope, page, dtype, q8, sessions, groups, seed=H + kv)
    _say(f"equal latents H={H} kv={kv} rope={rope} dtype={dtype} q8={q8}")
    d = device(gpu, c)
    plan = gpu.plan_attention(d["batch"], H, kv, rows=d["rows"], max_q_len=d["max_q_len"],
                              prefixes=d["shared"])
    lse = torch.zeros((d["rows"], H), device="cuda")
    out = gpu.latent_attention(plan, d["pages"], d["ql"], d["qr"], scale, rope_dim=rope,
                               dtype=dtype, q8=q8, lse=lse)
    got = out.double().cpu().numpy()
    wrong = got != row
    assert not wrong.any(), f"{wrong.sum()} of {wrong.size}, worst {np.abs(got / row - 1).max()}"
    want = []
    for b, (n0, n) in enumerate(zip(c.ctx, c.q)):
        p = int(c.prefix[c.group_of(b)]) if c.group_of(b) >= 0 else 0
        for i in range(n):
            keys = n0 + i + 1
            high = -(-p // 32) + -(-keys // 32)
            want += [np.log(high * np.exp(scale) + (p + keys - high))] * H
    np.testing.assert_allclose(lse.double().cpu().numpy().reshape(-1), want, rtol=1e-5, atol=1e-5)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,q8", FORMATS)
@pytest.mark.parametrize("H,kv,rope,page", SHAPES)
def test_only_the_row_is_rounded_to_16_bits(gpu, H, kv, rope, page, dtype, q8):
    """Random contents.  A weight e with 2^E <= e < 2^(E+1) leaves at most 2^(E-8) (bf16) or
    2^(E-11) (fp16) behind its high part, and the low part half a step of that: 2^-17 e or 2^-23 e.
    (fp16's subnormals: 2^-25 a key next to a largest weight of 2^6 or more, below 2^-19 of the mass
    for these 1,700 keys.)  Scores and sums in 32 bits: 1e-5 of the mass, for the reason that the
    other tests give.  Then half a step of the row, and half of fp16's smallest step."""
    sessions, groups = [(700, 1), (31, 4), (0, 1), (0, 40), (130, 1), (1500, 1)], [(3, 300), (1, 33)]
    c = make(H, kv, rope, page, dtype, q8, sessions, groups, seed=H + kv + 1)
    _say(f"one rounding H={H} kv={kv} rope={rope} dtype={dtype} q8={q8}")
    _, out, lse = call(gpu, c, device(gpu, c))
    o, l, mass = expect(c)
    before = (2.0 ** -17 + 2.0 ** -19 + 1e-5) * mass
    bound = before + ref.HALF_STEP[dtype] * (np.abs(o) + before) + 2.0 ** -25
    assert (np.abs(out.double().cpu().numpy() - o) <= bound).all()
    np.testing.assert_allclose(lse.double().cpu().numpy(), l, rtol=1e-5, atol=1e-5)
