"""Attention over the paged key-value cache where the weights of a row lie far apart: a token far above
all others whose value is zero, so that the row is made of the small weights alone."""
import pytest
import torch

from kv_reference import Batch, TYPE, near, say

F16, BF16 = 0, 1
# H, KH, D, DV, page: every kernel's width, filled and not
SHAPES = [(4, 4, 64, 64, 64), (8, 2, 128, 128, 16), (2, 2, 192, 128, 64), (2, 1, 256, 256, 32),
          (3, 3, 80, 96, 48), (4, 4, 48, 32, 16)]
FEW = [(3000, 1), (20, 1), (900, 3), (20000, 1)]
MANY = [(700, 129), (0, 300), (2500, 70)]


def above(c, gap, every, size):
    """Every `every`-th token from the first (0: the first alone) lies `gap` nats above the others,
    which lie within a few, and its value is zero; the others' values are between size / 2 and size."""
    t = TYPE[c.dtype]
    c.scale = 0.125
    c.q[..., 0] = 8  # (its column gives the score that the key's has)
    c.q[..., 1:] *= c.D ** -0.5
    c.k[..., 0] = torch.where(c.k[..., 0].isnan(), c.k[..., 0], 0)
    g = torch.Generator().manual_seed(5)
    v = (torch.rand(c.v.shape, generator=g) * size / 2 + size / 2).to(t)
    c.v = torch.where(c.v.isnan(), c.v, v)
    for b, n in enumerate(c.lens):
        for j in range(0, n, every) if every else range(min(n, 1)):
            at, slot = c.token(b, j)
            c.k[at, :, slot, 0], c.v[at, :, slot] = gap, 0


def hold(gpu, c, window, sinks):
    batch, cache, q = c.device(gpu)
    plan = gpu.plan_kv_attention(batch, cache, c.H, rows=c.rows, max_q_len=max(c.q_len), window=window,
                                 sinks=sinks)
    lse = torch.zeros((c.rows, c.H), device="cuda")
    out = gpu.kv_attention(plan, cache, 0, q, c.scale, lse=lse)
    want, want_lse, off, off_lse = c.expect(window, sinks)
    near(out, want, off, "out")
    near(lse, want_lse, off_lse, "lse")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("window,sinks", [(None, 0), (500, 4)])
@pytest.mark.parametrize("sessions", [FEW, MANY], ids=["few", "many"])
@pytest.mark.parametrize("H,KH,D,DV,page", SHAPES)
def test_one_token_far_above_the_others(gpu, H, KH, D, DV, page, sessions, window, sinks, dtype):
    for gap, size in ((12, 4), (17, 4), (21, 64), (26, 60000), (31, 60000)):
        say(f"far above {H} {KH} {D} {DV} {page} {dtype} {window} {gap}")
        c = Batch(H, KH, D, DV, page, dtype, sessions, seed=gap)
        above(c, gap, 0, size)
        hold(gpu, c, window, sinks)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("every", [3, 32, 70])
@pytest.mark.parametrize("sessions", [FEW, MANY], ids=["few", "many"])
@pytest.mark.parametrize("H,KH,D,DV,page", SHAPES)
def test_tokens_far_above_the_others_everywhere(gpu, H, KH, D, DV, page, sessions, every, dtype):
    for gap, size in ((14, 4), (19, 64), (28, 60000)):
        say(f"far above, every {every} {H} {KH} {D} {DV} {page} {dtype} {gap}")
        c = Batch(H, KH, D, DV, page, dtype, sessions[:3], seed=gap + every)
        above(c, gap, every, size)
        hold(gpu, c, 300 if every == 32 else None, 0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("H,KH,D,DV,page", SHAPES)
def test_scores_that_fall_and_rise(gpu, H, KH, D, DV, page, dtype):
    """Scores that rise by 40 nats towards the last token, fall as far, or do both in turn."""
    for shape in (lambda x: x, lambda x: -x, lambda x: (x * 40).sin()):
        say(f"falling and rising {H} {D} {dtype}")
        c = Batch(H, KH, D, DV, page, dtype, [(2000, 1), (600, 90), (300, 2)], seed=3)
        above(c, 0, 0, 4)
        for b, n in enumerate(c.lens):
            for j in range(n):
                at, slot = c.token(b, j)
                c.k[at, :, slot, 0] = float(40 * shape(torch.tensor(j / n)))
        hold(gpu, c, None, 0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_small_weights_and_values_that_are_not_finite(gpu, dtype):
    """An infinite value behind a small weight, in units that some rows of a block see in part: its
    column is not finite in the rows that see it, and no other."""
    for H, KH, D, DV, page in SHAPES[:2]:
        say(f"small weights, not finite {D} {dtype}")
        c = Batch(H, KH, D, DV, page, dtype, [(100, 1), (70, 5), (40, 200)], seed=4)
        above(c, 16, 0, 4)
        for b, n in enumerate(c.lens):
            for i, back in enumerate((0, 3, 33, 65)):
                at, slot = c.token(b, n - 1 - back)
                c.v[at, i % KH, slot, 5 * i] = [float("inf"), -float("inf")][i % 2]
        hold(gpu, c, None, 0)
        hold(gpu, c, 50, 2)
