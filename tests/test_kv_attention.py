"""Attention over the paged key-value cache against its definition in 64 bits."""
import pytest
import torch

from kv_reference import Batch, HALF_STEP, TYPE, near, say

F16, BF16 = 0, 1


def attend(gpu, c, window=None, sinks=0, info=True, **kw):
    batch, cache, q = c.device(gpu)
    plan = gpu.plan_kv_attention(batch, cache, c.H, rows=c.rows,
                                 max_q_len=max(c.q_len + [1]), window=window, sinks=sinks)
    if info:
        plan.read_info()
    out = torch.full((c.rows, c.H, c.DV), 7.0, dtype=TYPE[c.dtype], device="cuda")
    lse = torch.full((c.rows, c.H), 7.0, device="cuda")
    got = gpu.kv_attention(plan, cache, 0, q, c.scale, out=out, lse=lse, **kw)
    assert got is out
    torch.cuda.synchronize()
    return plan, out, lse


def hold(gpu, c, window=None, sinks=0, info=True):
    plan, out, lse = attend(gpu, c, window, sinks, info)
    want, want_lse, off, off_lse = c.expect(window, sinks)
    near(out, want, off, "out")
    near(lse, want_lse, off_lse, "lse")
    return plan


# H, KH, D, DV, page: heads of their own, groups of every kind, widths that fill a kernel and that
# do not, pages of one tile, odd numbers of tiles and many
SHAPES = [(8, 8, 64, 64, 64), (32, 8, 128, 128, 64), (16, 16, 192, 128, 64), (4, 4, 256, 256, 32),
          (1, 1, 16, 16, 16), (15, 3, 80, 96, 48), (16, 1, 128, 64, 16), (12, 2, 48, 240, 128),
          (10, 2, 112, 112, 16), (40, 1, 64, 32, 256), (7, 7, 160, 16, 80)]
# cached tokens and query rows: none, one, at and around the edges of tiles, units and pages
DECODE = [(0, 1), (15, 1), (16, 1), (31, 1), (32, 1), (0, 0), (63, 1), (64, 1), (700, 1), (127, 1),
          (128, 0), (1500, 1)]
DRAFTS = [(0, 2), (30, 4), (61, 5), (5, 0), (200, 1), (333, 3), (1000, 7)]
CHUNKS = [(0, 33), (100, 70), (0, 1), (0, 0), (17, 129), (411, 40), (640, 2)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("H,KH,D,DV,page", SHAPES)
def test_decode_rows(gpu, H, KH, D, DV, page, dtype):
    say(f"decode {H} {KH} {D} {DV} {page} {dtype}")
    hold(gpu, Batch(H, KH, D, DV, page, dtype, DECODE, seed=H + D))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("H,KH,D,DV,page", SHAPES)
def test_drafted_rows_and_chunks(gpu, H, KH, D, DV, page, dtype):
    say(f"chunks {H} {KH} {D} {DV} {page} {dtype}")
    hold(gpu, Batch(H, KH, D, DV, page, dtype, DRAFTS + CHUNKS, seed=H + D + 1))


@pytest.mark.gpu
@pytest.mark.parametrize("window,sinks", [(None, 0), (1, 0), (9, 2), (40, 33)])
@pytest.mark.parametrize("H,KH,D,DV,page", [(8, 8, 64, 64, 64), (4, 2, 128, 128, 16), (2, 2, 192, 128, 64),
                                            (2, 1, 256, 256, 32), (3, 3, 80, 96, 48)])
def test_drafted_rows_alone(gpu, H, KH, D, DV, page, window, sinks):
    """At most 16 rows a session and kv head: blocks of 16, of several positions each, with values
    that are not finite in the last token's."""
    say(f"drafts {H} {KH} {D} {DV} {page} {window}")
    c = Batch(H, KH, D, DV, page, BF16, DRAFTS, seed=H + D + 2)
    for b, n in enumerate(c.lens):
        at, slot = c.token(b, n - 1)
        c.v[at, 0, slot, b % DV] = float("inf")
    hold(gpu, c, window, sinks)


WINDOWS = [(1, 0), (1, 1), (31, 4), (32, 0), (33, 33), (64, 1), (100, 128), (257, 5), (5000, 3)]


@pytest.mark.gpu
@pytest.mark.parametrize("window,sinks", WINDOWS)
@pytest.mark.parametrize("H,KH,D,DV,page", [SHAPES[0], SHAPES[1], SHAPES[3], SHAPES[5]])
def test_windows_with_sinks(gpu, H, KH, D, DV, page, window, sinks):
    """With NaN in the keys and values of the tokens that no row sees any more."""
    dtype = (window + H) % 2
    say(f"window {H} {KH} {D} {DV} {page} {dtype} {window} {sinks}")
    c = Batch(H, KH, D, DV, page, dtype, DECODE + DRAFTS + CHUNKS, seed=window + sinks)
    for b in range(len(c.lens)):
        if c.q_len[b]:
            for j in (~c.sees(b, window, sinks).any(0)).nonzero().flatten().tolist():
                at, slot = c.token(b, j)
                c.k[at, :, slot] = c.v[at, :, slot] = float("nan")
    hold(gpu, c, window, sinks)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("H,KH,D,DV,page", [SHAPES[0], SHAPES[1], SHAPES[3], SHAPES[7]])
@pytest.mark.parametrize("window,sinks", [(None, 0), (40, 6)])
def test_values_that_are_not_finite_reach_the_rows_that_see_them(gpu, H, KH, D, DV, page, dtype,
                                                                 window, sinks):
    """An infinity or NaN in a column of a token's value, among it tokens that only some rows of a
    block see: the column of those rows is not finite, and no other."""
    say(f"not finite {H} {KH} {D} {DV} {page} {dtype} {window}")
    sessions = [(20, 9), (50, 40), (90, 1), (3, 2), (0, 150)]
    c = Batch(H, KH, D, DV, page, dtype, sessions, seed=5)
    bad = [float("inf"), -float("inf"), float("nan")]
    for b, n in enumerate(c.lens):
        for i, back in enumerate((0, 1, 5, 30, 45)):
            if back < n:
                at, slot = c.token(b, n - 1 - back)
                c.v[at, i % KH, slot, (3 * i + 5) % DV] = bad[i % 3]
    # weights of a seen token are above fp16's and fp32's smallest: scores within +-20
    c.q *= 0.5
    hold(gpu, c, window, sinks)


@pytest.mark.gpu
@pytest.mark.parametrize("H,KH,D,DV,page", [SHAPES[0], SHAPES[1], SHAPES[3]])
def test_keys_that_are_not_finite(gpu, H, KH, D, DV, page):
    """A NaN key makes the rows that see it NaN, no others; an infinite one gives a score of +-inf:
    weight 0, or a row of NaN."""
    c = Batch(H, KH, D, DV, page, F16, [(20, 9), (50, 40), (90, 1)], seed=6)
    say(f"keys not finite {H} {KH} {D}")
    for b in range(3):
        n = c.lens[b]
        at, slot = c.token(b, n - 1)
        c.k[at, 0, slot, 2] = float("nan")
        at, slot = c.token(b, 1)
        c.k[at, -1, slot, 1] = -float("inf")
    c.q[:, :, 1] = c.q[:, :, 1].abs() + 0.1  # its score is -inf for all rows
    plan, out, lse = attend(gpu, c)
    want, want_lse, off, off_lse = c.expect()
    near(out, want, off, "out")
    near(lse, want_lse, off_lse, "lse")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("H,KH,D,DV,page", SHAPES)
def test_a_mean_of_equal_values_is_the_value(gpu, H, KH, D, DV, page, dtype):
    """Whatever the weights are: they are off by 2^-17 each at most where they meet the values, the
    sums in 32 bits by less, so the row before its rounding is within 1e-5 of the value, and half a
    step of the type is 2^-12 of it at least."""
    say(f"equal values {H} {D} {dtype}")
    c = Batch(H, KH, D, DV, page, dtype, DECODE + DRAFTS + CHUNKS, seed=9)
    g = torch.Generator().manual_seed(1)
    row = ((8 + torch.randint(0, 8, (KH, DV), generator=g)) / 8).to(TYPE[dtype])
    c.v[:] = torch.where(c.v.isnan(), c.v, row[None, :, None])
    _, out, _ = attend(gpu, c)
    want = row.repeat_interleave(H // KH, 0)[None].expand(c.rows, H, DV)
    assert torch.equal(out.cpu(), want)


@pytest.mark.gpu
@pytest.mark.parametrize("H,KH,D,DV,page,dtype", [(8, 8, 64, 64, 64, F16), (32, 8, 128, 128, 64, BF16)])
def test_long_contexts_are_split_and_joined(gpu, H, KH, D, DV, page, dtype):
    say(f"long {H} {D}")
    c = Batch(H, KH, D, DV, page, dtype, [(20000, 1), (30001, 40), (5, 1), (9000, 3)], seed=11)
    plan = hold(gpu, c)
    assert plan.read_info()[4] > 0
    plan = hold(gpu, c, 12000, 70)
    assert plan.read_info()[4] > 0


@pytest.mark.gpu
def test_large_scores_and_a_rising_maximum(gpu):
    """Scores of hundreds, the largest ever later: the reference maximum is raised again and again."""
    c = Batch(8, 2, 64, 64, 16, BF16, [(600, 1), (300, 50)], seed=12, scale=1.0)
    say("rising maximum")
    for b in range(2):
        for j in range(c.lens[b]):
            at, slot = c.token(b, j)
            c.k[at, :, slot] = (c.q[0].float().mean(0) * (1 + j / 8)).to(TYPE[BF16])
    hold(gpu, c)


@pytest.mark.gpu
def test_many_sessions(gpu):
    """More sessions and blocks than the plan's tables hold on the chip."""
    sessions = [((i * 7) % 90, 1 if i % 5 else i % 3) for i in range(3100)]
    say("many sessions")
    c = Batch(2, 1, 16, 16, 16, F16, sessions, seed=13)
    hold(gpu, c)
    hold(gpu, c, 20, 2, info=False)


@pytest.mark.gpu
@pytest.mark.parametrize("window,sinks", [(None, 0), (50, 4)])
def test_calls_without_the_plans_info(gpu, window, sinks):
    c = Batch(32, 8, 128, 128, 64, BF16, DECODE + CHUNKS, seed=14)
    say("no info")
    _, a, la = attend(gpu, c, window, sinks, info=True)
    _, b, lb = attend(gpu, c, window, sinks, info=False)
    assert torch.equal(a, b) and torch.equal(la, lb)


@pytest.mark.gpu
def test_rows_past_the_batch_and_failed_plans_are_left_alone(gpu):
    c = Batch(8, 8, 64, 64, 64, F16, [(100, 1), (20, 3)], seed=15)
    say("rows past the batch")
    batch, cache, q = c.device(gpu)
    plan = gpu.plan_kv_attention(batch, cache, 8, rows=9, max_q_len=3)
    wide = torch.cat([q, torch.full((5, 8, 64), float("nan"), dtype=q.dtype, device="cuda")])
    out = torch.full((9, 8, 64), 7.0, dtype=q.dtype, device="cuda")
    lse = torch.full((9, 8), 7.0, device="cuda")
    gpu.kv_attention(plan, cache, 0, wide, c.scale, out=out, lse=lse)
    want, want_lse, off, off_lse = c.expect()
    near(out[:4], want, off, "out")
    near(lse[:4], want_lse, off_lse, "lse")
    assert (out[4:] == 7).all() and (lse[4:] == 7).all()
    # a session has more rows than max_q_len; more rows than the plan's
    for kw, why in ((dict(rows=4, max_q_len=2), "session 1"), (dict(rows=3, max_q_len=3), "rows")):
        plan = gpu.plan_kv_attention(batch, cache, 8, **kw)
        out.fill_(7)
        gpu.kv_attention(plan, cache, 0, wide[:kw["rows"]], c.scale, out=out[:kw["rows"]])
        assert (out == 7).all()
        with pytest.raises(gpu.MlaError, match=why):
            plan.read_info()


@pytest.mark.gpu
def test_empty_calls(gpu):
    say("empty")
    for sessions in ([], [(5, 0)], [(0, 0), (0, 0)]):
        c = Batch(8, 8, 64, 64, 64, F16, sessions)
        batch, cache, q = c.device(gpu)
        plan = gpu.plan_kv_attention(batch, cache, 8, rows=c.rows, max_q_len=1)
        assert gpu.kv_attention(plan, cache, 0, q, 0.1).shape == (0, 8, 64)


@pytest.mark.gpu
def test_a_layer_of_several_and_offsets_past_32_bits(gpu):
    """A pool of 6.4 GB: layer 1's last pages lie past 2^32 bytes and words of the first."""
    say("past 32 bits")
    H, KH, D, page, n = 4, 2, 128, 256, 12300
    pool = n + 3
    cache = gpu.PagedKVCache(2, pool, page, KH, D, dtype=BF16)
    assert cache.pages.numel() > 2 ** 31 and cache.pages[0].numel() * 2 > 2 ** 31
    c = Batch(H, KH, D, D, page, BF16, [(700, 1), (300, 60)], seed=16)
    batch, _, q = c.device(gpu)
    shift = pool - c.pool
    cache.pages[1, shift:] = c.storage()[0].cuda()
    i32 = lambda x: torch.tensor(list(x), dtype=torch.int32, device="cuda")
    batch = gpu.build_metadata(i32(c.ctx), i32(c.q_len), i32(c.cu), i32(c.ids + shift), page,
                               c.max_pages, pool, split_pages=64, max_work=4, max_rows=c.rows)
    plan = gpu.plan_kv_attention(batch, cache, H, rows=c.rows, max_q_len=60)
    want, _, off, _ = c.expect()
    near(gpu.kv_attention(plan, cache, 1, q, c.scale), want, off, "out")
    near(gpu.kv_attention(plan, cache, -1, q, c.scale), want, off, "out")


@pytest.mark.gpu
def test_another_stream(gpu):
    c = Batch(32, 8, 128, 128, 64, BF16, DECODE + CHUNKS, seed=17)
    say("another stream")
    batch, cache, q = c.device(gpu)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    plan = gpu.plan_kv_attention(batch, cache, 32, rows=c.rows, max_q_len=129, stream=s)
    out = gpu.kv_attention(plan, cache, 0, q, c.scale, stream=s)
    s.synchronize()
    want, _, off, _ = c.expect()
    near(out, want, off, "out")


@pytest.mark.gpu
def test_refusals(gpu):
    c = Batch(8, 4, 64, 48, 64, F16, [(100, 1), (20, 3)], seed=18)
    say("refusals")
    batch, cache, q = c.device(gpu)
    make = lambda **kw: gpu.plan_kv_attention(batch, cache, **{"n_heads": 8, "rows": 4, "max_q_len": 3, **kw})
    for kw in (dict(n_heads=6), dict(n_heads=0), dict(window=0), dict(window=-1), dict(sinks=2),
               dict(window=4, sinks=-1), dict(max_q_len=0), dict(rows=-1)):
        with pytest.raises(ValueError):
            make(**kw)
    plan = make()
    call = lambda **kw: gpu.kv_attention(**{"plan": plan, "cache": cache, "layer": 0, "q": q, "scale": 0.1, **kw})
    other = gpu.PagedKVCache(1, c.pool, 64, 4, 64, 64, dtype=F16)
    fewer = gpu.PagedKVCache(1, c.pool - 1, 64, 4, 64, 48, dtype=F16)
    typed = gpu.PagedKVCache(1, c.pool, 64, 4, 64, 48, dtype=BF16)
    wide = torch.zeros((4, 8, 128), dtype=torch.float16, device="cuda")
    for kw in (dict(cache=other), dict(cache=fewer), dict(cache=typed), dict(q=q[:3]), dict(q=q.bfloat16()),
               dict(q=q.cpu()), dict(q=wide[..., :64]), dict(out=torch.zeros_like(q)),
               dict(lse=torch.zeros((4, 8), dtype=torch.float16, device="cuda")),
               dict(workspace=torch.zeros(64, device="cuda"))):
        with pytest.raises(ValueError):
            call(**kw)
    for kw in (dict(scale=0.0), dict(scale=float("nan")), dict(scale=float("inf")),
               dict(workspace=torch.zeros(64, dtype=torch.uint8, device="cuda"))):
        with pytest.raises(gpu.MlaError):
            call(**kw)
    with pytest.raises(IndexError):
        call(layer=1)
    with pytest.raises(ValueError):
        gpu.plan_kv_attention(batch, fewer, 8, rows=4)
    for shape in ((1, 4, 24, 4, 64), (1, 4, 64, 4, 40), (1, 4, 64, 4, 272), (1, 4, 64, 0, 64)):
        with pytest.raises(ValueError):
            gpu.PagedKVCache(*shape)
    with pytest.raises(ValueError):
        gpu.PagedKVCache(1, 4, 64, 4, 64, storage=torch.zeros((1, 4, 8), dtype=torch.float16))
