"""Every instantiation of the planned attention kernel: both lists, each width, rope columns fixed
or not, both cache formats and types, the list that ran asserted by the plan's own counts."""
import numpy as np
import pytest
import torch

import latent_reference as ref
from cpp_inference_train_engine_amd.workloads import to_bits
from test_latent_attention import FORMATS, _say, call, device, make, put16


def expect(c):
    """(out, lse, mass) [rows, H, ..] in 64 bits, on the GPU; a row that sees a non-finite latent is
    NaN."""
    lat, key = (torch.from_numpy(x).cuda() for x in c.rows())
    bad = ~(lat.isfinite().all(1) & key.isfinite().all(1))
    lat, key = (torch.where(x.isfinite(), x, 0.0) for x in (lat, key))
    bits = lambda x: torch.from_numpy(ref.from_bits(x, c.dtype)).cuda()
    ql, qr = bits(c.ql), bits(c.qr).view(len(c.ql), c.H, c.rope)
    outs, at = [], 0
    for b, (n0, n) in enumerate(zip(c.ctx.tolist(), c.q.tolist())):
        g = c.group_of(b)
        p = int(c.prefix[g]) if g >= 0 else 0
        slots = np.concatenate([c.flat(c.prefix_pages[g], p) if p else np.zeros(0, int),
                                c.flat(c.own_pages[b], n0 + n)]).astype(int)
        slots = torch.from_numpy(slots).cuda()
        x, k = lat[slots], key[slots]
        q, r = ql[at:at + n].reshape(n * c.H, c.kv), qr[at:at + n].reshape(n * c.H, c.rope)
        s = ((q @ x.T + r @ k.T) * c.scale).view(n, c.H, len(slots))
        last = p + n0 + torch.arange(n, device="cuda")[:, None]
        unseen = torch.arange(len(slots), device="cuda")[None] > last
        s.masked_fill_(unseen[:, None], -np.inf)
        lse = torch.logsumexp(s, 2)
        w = torch.exp(s - lse[..., None]).view(n * c.H, len(slots))
        out, mass = ((w @ y).view(n, c.H, c.kv) for y in (x, x.abs()))
        hit = (~unseen & bad[slots][None]).any(1)
        out[hit], lse[hit] = np.nan, np.nan
        outs.append((out, lse, mass))
        at += n
    return tuple(torch.cat(x) for x in zip(*outs))


def check(c, out, lse, want, scores=1e-5):
    """Weights in two parts of the type are within 2^-17 of theirs (2^-19 of the mass for fp16's
    subnormals, for up to 1,700 keys); `scores`: what scores and sums in 32 bits carry into a
    weight.  Then half a step of the row, and half of fp16's smallest step."""
    o, l, mass = want
    before = (2.0 ** -17 + 2.0 ** -19 + scores) * mass
    bound = before + ref.HALF_STEP[c.dtype] * (o.abs() + before) + 2.0 ** -25
    nan = o.isnan()
    assert torch.equal(out.isnan(), nan) and torch.equal(lse.isnan(), l.isnan())
    excess = torch.where(nan, -1.0, (out.double() - o).abs() - bound)
    assert excess.max() <= 0, f"off by {excess.max()} more than the bound"
    assert ((lse.double() - l).abs() <= scores * (1 + l.abs()))[~l.isnan()].all()


# List K takes segments of up to 64 (query, head) rows, and others while it has room for them: past
# 4 blocks of 16 rows for each of its 1,024, 512 or 256 slots (kv up to 128, 256, 512; a prefix
# counts its sessions' rows again) only list R does.
LISTS = [  # H, kv, rope, page, rows of the chunk, list
    (8, 128, 16, 64, 40, "K"), (40, 128, 16, 64, 850, "R"), (16, 512, 64, 64, 3, "K"),
    (40, 512, 64, 64, 220, "R"), (8, 32, 8, 16, 40, "K"), (40, 32, 8, 16, 850, "R"),
    (40, 96, 24, 48, 850, "R"), (12, 128, 64, 16, 5, "K"), (40, 128, 64, 16, 850, "R"),
    (16, 160, 8, 32, 4, "K"), (40, 160, 40, 16, 430, "R"), (16, 256, 32, 32, 4, "K"),
    (40, 256, 32, 32, 430, "R"), (16, 288, 16, 32, 4, "K"), (40, 288, 16, 32, 220, "R"),
    (8, 384, 64, 64, 6, "K"), (128, 384, 64, 64, 70, "R"), (16, 512, 16, 64, 4, "K"),
    (40, 512, 48, 16, 220, "R")]
GROUPS = [(2, 100), (1, 70)]


def batch(H, kv, rope, page, dtype, q8, chunk, seed):
    """Behind two prefixes a decode row, a chunk and a decode row, then sessions of their own."""
    sessions = [(40, 1), (200, chunk), (70, 1), (0, 9), (0, 1), (600, 1), (31, 2)]
    return make(H, kv, rope, page, dtype, q8, sessions, GROUPS, seed=seed)


def ran(plan, on, H):
    info = plan.read_info()
    _say(info)
    assert (info[3] > 0) == (on == "R")
    if H <= 64:  # the decode rows
        assert info[2] > 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,q8", FORMATS)
@pytest.mark.parametrize("H,kv,rope,page,chunk,on", LISTS)
def test_every_list_and_width(gpu, H, kv, rope, page, chunk, on, dtype, q8):
    """With the launch of every job that the plan could have, and with that of its jobs alone."""
    c = batch(H, kv, rope, page, dtype, q8, chunk, seed=kv + rope)
    _say(f"list {on} H={H} kv={kv} rope={rope} dtype={dtype} q8={q8}")
    d = device(gpu, c)
    plan, out, lse = call(gpu, c, d)
    check(c, out, lse, expect(c))
    ran(plan, on, H)
    _, out2, lse2 = call(gpu, c, d, plan)
    assert torch.equal(out, out2) and torch.equal(lse, lse2)


def spoil(c, slots, word):
    """Column 3 of the tokens' latents becomes NaN (8 bits) or `word`."""
    lat, key = c.rows()
    x = lat[slots].astype(np.float32)
    kb = to_bits(key[slots].astype(np.float32), c.dtype).reshape(len(slots), c.rope)
    if c.q8:
        byte, k = ref.quantise(x, c.dtype)
        byte[:, 3] = 0x7F
        ref.q8_store(c.pool, c.page, c.kv, c.rope, slots, byte, kb, k)
    else:
        w = to_bits(x, c.dtype)
        w[:, 3] = word
        put16(c, slots, w, kb)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,q8", FORMATS)
@pytest.mark.parametrize("H,kv,rope,page,chunk,on", LISTS)
def test_nonfinite_latents_on_every_list(gpu, H, kv, rope, page, chunk, on, dtype, q8):
    """NaN, then infinities of both signs: in either half of a 64-key unit of the chunk's own tokens,
    at its end, in a whole unit, in a prefix, and as a row's only key."""
    nan, inf = ((0x7E00, 0x7C00), (0x7FC0, 0x7F80))[dtype]
    for words in ([nan] * 3,) if q8 else ([nan] * 3, [inf, inf | 0x8000, inf]):
        c = batch(H, kv, rope, page, dtype, q8, chunk, seed=kv + rope + 1)
        own = [c.flat(p, int(n)) for p, n in zip(c.own_pages, c.ctx + c.q)]
        spoil(c, own[1][[200 + chunk // 2, 200 + chunk - 1]], words[0])
        spoil(c, own[1][[200 + chunk * 3 // 4]], words[1])
        spoil(c, own[3][[4]], words[1])
        spoil(c, own[4], words[2])
        spoil(c, own[5][512:544], words[0])
        spoil(c, c.flat(c.prefix_pages[1], 70)[[69]], words[1])
        _say(f"non-finite, list {on} H={H} kv={kv} rope={rope} dtype={dtype} q8={q8} {words[0]:x}")
        plan, out, lse = call(gpu, c, device(gpu, c))
        want = expect(c)
        check(c, out, lse, want)
        seen = want[0].isnan().any(2).any(1)
        assert seen[1:1 + chunk].sum() == chunk - chunk // 2 and seen[1 + chunk]
        ran(plan, on, H)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,q8", FORMATS)
@pytest.mark.parametrize("H,kv,rope,page,chunk,on", LISTS)
def test_rising_scores_on_every_list(gpu, H, kv, rope, page, chunk, on, dtype, q8):
    """Scores climb by 40 nats along the keys and fall behind them: the reference maximum is raised
    again and again.  A score of 40 summed in 32 bits from kv + rope products is off by 40 *
    1.4e-6, in the weight and in the mass."""
    c = batch(H, kv, rope, page, dtype, q8, chunk, seed=kv + rope + 2)
    lat, key = c.rows()
    for pages, n in zip(list(c.prefix_pages) + list(c.own_pages), list(c.prefix) + list(c.ctx + c.q)):
        slots = c.flat(pages, int(n))
        x = lat[slots] * 0.1
        x[:, :4] += (20 * (1 - np.abs(np.arange(n) / n - 0.7)) / (c.scale * 4))[:, None]
        kb = to_bits((key[slots] * 0.1).astype(np.float32), dtype).reshape(len(slots), rope)
        if q8:
            byte, k = ref.quantise(x.astype(np.float32), dtype)
            ref.q8_store(c.pool, page, kv, rope, slots, byte, kb, k)
        else:
            put16(c, slots, to_bits(x.astype(np.float32), dtype), kb)
    u = np.zeros(kv)
    u[:4] = 2
    q = np.random.default_rng(1).standard_normal(c.ql.shape) * 0.05 + u
    c.ql[:] = to_bits(q.astype(np.float32), dtype)
    _say(f"rising, list {on} H={H} kv={kv} rope={rope} dtype={dtype} q8={q8}")
    plan, out, lse = call(gpu, c, device(gpu, c))
    check(c, out, lse, expect(c), scores=2 * 40 * 1.4e-6)
    ran(plan, on, H)


@pytest.mark.gpu
def test_plans_of_the_same_sizes_share_a_workspace(gpu):
    """One after the other on a stream, with other lengths behind the same sizes, host info read for
    one of them only: each call's rows are those of a workspace of its own."""
    lengths = [(500, 900, 20, 3000), (3000, 1, 1500, 40)]
    cases = [make(8, 128, 16, 64, 0, True, [(a, 1), (b, 5), (x, 1), (y, 1)], [(3, p)], seed=i)
             for i, ((a, b, x, y), p) in enumerate(zip(lengths, (700, 64)))]
    data = [device(gpu, c) for c in cases]
    _say("one workspace, two plans")
    alone = [call(gpu, c, d) for c, d in zip(cases, data)]
    ws = gpu.attention_workspace(alone[0][0])
    alone[0][0].read_info()
    for _ in range(2):
        for c, d, (plan, out, lse) in zip(cases, data, alone):
            _, out2, lse2 = call(gpu, c, d, plan, workspace=ws)
            assert torch.equal(out, out2) and torch.equal(lse, lse2)
    for c, (_, out, lse) in zip(cases, alone):
        check(c, out, lse, expect(c))
