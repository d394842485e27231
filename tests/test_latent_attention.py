"""Planned attention over the 16-bit and the 8-bit latent cache, with and without shared prefixes,
against the definition in 64 bits."""
import ctypes
from dataclasses import dataclass, replace

import numpy as np
import pytest

import latent_reference as ref
from cpp_inference_train_engine_amd.workloads import to_bits


def _say(*a):
    print(*a, flush=True)


@dataclass
class Case:
    """sessions: (own tokens before the call's rows, rows); groups: (sessions, prefix tokens)."""
    H: int
    kv: int
    rope: int
    page: int
    dtype: int
    q8: bool
    ctx: np.ndarray
    q: np.ndarray
    cu_groups: np.ndarray
    prefix: np.ndarray
    own_pages: list
    prefix_pages: list
    pool: np.ndarray
    ql: np.ndarray  # 16-bit words
    qr: np.ndarray

    @property
    def scale(self):
        return 1 / np.sqrt(self.kv / 2 + self.rope)

    def group_of(self, b):
        g = int(np.searchsorted(self.cu_groups, b, "right")) - 1
        return g if 0 <= g < len(self.prefix) else -1

    def flat(self, pages, n):
        """Flat slots of the first n tokens on a page list."""
        t = np.arange(n)
        return np.array(pages, int)[t // self.page] * self.page + t % self.page if n else t

    def rows(self):
        f = ref.q8_rows if self.q8 else ref.rows16
        return f(self.pool, self.page, self.kv, self.rope, self.dtype)


def make(H, kv, rope, page, dtype, q8, sessions, groups=(), seed=0, spare=2):
    """Contents N(0, 1); every slot that no key occupies holds NaN (or any bits)."""
    rng = np.random.default_rng(seed)
    ctx = np.array([c for c, _ in sessions])
    q = np.array([n for _, n in sessions])
    need = [-(-p // page) for _, p in groups] + [-(-(c + n) // page) for c, n in sessions]
    P = sum(need) + spare
    ids = rng.permutation(P)
    lists, at = [], 0
    for n in need:
        lists.append(ids[at:at + n])
        at += n
    G = len(groups)
    c = Case(H, kv, rope, page, dtype, q8, ctx, q,
             np.concatenate([[0], np.cumsum([n for n, _ in groups])]).astype(int),
             np.array([p for _, p in groups], int), lists[G:], lists[:G], None,
             to_bits(rng.standard_normal((int(q.sum()), H, kv), dtype=np.float32), dtype),
             to_bits(rng.standard_normal((int(q.sum()), H, rope), dtype=np.float32), dtype))
    used = np.concatenate([c.flat(l, n) for l, n in
                           zip(lists, [p for _, p in groups] + [int(a + b) for a, b in sessions])])
    n = len(used)
    x = rng.standard_normal((n, kv), dtype=np.float32)
    key = to_bits(rng.standard_normal((n, rope), dtype=np.float32), dtype).reshape(n, rope)
    if q8:
        c.pool = np.full((P, page * (kv + 2 * rope + kv // 32)), 0xFF, np.uint8)
        byte, k = ref.quantise(x, dtype)
        ref.q8_store(c.pool, page, kv, rope, used, byte, key, k)
    else:
        c.pool = np.full((P, page * (kv + rope)), 0x7FC0, np.uint16)
        put16(c, used, to_bits(x, dtype), key)
    return c


def put16(c, slots, bits, key):
    from cpp_inference_train_engine_amd.ops import latent_word, rope_word
    p, o = np.asarray(slots) // c.page, np.asarray(slots) % c.page
    c.pool[p[:, None], latent_word(o[:, None], np.arange(c.kv), c.page, c.kv, c.rope)] = bits
    c.pool[p[:, None], rope_word(o[:, None], np.arange(c.rope), c.page, c.kv, c.rope)] = key


def expect(c):
    """(out, lse, mass) [rows, H, ..] in 64 bits."""
    lat, key = c.rows()
    ql = ref.from_bits(c.ql, c.dtype)
    qr = ref.from_bits(c.qr, c.dtype).reshape(len(ql), c.H, c.rope)
    outs, at = [], 0
    for b, (n0, n) in enumerate(zip(c.ctx, c.q)):
        g = c.group_of(b)
        p = int(c.prefix[g]) if g >= 0 else 0
        slots = np.concatenate([c.flat(c.prefix_pages[g], p) if p else np.zeros(0, int),
                                c.flat(c.own_pages[b], int(n0 + n))]).astype(int)
        seen = np.arange(len(slots))[None] <= p + n0 + np.arange(n)[:, None]
        outs.append(ref.attention(ql[at:at + n], qr[at:at + n], lat[slots], key[slots], seen,
                                  c.scale))
        at += n
    return tuple(np.concatenate(x) for x in zip(*outs))


def device(gpu, c, rows=None, max_q_len=None):
    """Everything a call takes, on the GPU."""
    import torch
    i32 = lambda x: torch.tensor(np.asarray(x, np.int64).astype(np.int32), device="cuda")
    tdt = torch.float16 if c.dtype == 0 else torch.bfloat16
    half = lambda x: torch.from_numpy(np.ascontiguousarray(x).view(np.int16)).cuda().view(tdt)
    need = [len(p) for p in c.own_pages]
    total = int(c.q.sum())
    batch = gpu.build_metadata(
        i32(c.ctx), i32(c.q), i32(np.concatenate([[0], np.cumsum(need)])),
        i32(np.concatenate(c.own_pages + [np.zeros(1)])), c.page, max(need), len(c.pool),
        split_pages=4, max_work=4096, max_rows=total)
    shared = None
    if len(c.prefix):
        lens = [len(p) for p in c.prefix_pages]
        shared = gpu.SharedPrefixes(i32(c.cu_groups), i32(c.prefix),
                                    i32(np.concatenate([[0], np.cumsum(lens)])),
                                    i32(np.concatenate(c.prefix_pages)))
    pages = torch.from_numpy(c.pool).cuda() if c.q8 else half(c.pool)
    rows = total if rows is None else rows
    pad = np.zeros((rows - total,) + c.ql.shape[1:], np.uint16)
    return dict(batch=batch, shared=shared, pages=pages, rows=rows,
                max_q_len=int(c.q.max()) if max_q_len is None else max_q_len,
                ql=half(np.concatenate([c.ql, pad])),
                qr=half(np.concatenate([c.qr, pad[:, :, :1].repeat(c.rope, 2)]).reshape(rows, c.H, c.rope)))


def call(gpu, c, d, plan=None, **kw):
    import torch
    plan = plan or gpu.plan_attention(d["batch"], c.H, c.kv, rows=d["rows"],
                                      max_q_len=d["max_q_len"], prefixes=d["shared"])
    out = torch.full((d["rows"], c.H, c.kv), 5.0, dtype=d["ql"].dtype, device="cuda")
    lse = torch.full((d["rows"], c.H), 5.0, device="cuda")
    gpu.latent_attention(plan, d["pages"], d["ql"], d["qr"], c.scale, rope_dim=c.rope,
                         dtype=c.dtype, q8=c.q8, out=out, lse=lse, **kw)
    return plan, out, lse


def check(c, out, lse, want=None):
    """out: weights rounded to the 16-bit type (half a step of each, relative), the row rounded to
    it (half a step, and half of fp16's smallest step), and 1e-5 of the mass for fp32 scores: a
    score s summed from kv + rope <= 576 products is off by about |s| 2^-24 sqrt(576) = 1.4e-6 |s|,
    and |s| <= 8 here.  lse: the same 1e-5, absolute and relative."""
    o, l, mass = want or expect(c)
    half = ref.HALF_STEP[c.dtype]
    got, got_lse = out.double().cpu().numpy(), lse.double().cpu().numpy()
    bound = (half * (1 + half) + 1e-5) * mass + half * np.abs(o) + 2.0 ** -25
    nan = np.isnan(o)
    assert int((np.isnan(got) != nan).sum()) == 0
    excess = np.where(nan, 0, np.abs(got - o) - bound)
    assert excess.max(initial=-1) <= 0, f"off by {excess.max()} more than the bound"
    np.testing.assert_allclose(got_lse, l, rtol=1e-5, atol=1e-5)


SHAPES = [  # H, kv, rope, page
    (8, 128, 16, 64), (1, 32, 8, 16), (16, 64, 16, 32), (12, 96, 24, 48), (17, 128, 64, 16),
    (40, 128, 0, 64), (4, 160, 40, 16), (32, 256, 32, 32), (16, 512, 64, 64), (128, 512, 64, 64),
    (128, 224, 8, 128)]
FORMATS = [(0, False), (1, False), (0, True), (1, True)]  # dtype, 8-bit


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,q8", FORMATS)
@pytest.mark.parametrize("H,kv,rope,page", SHAPES)
def test_decode_rows(gpu, H, kv, rope, page, dtype, q8):
    """One row a session, keys from one to many, at tile and page edges."""
    n = [1, 2, 15, 16, 17, 31, 32, 33, page - 1, page, page + 1, 128, 129, 700, 1500]
    c = make(H, kv, rope, page, dtype, q8, [(k - 1, 1) for k in n], seed=H + kv)
    _say(f"decode H={H} kv={kv} rope={rope} page={page} dtype={dtype} q8={q8}")
    _, out, lse = call(gpu, c, device(gpu, c))
    check(c, out, lse)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,q8", FORMATS)
@pytest.mark.parametrize("H,kv,rope,page", SHAPES)
def test_mixed_rows(gpu, H, kv, rope, page, dtype, q8):
    """Decode rows, drafted tokens and chunks in one batch, sessions without rows among them, and
    rows past the batch's, which stay as they were."""
    sessions = [(0, 1), (40, 0), (3, 5), (700, 2), (0, 17), (99, 33), (page, 0), (1000, 9), (30, 1),
                (5, 70)]
    c = make(H, kv, rope, page, dtype, q8, sessions, seed=H + kv + 1)
    _say(f"mixed H={H} kv={kv} rope={rope} page={page} dtype={dtype} q8={q8}")
    total = int(c.q.sum())
    d = device(gpu, c, rows=total + 3)
    _, out, lse = call(gpu, c, d)
    check(c, out[:total], lse[:total])
    assert (out[total:] == 5).all() and (lse[total:] == 5).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,q8", FORMATS)
@pytest.mark.parametrize("H,kv,rope,page", SHAPES)
def test_shared_prefixes(gpu, H, kv, rope, page, dtype, q8):
    """Groups of one session, of several and of many, an empty group, a group without a prefix, a
    prefix of one token and one that ends inside a page; sessions with several rows and with none;
    sessions behind the last group."""
    groups = [(1, 40), (3, 1), (0, 64), (2, 0), (20, 700 + page // 2), (3, 5 * page), (2, 33)]
    rng = np.random.default_rng(3)
    sessions = [(int(rng.integers(0, 90)), 1) for _ in range(31)] + [(11, 1), (300, 1)]
    sessions[2], sessions[10], sessions[26], sessions[27], sessions[29] = (9, 4), (7, 0), (0, 3), (50, 20), (5, 0)
    sessions[30] = (6, 0)  # a group whose sessions have no rows
    c = make(H, kv, rope, page, dtype, q8, sessions, groups, seed=H + kv + 2)
    _say(f"shared H={H} kv={kv} rope={rope} page={page} dtype={dtype} q8={q8}")
    _, out, lse = call(gpu, c, device(gpu, c))
    check(c, out, lse)


@pytest.mark.gpu
@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("H,kv,rope,page,sessions,groups", [
    (8, 128, 16, 64, [(20000, 1)], []),                      # one long session
    (8, 128, 16, 64, [(9000, 1)] * 2 + [(5, 1)] * 300, []),  # many sessions, two long ones
    (8, 128, 16, 64, [(k, 1) for k in range(64)], [(64, 12000)]),
    (2, 32, 8, 16, [(3, 600)], []),                          # a chunk of many rows
    (128, 512, 64, 64, [(4000, 1), (30, 3)], []),
    (128, 512, 64, 64, [(k, 1) for k in range(5)], [(5, 3000)])])
def test_long_keys_and_many_sessions(gpu, H, kv, rope, page, sessions, groups, q8):
    c = make(H, kv, rope, page, 0, q8, sessions, groups, seed=len(sessions))
    _say(f"long H={H} kv={kv} sessions={len(sessions)} groups={groups} q8={q8}")
    d = device(gpu, c)
    plan, out, lse = call(gpu, c, d)
    check(c, out, lse)
    _say(plan.read_info())  # from here on the exact number of workgroups
    _, out2, lse2 = call(gpu, c, d, plan)
    assert (out2 == out).all() and (lse2 == lse).all()


@pytest.mark.gpu
@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("H,kv,rope,page", [(8, 128, 16, 64), (40, 64, 16, 32), (128, 512, 64, 64)])
def test_nonfinite_latents_reach_only_the_rows_that_see_them(gpu, H, kv, rope, page, q8):
    """NaN (16-bit cache: infinities too) in a chunk's own tokens and in a prefix."""
    sessions = [(40, 1), (200, 40), (0, 9), (70, 1), (5, 1), (0, 1), (600, 1)]
    c = make(H, kv, rope, page, 0, q8, sessions, [(2, 100), (1, 70)], seed=5)
    lat, key = c.rows()

    def spoil(slots, bits):
        byte, k = ref.quantise(lat[slots].astype(np.float32), 0)
        kb = to_bits(key[slots].astype(np.float32), 0).reshape(len(slots), rope)
        if q8:
            byte[:, 3] = 0x7F
            ref.q8_store(c.pool, page, kv, rope, slots, byte, kb, k)
        else:
            w = to_bits(lat[slots].astype(np.float32), 0)
            w[:, 3] = bits
            put16(c, slots, w, kb)

    spoil(c.flat(c.own_pages[1], 240)[[220, 236]], 0x7E00)
    spoil(c.flat(c.own_pages[2], 9)[[4]], 0x7E00)
    spoil(c.flat(c.own_pages[3], 71)[[30]], 0x7E00)
    spoil(c.flat(c.prefix_pages[1], 70)[[69]], 0x7E00)
    spoil(c.flat(c.own_pages[5], 1), 0x7E00)                     # a row's only key
    spoil(c.flat(c.own_pages[6], 601)[512:544], 0x7E00)          # all keys of a unit
    _say(f"non-finite H={H} kv={kv} q8={q8}")
    d = device(gpu, c)
    _, out, lse = call(gpu, c, d)
    check(c, out, lse)
    assert np.isnan(out.double().cpu().numpy()).any(axis=(1, 2)).sum() == 20 + 9 + 1 + 1 + 1
    if not q8:
        want = expect(c)
        spoil(c.flat(c.own_pages[1], 240)[[220, 236]], 0x7C00)
        spoil(c.flat(c.own_pages[2], 9)[[4]], 0xFC00)
        spoil(c.flat(c.own_pages[3], 71)[[30]], 0xFC00)
        spoil(c.flat(c.own_pages[5], 1), 0x7C00)
        d = device(gpu, c)
        _, out, lse = call(gpu, c, d)
        check(c, out, lse, want)


@pytest.mark.gpu
@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("H,kv,rope,page", [(8, 128, 16, 64), (40, 96, 16, 32), (128, 512, 64, 64)])
def test_scores_that_rise_along_the_keys(gpu, H, kv, rope, page, q8):
    """Scores that climb by 60 log2 units along the keys, then fall: the reference maximum is
    raised many times, and early keys end with weight zero.  Bound: as in check, with a score of
    60 log2 units (42 nats) carrying 42 * 1.4e-6 into each weight."""
    c = make(H, kv, rope, page, 0, q8, [(900, 1), (400, 20), (37, 1)], [(3, 300)], seed=9)
    lat, key = c.rows()
    u = np.zeros(kv)
    u[:4] = 1
    for flat in [c.flat(p, len(p) * page) for p in c.own_pages + c.prefix_pages]:
        n = len(flat)
        x = np.nan_to_num(lat[flat]) * 0.1
        x[:, :4] += (60 * (1 - np.abs(np.arange(n) / n - 0.7)) / (1.4427 * c.scale * 4 * 2))[:, None]
        kb = to_bits(np.nan_to_num(key[flat]).astype(np.float32), 0).reshape(n, rope)
        if q8:
            byte, k = ref.quantise(x.astype(np.float32), 0)
            ref.q8_store(c.pool, page, kv, rope, flat, byte, kb, k)
        else:
            put16(c, flat, to_bits(x.astype(np.float32), 0), kb)
    ql = np.random.default_rng(1).standard_normal(c.ql.shape) * 0.05 + 2 * u
    c.ql[:] = to_bits(ql.astype(np.float32), 0)
    _say(f"rising scores H={H} kv={kv} q8={q8}")
    _, out, lse = call(gpu, c, device(gpu, c))
    o, l, mass = expect(c)
    got = out.double().cpu().numpy()
    bound = (2 ** -11 * 1.001 + 42 * 1.4e-6 * 2) * mass + 2 ** -11 * np.abs(o) + 2.0 ** -25
    assert (np.abs(got - o) <= bound).all()
    np.testing.assert_allclose(lse.double().cpu().numpy(), l, rtol=1e-5, atol=1e-4)


@pytest.mark.gpu
def test_equals_the_framework_attention(gpu):
    """On a 16-bit cache, the decode and prefill entry points of the same batch and metadata; on an
    8-bit one, the same call over a 16-bit cache that holds what is read back, bit for bit."""
    import torch
    sessions = [(100, 1), (2000, 1), (0, 1), (50, 20), (777, 1)]
    c = make(8, 128, 16, 64, 0, False, sessions, seed=4)
    d = device(gpu, c)
    _say("against decode_attention and prefill_attention")
    _, out, lse = call(gpu, c, d)
    lse2 = torch.zeros_like(lse)
    want = gpu.decode_attention(d["batch"], d["pages"], d["ql"], d["qr"], c.scale, kv_rank=128,
                                rope_dim=16, lse=lse2)
    gpu.prefill_attention(d["batch"], d["pages"], d["ql"], d["qr"], c.scale, kv_rank=128,
                          rope_dim=16, max_q_len=20, out=want, lse=lse2)
    torch.testing.assert_close(out.float(), want, rtol=2e-3, atol=2e-3)
    # the page kernels sum the fp16-rounded weights (off by 2^-11 of each): so is their ln(sum)
    torch.testing.assert_close(lse, lse2, rtol=1e-5, atol=2.0 ** -11)
    q = make(8, 128, 16, 64, 0, True, sessions, seed=4)
    lat, key = q.rows()
    w = make(8, 128, 16, 64, 0, False, sessions, seed=4)
    n = np.arange(len(lat))
    put16(w, n, to_bits(lat.astype(np.float32), 0), to_bits(key.astype(np.float32), 0))
    a, b = call(gpu, q, device(gpu, q)), call(gpu, w, device(gpu, w))
    assert torch.equal(a[1], b[1]) and torch.equal(a[2], b[2])


@pytest.mark.gpu
def test_one_plan_many_calls_streams_and_graphs(gpu):
    """A plan serves other queries, other layers and other streams; a captured plan and call replay
    with new contents, eager work between; repeated calls give the same bits."""
    import torch
    c = make(8, 128, 16, 64, 0, True, [(k * 37, 1) for k in range(20)], [(12, 500)], seed=6)
    d = device(gpu, c)
    _say("plan reuse, side stream, graph")
    plan, out, lse = call(gpu, c, d)
    ws = gpu.attention_workspace(plan)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _, out2, lse2 = call(gpu, c, d, plan, workspace=ws)
    side.synchronize()
    assert torch.equal(out, out2) and torch.equal(lse, lse2)

    b = d["batch"]
    gout, glse = torch.zeros_like(out), torch.zeros_like(lse)
    warm = torch.cuda.Stream()
    warm.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(warm):
        gpu.plan_attention(b, c.H, c.kv, rows=d["rows"], max_q_len=1, prefixes=d["shared"])
    torch.cuda.current_stream().wait_stream(warm)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        gplan = gpu.plan_attention(b, c.H, c.kv, rows=d["rows"], max_q_len=1, prefixes=d["shared"])
        gpu.latent_attention(gplan, d["pages"], d["ql"], d["qr"], c.scale, rope_dim=16, q8=True,
                             out=gout, lse=glse, workspace=ws)
    rng = np.random.default_rng(8)
    for i in range(3):
        d["ql"].copy_(torch.from_numpy(rng.standard_normal(c.ql.shape)).half())
        _, eager, elses = call(gpu, c, d)
        gout.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(gout, eager) and torch.equal(glse, elses), i


@pytest.mark.gpu
@pytest.mark.parametrize("H,kv,rope,page,dtype,q8", [(2, 32, 8, 16, 1, False), (8, 128, 16, 64, 0, True)])
def test_more_sessions_than_the_plan_keeps_on_chip(gpu, H, kv, rope, page, dtype, q8):
    """The plan's tables of the segments lie in its own memory; sessions behind a prefix and
    without one, the longest own keys at the end."""
    rng = np.random.default_rng(12)
    sessions = [(int(k), 1) for k in rng.integers(0, 60, 3100)]
    sessions[7], sessions[1900], sessions[3099] = (9, 12), (20, 0), (63, 1)
    c = make(H, kv, rope, page, dtype, q8, sessions, [(5, 70), (2200, 200), (1, 3)], seed=13)
    _say(f"3100 sessions H={H} kv={kv} q8={q8}")
    d = device(gpu, c)
    plan, out, lse = call(gpu, c, d)
    check(c, out, lse)
    plan.read_info()
    _, out2, lse2 = call(gpu, c, d, plan)
    assert (out2 == out).all() and (lse2 == lse).all()


@pytest.mark.gpu
@pytest.mark.parametrize("H,kv,rope,page", [(8, 128, 16, 64), (128, 512, 64, 64)])
def test_a_batch_without_rows_or_without_sessions(gpu, H, kv, rope, page):
    import torch
    c = make(H, kv, rope, page, 0, True, [(30, 0), (100, 0)], [(2, 70)], seed=14)
    _say(f"no rows H={H}")
    d = device(gpu, c, rows=3, max_q_len=1)
    plan, out, lse = call(gpu, c, d)
    assert plan.read_info()[:1] == [0]
    assert (out == 5).all() and (lse == 5).all()
    _, out, lse = call(gpu, c, d, plan)
    assert (out == 5).all() and (lse == 5).all()
    _say("no sessions")
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    zero = torch.zeros(1, dtype=torch.int32, device="cuda")
    batch = gpu.build_metadata(none, none, zero, zero, page, 1, len(c.pool), max_rows=3)
    d = dict(d, batch=batch, shared=None)
    plan, out, lse = call(gpu, c, d)
    assert plan.read_info()[:1] == [0]
    assert (out == 5).all() and (lse == 5).all()


@pytest.mark.gpu
def test_a_graph_that_plans_a_growing_batch(gpu):
    """Metadata, plan and attention captured together: each replay is that of the lengths that the
    batch has then, eager calls between."""
    import torch
    rng = np.random.default_rng(15)
    full = [int(k) for k in rng.integers(60, 900, 12)]
    c = make(8, 128, 16, 64, 0, True, [(k, 1) for k in full], [(5, 300), (3, 10)], seed=16)
    d = device(gpu, c)
    need = [len(p) for p in c.own_pages]
    i32 = lambda x: torch.tensor(np.asarray(x, np.int64).astype(np.int32), device="cuda")
    ctx, q = i32(c.ctx), i32(c.q)
    cu_pages, ids = i32(np.concatenate([[0], np.cumsum(need)])), i32(np.concatenate(c.own_pages))
    out = torch.zeros((12, 8, 128), dtype=torch.float16, device="cuda")
    lse = torch.zeros((12, 8), device="cuda")

    def step(out, lse, ws=None):
        # (a session's page list may be longer than its keys need)
        batch = gpu.build_metadata(ctx, q, cu_pages, ids, c.page, max(need), len(c.pool),
                                   split_pages=4, max_work=4096, max_rows=12)
        plan = gpu.plan_attention(batch, 8, 128, rows=12, max_q_len=1, prefixes=d["shared"])
        gpu.latent_attention(plan, d["pages"], d["ql"], d["qr"], c.scale, rope_dim=16, q8=True,
                             out=out, lse=lse, workspace=ws)
        return plan

    _say("graph of a growing batch")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ws = gpu.attention_workspace(step(out, lse))
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(out, lse, ws)
    for share in (0.0, 0.3, 1.0, 0.6):
        now = (np.array(full) * share).astype(int)
        ctx.copy_(torch.from_numpy(now.astype(np.int32)))
        eager, elses = torch.zeros_like(out), torch.zeros_like(lse)
        step(eager, elses)
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager) and torch.equal(lse, elses), share
        want = expect(replace(c, ctx=now))
        check(c, out, lse, want)


@pytest.mark.gpu
@pytest.mark.parametrize("q8", [False, True])
def test_pages_past_32_bit_offsets(gpu, q8):
    """A session on the last pages of a pool of more than 4 GiB, and a prefix there, give the bits
    that the same contents give on its first pages; read back too."""
    import torch
    H, kv, rope, page, n = 16, 512, 64, 64, 300
    P = (1 << 32) // (page * ((kv + 2 * rope + kv // 32) if q8 else 2 * (kv + rope))) + 40
    _say(f"a pool of {P} pages q8={q8}")
    cache = (gpu.QuantizedLatentCache if q8 else gpu.PagedLatentCache)(1, P, page, kv, rope)
    append = gpu.append_latent_q8 if q8 else gpu.append_latent
    i32 = lambda x: torch.tensor(np.asarray(x, np.int64).astype(np.int32), device="cuda")
    torch.manual_seed(18)
    x, key = torch.randn(n, kv, device="cuda"), torch.randn(n, rope, device="cuda")
    lists = [np.arange(5), P - 1 - np.arange(5)]
    t = np.arange(n)
    for l in lists:
        append(cache, 0, x, key, i32(l[t // page] * page + t % page))
    if q8:
        got = [gpu.read_latent_q8(cache, 0, i32(l[t // page] * page + t % page)) for l in lists]
        assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])
        assert (got[0][0].float() - x).abs().max() < 0.5  # e4m3 of |x| < 8
    ql = torch.randn(1, H, kv, device="cuda").half().repeat(2, 1, 1)
    qr = torch.randn(1, H, rope, device="cuda").half().repeat(2, 1, 1)
    batch = gpu.build_metadata(i32([n - 1] * 2), i32([1, 1]), i32([0, 5, 10]),
                               i32(np.concatenate(lists)), page, 5, P, max_rows=2)
    shared = gpu.SharedPrefixes(i32([0, 1, 2]), i32([n, n]), i32([0, 5, 10]),
                                i32(np.concatenate(lists)))
    for prefixes in (None, shared):
        plan = gpu.plan_attention(batch, H, kv, rows=2, prefixes=prefixes)
        plan.read_info()
        out = gpu.latent_attention(plan, cache.layer(0), ql, qr, 0.05, rope_dim=rope, q8=q8)
        assert torch.equal(out[0], out[1]) and out.isfinite().all() and (out != 0).any()


@pytest.mark.gpu
def test_tensors_made_by_a_call_belong_to_its_stream(gpu):
    """Without out and workspace, on a stream that is not the current one: what the call makes is
    filled before its kernels run, however far behind the current stream is."""
    import torch
    c = make(8, 128, 16, 64, 0, True, [(k * 50, 1) for k in range(20)], [(12, 500)], seed=17)
    d = device(gpu, c)
    plan, want, _ = call(gpu, c, d)
    slots = torch.arange(64, dtype=torch.int32, device="cuda")
    cache = gpu.QuantizedLatentCache(1, len(c.pool), 64, 128, 16, storage=d["pages"][None])
    lat, key = gpu.read_latent_q8(cache, 0, slots)
    a = torch.randn(4096, 4096, device="cuda", dtype=torch.float16)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    _say("made on a side stream")
    for _ in range(20):
        b = a @ a  # the current stream is busy
    sided = gpu.plan_attention(d["batch"], 8, 128, rows=20, max_q_len=1, prefixes=d["shared"],
                               stream=side)
    got = gpu.latent_attention(sided, d["pages"], d["ql"], d["qr"], c.scale, rope_dim=16, q8=True,
                               stream=side)
    lat2, key2 = gpu.read_latent_q8(cache, 0, slots, stream=side)
    side.synchronize()
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    assert torch.equal(lat.view(torch.int16), lat2.view(torch.int16))
    assert torch.equal(key.view(torch.int16), key2.view(torch.int16))


@pytest.mark.gpu
def test_bad_batches_and_prefixes_fail_the_plan_and_write_nothing(gpu):
    """Every error that only the device arrays hold: the plan says which entry, and the call over
    it leaves its outputs alone."""
    import torch
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    c = make(8, 128, 16, 64, 0, False, [(10, 1), (20, 1), (30, 2)], [(2, 100)], seed=7)
    d = device(gpu, c)
    s, n = d["shared"], len(c.pool)
    ids = s.page_ids.tolist()

    def expect_bad(match, rows=d["rows"], max_q_len=2, batch=d["batch"], **kw):
        x = gpu.SharedPrefixes(**dict(dict(cu_groups=s.cu_groups, prefix_len=s.prefix_len,
                                           cu_pages=s.cu_pages, page_ids=s.page_ids), **kw))
        plan = gpu.plan_attention(batch, 8, 128, rows=rows, max_q_len=max_q_len, prefixes=x)
        with pytest.raises(gpu.MlaError, match=match) as e:
            plan.read_info()
        assert e.value.code == "invalid_argument"
        out = torch.full((rows, 8, 128), 5.0, dtype=torch.float16, device="cuda")
        lse = torch.full((rows, 8), 5.0, device="cuda")
        gpu.latent_attention(plan, d["pages"], d["ql"][:rows], d["qr"][:rows], c.scale,
                             rope_dim=16, out=out, lse=lse)
        assert (out == 5).all() and (lse == 5).all()

    _say("bad prefixes")
    expect_bad("entry 0", cu_groups=i32([0, 4]))
    expect_bad("entry 0", cu_groups=i32([-1, 2]))
    expect_bad("entry 0", cu_groups=i32([2, 1]))
    expect_bad("entry 1", cu_groups=i32([0, 2, 1]), prefix_len=i32([100, 0]), cu_pages=i32([0, 2, 2]))
    expect_bad("entry 0", prefix_len=i32([129]))
    expect_bad("entry 0", prefix_len=i32([-1]))
    expect_bad("entry 0", cu_pages=i32([0, 3]))
    expect_bad("entry 0", cu_pages=i32([-1, 2]))
    expect_bad("entry 0", cu_pages=i32([2, 0]))
    expect_bad("entry 0", page_ids=i32([ids[0], n]))
    expect_bad("entry 0", page_ids=i32([-1, ids[1]]))
    _say("bad rows")
    expect_bad("entry 3", max_q_len=1)  # the third session's two rows, behind one group
    expect_bad("more rows", rows=3)
    bad = gpu.build_metadata(i32([10]), i32([1]), i32([0, 1]), i32([n]), 64, 1, n, max_rows=1)
    expect_bad("metadata", rows=1, batch=bad, cu_groups=i32([0, 1]))


@pytest.mark.gpu
def test_a_plan_for_other_sizes_writes_nothing(gpu):
    c = make(8, 128, 16, 64, 0, False, [(10, 1), (20, 1)], seed=7)
    d = device(gpu, c)
    _say("plan of other sizes")
    plan = gpu.plan_attention(d["batch"], 8, 128, rows=2, max_q_len=2)
    replan = lambda q, words: gpu.AttentionPlan(d["batch"], 8, 128, 2, q, None, words)
    other = replan(1, plan.words)  # tables of the same size
    _, out, lse = call(gpu, c, d, other, workspace=gpu.attention_workspace(plan))
    assert (out == 5).all() and (lse == 5).all()
    plan.read_info()
    with pytest.raises(gpu.MlaError, match="host_info"):
        other._info = plan._info
        call(gpu, c, d, other, workspace=gpu.attention_workspace(plan))
    small = replan(2, plan.words[:64])
    with pytest.raises(gpu.MlaError, match="other sizes"):
        call(gpu, c, d, small, workspace=gpu.attention_workspace(plan))


def test_refusals_of_planned_attention():
    import cpp_inference_train_engine_amd as mla
    L = mla.lib()
    buf = ctypes.create_string_buffer(4096)
    a = ctypes.addressof(buf)
    a += -a % 256
    size = L.mla_attention_plan_bytes
    assert size(4, 4, 8, 128, 1, 0) > 0
    for bad in ((-1, 4, 8, 128, 1, 0), (4, -1, 8, 128, 1, 0), (4, 4, 0, 128, 1, 0),
                (4, 4, 8, 0, 1, 0), (4, 4, 8, 128, 0, 0), (4, 4, 8, 128, 1, -1),
                (4, 4, 8, 128, 1, 5), (4, 1 << 28, 8, 128, 1, 0), (1 << 22, 4, 8, 128, 1, 1),
                (2**31 - 1, 4, 8, 128, 1, 0), (4, 1 << 24, 64, 128, 1 << 24, 4)):
        assert size(*bad) == 0 and L.mla_attention_workspace_bytes(*bad) == 0
    names = ("stream", "B", "rows", "H", "kv", "page", "max_q", "cu_q", "cu_k", "info", "groups",
             "cu_groups", "prefix_len", "cu_pages", "ids", "n_ids", "pool", "plan", "bytes")

    def plan(**kw):
        v = dict(zip(names, (None, 4, 4, 8, 128, 64, 1, a, a, a, 1, a, a, a, a, 1, 10, a, 1 << 30)), **kw)
        return L.mla_plan_attention(*[v[n] for n in names])

    for kw in (dict(B=-1), dict(rows=-1), dict(H=0), dict(kv=0), dict(page=0), dict(max_q=0),
               dict(groups=-1), dict(groups=5), dict(n_ids=-1), dict(pool=-1), dict(cu_q=None),
               dict(cu_k=None), dict(info=None), dict(cu_groups=None), dict(prefix_len=None),
               dict(cu_pages=None), dict(ids=None), dict(plan=None), dict(plan=a + 4),
               dict(bytes=16)):
        assert plan(**kw) == 1, kw
    names2 = ("stream", "B", "rows", "H", "kv", "rope", "page", "max_q", "dtype", "fmt", "scale",
              "table", "max_pages", "pool", "pages", "ql", "qr", "groups", "cu_pages", "ids",
              "plan", "plan_bytes", "info", "out", "lse", "ws", "ws_bytes")

    def attend(**kw):
        v = dict(zip(names2, (None, 4, 4, 8, 128, 16, 64, 1, 0, 1, 0.1, a, 4, 10, a, a, a, 1, a, a,
                              a, 1 << 30, None, a, None, a, 1 << 40)), **kw)
        return L.mla_latent_attention(*[v[n] for n in names2])

    for kw in (dict(B=-1), dict(rows=-1), dict(H=0), dict(kv=0), dict(rope=-1), dict(page=0),
               dict(max_q=0), dict(dtype=2), dict(fmt=2), dict(scale=0.0), dict(scale=float("nan")),
               dict(scale=float("inf")), dict(max_pages=-1), dict(pool=-1), dict(groups=5),
               dict(table=None), dict(pages=None), dict(ql=None), dict(qr=None), dict(plan=None),
               dict(out=None), dict(ws=None), dict(cu_pages=None), dict(pages=a + 8),
               dict(ql=a + 2), dict(qr=a + 8), dict(out=a + 8), dict(plan=a + 8), dict(ws=a + 4),
               dict(plan_bytes=16), dict(ws_bytes=16), dict(info=a)):
        assert attend(**kw) == 1, kw
    for kw in (dict(kv=100), dict(kv=544), dict(rope=4), dict(rope=72), dict(page=40), dict(page=65552)):
        assert attend(**kw) == 3, kw
    assert attend(rows=0) == 0  # nothing to do
    st = L.mla_read_plan_info(None, None, a)
    assert st == 1


def test_python_wrappers_refuse_wrong_tensors(monkeypatch):
    import torch
    import cpp_inference_train_engine_amd as mla
    i = torch.zeros(8, dtype=torch.int32)
    rb = mla.RaggedBatch(B=2, page_size=64, max_pages=1, num_pool_pages=2, max_work=2, max_rows=2,
                         **{k: i for k in ("cu_seqlens_q", "cu_seqlens_k", "page_table",
                                           "slot_mapping", "num_splits", "cu_splits",
                                           "work_session", "work_split", "work_desc",
                                           "work_pages", "info")})
    monkeypatch.setattr(mla.ops, "_gpu", lambda: 0)
    with pytest.raises(ValueError, match="no plan"):
        mla.plan_attention(rb, 0, 128)
    with pytest.raises(ValueError, match="GPU"):
        mla.plan_attention(rb, 8, 128)
    with pytest.raises(ValueError, match="cu_groups"):
        mla.plan_attention(rb, 8, 128, prefixes=mla.SharedPrefixes(i, i[:1], i[:2], i))
    plan = mla.AttentionPlan(rb, 8, 128, 2, 1, None, i)
    q = torch.zeros((2, 8, 128), dtype=torch.float16)
    monkeypatch.setattr(mla.ops, "stream_handle", lambda stream=None: None)
    for pages in (q, torch.zeros((2, 9216)), torch.zeros((2, 9216), dtype=torch.float16)):
        with pytest.raises(ValueError, match="pages"):
            mla.latent_attention(plan, pages, q, q[:, :, :16], 0.1, rope_dim=16,
                                 out=q, workspace=i.view(torch.uint8))
    monkeypatch.setattr(torch.Tensor, "get_device", lambda t: 0)
    pages = torch.zeros((2, 9216), dtype=torch.float16)
    for ql in (q[:1], q.bfloat16(), q.transpose(0, 1)):
        with pytest.raises(ValueError, match="q_latent"):
            mla.latent_attention(plan, pages, ql, q[:, :, :16], 0.1, rope_dim=16,
                                 out=q, workspace=i.view(torch.uint8))
    with pytest.raises(ValueError, match="q_rope"):
        mla.latent_attention(plan, pages, q, q[:, :, :16], 0.1, rope_dim=16,  # not contiguous
                             out=q, workspace=i.view(torch.uint8))


@pytest.mark.gpu
@pytest.mark.parametrize("q8", [False, True])
def test_a_serving_run(gpu, q8):
    """As a server uses them: a prompt shared by all sessions is written once; sessions append
    their own tokens through the metadata's slots step by step -- a chunk, drafted tokens, single
    tokens -- and each step's attention is that of a cache that holds everything."""
    import torch
    H, kv, rope, page, P = 8, 128, 16, 64, 40
    rng = np.random.default_rng(11)
    dev = lambda x: torch.from_numpy(np.ascontiguousarray(x)).cuda()
    i32 = lambda x: dev(np.asarray(x, np.int32))
    cache = (gpu.QuantizedLatentCache if q8 else gpu.PagedLatentCache)(1, P, page, kv, rope)
    append = gpu.append_latent_q8 if q8 else gpu.append_latent

    def write(x, key, slots):
        append(cache, 0, dev(x), dev(key), slots)
        if not q8:
            return (to_bits(x, 0), to_bits(key, 0))
        lat, kk = gpu.read_latent_q8(cache, 0, slots)
        return lat.cpu().numpy().view(np.uint16), kk.cpu().numpy().view(np.uint16)

    draw = lambda n: (rng.standard_normal((n, kv)).astype(np.float32),
                      rng.standard_normal((n, rope)).astype(np.float32))
    ids = rng.permutation(P).astype(np.int32)
    prompt = 150
    pslots = ids[np.arange(prompt) // page] * page + np.arange(prompt) % page
    told = write(*draw(prompt), i32(pslots))
    B, per = 5, 6  # six pages for each session
    lists = [ids[3 + per * b:3 + per * b + per] for b in range(B)]
    own = [(np.zeros((0, kv), np.uint16), np.zeros((0, rope), np.uint16)) for _ in range(B)]
    ctx = np.zeros(B, int)
    for step, q in enumerate(([70, 1, 33, 9, 1], [4, 4, 4, 4, 4], [1] * 5, [1, 0, 1, 0, 130], [1] * 5)):
        q = np.array(q)
        _say(f"serving run q8={q8} step {step} rows {q.tolist()}")
        rows = int(q.sum())
        batch = gpu.build_metadata(i32(ctx), i32(q), i32(np.arange(B + 1) * per),
                                   i32(np.concatenate(lists)), page, per, P, max_rows=rows)
        x, key = draw(rows)
        lat, kk = write(x, key, batch.slot_mapping)
        at = 0
        for b in range(B):
            own[b] = tuple(np.concatenate([o, n[at:at + q[b]]]) for o, n in zip(own[b], (lat, kk)))
            at += q[b]
        shared = gpu.SharedPrefixes(i32([0, B]), i32([prompt]), i32([0, 3]), i32(ids[:3]))
        plan = gpu.plan_attention(batch, H, kv, max_q_len=int(q.max()), prefixes=shared)
        ql = dev(rng.standard_normal((rows, H, kv))).half()
        qr = dev(rng.standard_normal((rows, H, rope))).half()
        lse = torch.zeros((rows, H), device="cuda")
        out = gpu.latent_attention(plan, cache.layer(0), ql, qr, 0.1, rope_dim=rope, q8=q8, lse=lse)
        plan.read_info()
        want, at = [], 0
        for b in range(B):
            k16 = [ref.from_bits(np.concatenate([t, o]), 0) for t, o in zip(told, own[b])]
            seen = np.arange(prompt + ctx[b] + q[b])[None] <= prompt + ctx[b] + np.arange(q[b])[:, None]
            want.append(ref.attention(ql[at:at + q[b]].double().cpu().numpy(),
                                      qr[at:at + q[b]].double().cpu().numpy(), *k16, seen, 0.1))
            at += q[b]
        c = Case(H, kv, rope, page, 0, q8, None, None, None, None, None, None, None, None, None)
        check(c, out, lse, tuple(np.concatenate(w) for w in zip(*want)))
        ctx += q
