"""What the operators of the 8-bit latent cache and of shared prefixes are measured on.

Kinds (``case["kind"]``):
  write   quantise new tokens' latents into the paged 8-bit cache (``append_latent_q8``)
  read    the cached tokens of sessions read back as 16-bit rows (``read_latent_q8``)
  attend  attention of every query row of a batch over its paged cache (``latent_attention``):
          decode rows, rows of drafted tokens, prompt chunks; over the 8-bit cache or the 16-bit
          one, and with prefixes that groups of sessions share

``own`` chooses between the plain form (elementary torch operations in 32 bits, whatever the
storage type, rounded once at the end) and the package's calls.  Lengths follow from the case's
numbers alone; the seed draws the contents (cache, queries, new tokens, page permutation).  Cached
latents are kv_norm-ed, so N(0, 1).

The 8-bit cache: page p is one record of bytes.  A token's latent is cut into blocks of 32
columns; a block holds e4m3 values and one power of two, the smallest 2^k with max|x| <= 448 2^k,
k limited so that every value is one of the 16-bit type as well (fp16: -15..7, bf16: -117..119;
larger finite values saturate, infinities and NaN become NaN).  With t = slot / 16, n = slot % 16,
j = column / 32, g = column % 32 / 8, e = column % 8 and J = kv / 32:
  latent  byte t*16*kv + (j/2)*1024 + (16 g + n)*16 + (j%2)*8 + e   (a last odd j: (16 g + n)*8)
  rope    16-bit word (t*(rope/8) + c/8)*128 + n*8 + c%8, after the latents of the page
  scale   byte slot*J + j holds k + 127, after the rope keys of the page
"""
import math
import random

import torch

own = False

RANGE = {"f16": (-15, 7), "bf16": (-117, 119)}
TYPE = {"f16": torch.float16, "bf16": torch.bfloat16}


def _package():  # only where `own` is true: the plain forms need torch alone
    import cpp_inference_train_engine_amd as package
    return package


# ------------------------------------------------------------------------------- cases ----
BASE = dict(heads=8, kv=128, rope=16, page=64, dtype="f16")     # the benchmark's model
WIDE = dict(heads=128, kv=512, rope=64, page=64, dtype="bf16")  # the DeepSeek-like latent shape


def listed():
    return [
        # A decode step's append: one new token of each of 64 sessions.  Latency.
        dict(name="write_64", kind="write", tokens=64, run=1, **BASE),
        # A prefill step's append at the wide latent shape.
        dict(name="write_wide", kind="write", tokens=7001, run=777, **WIDE),
        # One session's cache read back, to move it or to extend it elsewhere.
        dict(name="read_1037", kind="read", tokens=1037, run=1037, **BASE),
        # Many sessions' caches read back at the wide latent shape.
        dict(name="read_wide", kind="read", tokens=60013, run=2501, **WIDE),
        # One user's chat turn: a single decode row.  Latency.
        _attend("q8_1", 1, 1040, 1040, 1, "q8", **BASE),
        # The headline decode batch, 64 ragged sessions, over the 8-bit cache.
        _attend("q8_64", 64, 128, 4096, 1, "q8", **BASE),
        # Long contexts of a busy server at the wide latent shape: the largest call.
        _attend("q8_wide", 64, 2048, 14000, 1, "q8", **WIDE),
        # Five drafted tokens of each of 24 sessions scored in one call.
        _attend("q8_draft", 24, 64, 4096, 5, "q8", **BASE),
        # Prompt chunks on cached contexts.
        _attend("q8_chunk", 4, 509, 2048, 509, "q8", **BASE),
        # 64 chats behind one long system prompt.
        _attend("shared_64", 64, 1, 700, 1, "16", groups=1, prefix=4000, **BASE),
        # Five tenants, each with its own prompt, 200 sessions, over the 8-bit cache.
        _attend("shared_groups", 200, 1, 900, 1, "q8", groups=5, prefix=2048, **BASE),
        # Many questions about one long document at the wide latent shape.
        _attend("shared_wide", 48, 16, 1000, 1, "16", groups=1, prefix=8191, **WIDE),
    ]


def _attend(name, sessions, low, high, q, cache, groups=0, prefix=0, **shape):
    """low..high: keys of a session's own pages; q: query rows of a session, all of them when
    the call scores a fixed number of drafted tokens or a chunk."""
    return dict(name=name, kind="attend", sessions=sessions, low=low, high=high, q=q, cache=cache,
                groups=groups, prefix=prefix, **shape)


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw(rng):
    shape = rng.choice([BASE, BASE, dict(BASE, heads=16, dtype="bf16"), WIDE,
                        dict(WIDE, heads=rng.choice([16, 32, 64, 128]), dtype="f16"), None, None])
    if shape is None:
        shape = dict(heads=rng.choice([1, 4, 8, 12, 20, 32, 40]),
                     kv=rng.choice([32, 64, 96, 128, 256, 384]), rope=rng.choice([8, 16, 32, 64]),
                     page=rng.choice([16, 32, 64, 128]), dtype=rng.choice(["f16", "bf16"]))
    kind = rng.choice(["write", "read", "decode", "decode", "draft", "chunk", "shared", "shared"])
    if kind in ("write", "read"):
        tokens = _log_int(rng, 1, 60000 if kind == "read" else 7000)
        return dict(kind=kind, tokens=tokens, run=_log_int(rng, 1, tokens), **shape)
    cache = rng.choice(["q8", "q8", "16"])
    if kind == "shared":
        b = _log_int(rng, 2, 256)
        c = _attend("", b, 1, _log_int(rng, 1, 3000), rng.choice([1, 1, 1, 4]), cache,
                    groups=min(b, _log_int(rng, 1, 16)), prefix=_log_int(rng, 16, 12000), **shape)
    elif kind == "chunk":
        q = _log_int(rng, 16, 700)
        c = _attend("", rng.randint(1, 8), q, q + _log_int(rng, 1, 3000), q, "q8", **shape)
    else:
        q = 1 if kind == "decode" else rng.randint(2, 9)
        lo = _log_int(rng, q, 2000)
        c = _attend("", _log_int(rng, 1, 300), lo, _log_int(rng, lo, 14000), q, "q8", **shape)
    del c["name"]
    c["high"] = max(c["high"], c["q"])
    c["low"] = max(c["low"], c["q"])
    return c


def draw(rng):
    most = work(next(c for c in listed() if c["name"] == "q8_wide"))
    while True:
        c = _draw(rng)
        w = work(c)
        if c["kind"] != "attend" or (w["flops"] <= most["flops"] and w["bytes"] <= most["bytes"]
                                     and _padded(c) <= 64 * 14000 * 700):
            return c


# --------------------------------------------------------------------- shapes of a case ----
def _rng_of(case):
    return random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))


def _lengths(case):
    """Keys in each session's own pages, its new tokens among them."""
    rng = _rng_of(case)
    low = max(case["low"], case["q"])
    return [rng.randint(low, max(low, case["high"])) for _ in range(case["sessions"])]


def _group_ends(case):
    """Sessions dealt to the groups in order, as evenly as they go."""
    b, n = case["sessions"], case["groups"]
    return [b * (i + 1) // n for i in range(n)]


def _prefix_lengths(case):
    """Each group's prefix, the first one as long as the case says."""
    rng = _rng_of(dict(case, what="prefix"))
    n, p = case["groups"], case["prefix"]
    return [p if i == 0 else rng.randint(max(1, p // 2), p) for i in range(n)]


def _prefix_of(case):
    """The prefix length of each session."""
    got, at = [], 0
    for end, n in zip(_group_ends(case), _prefix_lengths(case)):
        got += [n] * (end - at)
        at = end
    return got or [0] * case["sessions"]


def _padded(case):
    """Elements of the plain form's key rows and scores, which pad the sessions to the longest."""
    keys = max(a + b for a, b in zip(_lengths(case), _prefix_of(case)))
    return case["sessions"] * keys * (case["kv"] + case["rope"] + case["q"] * case["heads"])


def _token_bytes(case):
    kv, rope = case["kv"], case["rope"]
    return kv + 2 * rope + kv // 32 if case.get("cache", "q8") == "q8" else 2 * (kv + rope)


def work(case):
    kv, rope, n = case["kv"], case["rope"], case.get("tokens", 0)
    if case["kind"] == "write":  # fp32 rows in, packed rows out
        return {"bytes": n * (4 * (kv + rope) + _token_bytes(case) + 4), "flops": 0}
    if case["kind"] == "read":   # packed rows in, 16-bit rows out
        return {"bytes": n * (2 * (kv + rope) + _token_bytes(case) + 4), "flops": 0}
    lens, pre, q, heads = _lengths(case), _prefix_of(case), case["q"], case["heads"]
    rows = q * len(lens)
    seen = sum(q * (p + k - q) + q * (q + 1) // 2 for k, p in zip(lens, pre))
    keys = sum(lens) + sum(_prefix_lengths(case))
    return {"bytes": keys * _token_bytes(case) + rows * heads * (4 * kv + 2 * rope + 4),
            "flops": 2 * seen * heads * (2 * kv + rope)}


# ------------------------------------------------------------------------------- states ----
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _randn(gen, shape, dtype):
    return torch.empty(shape, dtype=dtype, device="cuda").normal_(generator=gen)


def _sections(case):
    """Bytes of a page's latents, rope keys and scales."""
    page, kv, rope = case["page"], case["kv"], case["rope"]
    return page * kv, 2 * page * rope, page * (kv // 32)


def _views(pages, case):
    """The three parts of the 8-bit records: e4m3 latents, 16-bit keys, scale bytes."""
    a, b, c = _sections(case)
    return {"latent": pages[:, :a].view(torch.float8_e4m3fn),
            "rope": pages[:, a:a + b].view(TYPE[case["dtype"]]), "scale": pages[:, a + b:]}


def _pool(case, gen, count):
    """A page pool in use: N(0, 1) latents and keys of every slot."""
    page, kv, rope, dt = case["page"], case["kv"], case["rope"], TYPE[case["dtype"]]
    if case.get("cache", "q8") == "16":
        return _randn(gen, (count, page * (kv + rope)), dt)
    pages = torch.empty((count, sum(_sections(case))), dtype=torch.uint8, device="cuda")
    v = _views(pages, case)
    v["rope"].copy_(_randn(gen, (count, page * rope), dt))
    values, k = _quantise(_randn(gen, (count * page, kv), torch.float32), case["dtype"])
    v["latent"].copy_(_layout(values, page, kv))
    v["scale"].copy_(k.view(count, -1))
    return pages


def _layout(rows, page, kv):
    """Token rows [count * page, kv] in the order of the page records: [count, page * kv]."""
    n, t, j = rows.shape[0] // page, page // 16, kv // 32
    x = rows.view(torch.uint8).view(n, t, 16, j, 4, 8)
    pairs = x[:, :, :, :j - j % 2].reshape(n, t, 16, j // 2, 2, 4, 8)
    pairs = pairs.permute(0, 1, 3, 5, 2, 4, 6).reshape(n, t, 512 * (j - j % 2))
    last = x[:, :, :, j - j % 2:].permute(0, 1, 3, 4, 2, 5).reshape(n, t, 512 * (j % 2))
    return torch.cat([pairs, last], 2).view(n, page * kv).view(rows.dtype)


def _slots(case, rng):
    """Flat slots of runs of consecutive tokens, each starting somewhere in a page of its own, in
    pages numbered in order of use; and the pages used."""
    page, n, run = case["page"], case["tokens"], case["run"]
    slots, used = [], 0
    while len(slots) < n:
        m, off = min(run, n - len(slots)), rng.randrange(page)
        slots += range(used * page + off, used * page + off + m)
        used += -(-(off + m) // page)
    return slots, used


def prepare(case, seed):
    gen = _gen(seed)
    page, kv, rope, heads = case["page"], case["kv"], case["rope"], case["heads"]
    dt = TYPE[case["dtype"]]
    s = dict(case=case)
    if case["kind"] != "attend":
        slots, used = _slots(case, _rng_of(case))
        perm = torch.randperm(used + 2, generator=gen, device="cuda")
        slots = torch.tensor(slots, device="cuda")
        s["slots"] = (perm[slots // page] * page + slots % page).to(torch.int32)
        s["pages"] = _pool(case, gen, used + 2)
        if case["kind"] == "write":
            s["ckv"] = _randn(gen, (case["tokens"], kv), torch.float32)
            s["krope"] = _randn(gen, (case["tokens"], rope), torch.float32)
        else:
            s["ckv"] = torch.empty((case["tokens"], kv), dtype=dt, device="cuda")
            s["krope"] = torch.empty((case["tokens"], rope), dtype=dt, device="cuda")
        if own:
            s["cache"] = _package().QuantizedLatentCache(
                1, used + 2, page, kv, rope, dtype=_code(case), storage=s["pages"][None])
        return s
    lens, pre, q = _lengths(case), _prefix_lengths(case), case["q"]
    need = [-(-n // page) for n in pre + lens]
    ids = torch.randperm(sum(need) + 1, generator=gen, device="cuda").to(torch.int32)[:sum(need)]
    ends = [sum(need[:i + 1]) for i in range(len(need))]
    g, b = len(pre), len(lens)
    rows = b * q
    s.update(rows=rows, pool=sum(need) + 1, max_pages=max(need[g:]),
             max_keys=max(a + c for a, c in zip(lens, _prefix_of(case))),
             ctx_len=_ints([n - q for n in lens]), q_len=_ints([q] * b), k_len=_ints(lens),
             cu_pages=_ints([0] + [e - sum(need[:g]) for e in ends[g:]]), page_ids=ids[sum(need[:g]):].clone(),
             cu_groups=_ints([0] + _group_ends(case)), prefix_len=_ints(pre),
             cu_prefix_pages=_ints([0] + ends[:g]), prefix_page_ids=ids[:sum(need[:g])].clone(),
             pages=_pool(case, gen, sum(need) + 1), ql=_randn(gen, (rows, heads, kv), dt),
             qr=_randn(gen, (rows, heads, rope), dt),
             out=torch.zeros((rows, heads, kv), dtype=dt, device="cuda"),
             lse=torch.zeros((rows, heads), dtype=torch.float32, device="cuda"))
    if own:  # the step's metadata and plan, which every layer's call uses
        mla = _package()
        s["batch"] = mla.build_metadata(s["ctx_len"], s["q_len"], s["cu_pages"], s["page_ids"],
                                        page, s["max_pages"], s["pool"], split_pages=64,
                                        max_work=sum(-(-n // 64) for n in need), max_rows=rows)
        shared = mla.SharedPrefixes(s["cu_groups"], s["prefix_len"], s["cu_prefix_pages"],
                                    s["prefix_page_ids"]) if g else None
        s["plan"] = mla.plan_attention(s["batch"], heads, kv, rows=rows, max_q_len=q,
                                       prefixes=shared)
        s["plan"].read_info()
        s["workspace"] = mla.attention_workspace(s["plan"])
    return s


def _code(case):
    return _package().DTYPE_F16 if case["dtype"] == "f16" else _package().DTYPE_BF16


def _scale(case):
    return 1 / math.sqrt(case["kv"] / 2 + case["rope"])


# --------------------------------------------------------------------------------- runs ----
def run(s):
    case = s["case"]
    if own:
        mla = _package()
        if case["kind"] == "write":
            mla.append_latent_q8(s["cache"], 0, s["ckv"], s["krope"], s["slots"])
            return _views(s["pages"], case)
        if case["kind"] == "read":
            mla.read_latent_q8(s["cache"], 0, s["slots"], ckv=s["ckv"], krope=s["krope"])
            return {"ckv": s["ckv"], "krope": s["krope"]}
        mla.latent_attention(s["plan"], s["pages"], s["ql"], s["qr"], _scale(case),
                             rope_dim=case["rope"], dtype=_code(case), q8=case["cache"] == "q8",
                             out=s["out"], lse=s["lse"], workspace=s["workspace"])
        return {"out": s["out"], "lse": s["lse"]}
    if case["kind"] == "write":
        return _plain_write(s, case)
    if case["kind"] == "read":
        lat, key = _tokens(s["pages"], case, s["slots"].long())
        return {"ckv": lat.to(s["ckv"].dtype), "krope": key.to(s["krope"].dtype)}
    return _plain_attend(s, case)


def _quantise(x, dtype):
    """e4m3 values and scale bytes of fp32 rows [n, kv]: [n, kv] float8 and [n, kv / 32] uint8."""
    lo, hi = RANGE[dtype]
    b = x.view(x.shape[0], -1, 32)
    fine = torch.isfinite(b)
    amax = torch.where(fine, b.abs(), 0.0).amax(2)
    m, e = torch.frexp(amax)  # amax = m 2^e with m in [0.5, 1); 448 = 0.875 * 2^9
    k = torch.where(m <= 0.875, e - 9, e - 8)
    k = torch.where(amax > 0, k, lo).clamp(lo, hi)
    y = torch.ldexp(b, -k[..., None]).clamp(-448.0, 448.0)
    y = torch.where(fine, y, math.nan).to(torch.float8_e4m3fn)
    return y.view(x.shape), (k + 127).to(torch.uint8)


def _latent_bytes(slot, case):
    """Byte offset of every latent column of page slots [n]: [n, kv]."""
    kv = case["kv"]
    r = torch.arange(kv, device="cuda")
    j, g, e = r // 32, r % 32 // 8, r % 8
    t, n = slot[:, None] // 16, slot[:, None] % 16
    odd = (kv // 32 % 2 == 1) & (j == kv // 32 - 1)
    inside = torch.where(odd, j * 512 + (16 * g + n) * 8,
                         j // 2 * 1024 + (16 * g + n) * 16 + j % 2 * 8) + e
    return t * 16 * kv + inside


def _rope_words(slot, case):
    """16-bit word offset of every rope column of page slots [n]: [n, rope]."""
    c = torch.arange(case["rope"], device="cuda")
    t, n = slot[:, None] // 16, slot[:, None] % 16
    return (t * (case["rope"] // 8) + c // 8) * 128 + n * 8 + c % 8


def _plain_write(s, case):
    page, kv = case["page"], case["kv"]
    v = _views(s["pages"], case)
    slots = s["slots"].long()
    p, o = slots[:, None] // page, slots % page
    values, k = _quantise(s["ckv"], case["dtype"])
    v["latent"].view(torch.uint8)[p, _latent_bytes(o, case)] = values.view(torch.uint8)
    v["rope"][p, _rope_words(o, case)] = s["krope"].to(v["rope"].dtype)
    j = torch.arange(kv // 32, device="cuda")
    v["scale"][p, o[:, None] * (kv // 32) + j] = k
    return v


def _tokens(pages, case, slots):
    """fp32 latents and rope keys of flat slots [n]."""
    page, kv, rope = case["page"], case["kv"], case["rope"]
    p, o = slots[:, None] // page, slots % page
    if case.get("cache", "q8") == "16":
        r, c = torch.arange(kv, device="cuda"), torch.arange(rope, device="cuda")
        t, n = o[:, None] // 16, o[:, None] % 16
        lat = ((t * (kv // 32) + r // 32) * 4 + r % 32 // 8) * 128 + n * 8 + r % 8
        key = page * kv + (t * (rope // 8) + c // 8) * 128 + n * 8 + c % 8
        return pages[p, lat].float(), pages[p, key].float()
    v = _views(pages, case)
    lat = v["latent"].view(torch.uint8)[p, _latent_bytes(o, case)].view(torch.float8_e4m3fn).float()
    j = torch.arange(kv // 32, device="cuda")
    k = v["scale"][p, o[:, None] * (kv // 32) + j].int() - 127
    lat = torch.ldexp(lat.view(-1, kv // 32, 32), k[..., None]).view(-1, kv)
    return lat, v["rope"][p, _rope_words(o, case)].float()


def _plain_attend(s, case):
    page, heads, q = case["page"], case["heads"], case["q"]
    kv, rope, b, keys = case["kv"], case["rope"], case["sessions"], s["max_keys"]
    at = torch.arange(keys, device="cuda")[None]           # key index: the prefix, then own keys
    session = torch.arange(b, device="cuda")
    if case["groups"]:
        group = torch.bucketize(session.int(), s["cu_groups"][1:], right=True)
        pre = s["prefix_len"][group].long()[:, None]
        first = s["cu_prefix_pages"][group].long()[:, None]
        shared = s["prefix_page_ids"][(first + at.clamp(max=pre - 1) // page).clamp(
            max=s["prefix_page_ids"].numel() - 1)].long() * page + at % page
    else:
        pre = torch.zeros((b, 1), dtype=torch.long, device="cuda")
        shared = torch.zeros((b, keys), dtype=torch.long, device="cuda")
    total = pre + s["k_len"].long()[:, None]
    mine = (at - pre).clamp(min=0).minimum(s["k_len"].long()[:, None] - 1)
    slot = s["page_ids"][s["cu_pages"][:-1].long()[:, None] + mine // page].long() * page + mine % page
    slot = torch.where(at < pre, shared, slot)
    lat, key = _tokens(s["pages"], case, slot.view(-1))
    lat, key = lat.view(b, keys, kv), key.view(b, keys, rope)
    ql = s["ql"].float().view(b, q * heads, kv)
    qr = s["qr"].float().view(b, q * heads, rope)
    scores = torch.bmm(ql, lat.transpose(1, 2))
    scores += torch.bmm(qr, key.transpose(1, 2))
    scores *= _scale(case)
    last = total - q + torch.arange(q, device="cuda")[None]  # [b, q]: the last key of each row
    hidden = at[:, None] > last[:, :, None]
    scores.view(b, q, heads, keys).masked_fill_(hidden[:, :, None], -math.inf)
    top = scores.amax(2, keepdim=True)
    scores.sub_(top).exp_()
    mass = scores.sum(2, keepdim=True)
    out = torch.bmm(scores, lat) / mass
    lse = top + mass.log()
    return {"out": out.view(b * q, heads, kv).to(s["out"].dtype), "lse": lse.view(b * q, heads)}


# -------------------------------------------------------------------------------- exact ----
def _exact_rows(pages, case):
    """All of a pool's token rows in 64 bits, [slots, kv] and [slots, rope], the records taken
    apart by their order."""
    page, kv, rope, n = case["page"], case["kv"], case["rope"], pages.shape[0]
    tiles, j = page // 16, kv // 32
    if case.get("cache", "q8") == "16":
        lat = pages[:, :page * kv].reshape(n, tiles, j, 4, 16, 8).permute(0, 1, 4, 2, 3, 5)
        key = pages[:, page * kv:].reshape(n, tiles, rope // 8, 16, 8).permute(0, 1, 3, 2, 4)
        return lat.reshape(n * page, kv).double(), key.reshape(n * page, rope).double()
    a, b, c = _sections(case)
    lat = pages[:, :a].reshape(n, tiles, 512 * j)
    even = lat[:, :, :512 * (j - j % 2)].reshape(n, tiles, j // 2, 4, 16, 2, 8)
    even = even.permute(0, 1, 4, 2, 5, 3, 6).reshape(n * page, 32 * (j - j % 2))
    odd = lat[:, :, 512 * (j - j % 2):].reshape(n, tiles, j % 2, 4, 16, 8)
    odd = odd.permute(0, 1, 4, 2, 3, 5).reshape(n * page, 32 * (j % 2))
    bits = torch.cat([even, odd], 1).int()
    power, frac = bits // 8 % 16, bits % 8
    size = torch.where(power == 0, frac / 8.0 * 2.0 ** -6,
                       (1 + frac.double() / 8) * torch.exp2(power.double() - 7))
    size = torch.where(bits % 128 == 127, math.nan, size) * torch.where(bits >= 128, -1.0, 1.0)
    scale = torch.exp2(pages[:, a + b:].reshape(n * page, j, 1).double() - 127)
    key = pages[:, a:a + b].reshape(n, tiles, rope // 8, 16, 16).permute(0, 1, 3, 2, 4)
    key = key.reshape(n * page, 2 * rope).view(TYPE[case["dtype"]])
    return (size.view(-1, j, 32) * scale).view(-1, kv), key.double()


def _exact_write(s, case):
    page, kv, rope = case["page"], case["kv"], case["rope"]
    lo, hi = RANGE[case["dtype"]]
    v = _views(s["pages"], case)
    slots = s["slots"].long()
    x = s["ckv"].double().view(-1, kv // 32, 32)
    k = torch.ceil(torch.log2(x.abs().amax(2) / 448)).clamp(lo, hi)
    y = (x / torch.exp2(k)[..., None]).clamp(-448, 448)
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    y = torch.round(y / step) * step
    tiles, j, n = page // 16, kv // 32, s["pages"].shape[0]
    rows = torch.empty((n * page, kv), dtype=torch.float64, device="cuda")
    old = v["latent"].double()
    even = old.view(n, tiles, 512 * j)[:, :, :512 * (j - j % 2)].reshape(n, tiles, j // 2, 4, 16, 2, 8)
    rows[:, :32 * (j - j % 2)] = even.permute(0, 1, 4, 2, 5, 3, 6).reshape(n * page, 32 * (j - j % 2))
    if j % 2:
        odd = old.view(n, tiles, 512 * j)[:, :, 512 * (j - 1):].reshape(n, tiles, 4, 16, 8)
        rows[:, 32 * (j - 1):] = odd.permute(0, 1, 3, 2, 4).reshape(n * page, 32)
    rows[slots] = y.view(-1, kv)
    keys = v["rope"].double().view(n, tiles, rope // 8, 16, 8).permute(0, 1, 3, 2, 4).reshape(n * page, rope)
    keys = keys.clone()
    keys[slots] = s["krope"].to(v["rope"].dtype).double()
    scale = v["scale"].reshape(n * page, j).clone()
    scale[slots] = (k + 127).to(torch.uint8)
    even = rows.view(n, tiles, 16, j, 4, 8)[:, :, :, :j - j % 2].reshape(n, tiles, 16, j // 2, 2, 4, 8)
    even = even.permute(0, 1, 3, 5, 2, 4, 6).reshape(n, tiles, 512 * (j - j % 2))
    odd = rows.view(n, tiles, 16, j, 4, 8)[:, :, :, j - j % 2:].permute(0, 1, 3, 4, 2, 5)
    lat = torch.cat([even, odd.reshape(n, tiles, 512 * (j % 2))], 2).view(n, page * kv)
    keys = keys.view(n, tiles, 16, rope // 8, 8).permute(0, 1, 3, 2, 4).reshape(n, page * rope)
    return {"latent": lat, "rope": keys, "scale": scale.view(n, page * j)}


def exact(case, seed):
    s = prepare(case, seed)
    page, kv, rope, heads = case["page"], case["kv"], case["rope"], case["heads"]
    if case["kind"] == "write":
        return _exact_write(s, case)
    if case["kind"] == "read":
        lat, key = _exact_rows(s["pages"], case)
        return {"ckv": lat[s["slots"].long()], "krope": key[s["slots"].long()]}
    q, cu, cp = case["q"], s["cu_pages"].tolist(), s["cu_prefix_pages"].tolist()
    ends, pre = _group_ends(case) if case["groups"] else [], _prefix_lengths(case)
    out = torch.zeros((s["rows"], heads, kv), dtype=torch.float64, device="cuda")
    lse = torch.zeros((s["rows"], heads), dtype=torch.float64, device="cuda")
    for b, n in enumerate(_lengths(case)):
        lat, key = _exact_rows(s["pages"][s["page_ids"][cu[b]:cu[b + 1]].long()], case)
        lat, key, p = lat[:n], key[:n], 0
        if ends:
            g = next(i for i, e in enumerate(ends) if b < e)
            p = pre[g]
            more = _exact_rows(s["pages"][s["prefix_page_ids"][cp[g]:cp[g + 1]].long()], case)
            lat, key = torch.cat([more[0][:p], lat]), torch.cat([more[1][:p], key])
        ql, qr = s["ql"][b * q:b * q + q].double(), s["qr"][b * q:b * q + q].double()
        x = (ql.reshape(q * heads, kv) @ lat.T + qr.reshape(q * heads, rope) @ key.T) * _scale(case)
        late = torch.arange(p + n, device="cuda")[None] > p + n - q + torch.arange(q, device="cuda")[:, None]
        x = x.view(q, heads, p + n).masked_fill(late[:, None], -math.inf)
        lse[b * q:b * q + q] = torch.logsumexp(x, -1)
        x = torch.exp(x - lse[b * q:b * q + q, :, None])
        out[b * q:b * q + q] = (x.view(q * heads, p + n) @ lat).view(q, heads, kv)
    return {"out": out, "lse": lse}
