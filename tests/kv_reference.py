"""The paged key-value cache's operators from their definitions in 64 bits, and batches for them."""
import numpy as np
import torch

TYPE = {0: torch.float16, 1: torch.bfloat16}
HALF_STEP = {0: 2.0 ** -11, 1: 2.0 ** -8}  # half a step of a 16-bit type, relative


def say(what):
    print(f"[case] {what}", flush=True)


# ------------------------------------------------------------------------------ append ----
def turned(x, positions, frequencies, start, adjacent):
    """Rows x [T, heads, dim] turned: a pair as a complex number, times exp(i p f)."""
    x = x.double().cpu()
    n = len(frequencies)
    if n == 0 or len(x) == 0:
        return x
    part = x[..., start:start + 2 * n]
    z = part.unflatten(-1, (n, 2)) if adjacent else part.unflatten(-1, (2, n)).transpose(-1, -2)
    angle = torch.as_tensor(positions).double()[:, None] * torch.as_tensor(frequencies, dtype=torch.float64)
    z = torch.view_as_complex(z.contiguous()) * torch.polar(torch.ones_like(angle), angle)[:, None]
    z = torch.view_as_real(z)
    z = z if adjacent else z.transpose(-1, -2)
    return torch.cat([x[..., :start], z.flatten(-2), x[..., start + 2 * n:]], -1)


def turned_tolerance(x, want, frequencies, start, adjacent, dtype):
    """cos and sin in 32 bits are off by 2^-21 at most (the revolution's rest is rounded to 32 bits,
    2^-25 of a revolution, 1.9e-7 rad, then the function's 2 ulp), the two products and their sum by
    three roundings of 2^-24: 2^-20 (|a| + |b|).  Then half a step of the type, its smallest for
    fp16's subnormals, 2^-25."""
    x = x.double().cpu().abs()
    n, pair = len(frequencies), torch.zeros_like(x)
    if n:
        i = torch.arange(n)
        a = start + (2 * i if adjacent else i)
        b = a + (1 if adjacent else n)
        pair[..., a] = pair[..., b] = x[..., a] + x[..., b]
    before = 2.0 ** -20 * pair
    return before + HALF_STEP[dtype] * (want.abs() + before) + (2.0 ** -25 if dtype == 0 else 0)


# --------------------------------------------------------------------------- attention ----
class Batch:
    """Sessions [(cached tokens, query rows)] over a page pool whose unused slots hold NaN."""

    def __init__(self, H, KH, D, DV, page, dtype, sessions, seed=0, spare=3, scale=None):
        self.H, self.KH, self.D, self.DV, self.page, self.dtype = H, KH, D, DV, page, dtype
        self.ctx, self.q_len = [s[0] for s in sessions], [s[1] for s in sessions]
        self.lens = [a + b for a, b in sessions]
        self.rows = sum(self.q_len)
        self.scale = D ** -0.5 if scale is None else scale
        g = torch.Generator().manual_seed(seed)
        need = [-(-n // page) for n in self.lens]
        self.pool = sum(need) + spare
        self.max_pages = max(need + [1])
        ids = torch.randperm(self.pool, generator=g)[:sum(need)]
        self.cu = np.concatenate([[0], np.cumsum(need)]).astype(np.int64)
        self.ids = ids
        t = TYPE[dtype]
        self.k = torch.full((self.pool, KH, page, D), float("nan"), dtype=t)
        self.v = torch.full((self.pool, KH, page, DV), float("nan"), dtype=t)
        for b, n in enumerate(self.lens):
            for p in range(need[b]):
                m, at = min(page, n - p * page), ids[self.cu[b] + p]
                self.k[at, :, :m] = torch.randn((KH, m, D), generator=g).to(t)
                self.v[at, :, :m] = torch.randn((KH, m, DV), generator=g).to(t)
        self.q = torch.randn((self.rows, H, D), generator=g).to(t)

    def token(self, b, j):
        """Page and slot of session b's token j."""
        return int(self.ids[self.cu[b] + j // self.page]), j % self.page

    def storage(self):
        return torch.cat([self.k.flatten(1), self.v.flatten(1)], 1)[None].contiguous()

    def device(self, gpu):
        i32 = lambda x: torch.tensor(list(x), dtype=torch.int32, device="cuda")
        batch = gpu.build_metadata(i32(self.ctx), i32(self.q_len), i32(self.cu), i32(self.ids),
                                   self.page, self.max_pages, self.pool, split_pages=64,
                                   max_work=max(1, sum(-(-n // (64 * self.page)) for n in self.lens)),
                                   max_rows=max(1, self.rows))
        cache = gpu.PagedKVCache(1, self.pool, self.page, self.KH, self.D, self.DV, dtype=self.dtype,
                                 storage=self.storage().cuda())
        return batch, cache, self.q.cuda()

    def sees(self, b, window, sinks):
        n, q = self.lens[b], self.q_len[b]
        distance = torch.arange(n - q, n)[:, None] - torch.arange(n)
        seen = distance >= 0
        if window is not None:
            seen &= (distance < window) | (torch.arange(n) < sinks)
        return seen

    def expect(self, window=None, sinks=0):
        """Rows, lse, and what may be off of both (see attention)."""
        to = lambda x: x.to("cuda" if torch.cuda.is_available() else "cpu")
        got = [to(torch.zeros((self.rows, self.H, *n), dtype=torch.float64)) for n in ((self.DV,), (), (self.DV,), ())]
        all_k, all_v, all_q = to(self.k), to(self.v), to(self.q)
        r0, G = 0, self.H // self.KH
        for b, (n, q) in enumerate(zip(self.lens, self.q_len)):
            if q == 0:
                continue
            ids = to(self.ids[self.cu[b]:self.cu[b + 1]])
            seen = to(self.sees(b, window, sinks))
            for h in range(self.H):
                k = all_k[ids, h // G].reshape(-1, self.D)[:n]
                v = all_v[ids, h // G].reshape(-1, self.DV)[:n]
                for to_, x in zip(got, attention(all_q[r0:r0 + q, h], k, v, seen, self.scale, self.dtype)):
                    to_[r0:r0 + q, h] = x
            r0 += q
        return [x.cpu() for x in got]


def attention(x, k, v, seen, scale, dtype):
    """Rows, lse, and what may be off of both, of one head's rows x over keys k and values v.

    A score sums its products in 32 bits, at most 8 steps of 32 (5 levels each): 13 roundings of
    2^-24 of sum |q k|, and one more each for its scale and its distance from the maximum: within
    2^-20 of s = scale sum |q k|, twice that between two scores.  Exponentials 2^-22.  The weight's
    two parts 2^-17.  Sums over n keys: n / 16 additions of 2^-24.  All of it of the mass of
    absolute values.  Then half a step of the row, and half of fp16's smallest step."""
    x, k, v, n = x.double(), k.double(), v.double(), len(k)
    s = torch.where(seen, x @ k.T * scale, -torch.inf)
    lse, w = torch.logsumexp(s, 1), torch.softmax(s, 1)
    # (a value that a row does not see adds nothing to it, whatever it is)
    fine = torch.where(torch.isfinite(v), v, 0.0)
    hit = seen.double() @ (~torch.isfinite(v)).double() > 0
    out, mass = torch.where(hit, torch.nan, w @ fine), w @ fine.abs()
    size = torch.where(seen, (x.abs() @ k.abs().T) * scale, 0.0)
    size = torch.nan_to_num(size, nan=0.0, posinf=0.0).amax(1)
    weights = 2.0 ** -19 * size + 2.0 ** -21 + n / 16 * 2.0 ** -24
    before = (2 * weights + 2.0 ** -17)[:, None] * mass
    o = torch.nan_to_num(out, nan=0.0, posinf=0.0, neginf=0.0)
    off = before + HALF_STEP[dtype] * (o.abs() + before) + 2.0 ** -25
    return out, lse, off, weights + 2.0 ** -22 * (1 + torch.nan_to_num(lse).abs())


def near(got, want, off, what):
    """Finite in the same places (what is not is NaN or an infinity), and there within `off`."""
    got = got.double().cpu()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    fine = torch.isfinite(want)
    assert torch.equal(torch.isfinite(got), fine), f"{what}: finite in other places"
    wrong = fine & ((got - want).abs() > off)
    assert not wrong.any(), (f"{what}: {int(wrong.sum())} of {wrong.numel()} off, first at "
                             f"{wrong.nonzero()[0].tolist()}, worst by "
                             f"{float(((got - want).abs() / off)[fine].max()):.3g} times what may be")
