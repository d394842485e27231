"""The key-value cache's operators together, as a server uses them: metadata, append with rotation and
attention step after step, in full layers and in layers with a window, eagerly and captured."""
import numpy as np
import pytest
import torch

from kv_reference import TYPE, attention, near, say, turned, turned_tolerance

F16, BF16 = 0, 1
i32 = lambda x: torch.tensor(list(x), dtype=torch.int32, device="cuda")


class Server:
    """Sessions over one pool; layer 0 attends in full, layer 1 through a window with sinks."""

    WINDOW, SINKS = 24, 3

    def __init__(self, gpu, H, KH, D, DV, page, dtype, sessions, most, seed):
        self.gpu, self.shape, self.dtype = gpu, (H, KH, D, DV), dtype
        self.page, self.most = page, -(-most // page)
        self.cache = gpu.PagedKVCache(2, sessions * self.most + 1, page, KH, D, DV, dtype=dtype)
        self.cache.pages.fill_(float("nan"))  # nothing may depend on slots that were never written
        self.g = torch.Generator(device="cuda").manual_seed(seed)
        ids = torch.randperm(sessions * self.most + 1, generator=self.g, device="cuda")
        self.ids = ids[:sessions * self.most].to(torch.int32)
        self.cu = i32(np.arange(sessions + 1) * self.most)
        self.start, self.adjacent = (0, False) if D % 32 == 0 else (D // 2, True)
        pairs = D // 2 if self.start == 0 else D // 4
        self.frequencies = [10000.0 ** (-i / pairs) for i in range(pairs)]
        self.rotation = gpu.Rotation(self.frequencies, self.start, self.adjacent)
        self.ctx = [0] * sessions

    def step(self, counts):
        """counts[b] new tokens of each session through both layers, checked."""
        gpu, (H, KH, D, DV), c = self.gpu, self.shape, self.cache
        rows = sum(counts)
        batch = gpu.build_metadata(i32(self.ctx), i32(counts), self.cu, self.ids, self.page, self.most,
                                   c.num_pages, max_rows=max(rows, 1))
        at = [n + i for n, q in zip(self.ctx, counts) for i in range(q)]
        plans = [gpu.plan_kv_attention(batch, c, H, rows=rows, max_q_len=max(counts)),
                 gpu.plan_kv_attention(batch, c, H, rows=rows, max_q_len=max(counts), window=self.WINDOW,
                                       sinks=self.SINKS)]
        for layer, plan in enumerate(plans):
            x = torch.randn((rows, (H + KH) * D + KH * DV), generator=self.g, device="cuda").to(TYPE[self.dtype])
            q, k, v = x.split([H * D, KH * D, KH * DV], 1)
            k, v = k.unflatten(1, (KH, D)), v.unflatten(1, (KH, DV))
            q = gpu.append_kv(c, layer, k, v, batch.slot_mapping, rotation=self.rotation, positions=i32(at),
                              q=q.unflatten(1, (H, D)))
            lse = torch.zeros((rows, H), device="cuda")
            out = gpu.kv_attention(plan, c, layer, q, D ** -0.5, lse=lse)
            want = turned(k, at, self.frequencies, self.start, self.adjacent)
            off = turned_tolerance(k, want, self.frequencies, self.start, self.adjacent, self.dtype)
            self.check(layer, counts, q, out, lse, want, off, v)
        self.ctx = [a + b for a, b in zip(self.ctx, counts)]

    def check(self, layer, counts, q, out, lse, new_k, off_k, new_v):
        """The new tokens are in the cache, and the rows are those of all that it holds."""
        H, KH, D, DV = self.shape
        r = 0
        for b, n in enumerate(counts):
            if n == 0:
                continue
            total, ids = self.ctx[b] + n, self.ids[b * self.most:(b + 1) * self.most].long()
            k = self.cache.keys(layer)[ids].transpose(0, 1).reshape(KH, -1, D)[:, :total]
            v = self.cache.values(layer)[ids].transpose(0, 1).reshape(KH, -1, DV)[:, :total]
            near(k[:, -n:].transpose(0, 1), new_k[r:r + n], off_k[r:r + n], "keys")
            assert torch.equal(v[:, -n:].transpose(0, 1), new_v[r:r + n])
            far = torch.arange(total - n, total)[:, None] - torch.arange(total)
            seen = far >= 0
            if layer == 1:
                seen &= (far < self.WINDOW) | (torch.arange(total) < self.SINKS)
            for h in range(H):
                g = h // (H // KH)
                w = [x.cpu() for x in attention(q[r:r + n, h], k[g], v[g], seen.cuda(), D ** -0.5, self.dtype)]
                near(out[r:r + n, h], w[0], w[2], f"layer {layer} session {b} head {h}")
                near(lse[r:r + n, h], w[1], w[3], "lse")
            r += n


@pytest.mark.gpu
@pytest.mark.parametrize("H,KH,D,DV,page,dtype", [(8, 8, 64, 64, 64, F16), (8, 2, 128, 128, 32, BF16),
                                                  (4, 4, 192, 128, 16, BF16), (6, 2, 80, 48, 16, F16)])
def test_prompts_decode_steps_and_drafts(gpu, H, KH, D, DV, page, dtype):
    say(f"server {H} {KH} {D} {DV} {page} {dtype}")
    s = Server(gpu, H, KH, D, DV, page, dtype, sessions=4, most=220, seed=H + D)
    for counts in ([50, 1, 0, 130], [1, 40, 1, 1], [1, 1, 1, 0], [4, 5, 2, 1], [1, 1, 1, 1], [33, 1, 60, 3]):
        s.step(counts)


@pytest.mark.gpu
@pytest.mark.parametrize("window,sinks", [(None, 0), (100, 5)])
def test_a_captured_step_of_a_growing_batch(gpu, window, sinks):
    """Metadata, plan, append and attention captured once and replayed for other lengths, tokens and
    rows, with eager work between: each replay gives what the eager step gives."""
    say(f"captured {window}")
    H, KH, D, page, full = 16, 4, 128, 32, [400, 37, 1000, 64, 5, 251]
    B, most = len(full), 32
    rows = B
    cache = gpu.PagedKVCache(1, B * most, page, KH, D, dtype=BF16)
    other = gpu.PagedKVCache(1, B * most, page, KH, D, dtype=BF16)
    g = torch.Generator(device="cuda").manual_seed(1)
    cache.pages.copy_(torch.randn(cache.pages.shape, generator=g, device="cuda"))
    ids = torch.randperm(B * most, generator=g, device="cuda").to(torch.int32)
    cu, ctx, one = i32(np.arange(B + 1) * most), i32(full), i32([1] * B)
    rotation = gpu.Rotation.of_theta(D // 2, adjacent=False)
    x = torch.zeros((rows, (H + 2 * KH), D), dtype=torch.bfloat16, device="cuda")
    out = torch.zeros((rows, H, D), dtype=torch.bfloat16, device="cuda")
    lse, turned_q = torch.zeros((rows, H), device="cuda"), torch.empty_like(out)
    keep = {}

    def step(cache, out, lse, q_out, ws=None):
        batch = gpu.build_metadata(ctx, one, cu, ids, page, most, B * most, max_rows=rows, max_work=512)
        plan = gpu.plan_kv_attention(batch, cache, H, rows=rows, max_q_len=1, window=window, sinks=sinks)
        gpu.append_kv(cache, 0, x[:, H:H + KH], x[:, H + KH:], batch.slot_mapping, rotation=rotation,
                      positions=ctx, q=x[:, :H], q_out=q_out)
        gpu.kv_attention(plan, cache, 0, q_out, D ** -0.5, out=out, lse=lse, workspace=ws)
        return batch, plan

    _, plan = step(cache, out, lse, turned_q)
    ws = gpu.kv_attention_workspace(plan)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        keep["step"] = step(cache, out, lse, turned_q, ws)
    for i, share in enumerate((0.0, 0.3, 1.0, 0.6)):
        ctx.copy_((torch.tensor(full) * share).to(torch.int32))
        x.copy_(torch.randn(x.shape, generator=g, device="cuda"))
        other.pages.copy_(cache.pages)
        eager, elses, eq = torch.zeros_like(out), torch.zeros_like(lse), torch.empty_like(out)
        step(other, eager, elses, eq)
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager) and torch.equal(lse, elses), share
        assert torch.equal(cache.pages, other.pages) and torch.equal(turned_q, eq)
    assert keep["step"][1].read_info()[0] > 0 and keep["step"][1].info is None


@pytest.mark.gpu
def test_two_streams_with_workspaces_of_their_own(gpu):
    """Calls of one plan that may run at once."""
    say("two streams")
    from kv_reference import Batch
    c = Batch(32, 8, 128, 128, 64, BF16, [(3000, 1), (500, 1), (2000, 60), (10, 3)], seed=2)
    batch, cache, q = c.device(gpu)
    plan = gpu.plan_kv_attention(batch, cache, 32, rows=c.rows, max_q_len=60)
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [torch.zeros((c.rows, 32, 128), dtype=torch.bfloat16, device="cuda") for _ in streams]
    spaces = [gpu.kv_attention_workspace(plan) for _ in streams]
    torch.cuda.synchronize()
    for _ in range(10):
        for s, o, w in zip(streams, outs, spaces):
            gpu.kv_attention(plan, cache, 0, q, c.scale, out=o, workspace=w, stream=s)
    torch.cuda.synchronize()
    want, _, off, _ = c.expect()
    near(outs[0], want, off, "out")
    assert torch.equal(outs[0], outs[1])
