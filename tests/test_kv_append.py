"""Appending to the paged key-value cache, with the rotation, against its definition in 64 bits."""
import pytest
import torch

from kv_reference import TYPE, near, say, turned, turned_tolerance

F16, BF16 = 0, 1
ROWS = [torch.float32, torch.float16, torch.bfloat16]


def fill(cache, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    cache.pages.copy_(torch.randn(cache.pages.shape, device="cuda", generator=g))
    return cache.pages.clone()


def check(gpu, KH, D, DV, page, dtype, T, rot, rows, H=0, seed=0, view=None, far=5000, pool=None,
          layers=2, layer=1):
    """One append of T rows; `view` makes the rows tensors from (generator, shape)."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    pool = pool or -(-T // page) + 3
    cache = gpu.PagedKVCache(layers, pool, page, KH, D, DV, dtype=dtype)
    before = fill(cache, seed + 1)
    make = view or (lambda shape: torch.randn(shape, device="cuda", generator=g).to(rows))
    k, v = make((T, KH, D)), make((T, KH, DV))
    q = make((T, H, D)) if H else None
    slots = torch.randperm(pool * page, generator=g, device="cuda")[:T].to(torch.int32)
    if T > 3:  # rows without a place
        slots[1], slots[T // 2], slots[T - 1] = -1, pool * page, 2 ** 31 - 1
    at = torch.randint(0, far, (T,), generator=g, device="cuda").to(torch.int32)
    frequencies, start, adjacent = rot
    rotation = gpu.Rotation(frequencies, start, adjacent) if frequencies else None
    got = gpu.append_kv(cache, layer, k, v, slots, rotation=rotation, positions=at, q=q)
    torch.cuda.synchronize()
    want = turned(k, at.cpu(), frequencies, start, adjacent)
    off = turned_tolerance(k, want, frequencies, start, adjacent, dtype)
    s = slots.cpu().long()
    kept = ((s >= 0) & (s < pool * page)).nonzero().flatten()
    at_page, at_slot = (s[kept] // page).cuda(), (s[kept] % page).cuda()
    near(cache.keys(layer)[at_page, :, at_slot], want[kept], off[kept], "keys")
    assert torch.equal(cache.values(layer)[at_page, :, at_slot], v.to(TYPE[dtype])[kept.cuda()])
    # everything else is as it was
    keys, values = cache.keys(layer).clone(), cache.values(layer).clone()
    old = gpu.PagedKVCache(layers, pool, page, KH, D, DV, dtype=dtype, storage=before)
    keys[at_page, :, at_slot] = old.keys(layer)[at_page, :, at_slot]
    values[at_page, :, at_slot] = old.values(layer)[at_page, :, at_slot]
    assert torch.equal(keys, old.keys(layer)) and torch.equal(values, old.values(layer))
    for other in range(layers):
        if other != layer:
            assert torch.equal(cache.layer(other), old.layer(other))
    if H:
        want = turned(q, at.cpu(), frequencies, start, adjacent)
        near(got, want, turned_tolerance(q, want, frequencies, start, adjacent, dtype), "q")
    else:
        assert got is None


def rates(n, theta=10000.0):
    return [theta ** (-i / n) for i in range(n)]


ROTATIONS = [([], 0, True), (rates(8), 48, True), (rates(32), 0, False), (rates(32), 0, True),
             (rates(5), 2, True), (rates(5), 2, False), (rates(12), 24, False), (rates(16), 8, False)]


@pytest.mark.gpu
@pytest.mark.parametrize("rot", range(len(ROTATIONS)))
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("rows", ROWS)
def test_rotations_and_types(gpu, rot, dtype, rows):
    say(f"append rotation {rot} {dtype} {rows}")
    check(gpu, 3, 64, 48, 32, dtype, 37, ROTATIONS[rot], rows, H=6, seed=rot)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [0, 1, 2, 64, 1111])
@pytest.mark.parametrize("KH,D,DV,page,H", [(8, 64, 64, 64, 0), (8, 128, 128, 64, 32), (1, 16, 16, 16, 1),
                                            (16, 192, 128, 48, 16), (2, 256, 256, 16, 24)])
def test_sizes(gpu, KH, D, DV, page, H, T):
    say(f"append sizes {KH} {D} {DV} {page} {H} {T}")
    check(gpu, KH, D, DV, page, BF16, T, (rates(D // 2, 5e5), 0, False), torch.bfloat16, H=H, seed=T)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("adjacent", [True, False])
@pytest.mark.parametrize("shift", [0, 1])
def test_slices_of_one_projection(gpu, rows, adjacent, shift):
    """q, k and v as slices of packed rows, at multiples of 16 bytes and not."""
    say(f"append packed {rows} {adjacent} {shift}")
    g = torch.Generator(device="cuda").manual_seed(3)
    T, H, KH, D, DV = 50, 8, 2, 64, 32
    packed = torch.randn((T, 8 * 64 + 2 * 64 + 2 * 32 + 8), device="cuda", generator=g).to(rows)
    at = {(T, KH, D): 512 + shift, (T, KH, DV): 640 + shift, (T, H, D): shift}
    view = lambda shape: packed[:, at[shape]:at[shape] + shape[1] * shape[2]].unflatten(1, shape[1:])
    check(gpu, KH, D, DV, 16, F16, T, (rates(16), 16, adjacent), rows, H=H, view=view)
    # heads outside tokens: [heads, T, columns], and one row for every token
    other = lambda shape: torch.randn((shape[1], T, shape[2]), device="cuda", generator=g).to(rows).transpose(0, 1)
    check(gpu, KH, D, DV, 16, F16, T, (rates(16), 16, adjacent), rows, H=H, view=other)
    same = lambda shape: torch.randn((1, *shape[1:]), device="cuda", generator=g).to(rows).expand(shape)
    check(gpu, KH, D, DV, 16, F16, T, (rates(16), 16, adjacent), rows, H=H, view=same)


@pytest.mark.gpu
@pytest.mark.parametrize("far", [2, 131072, 2 ** 31 - 1])
def test_far_positions(gpu, far):
    say(f"append far {far}")
    check(gpu, 2, 128, 64, 64, F16, 200, (rates(64), 0, True), torch.float32, H=2, far=far)


@pytest.mark.gpu
def test_values_that_are_not_finite_and_overflow(gpu):
    say("append not finite")
    cache = gpu.PagedKVCache(1, 2, 16, 1, 16, 16, dtype=F16)
    x = torch.zeros((4, 1, 16), device="cuda")
    x[0, 0, :4] = torch.tensor([float("inf"), -float("inf"), float("nan"), 1e6])
    x[1, 0, :3] = torch.tensor([65519.9, 65520.0, 2.0 ** -25 * 1.01])
    gpu.append_kv(cache, 0, x, x, torch.tensor([3, 20, 4, 5], dtype=torch.int32, device="cuda"))
    want = x.half()
    for got in (cache.keys(0), cache.values(0)):
        for i, (p, s) in enumerate([(0, 3), (1, 4), (0, 4), (0, 5)]):
            assert torch.equal(got[p, 0, s].nan_to_num(7, 8, 9), want[i, 0].nan_to_num(7, 8, 9))


@pytest.mark.gpu
def test_offsets_past_32_bits(gpu):
    say("append past 32 bits")
    T = 70
    cache = gpu.PagedKVCache(1, 12300, 256, 4, 128, 128, dtype=BF16)
    assert cache.pages.numel() > 2 ** 31
    x = torch.randn((T, 4, 128), device="cuda")
    slots = (12300 * 256 - T + torch.arange(T, device="cuda")).to(torch.int32)
    gpu.append_kv(cache, 0, x, x, slots)
    got = cache.keys(0)[12299, :, -T:].transpose(0, 1), cache.values(0)[12299, :, -T:].transpose(0, 1)
    assert torch.equal(got[0], x.bfloat16()) and torch.equal(got[1], x.bfloat16())
    assert not cache.pages[0, :12299:64].any()


@pytest.mark.gpu
def test_refusals(gpu):
    say("append refusals")
    cache = gpu.PagedKVCache(1, 4, 16, 2, 32, 16, dtype=F16)
    i32 = lambda n: torch.arange(n, dtype=torch.int32, device="cuda")
    k, v, q = (torch.zeros((5, h, d), device="cuda") for h, d in ((2, 32), (2, 16), (4, 32)))
    rot = gpu.Rotation.of_theta(8)
    call = lambda **kw: gpu.append_kv(**{"cache": cache, "layer": 0, "k": k, "v": v, "slot_mapping": i32(5),
                                         "rotation": rot, "positions": i32(5), **kw})
    call()
    bad = torch.zeros((5, 2, 64), device="cuda")
    for kw in (dict(k=k.double()), dict(v=v.half()), dict(q=q.half()), dict(k=k[:, :1]), dict(v=v[:4]),
               dict(k=bad[..., ::2]), dict(k=k.cpu()), dict(slot_mapping=i32(4)), dict(positions=None),
               dict(positions=i32(4)), dict(slot_mapping=i32(5).long()), dict(positions=i32(5).float()),
               dict(q=q, q_out=torch.zeros((5, 4, 32), device="cuda")), dict(q=q[..., :16]),
               dict(rotation=gpu.Rotation(torch.ones(4, dtype=torch.float64)))):
        with pytest.raises(ValueError):
            call(**kw)
    h = torch.zeros((5, 4, 32), dtype=torch.float16, device="cuda")
    with pytest.raises(gpu.MlaError, match="overlaps"):
        call(k=k.half(), v=v.half(), q=h, q_out=h)
    for r in (gpu.Rotation.of_theta(17), gpu.Rotation.of_theta(8, start=18), gpu.Rotation.of_theta(4, start=1),
              gpu.Rotation.of_theta(4, start=-2)):
        with pytest.raises(gpu.MlaError):
            call(rotation=r)
    with pytest.raises(ValueError):
        gpu.Rotation(torch.ones(4, device="cuda"))
    with pytest.raises(IndexError):
        call(layer=1)
