"""The MLA latent-cache operators on the GPU against plain 64-bit implementations."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

E4M3 = torch.float8_e4m3fn


def rotated(x, cos, sin):
    """The rotary embedding of interleaved pairs, as a product of complex numbers."""
    x, cos, sin = x.double(), cos.double(), sin.double()
    z = torch.complex(x[..., 0::2], x[..., 1::2]) * torch.complex(cos[..., :32], sin[..., :32])
    return torch.cat([z.real, z.imag], -1)


def tables(rows, dtype=torch.float32):
    ang = torch.arange(rows, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, 64, 2).double() / 64)
    ang = torch.cat([ang, ang], -1)
    return ang.cos().to(dtype).cuda(), ang.sin().to(dtype).cuda()


def make_cache(pages, page, dtype, fill=None):
    """A cache whose bytes are all `fill` values first (NaN by default: nothing may depend on unwritten rows)."""
    from pithtrain_b200.operators.mla import LatentCache
    c = LatentCache.allocate(pages, page, dtype)
    bad = float("nan") if fill is None else fill
    c.latent.copy_(torch.full((1,), bad, device="cuda").expand(c.latent.shape).to(dtype))
    c.rope.fill_(bad)
    if c.scale is not None:
        c.scale.fill_(bad)
    return c


def stored(cache):
    """Values that the cache stands for, fp64 [slots, 512] and [slots, 64]."""
    c = cache.latent.float().double().reshape(-1, 512)
    if cache.scale is not None:
        c = c * cache.scale.double().reshape(-1, 1)
    return c, cache.rope.double().reshape(-1, 64)


def check():
    from pithtrain_b200 import kernels
    torch.cuda.synchronize()
    kernels.check_device_status()


# fp32 arithmetic in front of one rounding: the error is half a step of the stored type, relative to the value, plus
# about 20 fp32 roundings (a 512-term sum, a reciprocal root, three products), below 2^-18 relative.
def assert_rounded(got, want, half_step, what, floor=0.0):
    excess = (got.double() - want).abs() - ((half_step + 2.0 ** -18) * want.abs() + floor)
    assert excess.max().item() <= 0, (what, excess.max().item())


@pytest.mark.parametrize("dtype", [torch.bfloat16, E4M3])
@pytest.mark.parametrize("shape,page", [((1, 1), 16), ((3, 5), 32), ((1, 129), 64), ((2, 4001), 192)])
@pytest.mark.parametrize("cs,positions,weight", [(torch.float32, True, torch.bfloat16),
                                                 (torch.bfloat16, False, torch.float32)])
def test_write_then_read(cuda_device, dtype, shape, page, cs, positions, weight):
    from pithtrain_b200.operators.mla import latent_cache_read, latent_cache_write
    g = torch.Generator(device="cuda").manual_seed(sum(shape) + page)
    B, S = shape
    pages = -(-B * S // page) + 2
    cache = make_cache(pages, page, dtype)
    proj = torch.randn(B, S, 576, generator=g, device="cuda").mul_(3).bfloat16()
    w = (1 + 0.2 * torch.randn(512, generator=g, device="cuda")).to(weight)
    cos, sin = tables(5000, cs)
    pos = torch.randint(0, 5000, (B, S), generator=g, device="cuda")
    slots = torch.randperm(pages * page, generator=g, device="cuda")[: B * S].view(B, S)
    skipped = torch.rand(B, S, generator=g, device="cuda") < 0.2
    slots = torch.where(skipped, -1, slots)
    before = [t.clone().view(torch.uint8) for t in (cache.latent, cache.rope)]
    rot = (cos, sin) if positions else (cos[pos], sin[pos])
    latent_cache_write(cache, slots, proj[..., :512], proj[..., None, 512:], w, *rot, 1e-6,
                       position_ids=pos if positions else None)
    check()
    x = proj[..., :512].double()
    c = x / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w.double()
    r = rotated(proj[..., 512:], cos[pos], sin[pos])
    got_c, got_r = stored(cache)
    kept = ~skipped
    at = slots[kept]
    assert_rounded(got_r[at], r[kept], 2.0 ** -8, "rope", floor=2.0 ** -20 * 4)  # a sum of two products may cancel
    if dtype == torch.bfloat16:
        assert_rounded(got_c[at], c[kept], 2.0 ** -8, "latent")
    else:
        scale = cache.scale.reshape(-1)[at].double()
        assert torch.equal(scale, 2.0 ** torch.ceil(torch.log2(c[kept].abs().amax(-1) / 448)))
        # half a step of e4m3: 2^-4 of the value, or 2^-10 of the scale below its smallest normal value
        assert_rounded(got_c[at], c[kept], 2.0 ** -4, "latent", floor=(scale * 2.0 ** -10)[:, None])
    untouched = torch.ones(pages * page, dtype=torch.bool, device="cuda")
    untouched[at] = False
    for now, old in zip((cache.latent, cache.rope), before):  # rows of other tokens stay as they were, to the bit
        now = now.view(torch.uint8).reshape(pages * page, -1)
        assert torch.equal(now[untouched], old.reshape(pages * page, -1)[untouched])
    lat, pe = latent_cache_read(cache, slots)
    check()
    assert lat.shape == (B, S, 512) and pe.shape == (B, S, 64)
    assert torch.equal(lat[kept].double(), got_c[at]) and torch.equal(pe[kept].double(), got_r[at])
    assert not lat[skipped].any() and not pe[skipped].any()


def test_write_keeps_zero_rows_and_marks_infinite_ones(cuda_device):
    from pithtrain_b200.operators.mla import latent_cache_write
    cache = make_cache(2, 16, E4M3)
    x = torch.zeros(1, 3, 512, device="cuda", dtype=torch.bfloat16)
    x[0, 1, 7] = float("inf")
    x[0, 2, 7] = float("nan")
    cos, sin = tables(8)
    latent_cache_write(cache, torch.tensor([[3, 4, 5]], device="cuda"), x, x[..., :64].contiguous(),
                       torch.ones(512, device="cuda"), cos, sin, 1e-6)
    check()
    c, _ = stored(cache)
    assert not c[3].any()
    assert c[4].isnan().any() and c[5].isnan().any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, E4M3])
def test_a_layer_of_a_larger_cache_and_another_stream(cuda_device, dtype):
    """Pages of several layers side by side: strided planes, written and read on a side stream."""
    from pithtrain_b200.operators.mla import LatentCache, latent_cache_read, latent_cache_write
    g = torch.Generator(device="cuda").manual_seed(5)
    lat = torch.zeros(4, 3, 32, 512, device="cuda").to(dtype)
    rope = torch.zeros(4, 3, 32, 64, device="cuda", dtype=torch.bfloat16)
    scale = torch.ones(4, 3, 32, device="cuda") if dtype == E4M3 else None
    cache = LatentCache(lat[:, 1], rope[:, 1], None if scale is None else scale[:, 1])
    x = torch.randn(1, 50, 576, generator=g, device="cuda").bfloat16()
    slots = torch.randperm(128, generator=g, device="cuda")[:50].view(1, 50)
    cos, sin = tables(50)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        latent_cache_write(cache, slots, x[..., :512], x[..., 512:], torch.ones(512, device="cuda"), cos, sin, 1e-6)
        got, pe = latent_cache_read(cache, slots)
    torch.cuda.current_stream().wait_stream(side)
    check()
    c = x[..., :512].double()
    c = c / (c.square().mean(-1, keepdim=True) + 1e-6).sqrt()
    top = c.abs().amax(-1, keepdim=True) / 448
    assert_rounded(got, c, 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -4, "latent", floor=top * 2.0 ** -9)
    assert_rounded(pe, rotated(x[..., 512:], cos, sin), 2.0 ** -8, "rope", floor=2.0 ** -18)
    assert not lat[:, 0].float().any() and not lat[:, 2].float().any() and not rope[:, 0].any()


def test_indices_out_of_range_are_reported(cuda_device):
    """The kernels check every index themselves: nothing outside the cache is touched, the host learns of it."""
    from pithtrain_b200 import kernels
    from pithtrain_b200.operators.mla import latent_cache_read, latent_cache_write
    cache = make_cache(2, 16, torch.bfloat16, fill=1.0)
    x = torch.ones(1, 2, 576, device="cuda", dtype=torch.bfloat16)
    cos, sin = tables(4)
    w = torch.ones(512, device="cuda")
    pos = torch.tensor([[0, 1]], device="cuda")
    latent_cache_write(cache, torch.tensor([[32, 1 << 40]], device="cuda"), x[..., :512], x[..., 512:], w, cos, sin,
                       1e-6, position_ids=pos)
    with pytest.raises(RuntimeError, match="a slot given to a latent-cache operator is out of range"):
        kernels.check_device_status()
    for bad in ([[0, 4]], [[-1, 0]]):
        latent_cache_write(cache, torch.tensor([[-1, -2]], device="cuda") + 2, x[..., :512], x[..., 512:], w, cos, sin,
                           1e-6, position_ids=torch.tensor(bad, device="cuda"))
        with pytest.raises(RuntimeError, match="a position given"):
            kernels.check_device_status()
    latent_cache_read(cache, torch.tensor([5, 32], device="cuda"))
    with pytest.raises(RuntimeError, match="a slot given"):
        kernels.check_device_status()
    assert (cache.latent.float()[0, 2:] == 1).all() and (cache.latent.float()[1] == 1).all()
    check()
