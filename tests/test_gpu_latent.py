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


# ---------------------------------------------------------------------------------------------------- attention
def quantised(latent):
    """e4m3 rows and their power-of-two factors."""
    scale = 2.0 ** torch.ceil(torch.log2(latent.abs().amax(-1).clamp_min(1e-30) / 448))
    return (latent / scale[..., None]).to(E4M3), scale


def filled_cache(g, lens, page, dtype, spare=3, spread=1.0):
    """A cache with random rows for sequences of the given lengths, in random pages; every row that no sequence owns is
    NaN, and so are the table's entries behind a sequence's last page out of range. Returns (cache, table)."""
    cache = make_cache(sum(-(-n // page) for n in lens) + spare, page, dtype)
    order = torch.randperm(cache.num_pages, generator=g, device="cuda").int()
    cols = max(1, max(-(-n // page) for n in lens)) + 1
    table = torch.full((len(lens), cols), 1 << 30, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(lens):
        need = -(-n // page)
        table[b, :need] = order[at: at + need]
        at += need
        rows = slots_of(table[b], n, page)
        c = torch.randn(n, 512, generator=g, device="cuda") * (1 + spread * torch.rand(n, 1, generator=g, device="cuda"))
        if dtype == E4M3 and n:
            c8, scale = quantised(c)
            cache.latent.view(torch.uint8).view(-1, 512)[rows] = c8.view(torch.uint8)
            cache.scale.view(-1)[rows] = scale
        elif n:
            cache.latent.view(-1, 512)[rows] = c.bfloat16()
        if n:
            cache.rope.view(-1, 64)[rows] = torch.randn(n, 64, generator=g, device="cuda").bfloat16()
    return cache, table


def slots_of(pages, n, page):
    i = torch.arange(n, device="cuda")
    return pages[i // page].long() * page + i % page


def visible(S, n, nq, tree=None):
    """bool [S, n]: which keys a sequence's token sees."""
    i, k = torch.arange(S, device="cuda")[:, None], torch.arange(n, device="cuda")
    if tree is None:
        seen = k <= n - nq + i
    else:
        j = k - (n - nq)
        seen = (j < 0) | tree[:, j.clamp(0, S - 1)]
    return seen & (i < nq)


def attention_reference(query, cache, table, lens, scale, query_lens=None, tree=None):
    """fp64 (out, log2 lse) and a bound of the kernel's error for every element of out, and for lse.

    Weights: rounded once to 8 significant bits (2^-8 relative); scores: fp32 sums of 576 products, relative to the sum of
    their magnitudes 576 * 2^-24, times two for numerator and denominator; exp2, log2 and the scaling: 2^-18. With an 8-bit
    cache the split query is exact to 2^-21 of its largest element, and a weight to 2^-20 of the largest of its row (2^-18
    where row factors differ by up to 4). The result is rounded to bf16: 2^-8."""
    B, S, H, _ = query.shape
    out = torch.zeros(B, S, H, 512, dtype=torch.float64, device="cuda")
    lse = torch.full((B, H, S), -math.inf, dtype=torch.float64, device="cuda")
    tol, tol_lse = torch.zeros_like(out), torch.zeros_like(lse)
    c_all, r_all = stored(cache)
    for b, n in enumerate(lens):
        nq = S if query_lens is None else query_lens[b]
        if n == 0 or nq == 0:
            continue
        rows = slots_of(table[b], n, cache.page_size)
        c, r = c_all[rows], r_all[rows]
        keys = torch.cat([c, r], -1)
        seen = visible(S, n, nq, None if tree is None else tree[b])
        for h in range(H):
            q = query[b, :, h].double()
            s = (q @ keys.T * scale).masked_fill(~seen, -math.inf)
            size = (q.abs() @ keys.abs().T * scale).masked_fill(~seen, 0).amax(-1)
            delta = size * 576 * 2.0 ** -24 + 2.0 ** -18
            floor = 0.0
            if cache.scale is not None:
                delta = delta + scale * 512 * 2.0 ** -21 * q[:, :512].abs().amax(-1) * c.abs().max()
                floor = 2.0 ** -16
            top = s.amax(-1, keepdim=True)
            p = torch.exp(s - torch.where(top.isinf(), 0, top))
            total = p.sum(-1, keepdim=True)
            some = (total > 0)
            total = torch.where(some, total, 1)
            out[b, :, h] = p @ c / total
            lse[b, h] = torch.where(some[:, 0], (top[:, 0] + total[:, 0].log()) / math.log(2), -math.inf)
            tol[b, :, h] = 2.0 ** -8 * out[b, :, h].abs() + (2.0 ** -8 + 2 * delta[:, None]) * (p @ c.abs()) / total \
                + floor * (seen.double() @ c.abs()) / total
            tol_lse[b, h] = 2 * delta + 2.0 ** -20 * lse[b, h].abs().nan_to_num(0, 0, 0)
    return out, lse, tol, tol_lse


def run_attention(query, cache, table, lens, scale, query_lens=None, tree=None):
    from pithtrain_b200.operators.mla import latent_attention
    i32 = lambda v: None if v is None else torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    return latent_attention(query, cache, table, i32(lens), scale, query_lens=i32(query_lens), tree_mask=tree,
                            return_lse=True)


def assert_attention(query, cache, table, lens, scale, query_lens=None, tree=None, got=None):
    o, l = run_attention(query, cache, table, lens, scale, query_lens, tree) if got is None else got
    check()
    ro, rl, tol, tol_lse = attention_reference(query, cache, table, lens, scale, query_lens, tree)
    assert not o.isnan().any(), "NaN in the output"
    assert ((o.double() - ro).abs() - tol).max().item() <= 0, ((o.double() - ro).abs() - tol).max().item()
    fin = rl.isfinite()
    assert torch.equal(l.isfinite(), fin) and not l.isnan().any()
    assert ((l.double() - rl)[fin].abs() <= tol_lse[fin]).all()
    return o, l


def random_tree(g, B, S):
    """Ancestors of every node (and itself) of random trees."""
    mask = torch.zeros(B, S, S, dtype=torch.bool)
    parent = torch.rand(B, S, generator=g)
    for b in range(B):
        for j in range(S):
            if j:
                mask[b, j] = mask[b, int(parent[b, j] * j)]
            mask[b, j, j] = True
    return mask.cuda()


SCALE = 192 ** -0.5


@pytest.mark.parametrize("dtype", [torch.bfloat16, E4M3])
@pytest.mark.parametrize("S,H,lens,page", [
    (1, 16, [1], 16), (1, 16, [77], 64), (1, 16, [64, 0, 65, 1, 128, 129, 63], 32), (1, 16, [4097, 3, 1500], 64),
    (1, 1, [300, 2], 16), (1, 2, [129], 192), (3, 5, [40, 3, 700], 128), (2, 16, [5, 1100], 32), (4, 16, [260, 4], 64),
    (1, 128, [513, 90], 64), (7, 16, [900, 7, 8], 16), (100, 4, [100], 64), (33, 16, [33, 2000], 128),
    (1, 16, list(range(1, 400, 2)), 16), (1, 16, [9000, 20000, 31000], 64), (2, 16, [5000, 100, 9999, 17000], 32),
    (16, 16, [2100, 700], 64)])  # the last ones: several tiles and pieces for every CTA
def test_attention_causal(cuda_device, dtype, S, H, lens, page):
    g = torch.Generator(device="cuda").manual_seed(1000 * S + H + len(lens))
    cache, table = filled_cache(g, lens, page, dtype)
    q = torch.randn(len(lens), S, H, 576, generator=g, device="cuda").bfloat16()
    assert_attention(q, cache, table, lens, SCALE)


@pytest.mark.parametrize("dtype", [torch.bfloat16, E4M3])
@pytest.mark.parametrize("S,H,lens,qlens,page", [
    (13, 16, [13, 500, 1025], None, 64), (5, 2, [5, 64, 66], None, 16), (48, 16, [300], None, 32),
    (9, 16, [200, 9, 3, 0], [9, 4, 0, 0], 64), (20, 8, [20, 129, 260], [20, 1, 7], 128)])
def test_attention_tree(cuda_device, dtype, S, H, lens, qlens, page):
    g = torch.Generator(device="cuda").manual_seed(S + H)
    cache, table = filled_cache(g, lens, page, dtype)
    q = torch.randn(len(lens), S, H, 576, generator=g, device="cuda").bfloat16()
    tree = random_tree(torch.Generator().manual_seed(S), len(lens), S)
    assert_attention(q, cache, table, lens, SCALE, qlens, tree)
    tree = torch.rand(tree.shape, generator=g, device="cuda") < 0.3       # any mask; rows that see only the prefix
    assert_attention(q, cache, table, lens, SCALE, qlens, tree)
    assert_attention(q, cache, table, lens, SCALE, qlens, torch.zeros_like(tree))


@pytest.mark.parametrize("dtype", [torch.bfloat16, E4M3])
def test_attention_of_a_padded_batch(cuda_device, dtype):
    """Sequences with fewer new tokens than the batch's S, with none, and with more tokens than keys (rows that see
    nothing); queries without a token are NaN."""
    g = torch.Generator(device="cuda").manual_seed(3)
    lens, qlens = [300, 65, 0, 3, 1000], [5, 1, 0, 5, 0]
    cache, table = filled_cache(g, lens, 32, dtype)
    q = torch.randn(5, 5, 8, 576, generator=g, device="cuda").bfloat16()
    for b, n in enumerate(qlens):
        q[b, n:] = float("nan")
    o, l = run_attention(q, cache, table, lens, SCALE, qlens)
    assert_attention(q.nan_to_num(0), cache, table, lens, SCALE, qlens, got=(o, l))
    for b, n in enumerate(qlens):
        assert not o[b, n:].any() and (l[b, :, n:] == -math.inf).all()
    assert not o[3, :2].any() and o[3, 2:].any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, E4M3])
def test_attention_with_large_scores_and_one_key_above_all(cuda_device, dtype):
    """Scores of several hundred, a maximum that rises late and often, and one key that outweighs all others."""
    g = torch.Generator(device="cuda").manual_seed(11)
    lens = [3000]
    cache, table = filled_cache(g, lens, 64, dtype)
    q = torch.randn(1, 1, 16, 576, generator=g, device="cuda").bfloat16()
    q[0, 0, 8:] *= 30
    rows = slots_of(table[0], 3000, 64)
    top = q[0, 0, 0, 512:] * 3                                           # key 2900 agrees with head 0
    cache.rope.view(-1, 64)[rows[2900]] = top
    rising = torch.linspace(0, 6, 3000, device="cuda")[:, None] * q[0, 0, 1, 512:].float()
    cache.rope.view(-1, 64)[rows] += rising.bfloat16()
    assert_attention(q, cache, table, lens, SCALE)


@pytest.mark.parametrize("dtype", [torch.bfloat16, E4M3])
def test_a_key_that_is_not_finite_reaches_only_the_rows_that_see_it(cuda_device, dtype):
    g = torch.Generator(device="cuda").manual_seed(12)
    S, H, lens = 6, 16, [150, 64]
    cache, table = filled_cache(g, lens, 64, dtype)
    q = torch.randn(2, S, H, 576, generator=g, device="cuda").bfloat16()
    tree = random_tree(torch.Generator().manual_seed(2), 2, S)
    tree[:, 5, :5] = False                                               # token 5 sees itself only
    want = assert_attention(q, cache, table, lens, SCALE, None, tree)[0]
    for b in range(2):                                                   # new token 5's row of both sequences
        row = slots_of(table[b], lens[b], 64)[lens[b] - 1]
        cache.latent.view(-1, 512).view(torch.uint8)[row] = 0x7F if dtype == E4M3 else 0xFF
    o = run_attention(q, cache, table, lens, SCALE, None, tree)[0]
    check()
    assert torch.equal(o[:, :5], want[:, :5]) and o[:, 5].isnan().all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, E4M3])
@pytest.mark.parametrize("first", [10, 140])
def test_keys_that_are_not_finite_in_several_tiles(cuda_device, dtype, first):
    """New tokens that span more than one tile of keys, three of them with values that are not finite: the rows in front of
    the first see none of them."""
    g = torch.Generator(device="cuda").manual_seed(first)
    S, H, lens = 200, 2, [500, 230]
    cache, table = filled_cache(g, lens, 16, dtype)
    q = torch.randn(2, S, H, 576, generator=g, device="cuda").bfloat16()
    want = assert_attention(q, cache, table, lens, SCALE)[0]
    for b in range(2):
        rows = slots_of(table[b], lens[b], 16)[lens[b] - S:]
        for at, column in ((first, 0), (first + 1, 511), (first + 50, 200)):
            cache.latent.view(-1, 512).view(torch.uint8).view(-1, 512, 1 if dtype == E4M3 else 2)[rows[at], column] = \
                0x7F if dtype == E4M3 else 0xFF
    o = run_attention(q, cache, table, lens, SCALE)[0]
    check()
    assert torch.equal(o[:, :first], want[:, :first]) and o[:, first:].isnan().any(-1).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, E4M3])
@pytest.mark.parametrize("S", [1, 2])
def test_sequences_without_keys_between_others(cuda_device, dtype, S):
    """Every other sequence is empty, and the queries' sizes differ from sequence to sequence (as do an 8-bit query's factors)."""
    r = torch.Generator().manual_seed(S)
    lens = [0 if b % 2 else int(torch.randint(S, 200, (), generator=r)) for b in range(500)]
    g = torch.Generator(device="cuda").manual_seed(S)
    cache, table = filled_cache(g, lens, 32, dtype)
    q = torch.randn(500, S, 16, 576, generator=g, device="cuda")
    q = (q * 2.0 ** torch.randint(-6, 3, (500, 1, 16, 1), generator=g, device="cuda")).bfloat16()
    o, l = assert_attention(q, cache, table, lens, SCALE)
    assert not o[1::2].any() and (l[1::2] == -math.inf).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, E4M3])
@pytest.mark.parametrize("B,S,H,longest,page,kind", [
    (170, 2, 16, 400, 16, "causal"), (60, 5, 16, 700, 32, "tree"), (300, 1, 16, 300, 192, "causal"),
    (160, 2, 16, 128, 64, "padded"), (45, 13, 8, 1500, 320, "tree"), (30, 16, 16, 600, 48 * 4, "padded"),
    (400, 1, 16, 100, 16, "causal"), (200, 2, 16, 60, 64, "padded"),   # no sequence can pass 128 keys
    (90, 2, 16, 700, 64, "causal"), (140, 1, 16, 900, 16, "padded"), (1, 1, 16, 300, 32, "causal"),
    (100, 4, 4, 1000, 128, "tree")])  # one CTA each for most of these
def test_many_sequences_of_uneven_lengths(cuda_device, dtype, B, S, H, longest, page, kind):
    """Several pieces for every CTA, some of them without keys, and every way of counting pages."""
    r = torch.Generator().manual_seed(B + S + page)
    lens = torch.randint(S if kind == "tree" else 0, longest + 1, (B,), generator=r).tolist()
    qlens = torch.randint(0, S + 1, (B,), generator=r).tolist() if kind == "padded" else None
    g = torch.Generator(device="cuda").manual_seed(B)
    cache, table = filled_cache(g, lens, page, dtype)
    q = torch.randn(B, S, H, 576, generator=g, device="cuda").bfloat16()
    assert_attention(q, cache, table, lens, SCALE, qlens, random_tree(r, B, S) if kind == "tree" else None)


def test_a_row_factor_that_is_not_finite_reaches_only_the_rows_that_see_it(cuda_device):
    g = torch.Generator(device="cuda").manual_seed(17)
    S, H, lens = 4, 16, [300, 70]
    for bad in (float("nan"), float("inf")):
        cache, table = filled_cache(g, lens, 32, E4M3)
        q = torch.randn(2, S, H, 576, generator=g, device="cuda").bfloat16()
        want = assert_attention(q, cache, table, lens, SCALE)[0]
        cache.scale.view(-1)[slots_of(table[0], 300, 32)[298]] = bad    # the third new token of the first sequence
        o = run_attention(q, cache, table, lens, SCALE)[0]
        check()
        assert torch.equal(o[0, :2], want[0, :2]) and torch.equal(o[1], want[1]) and o[0, 2:].isnan().all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, E4M3])
@pytest.mark.parametrize("S", [1, 4])
def test_a_query_that_is_not_finite_stays_in_its_row(cuda_device, dtype, S):
    g = torch.Generator(device="cuda").manual_seed(18)
    lens = [700, 64]
    cache, table = filled_cache(g, lens, 64, dtype)
    q = torch.randn(2, S, 16, 576, generator=g, device="cuda").bfloat16()
    want = assert_attention(q, cache, table, lens, SCALE)[0]
    bad = [(0, 0, 3, 17, "nan"), (0, S - 1, 5, 500, "inf"), (1, 0, 7, 570, "nan"), (1, S - 1, 8, 0, "-inf")]
    hit = torch.zeros(2, S, 16, dtype=torch.bool, device="cuda")
    for b, s, h, d, v in bad:
        q[b, s, h, d] = float(v)
        hit[b, s, h] = True
    o = run_attention(q, cache, table, lens, SCALE)[0]
    check()
    assert torch.equal(o[~hit], want[~hit]) and o[hit].isnan().any(-1).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, E4M3])
def test_attention_takes_strided_inputs_and_repeats_to_the_bit(cuda_device, dtype):
    from pithtrain_b200.operators.mla import LatentCache
    g = torch.Generator(device="cuda").manual_seed(13)
    lens = [700, 1, 2100]
    cache, table = filled_cache(g, lens, 64, dtype)
    q = torch.randn(3, 2, 16, 576, generator=g, device="cuda").bfloat16()
    o, l = assert_attention(q, cache, table, lens, SCALE)
    again = run_attention(q, cache, table, lens, SCALE)
    assert torch.equal(o, again[0]) and torch.equal(l, again[1])
    wide_q = torch.zeros(2, 3, 17, 640, device="cuda", dtype=torch.bfloat16)[:, :, 1:, 32:608].transpose(0, 1)
    wide_q.copy_(q)
    wide_t = torch.full((3, table.shape[1] + 5), -1, dtype=torch.int32, device="cuda")[:, 2:2 + table.shape[1]]
    wide_t.copy_(table)
    lat = torch.zeros(cache.num_pages, 2, 64, 512, device="cuda").to(dtype)
    rope = torch.zeros(cache.num_pages, 2, 64, 64, device="cuda", dtype=torch.bfloat16)
    lat[:, 1] = cache.latent
    rope[:, 1] = cache.rope
    scale = None
    if cache.scale is not None:
        scale = torch.zeros(cache.num_pages, 64, 2, device="cuda")[..., 1]
        scale.copy_(cache.scale)
    layer = LatentCache(lat[:, 1], rope[:, 1], scale)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = run_attention(wide_q, layer, wide_t, lens, SCALE)
    torch.cuda.current_stream().wait_stream(side)
    check()
    assert torch.equal(o, other[0]) and torch.equal(l, other[1])


def test_attention_in_a_graph_and_beside_another_call(cuda_device):
    """One captured call, replayed with other lengths, pages and queries; a second captured call replayed beside it."""
    from pithtrain_b200.operators.mla import latent_attention
    g = torch.Generator(device="cuda").manual_seed(14)
    cache, table = filled_cache(g, [2000, 1500], 64, torch.bfloat16)
    cache8, table8 = filled_cache(g, [1800, 900], 64, E4M3)
    q = torch.randn(2, 1, 16, 576, generator=g, device="cuda").bfloat16()
    lens = torch.tensor([1, 2], dtype=torch.int32, device="cuda")
    latent_attention(q, cache, table, lens, SCALE)
    latent_attention(q, cache8, table8, lens, SCALE)
    torch.cuda.synchronize()
    graphs = []
    for c, t in ((cache, table), (cache8, table8)):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            res = latent_attention(q, c, t, lens, SCALE, return_lse=True)
        graphs.append((graph, res))
    side = torch.cuda.Stream()
    for step in ([1700, 800], [0, 65], [1000, 900]):
        lens.copy_(torch.tensor(step, dtype=torch.int32))
        q.copy_(torch.randn(q.shape, generator=g, device="cuda"))
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            for _ in range(5):
                graphs[1][0].replay()
        for _ in range(5):
            graphs[0][0].replay()
        torch.cuda.synchronize()
        assert_attention(q, cache, table, step, SCALE, got=graphs[0][1])
        assert_attention(q, cache8, table8, step, SCALE, got=graphs[1][1])


def test_pages_and_lengths_out_of_range_are_reported(cuda_device):
    from pithtrain_b200 import kernels
    from pithtrain_b200.operators.mla import latent_attention
    g = torch.Generator(device="cuda").manual_seed(15)
    cache, table = filled_cache(g, [100, 50], 64, torch.bfloat16)
    q = torch.randn(2, 1, 16, 576, generator=g, device="cuda").bfloat16()
    lens = torch.tensor([100, 50], dtype=torch.int32, device="cuda")
    for bad in (-1, cache.num_pages, 1 << 30):
        t = table.clone()
        t[0, 1] = bad
        latent_attention(q, cache, t, lens, SCALE)
        with pytest.raises(RuntimeError, match="a page of the block table"):
            kernels.check_device_status()
    for bad in ([100, -1], [table.shape[1] * 64 + 1, 50]):
        t = table.clamp(max=cache.num_pages - 1)
        latent_attention(q, cache, t, torch.tensor(bad, dtype=torch.int32, device="cuda"), SCALE)
        with pytest.raises(RuntimeError, match="a sequence length"):
            kernels.check_device_status()
    latent_attention(q, cache, table, lens, SCALE, query_lens=torch.tensor([2, 0], dtype=torch.int32, device="cuda"))
    with pytest.raises(RuntimeError, match="a sequence length"):
        kernels.check_device_status()
    assert_attention(q, cache, table, [100, 50], SCALE)


def test_a_cache_of_more_than_2_31_elements(cuda_device):
    """Offsets behind 2^32 bytes and 2^31 elements, written, read and attended to."""
    from pithtrain_b200.operators.mla import LatentCache, latent_cache_read, latent_cache_write
    pages, page = 68000, 64
    cache = LatentCache(torch.empty(pages, page, 512, dtype=torch.bfloat16, device="cuda"),
                        torch.empty(pages, page, 64, dtype=torch.bfloat16, device="cuda"))
    g = torch.Generator(device="cuda").manual_seed(16)
    n = 300
    table = (pages - 1 - torch.arange(5, device="cuda")).int()[None]
    slots = slots_of(table[0], n, page)[None]
    assert slots.min().item() * 512 > 2 ** 31
    x = torch.randn(1, n, 576, generator=g, device="cuda").bfloat16()
    cos, sin = tables(n)
    latent_cache_write(cache, slots, x[..., :512], x[..., 512:], torch.ones(512, device="cuda"), cos, sin, 1e-6)
    lat, pe = latent_cache_read(cache, slots)
    check()
    assert torch.equal(lat[0], cache.latent.view(-1, 512)[slots[0]])
    q = torch.randn(1, 1, 16, 576, generator=g, device="cuda").bfloat16()
    o, l = run_attention(q, cache, table, [n], SCALE)
    small, t = filled_cache(g, [n], page, torch.bfloat16)
    small.latent.view(-1, 512)[slots_of(t[0], n, page)] = lat[0]
    small.rope.view(-1, 64)[slots_of(t[0], n, page)] = pe[0]
    assert_attention(q, small, t, [n], SCALE, got=(o, l))


# ---------------------------------------------------------------------------------------------------- projections
# One rounding to bf16 (2^-8 of the value) behind an fp32 sum of K products (K * 2^-24 of the sum of their magnitudes).
def assert_product(got, x, w, what):
    want = torch.einsum("bshk,hkn->bshn", x.double(), w.double())
    size = torch.einsum("bshk,hkn->bshn", x.double().abs(), w.double().abs())
    excess = (got.double() - want).abs() - (2.0 ** -8 * want.abs() + x.shape[-1] * 2.0 ** -24 * size)
    assert excess.max().item() <= 0, (what, excess.max().item())


@pytest.mark.parametrize("B,S,H", [(1, 1, 16), (1, 1, 1), (3, 1, 16), (33, 1, 5), (2, 65, 16), (1, 129, 2), (1, 700, 16),
                                   (3, 130, 16), (64, 5, 16), (1, 300, 128)])
def test_query_and_output_projections(cuda_device, B, S, H):
    from pithtrain_b200.operators.mla import latent_output, latent_query
    g = torch.Generator(device="cuda").manual_seed(B * S + H)
    w = (torch.randn(H * 256, 512, generator=g, device="cuda") / 20).bfloat16()
    heads = w.view(H, 256, 512)
    q = torch.randn(B, S, H, 192, generator=g, device="cuda").bfloat16()
    cos, sin = tables(3000)
    pos = torch.randint(0, 3000, (B, S), generator=g, device="cuda")
    out = latent_query(q, w, cos, sin, position_ids=pos)
    check()
    assert out.shape == (B, S, H, 576) and out.is_contiguous()
    assert_product(out[..., :512], q[..., :128], heads[:, :128], "query")
    turned = rotated(q[..., 128:], cos[pos][:, :, None], sin[pos][:, :, None])
    assert_rounded(out[..., 512:], turned, 2.0 ** -8, "rope", floor=2.0 ** -20)
    a = torch.randn(B, S, H, 512, generator=g, device="cuda").bfloat16()
    y = latent_output(a, w)
    check()
    assert y.shape == (B, S, H, 128) and y.is_contiguous()
    assert_product(y, a, heads[:, 128:].transpose(1, 2), "output")


@pytest.mark.parametrize("cs", [torch.float32, torch.bfloat16])
def test_projections_take_strided_views(cuda_device, cs):
    """Head and sequence slices of larger tensors, tables gathered beforehand, a weight with padded rows."""
    from pithtrain_b200.operators.mla import latent_output, latent_query
    g = torch.Generator(device="cuda").manual_seed(21)
    B, S, H = 3, 150, 4
    w = torch.randn(H * 256, 640, generator=g, device="cuda").div(20).bfloat16()[:, 64:576]
    q = torch.randn(S, B, 9, 200, generator=g, device="cuda").bfloat16()[:, :, 3:7, 8:].transpose(0, 1)
    cos, sin = (t[None] for t in tables(S, cs))
    out = latent_query(q, w, cos, sin)
    a = torch.randn(B, 2 * S, H, 512, generator=g, device="cuda").bfloat16()[:, S:]
    y = latent_output(a, w)
    check()
    heads = w.reshape(H, 256, 512)
    assert_product(out[..., :512], q[..., :128], heads[:, :128], "query")
    assert_rounded(out[..., 512:], rotated(q[..., 128:], cos[:, :, None], sin[:, :, None]), 2.0 ** -8, "rope",
                   floor=2.0 ** -20)
    assert_product(y, a, heads[:, 128:].transpose(1, 2), "output")


def test_projection_reports_a_position_out_of_range(cuda_device):
    from pithtrain_b200 import kernels
    from pithtrain_b200.operators.mla import latent_query
    cos, sin = tables(10)
    w = torch.zeros(256, 512, device="cuda", dtype=torch.bfloat16)
    q = torch.zeros(1, 2, 1, 192, device="cuda", dtype=torch.bfloat16)
    for bad in (10, -1, 1 << 40):
        latent_query(q, w, cos, sin, position_ids=torch.tensor([[0, bad]], device="cuda"))
        with pytest.raises(RuntimeError, match="a position given"):
            kernels.check_device_status()


# ---------------------------------------------------------------------------------------------------- all together
class Layer:
    """The weights of an MLA layer between its input projections and o_proj, and the expanded form in 64 bits."""

    def __init__(self, g, H):
        self.H = H
        self.norm = (1 + 0.1 * torch.randn(512, generator=g, device="cuda")).bfloat16()
        self.kv_b = torch.randn(H * 256, 512, generator=g, device="cuda").div(512 ** 0.5).bfloat16()
        self.cos, self.sin = tables(4096)

    def expanded(self, q, proj, seen, pos):
        """q [n, H, 192], proj [n, 576] of all n tokens of a sequence, seen [n, n], pos [n] -> [n, H, 128]."""
        x = proj[:, :512].double()
        c = x / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt() * self.norm.double()
        kv = torch.einsum("nr,hdr->nhd", c, self.kv_b.double().view(self.H, 256, 512))
        cos, sin = self.cos[pos], self.sin[pos]
        r = rotated(proj[:, 512:], cos, sin)
        qr = rotated(q[..., 128:], cos[:, None], sin[:, None])
        s = torch.einsum("ihd,nhd->hin", q[..., :128].double(), kv[..., :128]) + torch.einsum("ihd,nd->hin", qr, r)
        return torch.einsum("hin,nhd->ihd", torch.softmax((s * SCALE).masked_fill(~seen, -math.inf), -1), kv[..., 128:])


def close_to(got, want, dtype, what):
    """Against the expanded form in 64 bits. Four bf16 roundings in a row (latent, query, weights and result of attention,
    output) of half a step each, 2^-8 relative, act on sums of many terms whose rounding errors are independent, so that
    the relative 2-norm error is at most 4 * 2^-8 (all in the same direction); an 8-bit latent row adds 2^-4."""
    rel = ((got.double() - want).norm() / want.norm()).item()
    bound = 4 * 2.0 ** -8 + (2.0 ** -4 if dtype == E4M3 else 0)
    assert rel <= bound, (what, rel, bound)


@pytest.mark.parametrize("dtype", [torch.bfloat16, E4M3])
def test_prompt_tokens_drafts_and_the_expanded_form(cuda_device, dtype):
    """A ragged batch as a sampling loop runs it: prompts in two chunks, three single tokens, then a tree of drafts over
    everything so far; each compared with the expanded form over all tokens of the sequence."""
    from pithtrain_b200.operators import mla
    g = torch.Generator(device="cuda").manual_seed(30)
    H, page, B, D = 16, 32, 2, 6
    layer = Layer(g, H)
    prompts, total = [75, 130], [75 + 3 + D, 130 + 3 + D]
    pages = [-(-n // page) for n in total]
    cache = make_cache(sum(pages) + 1, page, dtype)
    order = torch.randperm(cache.num_pages, generator=g, device="cuda").int()
    table = torch.full((B, max(pages)), -1, dtype=torch.int32, device="cuda")
    table[0, : pages[0]], table[1, : pages[1]] = order[: pages[0]], order[pages[0]: sum(pages)]
    q = [torch.randn(n, H, 192, generator=g, device="cuda").bfloat16() for n in total]
    proj = [torch.randn(n, 576, generator=g, device="cuda").bfloat16() for n in total]
    tree = random_tree(torch.Generator().manual_seed(4), B, D)
    depth = tree.sum(-1) - 1

    def step(first, counts, mask=None, positions=None):
        S = max(counts)
        take = lambda xs: torch.stack([torch.cat([x[f:f + n], x.new_zeros(S - n, *x.shape[1:])])  # noqa: E731
                                       for x, f, n in zip(xs, first, counts)])
        qs, ps = take(q), take(proj)
        at = torch.tensor(first, device="cuda")[:, None] + torch.arange(S, device="cuda")
        pos = at if positions is None else positions
        real = torch.arange(S, device="cuda") < torch.tensor(counts, device="cuda")[:, None]
        slot = torch.gather(table.long(), 1, (at // page).clamp(max=table.shape[1] - 1)) * page + at % page
        mla.latent_cache_write(cache, torch.where(real, slot, -1), ps[..., :512], ps[..., 512:], layer.norm, layer.cos,
                               layer.sin, 1e-6, position_ids=pos)
        query = mla.latent_query(qs, layer.kv_b, layer.cos, layer.sin, position_ids=pos)
        lens = torch.tensor([f + n for f, n in zip(first, counts)], dtype=torch.int32, device="cuda")
        attn = mla.latent_attention(query, cache, table, lens, SCALE, tree_mask=mask,
                                    query_lens=torch.tensor(counts, dtype=torch.int32, device="cuda"))
        return mla.latent_output(attn, layer.kv_b)

    results = [[], []]
    for first, counts in (([0, 0], [64, 64]), ([64, 64], [11, 66])):          # the prompts' chunks
        y = step(first, counts)
        for b in range(B):
            results[b].append(y[b, : counts[b]])
    for i in range(3):
        y = step([n + i for n in prompts], [1, 1])
        for b in range(B):
            results[b].append(y[b])
    base = [n + 3 for n in prompts]
    y = step(base, [D, D], tree, torch.tensor(base, device="cuda")[:, None] + depth)
    check()
    for b in range(B):
        results[b].append(y[b])
        n = total[b]
        seen = torch.ones(n, n, dtype=torch.bool, device="cuda").tril()
        seen[base[b]:, base[b]:] = tree[b]
        pos = torch.arange(n, device="cuda")
        pos[base[b]:] = base[b] + depth[b]
        want = layer.expanded(q[b], proj[b], seen, pos)
        close_to(torch.cat(results[b]), want, dtype, f"sequence {b}")

    # the expanded form of the library over the cached prefix agrees with what was decoded from the cache
    b, n = 1, prompts[1]
    latent, pe = mla.latent_cache_read(cache, slots_of(table[b], n, page)[None])
    kv = (latent @ layer.kv_b.T).view(1, n, H, 256)
    key = torch.cat([kv[..., :128], pe[:, :, None].expand(1, n, H, 64)], -1)
    cos, sin = layer.cos[:n, None], layer.sin[:n, None]
    query = torch.cat([q[b][:n, :, :128], rotated(q[b][:n, :, 128:], cos, sin).bfloat16()], -1)[None]
    got = mla.MLA(H, 192, 128, SCALE)(query, key, kv[..., 128:].contiguous())
    check()
    close_to(got[0], torch.cat(results[b])[:n].double(), torch.bfloat16, "expanded over the cache")


def test_a_captured_decoding_step_is_the_eager_one(cuda_device):
    """All five operators of a step in one graph, replayed for several tokens with new contents in the same tensors."""
    from pithtrain_b200.operators import mla
    g = torch.Generator(device="cuda").manual_seed(40)
    H, page, B = 16, 64, 3
    layer = Layer(g, H)
    lens0 = [200, 5, 63]
    caches = []
    for _ in range(2):
        gen = torch.Generator(device="cuda").manual_seed(41)
        caches.append(filled_cache(gen, [n + 8 for n in lens0], page, E4M3))
    table = caches[0][1]
    q = torch.empty(B, 1, H, 192, dtype=torch.bfloat16, device="cuda")
    proj = torch.empty(B, 1, 576, dtype=torch.bfloat16, device="cuda")
    slots, pos = torch.zeros(B, 1, dtype=torch.int64, device="cuda"), torch.zeros(B, 1, dtype=torch.int64, device="cuda")
    lens = torch.zeros(B, dtype=torch.int32, device="cuda")

    def step(cache):
        mla.latent_cache_write(cache, slots, proj[..., :512], proj[..., 512:], layer.norm, layer.cos, layer.sin, 1e-6,
                               position_ids=pos)
        query = mla.latent_query(q, layer.kv_b, layer.cos, layer.sin, position_ids=pos)
        latent, pe = mla.latent_cache_read(cache, slots)
        return mla.latent_output(mla.latent_attention(query, cache, table, lens, SCALE), layer.kv_b), latent, pe

    def fill(i):
        n = torch.tensor([v + i for v in lens0], device="cuda")
        pos.copy_(n[:, None])
        lens.copy_(n + 1)
        slots.copy_(torch.gather(table.long(), 1, (n // page)[:, None]) * page + (n % page)[:, None])
        gen = torch.Generator(device="cuda").manual_seed(50 + i)
        q.copy_(torch.randn(q.shape, generator=gen, device="cuda"))
        proj.copy_(torch.randn(proj.shape, generator=gen, device="cuda"))

    fill(0)
    step(caches[0][0])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = step(caches[0][0])
    for i in range(6):
        fill(i)
        graph.replay()
        want = step(caches[1][0])
        check()
        for a, b in zip(res, want):
            assert torch.equal(a, b)
    for a, b in zip((caches[0][0].latent, caches[0][0].rope), (caches[1][0].latent, caches[1][0].rope)):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
