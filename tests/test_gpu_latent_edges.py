"""The MLA latent-cache operators where calls, streams and values meet: cases beside those of test_gpu_latent.py."""

import math
import time

import pytest
import torch

from test_gpu_latent import (E4M3, SCALE, assert_attention, assert_product, assert_rounded, check, filled_cache, make_cache,
                             quantised, random_tree, rotated, run_attention, slots_of, stored, tables, visible)

pytestmark = pytest.mark.gpu


def test_an_error_that_another_stream_records_while_parts_are_merged(cuda_device):
    """Attention whose parts are merged, beside a stream that records a bad slot at some moment of it: the call is done or
    skipped as a whole, the error is reported, and the next call is right."""
    from pithtrain_b200 import kernels
    from pithtrain_b200.operators.mla import LatentCache, latent_attention, latent_cache_write
    g = torch.Generator(device="cuda").manual_seed(60)
    lens = [3000, 1, 2500, 700]
    cache, table = filled_cache(g, lens, 64, torch.bfloat16)
    q = torch.randn(4, 1, 16, 576, generator=g, device="cuda").bfloat16()
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    other = LatentCache.allocate(1, 16)
    x = torch.ones(1, 1, 576, device="cuda", dtype=torch.bfloat16)
    cos, sin = tables(1)
    bad = torch.full((1, 1), 16, device="cuda")
    w = torch.ones(512, device="cuda")
    attend = lambda: latent_attention(q, cache, table, n, SCALE)  # noqa: E731
    record = lambda: latent_cache_write(other, bad, x[..., :512], x[..., 512:], w, cos, sin, 1e-6)  # noqa: E731
    attend()
    torch.cuda.synchronize()
    graphs = []
    for call, times in ((attend, 20), (record, 1)):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            for _ in range(times):
                call()
        graphs.append(graph)
    side = torch.cuda.Stream()
    for i in range(40):
        with torch.cuda.stream(side):
            torch.cuda._sleep(5000 * i)
            graphs[1].replay()
        graphs[0].replay()
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match="a slot given"):
            kernels.check_device_status()
    assert_attention(q, cache, table, lens, SCALE)


def one_context(g, n, page, dtype, mean):
    """(cache, table [1, pages]) of one context whose latent vectors have a common part."""
    cache = make_cache(-(-n // page), page, dtype, fill=0.0)
    c = mean + torch.randn(cache.num_pages * page, 512, generator=g, device="cuda")
    if dtype == E4M3:
        c8, scale = quantised(c)
        cache.latent.copy_(c8.view(cache.latent.shape))
        cache.scale.copy_(scale.view(cache.scale.shape))
    else:
        cache.latent.copy_(c.view(cache.latent.shape))
    return cache, torch.randperm(cache.num_pages, generator=g, device="cuda").int()[None]


def shared_context_reference(query, cache, table, n, tree=None):
    """fp64 (out [B,S,H,512], log2 lse [B,H,S]) where all sequences read the same n keys."""
    B, S, H, _ = query.shape
    rows = table[0].long()[torch.arange(n, device="cuda") // cache.page_size] * cache.page_size \
        + torch.arange(n, device="cuda") % cache.page_size
    c_all, r_all = stored(cache)
    c, keys = c_all[rows], torch.cat([c_all[rows], r_all[rows]], -1)
    out = torch.empty(B, S, H, 512, dtype=torch.float64, device="cuda")
    lse = torch.empty(B, H, S, dtype=torch.float64, device="cuda")
    for b in range(B):
        seen = visible(S, n, S, None if tree is None else tree[b])
        for i in range(0, S, 16):
            s = torch.einsum("ihd,nd->ihn", query[b, i:i + 16].double() * SCALE, keys)
            s.masked_fill_(~seen[i:i + 16, None], -math.inf)
            lse[b, :, i:i + 16] = (torch.logsumexp(s, -1) / math.log(2)).T
            out[b, i:i + 16] = torch.softmax(s, -1) @ c
    return out, lse


@pytest.mark.parametrize("dtype", [torch.bfloat16, E4M3])
@pytest.mark.parametrize("B,S,n,spread", [(148, 1, 100_000, 0.7), (148, 1, 30_000, 0.0), (16, 13, 100_000, 0.7),
                                          (1, 256, 100_000, 2.0), (148, 2, 131_071, 1.0)])
def test_many_small_weights_behind_a_large_one(cuda_device, dtype, B, S, n, spread):
    """The first key outweighs each other key by 9 to 16 nats, and the others have a common part that makes up as much as all of
    the result; a piece of the work is a whole context, or most of one. The bound has no term that grows with the keys: of the
    result's norm 2^-8 for its rounding to bf16, 2^-9 for the rounding of large weights (bf16: 2^-9 too) and 2^-9 for what is
    left of the small ones, 2^-7 in all. Scores and row sums are fp32: sums of 576 products below 32 in magnitude."""
    g = torch.Generator(device="cuda").manual_seed(B + S + n)
    cache, table = one_context(g, n, 64, dtype, 1.0)
    H = 16
    q = torch.zeros(B, S, H, 576, device="cuda")
    q[..., :512] = torch.randn(B, S, H, 512, generator=g, device="cuda") * (spread / (SCALE * 512 ** 0.5))
    q[..., 512] = torch.linspace(9, 16, B * S * H, device="cuda").view(B, S, H)
    q = q.bfloat16()
    first = table[0, 0].item() * 64
    cache.rope.view(-1, 64)[first, 0] = 1 / SCALE
    tree = random_tree(torch.Generator().manual_seed(S), B, S) if B > 1 and S > 2 else None
    o, l = run_attention(q, cache, table.expand(B, -1), [n] * B, SCALE, None, tree)
    check()
    want, lse = shared_context_reference(q, cache, table, n, tree)
    rel = (o.double() - want).norm(dim=-1) / want.norm(dim=-1)
    assert rel.max().item() <= 2.0 ** -7, rel.max().item()
    assert (l.double() - lse).abs().max().item() <= 2.0 ** -8


@pytest.mark.parametrize("dtype", [torch.bfloat16, E4M3])
def test_a_cache_that_was_parked_and_taken_back(cuda_device, dtype):
    """The planes' memory is released, taken by others, and allocated anew: the operators use the new place, and leave what
    lies at the old one alone."""
    from pithtrain_b200.operators.mla import latent_cache_read, latent_cache_write
    g = torch.Generator(device="cuda").manual_seed(70)
    cache, table = filled_cache(g, [3000], 64, dtype)
    q = torch.randn(1, 1, 16, 576, generator=g, device="cuda").bfloat16()
    assert_attention(q, cache, table, [3000], SCALE)
    planes = [t for t in (cache.latent, cache.rope, cache.scale) if t is not None]
    copies = [t.view(torch.uint8).clone() for t in planes]
    sizes = [t.untyped_storage().nbytes() for t in planes]
    for t in planes:
        t.untyped_storage().resize_(0)
    with pytest.raises(RuntimeError, match="released"):
        run_attention(q, cache, table, [3000], SCALE)
    others = [torch.full((n,), 77, dtype=torch.uint8, device="cuda") for n in sizes]
    for t, n, c in zip(planes, sizes, copies):
        t.untyped_storage().resize_(n)
        t.view(torch.uint8).copy_(c)
    assert_attention(q, cache, table, [3000], SCALE)
    x = torch.randn(1, 4, 576, generator=g, device="cuda").bfloat16()
    cos, sin = tables(4)
    slots = torch.tensor([[0, 65, 5, 99]], device="cuda")
    latent_cache_write(cache, slots, x[..., :512], x[..., 512:], torch.ones(512, device="cuda"), cos, sin, 1e-6)
    got = latent_cache_read(cache, slots)[0]
    check()
    assert torch.equal(got[0].double(), stored(cache)[0][slots[0]]) and got.any()
    assert all((o == 77).all() for o in others)


def test_an_index_error_reaches_a_later_call_without_a_sync(cuda_device):
    """A loop that never asks for the status stops at a later call of these operators, or of the training operators; a capture
    that begins in between is not disturbed."""
    from pithtrain_b200.operators.attention import flash_attn_func
    from pithtrain_b200.operators.mla import LatentCache, latent_cache_read, latent_cache_write
    cache = LatentCache.allocate(1, 16)
    x = torch.ones(1, 1, 576, device="cuda", dtype=torch.bfloat16)
    cos, sin = tables(1)
    w = torch.ones(512, device="cuda")
    good = torch.zeros(1, 1, dtype=torch.int64, device="cuda")

    def write(slot):
        latent_cache_write(cache, good + slot, x[..., :512], x[..., 512:], w, cos, sin, 1e-6)

    check()
    write(16)
    with pytest.raises(RuntimeError, match="a slot given"):
        for _ in range(50):
            time.sleep(0.003)
            latent_cache_read(cache, good)
    write(3)
    check()
    assert (latent_cache_read(cache, good + 3)[0] != 0).all()
    time.sleep(0.02)
    write(16)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rows = latent_cache_read(cache, good + 3)[0]
    q = torch.randn(1, 128, 2, 128, device="cuda").bfloat16()
    with pytest.raises(RuntimeError, match="a slot given"):
        flash_attn_func(q, q, q, causal=True)
    graph.replay()
    check()
    assert (rows != 0).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, E4M3])
def test_a_sequence_alone_and_in_batches_that_cut_it_differently(cuda_device, dtype):
    """The rounding of the weights is all that other sequences may change: at most 2^-8 of each weight in either call, and a
    rounding of the result in each (2^-8), 2^-8 of a norm each time; in 8 bits 2^-9 more for what is left of small weights. The
    LSE differs by fp32 rounding of scores and sums only. Repeated calls agree to the bit."""
    g = torch.Generator(device="cuda").manual_seed(80)
    n = 5000
    cache, table = one_context(g, n, 64, dtype, 0.5)
    q = torch.randn(1, 1, 16, 576, generator=g, device="cuda").bfloat16() * 2
    cache.rope.normal_(generator=g)
    alone, lse = assert_attention(q, cache, table, [n], SCALE)
    want, _ = shared_context_reference(q, cache, table, n)
    rows = table[0].long()[torch.arange(n, device="cuda") // 64] * 64 + torch.arange(n, device="cuda") % 64
    s = torch.einsum("hd,nd->hn", q[0, 0].double() * SCALE, torch.cat([t[rows] for t in stored(cache)], -1))
    size = (torch.softmax(s, -1) @ stored(cache)[0][rows].abs()).norm(dim=-1)     # of the weighted sum of magnitudes
    bound = 2 * (2.0 ** -8 * size + 2.0 ** -8 * want[0, 0].norm(dim=-1) + (2.0 ** -9 * size if dtype == E4M3 else 0))
    for others in ([], [1], [n] * 3, [77] * 200, [n] * 147, [4000, 3, 2500] * 40):
        lens = others + [n]
        batch = torch.randn(len(lens), 1, 16, 576, generator=g, device="cuda").bfloat16()
        batch[-1] = q[0]
        o, l = run_attention(batch, cache, table.expand(len(lens), -1), lens, SCALE)
        again = run_attention(batch, cache, table.expand(len(lens), -1), lens, SCALE)
        check()
        assert torch.equal(o, again[0]) and torch.equal(l, again[1])
        assert ((o[-1, 0].double() - alone[0, 0].double()).norm(dim=-1) <= bound).all()
        assert (l[-1] - lse[0]).abs().max().item() <= 2.0 ** -10


@pytest.mark.parametrize("dtype", [torch.bfloat16, E4M3])
@pytest.mark.parametrize("k", [118, 110, -90, -98])
def test_queries_of_any_magnitude(cuda_device, dtype, k):
    """A query times 2^k with a softmax scale of 2^-k gives the same scores: the same results, to the bit, as long as no product
    leaves the range of fp32."""
    from pithtrain_b200.operators.mla import latent_attention
    g = torch.Generator(device="cuda").manual_seed(90)
    lens = [900, 70]
    cache, table = filled_cache(g, lens, 64, dtype)
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    for S in (1, 3):
        q = torch.randn(2, S, 16, 576, generator=g, device="cuda").clamp(-4, 4).bfloat16()
        q = torch.where(q.abs() < 2.0 ** -8, torch.ones_like(q), q)
        want = latent_attention(q, cache, table, n, SCALE)
        got = latent_attention((q.double() * 2.0 ** k).bfloat16(), cache, table, n, SCALE * 2.0 ** -k)
        check()
        assert torch.equal(got, want)


def test_rows_with_the_least_factor(cuda_device):
    """Rows so small that their factor is the least one, 2^-100: read back and attended to as what is stored."""
    from pithtrain_b200.operators.mla import LatentCache, latent_cache_read, latent_cache_write
    g = torch.Generator(device="cuda").manual_seed(100)
    n = 200
    cache = LatentCache.allocate(4, 64, E4M3)
    x = torch.randn(1, n, 576, generator=g, device="cuda").bfloat16()
    cos, sin = tables(n)
    latent_cache_write(cache, torch.arange(n, device="cuda")[None], x[..., :512], x[..., 512:],
                       torch.full((512,), 2.0 ** -95, device="cuda"), cos, sin, 1e-6)
    check()
    assert (cache.scale.view(-1)[:n] == 2.0 ** -100).all()
    assert torch.equal(latent_cache_read(cache, torch.arange(n, device="cuda"))[0].double(), stored(cache)[0][:n])
    q = torch.randn(1, 2, 16, 576, generator=g, device="cuda").bfloat16()
    table = torch.arange(4, dtype=torch.int32, device="cuda")[None]
    o, _ = assert_attention(q, cache, table, [n], SCALE)
    assert o.any()


def test_a_negative_row_factor_reaches_only_the_rows_that_see_it(cuda_device):
    g = torch.Generator(device="cuda").manual_seed(101)
    cache, table = filled_cache(g, [300], 32, E4M3)
    q = torch.randn(1, 4, 16, 576, generator=g, device="cuda").bfloat16()
    want = assert_attention(q, cache, table, [300], SCALE)[0]
    row = table[0, 298 // 32].long() * 32 + 298 % 32
    cache.scale.view(-1)[row] *= -1
    o = run_attention(q, cache, table, [300], SCALE)[0]
    check()
    assert torch.equal(o[0, :2], want[0, :2]) and o[0, 2:].isnan().all()


def odd_axes(t):
    """The same elements with strides of 3 on every axis of one element."""
    return t.as_strided(t.shape, [3 if n == 1 else s for n, s in zip(t.shape, t.stride())], t.storage_offset())


@pytest.mark.parametrize("dtype", [torch.bfloat16, E4M3])
@pytest.mark.parametrize("B,S,H", [(1, 1, 1), (5, 1, 16), (1, 7, 2), (3, 4, 1)])
def test_strides_of_axes_of_one_element_say_nothing(cuda_device, dtype, B, S, H):
    from pithtrain_b200.operators import mla
    g = torch.Generator(device="cuda").manual_seed(B + S + H)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda").bfloat16()  # noqa: E731
    kv, pe, q, w = rnd(B, S, 512), rnd(B, S, 1, 64), rnd(B, S, H, 192), rnd(H * 256, 512)
    cos, sin = tables(S)
    slots = torch.randperm(64, generator=g, device="cuda")[: B * S].view(B, S)
    pos = torch.arange(S, device="cuda")[None]
    lens = torch.tensor([64 if b == 0 else 40 for b in range(B)], dtype=torch.int32, device="cuda")
    table = torch.zeros(B, 1, dtype=torch.int32, device="cuda")
    results = []
    for turn in (lambda t: t, odd_axes):
        gen = torch.Generator(device="cuda").manual_seed(1)
        cache, _ = one_context(gen, 64, 64, dtype, 0.0)
        planes = [turn(t) if t is not None else None for t in (cache.latent, cache.rope, cache.scale)]
        one = mla.LatentCache(*planes)
        for c, s, p in ((cos, sin, pos), (cos[None], sin[None], None)):
            mla.latent_cache_write(one, turn(slots), turn(kv), turn(pe), torch.ones(512, device="cuda"), turn(c), turn(s),
                                   1e-6, position_ids=None if p is None else turn(p))
            query = mla.latent_query(turn(q), w, turn(c), turn(s), None if p is None else turn(p))
        o = mla.latent_attention(turn(query), one, turn(table), lens, SCALE)
        y = mla.latent_output(turn(o), w)
        check()
        results.append([cache.latent.view(torch.uint8), cache.rope, query, o, y, *mla.latent_cache_read(one, turn(slots))])
    for a, b in zip(*results):
        assert torch.equal(a, b)


# The persistent projection kernel: batches that are not one token axis, more (batch, head) groups than SMs, and token counts
# that are no multiple of a tile.
@pytest.mark.parametrize("B,S,H", [(5, 300, 16), (10, 300, 16), (3, 4095, 2), (40, 129, 8), (2, 700, 80)])
def test_projections_of_batches_that_are_no_single_token_axis(cuda_device, B, S, H):
    from pithtrain_b200.operators.mla import latent_output, latent_query
    g = torch.Generator(device="cuda").manual_seed(B * S + H)
    w = (torch.randn(H * 256, 512, generator=g, device="cuda") / 20).bfloat16()
    heads = w.view(H, 256, 512)
    q = torch.randn(B, 2 * S, H, 192, generator=g, device="cuda").bfloat16()[:, S:]
    cos, sin = tables(3000)
    pos = torch.randint(0, 3000, (B, S), generator=g, device="cuda")
    out = latent_query(q, w, cos, sin, position_ids=pos)
    check()
    assert_product(out[..., :512], q[..., :128], heads[:, :128], "query")
    turned = rotated(q[..., 128:], cos[pos][:, :, None], sin[pos][:, :, None])
    assert_rounded(out[..., 512:], turned, 2.0 ** -8, "rope", floor=2.0 ** -20)
    gathered = latent_query(q, w, cos[pos], sin[pos])
    assert torch.equal(out, gathered)
    del q, turned, gathered, out
    a = torch.randn(B, 2 * S, H, 512, generator=g, device="cuda").bfloat16()[:, S:]
    y = latent_output(a, w)
    check()
    for b in range(B):
        assert_product(y[b:b + 1], a[b:b + 1], heads[:, 128:].transpose(1, 2), "output")


@pytest.mark.parametrize("bad", [4096, -1, 1 << 40])
def test_a_position_out_of_range_among_many(cuda_device, bad):
    """Reported by the warps that rotate tokens beside the GEMM of many; the next call is right."""
    from pithtrain_b200 import kernels
    from pithtrain_b200.operators.mla import latent_query
    g = torch.Generator(device="cuda").manual_seed(110)
    B, S, H, at = 2, 2500, 16, (1, 1234)
    w = (torch.randn(H * 256, 512, generator=g, device="cuda") / 20).bfloat16()
    q = torch.randn(B, S, H, 192, generator=g, device="cuda").bfloat16()
    cos, sin = tables(4096)
    pos = torch.randint(0, 4096, (B, S), generator=g, device="cuda")
    want = latent_query(q, w, cos, sin, position_ids=pos)
    off = pos.clone()
    off[at] = bad
    latent_query(q, w, cos, sin, position_ids=off)
    with pytest.raises(RuntimeError, match="a position given"):
        kernels.check_device_status()
    assert torch.equal(latent_query(q, w, cos, sin, position_ids=pos), want)
    check()


def step_inputs(g, dtype, B, H, n):
    """A layer of a larger cache with n keys a sequence, and the tensors of a decoding step: (planes, args)."""
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda").bfloat16()  # noqa: E731
    pages = B * (-(-n // 64) + 1)
    lat, rope = torch.zeros(pages, 2, 64, 512, device="cuda").to(dtype), torch.zeros(pages, 2, 64, 64, device="cuda").bfloat16()
    scale = torch.ones(pages, 2, 64, device="cuda") if dtype == E4M3 else None
    planes = [t[:, 1] if t is not None else None for t in (lat, rope, scale)]
    table = torch.randperm(pages, generator=g, device="cuda").int().view(B, -1)
    slots = torch.stack([slots_of(t, n, 64) for t in table])
    cos, sin = tables(n + 1)
    return planes, dict(slots=slots, proj=rnd(B, n, 576), q=rnd(B, 1, H, 192), table=table, w=rnd(H * 256, 512) / 20,
                        lens=torch.full((B,), n, dtype=torch.int32, device="cuda"), cos=cos, sin=sin, norm=rnd(512),
                        pos=torch.arange(n, device="cuda")[None])


@pytest.mark.parametrize("dtype", [torch.bfloat16, E4M3])
def test_a_compiled_step_is_the_eager_one(cuda_device, dtype):
    """All five operators inside torch.compile(fullgraph=True): one graph, the same results, the same cache."""
    from pithtrain_b200.operators import mla

    def step(cache, a):
        mla.latent_cache_write(cache, a["slots"], a["proj"][..., :512] * 1.0, a["proj"][..., 512:], a["norm"], a["cos"],
                               a["sin"], 1e-6, position_ids=a["pos"])
        query = mla.latent_query(a["q"] * 1.0, a["w"], a["cos"], a["sin"], position_ids=a["pos"][:, -1:])
        latent, pe = mla.latent_cache_read(cache, a["slots"][:, -3:])
        o, lse = mla.latent_attention(query, cache, a["table"], a["lens"], SCALE, return_lse=True)
        only = mla.latent_attention(query, cache, a["table"], a["lens"], SCALE, query_lens=torch.ones_like(a["lens"]))
        return mla.latent_output(o, a["w"]) + 0.0, lse, only, latent, pe

    results = []
    torch._dynamo.reset()
    for fn in (step, torch.compile(step, fullgraph=True)):
        g = torch.Generator(device="cuda").manual_seed(120)
        planes, a = step_inputs(g, dtype, 3, 16, 200)
        with torch.no_grad():
            out = fn(mla.LatentCache(*planes), a)
        check()
        results.append([*out, *(t.contiguous().view(torch.uint8) for t in planes if t is not None)])
    for a, b in zip(*results):
        assert a.shape == b.shape and a.dtype == b.dtype and torch.equal(a, b)
    assert results[0][0].any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, E4M3])
def test_fake_kernels_describe_the_real_outputs(cuda_device, dtype):
    from pithtrain_b200.operators.mla import latent
    g = torch.Generator(device="cuda").manual_seed(121)
    planes, a = step_inputs(g, dtype, 2, 4, 70)
    # the schema check compares inputs before and after with operations that PyTorch has not for 8-bit floats
    utils = ("test_schema", "test_faketensor") if dtype == torch.bfloat16 else ("test_faketensor",)
    pos = a["pos"][:, -1:]
    query = latent.latent_query_op(a["q"], a["w"], a["cos"], a["sin"], pos)
    with torch.no_grad():
        torch.library.opcheck(latent.latent_cache_write_op, (*planes, a["slots"], a["proj"][..., :512], a["proj"][..., 512:],
                                                             a["norm"], a["cos"], a["sin"], 1e-6, a["pos"]), test_utils=utils)
        torch.library.opcheck(latent.latent_cache_read_op, (*planes, a["slots"]), test_utils=utils)
        for lse in (False, True):
            torch.library.opcheck(latent.latent_attention_op, (query, *planes, a["table"], a["lens"], SCALE, None, None, lse),
                                  test_utils=utils)
        torch.library.opcheck(latent.latent_query_op, (a["q"], a["w"], a["cos"], a["sin"], pos), test_utils=utils)
        torch.library.opcheck(latent.latent_output_op, (query[..., :512], a["w"]), test_utils=utils)
    check()
