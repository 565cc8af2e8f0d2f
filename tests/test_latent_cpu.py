"""Argument checks of the MLA latent-cache operators that need no GPU: the Python layer and the C ABI."""

import ctypes

import pytest
import torch

from pithtrain_b200.operators import mla

BF = torch.bfloat16


def cache(dtype=BF, pages=2, page=16):
    return mla.LatentCache.allocate(pages, page, dtype, device="cpu")


def write_args(B=1, S=2):
    return dict(slots=torch.zeros(B, S, dtype=torch.int64), compressed_kv=torch.zeros(B, S, 512, dtype=BF),
                k_pe=torch.zeros(B, S, 64, dtype=BF), norm_weight=torch.ones(512), cos=torch.ones(8, 64),
                sin=torch.zeros(8, 64), eps=1e-6)


def test_cache_planes_are_checked():
    c = cache(torch.float8_e4m3fn, 3, 32)
    assert (c.num_pages, c.page_size) == (3, 32) and c.scale.shape == (3, 32)
    lat, rope, scale = torch.zeros(2, 16, 512, dtype=BF), torch.zeros(2, 16, 64, dtype=BF), torch.ones(2, 16)
    with pytest.raises(ValueError, match="page_size"):
        cache(page=48)
    with pytest.raises(ValueError, match="has none"):
        mla.LatentCache(lat, rope, scale)
    with pytest.raises(ValueError, match="scale plane"):
        mla.LatentCache(lat.to(torch.float8_e4m3fn), rope)
    with pytest.raises(ValueError, match="512"):
        mla.LatentCache(lat[..., :256], rope)
    with pytest.raises(ValueError, match="rope must be"):
        mla.LatentCache(lat, rope[:1])
    with pytest.raises(TypeError, match="bfloat16"):
        mla.LatentCache(lat.float(), rope)


@pytest.mark.parametrize("change,error,text", [
    (dict(compressed_kv=torch.zeros(1, 2, 256, dtype=BF)), ValueError, "compressed_kv must be"),
    (dict(compressed_kv=torch.zeros(1, 2, 512)), TypeError, "must be bfloat16"),
    (dict(k_pe=torch.zeros(1, 3, 64, dtype=BF)), ValueError, "k_pe must be"),
    (dict(slots=torch.zeros(1, 2, dtype=torch.int32)), TypeError, "slots must be int64"),
    (dict(slots=torch.zeros(2, 1, dtype=torch.int64)), ValueError, "slots has shape"),
    (dict(norm_weight=torch.ones(64)), ValueError, "norm_weight"),
    (dict(cos=torch.ones(1, 64), sin=torch.ones(1, 64)), ValueError, "rows"),
    (dict(cos=torch.ones(8, 64), sin=torch.ones(8, 64, dtype=BF)), TypeError, "cos and sin"),
    (dict(cos=torch.ones(1, 2, 64), sin=torch.ones(1, 2, 64), position_ids=torch.zeros(1, 2, dtype=torch.int64)),
     ValueError, "tables"),
    (dict(position_ids=torch.zeros(1, 3, dtype=torch.int64)), ValueError, "position_ids has shape"),
    (dict(position_ids=torch.zeros(1, 2, dtype=torch.int32)), TypeError, "position_ids must be int64"),
    (dict(), RuntimeError, "no CPU fallback"),
])
def test_write_refuses(change, error, text):
    with pytest.raises(error, match=text):
        mla.latent_cache_write(cache(), **{**write_args(), **change})


def test_read_refuses():
    with pytest.raises(TypeError, match="int64"):
        mla.latent_cache_read(cache(), torch.zeros(2, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        mla.latent_cache_read(cache(), torch.zeros(2, dtype=torch.int64))


def test_inputs_that_need_gradients_are_refused():
    a = write_args()
    a["norm_weight"].requires_grad_()
    with pytest.raises(RuntimeError, match="no gradient"):
        mla.latent_cache_write(cache(), **a)
    with torch.no_grad(), pytest.raises(RuntimeError, match="no CPU fallback"):
        mla.latent_cache_write(cache(), **a)


def cabi_cache(a):
    a.cache.latent = a.cache.rope = 0x1000
    a.cache.dtype, a.cache.pages, a.cache.page_size = 0, 2, 16
    for s, d in ((a.cache.latent_stride, 512), (a.cache.rope_stride, 64)):
        s[0], s[1] = 16 * d, d


def test_cabi_refuses_on_the_host(built_library):
    from pithtrain_b200 import _lib
    lib = _lib.load()
    assert lib.pith_latent_write(None, None) < 0 and b"null args" in lib.pith_last_error()
    w = _lib.LatentWriteArgs()
    w.B, w.S = 1, 2
    cabi_cache(w)
    assert lib.pith_latent_write(ctypes.byref(w), None) < 0 and b"null tensor" in lib.pith_last_error()
    w.cache.page_size = 24
    assert lib.pith_latent_write(ctypes.byref(w), None) < 0 and b"page_size" in lib.pith_last_error()
    w.cache.page_size, w.cache.dtype = 16, 2
    assert lib.pith_latent_write(ctypes.byref(w), None) < 0 and b"null cache plane" in lib.pith_last_error()
    w.cache.dtype, w.cache.latent = 0, 0x1008
    assert lib.pith_latent_write(ctypes.byref(w), None) < 0 and b"16-byte aligned" in lib.pith_last_error()
    w.cache.latent, w.S = 0x1000, 0
    assert lib.pith_latent_write(ctypes.byref(w), None) == 0               # no tokens: nothing to do
    r = _lib.LatentReadArgs()
    cabi_cache(r)
    assert lib.pith_latent_read(ctypes.byref(r), None) == 0
    r.n = 1
    assert lib.pith_latent_read(ctypes.byref(r), None) < 0 and b"null tensor" in lib.pith_last_error()


def test_struct_sizes_match_the_header(built_library):
    import subprocess
    import tempfile
    from pathlib import Path
    from pithtrain_b200 import _lib
    root = Path(__file__).resolve().parent.parent
    names = {"pith_latent_cache": _lib.LatentCacheArgs, "pith_latent_write_args": _lib.LatentWriteArgs,
             "pith_latent_read_args": _lib.LatentReadArgs, "pith_latent_attn_args": _lib.LatentAttnArgs,
             "pith_latent_proj_args": _lib.LatentProjArgs}
    src = '#include <stdio.h>\n#include "pith_b200.h"\nint main(void) {%s return 0; }' % "".join(
        f'printf("%zu\\n", sizeof({n}));' for n in names)
    with tempfile.TemporaryDirectory() as d:
        (Path(d) / "s.c").write_text(src)
        subprocess.run(["gcc", "-I", str(root / "include"), f"{d}/s.c", "-o", f"{d}/s"], check=True)
        got = subprocess.run([f"{d}/s"], capture_output=True, text=True, check=True).stdout.split()
    assert [int(x) for x in got] == [ctypes.sizeof(t) for t in names.values()]


def test_status_string_of_an_index(built_library):
    from pithtrain_b200 import _lib
    lib = _lib.load()
    for detail, text in ((1, b"a slot"), (2, b"a position"), (3, b"a page"), (4, b"a sequence length")):
        assert text in lib.pith_status_string((5 << 24) | detail)


def attn_args(B=2, S=3, H=4):
    return dict(query=torch.zeros(B, S, H, 576, dtype=BF), block_table=torch.zeros(B, 2, dtype=torch.int32),
                seq_lens=torch.zeros(B, dtype=torch.int32), softmax_scale=0.1)


@pytest.mark.parametrize("change,error,text", [
    (dict(query=torch.zeros(2, 3, 4, 512, dtype=BF)), ValueError, "query must be"),
    (dict(query=torch.zeros(2, 3, 4, 576)), TypeError, "query must be bfloat16"),
    (dict(block_table=torch.zeros(2, 2, dtype=torch.int64)), TypeError, "int32"),
    (dict(block_table=torch.zeros(1, 2, dtype=torch.int32)), ValueError, "block_table must be"),
    (dict(block_table=torch.zeros(2, 0, dtype=torch.int32)), ValueError, "block_table must be"),
    (dict(block_table=torch.zeros(2, 4, dtype=torch.int32)[:, ::2]), ValueError, "block_table must be"),
    (dict(seq_lens=torch.zeros(3, dtype=torch.int32)), ValueError, "seq_lens has shape"),
    (dict(query_lens=torch.zeros(2, dtype=torch.int64)), TypeError, "query_lens must be int32"),
    (dict(query_lens=torch.zeros(1, dtype=torch.int32)), ValueError, "query_lens has shape"),
    (dict(tree_mask=torch.zeros(2, 3, 3)), TypeError, "tree_mask must be bool"),
    (dict(tree_mask=torch.zeros(2, 3, 4, dtype=torch.bool)), ValueError, "tree_mask has shape"),
    (dict(softmax_scale=0.0), ValueError, "softmax_scale"),
    (dict(softmax_scale=float("nan")), ValueError, "softmax_scale"),
    (dict(), RuntimeError, "no CPU fallback"),
])
def test_attention_refuses(change, error, text):
    a = {**attn_args(), **change}
    with pytest.raises(error, match=text):
        mla.latent_attention(a.pop("query"), cache(), a.pop("block_table"), a.pop("seq_lens"), a.pop("softmax_scale"), **a)


def test_cabi_attention_refuses_on_the_host(built_library):
    from pithtrain_b200 import _lib
    lib = _lib.load()
    assert lib.pith_latent_attn(None, None) < 0 and b"null args" in lib.pith_last_error()
    a = _lib.LatentAttnArgs()
    cabi_cache(a)
    a.B, a.Sq, a.H, a.table_cols = 1, 1, 16, 4
    assert lib.pith_latent_attn(ctypes.byref(a), None) < 0 and b"softmax_scale" in lib.pith_last_error()
    a.softmax_scale = 0.1
    assert lib.pith_latent_attn(ctypes.byref(a), None) < 0 and b"null tensor" in lib.pith_last_error()
    a.q = a.out = a.block_table = a.seq_lens = a.workspace = 0x1000
    a.q_stride[2] = 4
    assert lib.pith_latent_attn(ctypes.byref(a), None) < 0 and b"16-byte aligned" in lib.pith_last_error()
    a.q_stride[2], a.table_cols = 576, 1 << 30
    assert lib.pith_latent_attn(ctypes.byref(a), None) < 0 and b"too many keys" in lib.pith_last_error()
    a.H = 0
    assert lib.pith_latent_attn(ctypes.byref(a), None) == 0


@pytest.mark.parametrize("change,error,text", [
    (dict(q=torch.zeros(1, 2, 4, 128, dtype=BF)), ValueError, "q must be"),
    (dict(q=torch.zeros(1, 2, 4, 192)), TypeError, "must be bfloat16"),
    (dict(kv_b_weight=torch.zeros(4 * 256, 512)), TypeError, "must be bfloat16"),
    (dict(kv_b_weight=torch.zeros(3 * 256, 512, dtype=BF)), ValueError, "kv_b_weight must be"),
    (dict(cos=torch.ones(2, 64), sin=torch.ones(2, 32)), ValueError, "cos and sin"),
    (dict(position_ids=torch.zeros(2, 2, dtype=torch.int64)), ValueError, "position_ids has shape"),
    (dict(), RuntimeError, "no CPU fallback"),
])
def test_query_projection_refuses(change, error, text):
    a = dict(q=torch.zeros(1, 2, 4, 192, dtype=BF), kv_b_weight=torch.zeros(4 * 256, 512, dtype=BF),
             cos=torch.ones(8, 64), sin=torch.ones(8, 64))
    with pytest.raises(error, match=text):
        mla.latent_query(**{**a, **change})


def test_output_projection_refuses():
    w = torch.zeros(4 * 256, 512, dtype=BF)
    with pytest.raises(ValueError, match="attn must be"):
        mla.latent_output(torch.zeros(1, 2, 4, 576, dtype=BF), w)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        mla.latent_output(torch.zeros(1, 2, 4, 512, dtype=BF), w)
    with pytest.raises(RuntimeError, match="no gradient"):
        mla.latent_output(torch.zeros(1, 2, 4, 512, dtype=BF), w.requires_grad_())


def test_cabi_projections_refuse_on_the_host(built_library):
    from pithtrain_b200 import _lib
    lib = _lib.load()
    a = _lib.LatentProjArgs()
    for entry in (lib.pith_latent_query, lib.pith_latent_output):
        assert entry(None, None) < 0 and b"null args" in lib.pith_last_error()
        a.B, a.S, a.H = 1, 0, 4
        assert entry(ctypes.byref(a), None) == 0
        a.S = 1
        assert entry(ctypes.byref(a), None) < 0 and b"null tensor" in lib.pith_last_error()
    a.x = a.weight = a.out = a.cos = a.sin = 0x1000
    a.cs_stride[1] = 2
    assert lib.pith_latent_query(ctypes.byref(a), None) < 0 and b"multiples of 4" in lib.pith_last_error()
    a.cs_stride[1], a.cs_dtype = 64, 2
    assert lib.pith_latent_query(ctypes.byref(a), None) < 0 and b"bf16 or fp32" in lib.pith_last_error()


@pytest.mark.parametrize("dtype", [BF, torch.float8_e4m3fn])
def test_a_cache_whose_memory_moves(dtype):
    """The address that a call gets is the planes' present one; planes without memory, or of another form, are refused."""
    c = cache(dtype, 3, 32)
    planes = [c.latent, c.rope] + ([c.scale] if c.scale is not None else [])
    addresses = lambda: tuple(t.data_ptr() for t in planes)  # noqa: E731
    assert c.flat[: len(planes)] == addresses()
    keep = []
    for t in planes:                                           # released, and taken back elsewhere
        size, old = t.untyped_storage().nbytes(), t.data_ptr()
        t.untyped_storage().resize_(0)
        with pytest.raises(RuntimeError, match="released"):
            c.flat
        keep.append(torch.empty(size, dtype=torch.uint8))
        t.untyped_storage().resize_(size)
        t.set_(torch.zeros_like(t)) if t.data_ptr() == old else None
        assert c.flat[: len(planes)] == addresses()
    c.latent.data = torch.zeros(3, 2, 32, 512).to(dtype)[:, 1]   # a layer of a larger tensor now
    assert c.flat[: len(planes)] == addresses() and c.flat[6:8] == (2 * 32 * 512, 512)
    c.latent.data = torch.zeros(2, 32, 512).to(dtype)
    with pytest.raises(ValueError, match="rope must be"):
        c.flat


def test_a_moved_cache_is_not_written_at_its_old_place():
    c = cache()
    old = c.flat[0]
    parked = c.latent.data
    c.latent.data = torch.zeros(2, 16, 512, dtype=BF)
    assert parked.data_ptr() == old and c.flat[0] == c.latent.data_ptr() != old


def calls():
    """Every operator as (call, its differentiable inputs by name)."""
    c8 = cache(torch.float8_e4m3fn)
    w = write_args()
    w["norm_weight"] = torch.ones(512)
    at = attn_args()
    pr = dict(q=torch.zeros(1, 2, 4, 192, dtype=BF), kv_b_weight=torch.zeros(4 * 256, 512, dtype=BF), cos=torch.ones(8, 64),
              sin=torch.ones(8, 64))
    out = dict(attn=torch.zeros(1, 2, 4, 512, dtype=BF), kv_b_weight=torch.zeros(4 * 256, 512, dtype=BF))
    slots = torch.zeros(2, dtype=torch.int64)
    return {
        "latent_cache_write": (lambda a, c: mla.latent_cache_write(c, **a), w, cache()),
        "latent_cache_read": (lambda a, c: mla.latent_cache_read(c, slots), {}, c8),
        "latent_attention": (lambda a, c: mla.latent_attention(a["query"], c, a["block_table"], a["seq_lens"],
                                                               a["softmax_scale"]), at, c8),
        "latent_query": (lambda a, c: mla.latent_query(**a), pr, None),
        "latent_output": (lambda a, c: mla.latent_output(**a), out, None)}


@pytest.mark.parametrize("name", ["latent_cache_write", "latent_cache_read", "latent_attention", "latent_query",
                                  "latent_output"])
def test_every_input_that_wants_a_gradient_is_refused(name):
    from torch.autograd import forward_ad
    call, args, c = calls()[name]
    floating = [k for k, v in args.items() if torch.is_tensor(v) and v.is_floating_point()]
    assert floating or name == "latent_cache_read"
    for key in floating:
        with pytest.raises(RuntimeError, match="no gradient"):
            call({**args, key: args[key].clone().requires_grad_()}, c)
        with forward_ad.dual_level(), torch.no_grad():
            dual = forward_ad.make_dual(args[key], torch.ones_like(args[key]))
            with pytest.raises(RuntimeError, match="no gradient"):
                call({**args, key: dual}, c)
            with pytest.raises(RuntimeError, match="no CPU fallback"):   # other duals do no harm
                call(args, c)
    if c is not None:
        with pytest.raises(RuntimeError, match="no gradient"):
            call(args, mla.LatentCache(c.latent, c.rope.clone().requires_grad_(), c.scale))
        with torch.no_grad(), pytest.raises(RuntimeError, match="no CPU fallback"):
            call(args, c)


def test_cabi_projections_name_the_argument_that_is_off(built_library):
    from pithtrain_b200 import _lib
    lib = _lib.load()
    for entry, name in ((lib.pith_latent_query, b"q must"), (lib.pith_latent_output, b"attn must")):
        a = _lib.LatentProjArgs()
        a.B, a.S, a.H = 2, 3, 4
        a.x = a.weight = a.out = a.cos = a.sin = 0x1000
        a.cs_stride[1], a.weight_stride = 64, 512
        a.x_stride[0], a.x_stride[1], a.x_stride[2] = 3 * 4 * 512, 4 * 512, 512
        for field, value, text in (("x", 0x1008, name + b" be 16-byte aligned"),
                                   ("weight", 0x1004, b"kv_b_weight must be 16-byte aligned"),
                                   ("weight_stride", 516, b"kv_b_weight must be"), ("weight_stride", 0, b"kv_b_weight")):
            old = getattr(a, field)
            setattr(a, field, value)
            assert entry(ctypes.byref(a), None) < 0 and text in lib.pith_last_error(), (text, lib.pith_last_error())
            setattr(a, field, old)
        for i in range(3):
            old = a.x_stride[i]
            a.x_stride[i] = 516
            assert entry(ctypes.byref(a), None) < 0 and name + b" be 16-byte" in lib.pith_last_error()
            a.x_stride[i] = 0
            assert entry(ctypes.byref(a), None) < 0 and name + b" not repeat" in lib.pith_last_error()
            a.x_stride[i] = old


@pytest.mark.parametrize("name", ["latent_cache_write", "latent_cache_read", "latent_attention", "latent_query",
                                  "latent_output"])
def test_a_traced_call_is_one_op(name):
    """torch.compile(fullgraph=True) sees one custom op, whose fake kernel knows the result; run, it is the kernel's call."""
    call, args, c = calls()[name]
    seen = []

    def backend(gm, inputs):
        seen.extend(n for n in gm.graph.nodes if n.op == "call_function" and "pithtrain_b200" in str(n.target))
        return gm.forward

    torch._dynamo.reset()
    fn = torch.compile(lambda a: call(a, c), backend=backend, fullgraph=True)
    with torch.no_grad(), pytest.raises(RuntimeError, match="no CPU fallback"):
        fn(args)
    assert [str(n.target).split(".")[1] for n in seen] == [name]
