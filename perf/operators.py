"""Cases of the latent-cache operators of multi-head latent attention (MLA): writing the cache (RMSNorm, rotary
embedding, optionally 8-bit), reading rows back, folding the key projection into the query, attention over the paged
latent cache (one token, several, a tree of drafted tokens), and the value projection of its result.

``run`` computes them in plain 32-bit torch, or with ``own`` set by the library's operators; ``exact`` in 64 bits.
Sizes are DeepSeek-V2-Lite's (16 heads, latent 512, rope 64, nope 128, v 128) and other head counts."""

import math
import os
import sys

import numpy as np
import torch

own = False
PACKAGE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "pith-train_b200")

LATENT, ROPE, NOPE, VDIM = 512, 64, 128, 128
EPS = 1e-6
E4M3_MAX = 448.0


# ---------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one decoding step of 64 sequences: latency
        {"name": "write_decode_bf16", "op": "write", "tokens": 64, "cache": "bf16", "page": 64},
        # a prompt goes into an 8-bit cache and its rows are read back for the expanded form
        {"name": "write_read_prompt_e4m3", "op": "write_read", "tokens": 8191, "cache": "e4m3", "page": 64},
        # a long cached prefix is gathered for the expanded form of the next chunk
        {"name": "read_prefix_bf16", "op": "read", "tokens": 32768, "cache": "bf16", "page": 64},
        # one decoding step: the weights are what has to be read
        {"name": "query_decode", "op": "query", "batch": 32, "seq": 1, "heads": 16},
        # a chunk of a prompt, not a multiple of any tile
        {"name": "query_prompt", "op": "query", "batch": 1, "seq": 4095, "heads": 16},
        {"name": "output_decode", "op": "output", "batch": 32, "seq": 1, "heads": 16},
        {"name": "output_prompt", "op": "output", "batch": 1, "seq": 4095, "heads": 16},
        # a single sequence just after a short prompt: the smallest call
        {"name": "attn_single_bf16", "op": "attn", "batch": 1, "seq": 1, "heads": 16, "min_len": 77, "max_len": 77,
         "cache": "bf16", "page": 64, "tree": False},
        # a serving batch in the middle of its generations, ragged
        {"name": "attn_decode_bf16", "op": "attn", "batch": 64, "seq": 1, "heads": 16, "min_len": 130, "max_len": 8191,
         "cache": "bf16", "page": 64, "tree": False},
        # few very long contexts in an 8-bit cache
        {"name": "attn_long_e4m3", "op": "attn", "batch": 8, "seq": 1, "heads": 16, "min_len": 9000, "max_len": 131071,
         "cache": "e4m3", "page": 64, "tree": False},
        # trees of 13 drafted tokens
        {"name": "attn_tree_e4m3", "op": "attn", "batch": 16, "seq": 13, "heads": 16, "min_len": 500, "max_len": 4097,
         "cache": "e4m3", "page": 64, "tree": True},
        # a chunk of a prompt behind a cached prefix
        {"name": "attn_chunk_bf16", "op": "attn", "batch": 1, "seq": 250, "heads": 16, "min_len": 6001, "max_len": 6001,
         "cache": "bf16", "page": 64, "tree": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["write", "write_read", "read", "query", "output", "attn", "attn", "attn", "attn"])
    cache, page = rng.choice(["bf16", "e4m3"]), rng.choice([16, 32, 64, 128])
    if op == "write":
        return {"op": op, "tokens": _log(rng, 1, 8191), "cache": "bf16", "page": page}
    if op in ("write_read", "read"):
        return {"op": op, "tokens": _log(rng, 1, 8191 if op == "write_read" else 32768), "cache": cache, "page": page}
    heads = rng.choice([1, 2, 4, 5, 8, 16, 16, 16])
    if op in ("query", "output"):
        batch = _log(rng, 1, 64)
        return {"op": op, "batch": batch, "seq": _log(rng, 1, max(1, 4095 // batch)), "heads": heads}
    kind = rng.choice(["decode", "few", "tree", "chunk"])
    seq = {"decode": 1, "few": rng.randint(2, 8), "tree": rng.randint(2, 48), "chunk": _log(rng, 16, 250)}[kind]
    batch = {"decode": _log(rng, 1, 128), "few": _log(rng, 1, 48), "tree": _log(rng, 1, 16), "chunk": 1}[kind]
    # at most 250,000 cached tokens a pass, and no more row-key pairs than the chunk of a prompt has
    most = min(131071, 250000 // batch, 220 * 16 * 6001 // (batch * seq * heads))
    top = _log(rng, max(seq, min(64, most)), max(seq, most))
    low = rng.randint(seq, max(seq, top))
    return {"op": "attn", "batch": batch, "seq": seq, "heads": heads, "min_len": min(low, top), "max_len": top,
            "cache": cache, "page": page, "tree": kind == "tree"}


def _lens(case):
    """Ragged lengths between min_len and max_len, spread evenly by the golden ratio; the first is the longest."""
    b = np.arange(case["batch"])
    frac = np.mod(1.0 - b * 0.6180339887498949, 1.0)
    frac[0] = 1.0
    return (case["min_len"] + np.floor(frac * (case["max_len"] - case["min_len"]))).astype(np.int64)


def _pairs(case):
    """Visible (query token, key) pairs; a tree's token sees half of the drafted ones on average."""
    n, s = _lens(case), case["seq"]
    return int((s * (n - s)).sum() + case["batch"] * s * (s + 1) // 2)


def work(case):
    op = case["op"]
    if op in ("write", "write_read", "read"):
        t = case["tokens"]
        stored = 2 * LATENT + 2 * ROPE if case["cache"] == "bf16" else LATENT + 4 + 2 * ROPE
        plain = 2 * (LATENT + ROPE)
        tables = 2 * 4 * ROPE
        moved = {"write": plain + tables + stored + 8, "read": stored + plain + 8,
                 "write_read": plain + tables + 2 * stored + plain + 8}[op]
        return {"bytes": t * moved, "flops": t * (6 * LATENT + 4 * ROPE)}
    if op in ("query", "output"):
        rows = case["batch"] * case["seq"] * case["heads"]
        weights = case["heads"] * NOPE * LATENT * 2
        row = 2 * (NOPE + ROPE) + 2 * (LATENT + ROPE) if op == "query" else 2 * LATENT + 2 * VDIM
        return {"bytes": rows * row + weights, "flops": 2 * rows * NOPE * LATENT}
    keys = int(_lens(case).sum())
    row = 2 * (LATENT + ROPE) if case["cache"] == "bf16" else LATENT + 4 + 2 * ROPE
    rows = case["batch"] * case["seq"] * case["heads"]
    return {"bytes": keys * row + rows * 2 * (LATENT + ROPE + LATENT),
            "flops": 2 * _pairs(case) * case["heads"] * (2 * LATENT + ROPE)}


# ---------------------------------------------------------------------------------------------------- inputs
def _normal(gen, *shape, std=1.0):
    return torch.randn(*shape, generator=gen, device="cuda") * std


def _tables(n):
    """cos / sin tables of the rotary embedding, angles in 64 bits."""
    freq = 10000.0 ** (-torch.arange(0, ROPE, 2, dtype=torch.float64, device="cuda") / ROPE)
    ang = torch.arange(n, dtype=torch.float64, device="cuda")[:, None] * freq
    ang = torch.cat([ang, ang], -1)
    return ang.cos().float(), ang.sin().float()


def _planes(case, gen, pages):
    """A cache holding normalised latent vectors and rotated keys."""
    page = case["page"]
    latent = _normal(gen, pages, page, LATENT)
    rope = _normal(gen, pages, page, ROPE).bfloat16()
    if case["cache"] == "bf16":
        return latent.bfloat16(), rope, None
    e = torch.frexp(latent.abs().amax(-1) / E4M3_MAX)
    scale = torch.ldexp(torch.ones_like(e.mantissa), e.exponent - (e.mantissa == 0.5).int())
    return (latent / scale[..., None]).to(torch.float8_e4m3fn), rope, scale


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op = case["op"]
    s = {"case": case}
    if op in ("write", "write_read", "read"):
        t = case["tokens"]
        pages = -(-t // case["page"]) + 3
        s["latent"], s["rope"], s["scale"] = _planes(case, gen, pages)
        s["slots"] = torch.randperm(pages * case["page"], generator=gen, device="cuda")[:t].view(1, t)
        if op != "read":
            both = _normal(gen, 1, t, LATENT + ROPE, std=1.3).bfloat16()
            s["kv"], s["pe"] = both[..., :LATENT], both[..., LATENT:]
            s["norm"] = (1 + 0.1 * _normal(gen, LATENT)).bfloat16()
            s["cos"], s["sin"] = _tables(8192)
            s["pos"] = torch.randint(0, 8192, (1, t), generator=gen, device="cuda")
    elif op in ("query", "output"):
        b, q, h = case["batch"], case["seq"], case["heads"]
        s["weight"] = _normal(gen, h * (NOPE + VDIM), LATENT, std=LATENT ** -0.5).bfloat16()
        if op == "query":
            s["q"] = _normal(gen, b, q, h, NOPE + ROPE).bfloat16()
            s["cos"], s["sin"] = _tables(8192)
            s["pos"] = torch.randint(0, 8192, (b, q), generator=gen, device="cuda")
        else:
            s["attn"] = _normal(gen, b, q, h, LATENT, std=0.3).bfloat16()
    else:
        b, q, h, page = case["batch"], case["seq"], case["heads"], case["page"]
        lens = _lens(case)
        need = -(-lens // page)
        pages = int(need.sum()) + 5
        s["latent"], s["rope"], s["scale"] = _planes(case, gen, pages)
        order = torch.randperm(pages, generator=gen, device="cuda").int()
        first = torch.from_numpy(np.cumsum(need) - need).cuda()
        column = torch.arange(int(need.max()), device="cuda")
        table = order[(first[:, None] + column).clamp(max=pages - 1)]
        s["table"] = torch.where(column < torch.from_numpy(need).cuda()[:, None], table, -1).int().contiguous()
        s["lens"] = torch.from_numpy(lens).cuda().int()
        s["query"] = _normal(gen, b, q, h, LATENT + ROPE).bfloat16()
        s["sm_scale"] = (NOPE + ROPE) ** -0.5
        s["tree"] = None
        if case["tree"]:
            # node 0 is the root; the parent of node j is an earlier node
            parent = (torch.rand(b, q, generator=gen, device="cuda") * torch.arange(q, device="cuda")).long()
            mask = torch.zeros(b, q, q, dtype=torch.bool, device="cuda")
            rows = torch.arange(b, device="cuda")
            mask[:, 0, 0] = True
            for j in range(1, q):
                mask[:, j] = mask[rows, parent[:, j]]
                mask[:, j, j] = True
            s["tree"] = mask
    if own:
        if PACKAGE not in sys.path:
            sys.path.insert(0, PACKAGE)
        from pithtrain_b200.operators.mla import LatentCache
        if "latent" in s:
            s["handle"] = LatentCache(s["latent"], s["rope"], s["scale"])
    return s


# ---------------------------------------------------------------------------------------------------- plain form
def _rotate(x, cos, sin):
    x = x.float()
    even, odd = x[..., 0::2], x[..., 1::2]
    half = ROPE // 2
    return torch.cat([even * cos[..., :half] - odd * sin[..., :half], odd * cos[..., half:] + even * sin[..., half:]], -1)


def _plain_write(s):
    x = s["kv"].float()
    c = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * s["norm"].float()
    r = _rotate(s["pe"], s["cos"][s["pos"]], s["sin"][s["pos"]])
    slots = s["slots"].reshape(-1)
    latent, rope = s["latent"].view(-1, LATENT), s["rope"].view(-1, ROPE)
    rope[slots] = r.view(-1, ROPE).bfloat16()
    c = c.view(-1, LATENT)
    if s["scale"] is None:
        latent[slots] = c.bfloat16()
        return
    e = torch.frexp(c.abs().amax(-1) / E4M3_MAX)
    scale = torch.ldexp(torch.ones_like(e.mantissa), e.exponent - (e.mantissa == 0.5).int())
    s["scale"].view(-1)[slots] = scale
    latent.view(torch.uint8)[slots] = (c / scale[:, None]).to(torch.float8_e4m3fn).view(torch.uint8)


def _plain_rows(s, slots):
    """Cached rows in 32 bits."""
    latent = s["latent"].view(-1, LATENT)
    if s["scale"] is None:
        c = latent[slots].float()
    else:
        c = latent.view(torch.uint8)[slots].view(torch.float8_e4m3fn).float() * s["scale"].view(-1)[slots][..., None]
    return c, s["rope"].view(-1, ROPE)[slots].float()


def _plain_attention(s):
    q = s["query"].float()
    b, t, h, _ = q.shape
    page = s["latent"].shape[1]
    n = torch.arange(s["table"].shape[1] * page, device="cuda")
    lens = s["lens"].long()
    slots = s["table"].long().repeat_interleave(page, 1) * page + n % page
    there = n < lens[:, None]
    c, r = _plain_rows(s, torch.where(there, slots, 0))
    c = torch.where(there[..., None], c, 0)
    first = lens - t
    i = torch.arange(t, device="cuda")
    if s["tree"] is None:
        seen = n <= (first[:, None] + i)[..., None]
    else:
        j = n - first[:, None]
        drafted = torch.gather(s["tree"], 2, j.clamp(0, t - 1)[:, None, :].expand(b, t, n.numel()))
        seen = (j < 0)[:, None, :] | drafted
    seen = (seen & there[:, None, :])[:, :, None, :].expand(b, t, h, n.numel()).reshape(b, t * h, n.numel())
    keys = torch.cat([c, r], -1)
    score = torch.matmul(q.view(b, t * h, LATENT + ROPE), keys.transpose(1, 2)) * s["sm_scale"]
    score = torch.where(seen, score, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, 0, top))
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, c) / torch.where(total == 0, 1, total)
    return out.view(b, t, h, LATENT).bfloat16()


def run(s):
    op = s["case"]["op"]
    if own:
        return _own(op, s)
    if op == "write":
        _plain_write(s)
        return s["latent"], s["rope"]
    if op in ("read", "write_read"):
        if op == "write_read":
            _plain_write(s)
        c, r = _plain_rows(s, s["slots"])
        return c.bfloat16(), r.bfloat16()
    if op == "query":
        q, h = s["q"].float(), s["case"]["heads"]
        w = s["weight"].float().view(h, NOPE + VDIM, LATENT)[:, :NOPE]
        cos, sin = s["cos"][s["pos"]][:, :, None], s["sin"][s["pos"]][:, :, None]
        folded = torch.matmul(q[..., :NOPE].transpose(1, 2), w).transpose(1, 2)
        return torch.cat([folded, _rotate(q[..., NOPE:], cos, sin)], -1).bfloat16()
    if op == "output":
        h = s["case"]["heads"]
        w = s["weight"].float().view(h, NOPE + VDIM, LATENT)[:, NOPE:]
        return torch.matmul(s["attn"].float().transpose(1, 2), w.transpose(1, 2)).transpose(1, 2).bfloat16()
    return _plain_attention(s)


# ---------------------------------------------------------------------------------------------------- own calls
def _own(op, s):
    from pithtrain_b200.operators import mla
    if op in ("write", "write_read"):
        mla.latent_cache_write(s["handle"], s["slots"], s["kv"], s["pe"], s["norm"], s["cos"], s["sin"], EPS,
                               position_ids=s["pos"])
        if op == "write":
            return s["latent"], s["rope"]
    if op in ("read", "write_read"):
        return mla.latent_cache_read(s["handle"], s["slots"])
    if op == "query":
        return mla.latent_query(s["q"], s["weight"], s["cos"], s["sin"], position_ids=s["pos"])
    if op == "output":
        return mla.latent_output(s["attn"], s["weight"])
    return mla.latent_attention(s["query"], s["handle"], s["table"], s["lens"], s["sm_scale"], tree_mask=s["tree"])


# ---------------------------------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]

    def turned(x, cos, sin):
        z = torch.complex(x[..., 0::2].double(), x[..., 1::2].double())
        z = z * torch.complex(cos[..., : ROPE // 2].double(), sin[..., : ROPE // 2].double())
        return torch.cat([z.real, z.imag], -1)

    def stored(slots):
        c = s["latent"].view(-1, LATENT)[slots].double() if s["scale"] is None else \
            s["latent"].view(torch.uint8).view(-1, LATENT)[slots].view(torch.float8_e4m3fn).double() \
            * s["scale"].view(-1)[slots].double()[..., None]
        return c, s["rope"].view(-1, ROPE)[slots].double()

    if op == "read":
        return stored(s["slots"])
    if op in ("write", "write_read"):
        x = s["kv"].double()
        c = x / torch.sqrt((x ** 2).sum(-1, keepdim=True) / LATENT + EPS) * s["norm"].double()
        r = turned(s["pe"], s["cos"][s["pos"]], s["sin"][s["pos"]])
        if op == "write":
            latent, rope = s["latent"].double(), s["rope"].double()
            latent.view(-1, LATENT)[s["slots"][0]] = c[0]
            rope.view(-1, ROPE)[s["slots"][0]] = r[0]
            return latent, rope
        return (None if case["cache"] == "e4m3" else c), r  # the value that an 8-bit rounding picks has no exact form
    if op in ("query", "output"):
        w = s["weight"].double().view(case["heads"], NOPE + VDIM, LATENT)
        if op == "output":
            return torch.einsum("bshr,hvr->bshv", s["attn"].double(), w[:, NOPE:])
        folded = torch.einsum("bshd,hdr->bshr", s["q"][..., :NOPE].double(), w[:, :NOPE])
        return torch.cat([folded, turned(s["q"][..., NOPE:], s["cos"][s["pos"]].unsqueeze(2),
                                         s["sin"][s["pos"]].unsqueeze(2))], -1)
    b, t, h, page = case["batch"], case["seq"], case["heads"], case["page"]
    out = torch.zeros(b, t, h, LATENT, dtype=torch.float64, device="cuda")
    for i, length in enumerate(_lens(case).tolist()):
        n = torch.arange(length, device="cuda")
        c, r = stored(s["table"][i].long()[n // page] * page + n % page)
        q = s["query"][i].double()
        for token in range(t):
            score = (q[token, :, :LATENT] @ c.T + q[token, :, LATENT:] @ r.T) * s["sm_scale"]
            if s["tree"] is None:
                hidden = n > length - t + token
            else:
                hidden = torch.zeros(length, dtype=torch.bool, device="cuda")
                hidden[length - t:] = ~s["tree"][i, token]
            out[i, token] = torch.softmax(score.masked_fill(hidden, -math.inf), -1) @ c
    return out
