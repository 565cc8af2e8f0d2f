"""Sampling from an MLA layer: a paged cache of the shared latent vectors, and attention in the absorbed form over it.

The training path expands every token's 512-wide latent vector into keys and values of all heads
(``kv_b_proj``, pithtrain/models/deepseek_v2_lite.py:426-454) and attends to those (``MLA``). Token by token that would
recompute or store ``16 * (192 + 128)`` values a token. Here a token costs 512 + 64: its normalised latent vector ``c``
and the rotated key ``r`` that all heads share. With ``W_k[h] [128, 512]`` and ``W_v[h] [128, 512]`` the two halves of
head h's block of ``kv_b_proj.weight``,

    q_nope . (W_k c) = (q_nope W_k) . c        and        sum_n p_n W_v c_n = W_v (sum_n p_n c_n),

so the query takes ``W_k`` in, attention runs on the latent vectors themselves, and its result goes through ``W_v``.

These operators have no gradients (training keeps the expanded form): under grad mode, inputs that require one are
refused, and so are tangents of forward-mode differentiation. Sizes are DeepSeek-V2-Lite's (latent 512, rope 64, nope
128, v 128), any number of heads; bf16, CUDA only. Indices are read on the device, so a slot, page, position or length
out of range cannot raise at the call: nothing outside the tensors is touched, the error is recorded, and later kernels
of the library skip their work, so that their outputs hold nothing. A later call of these or the attention operators
raises as soon as the news has reached the host (about ten milliseconds; not while a graph is being captured, and
replays do not look); ``pithtrain_b200.kernels.check_device_status()`` waits and raises at once. A sampling loop calls
it where it fetches its tokens.
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch
from torch.autograd import forward_ad

from ... import _lib, kernels

_is_compiling = torch.compiler.is_compiling


def _refuse_gradients(what: str, *inputs) -> None:
    """Raises where one of the inputs (tensors or None) wants a gradient: backward under grad mode, or forward mode. The operators
    come here only if there may be one: as a loop over all inputs it costs an eager call half a microsecond."""
    if torch.is_grad_enabled():
        for t in inputs:
            if t is not None and t.requires_grad:
                raise RuntimeError(f"{what} has no gradient: call it under torch.no_grad()")
    if forward_ad._current_level >= 0:
        for t in inputs:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise RuntimeError(f"{what} has no gradient: forward-mode differentiation would lose a tangent here")


class LatentCache:
    """Planes of a paged latent cache: ``latent`` [pages, page_size, 512] (bfloat16 or float8_e4m3fn), ``rope``
    [pages, page_size, 64] bfloat16, and for float8_e4m3fn ``scale`` [pages, page_size] float32 (a row's values are
    stored * scale; scales are not negative, and attention takes those below 2^-100, which ``latent_cache_write`` does not
    store, as 2^-100). A slot is ``page * page_size + row``. ``page_size`` is 16, 32 or a multiple of 64; planes may be
    strided (a layer of a larger tensor) as long as rows are contiguous. The planes' memory may move between calls (a storage
    released and taken back, ``set_``, ``.data``): every call looks where they are. Where they stay, shapes and strides do too.
    """

    def __init__(self, latent: torch.Tensor, rope: torch.Tensor, scale: torch.Tensor | None = None):
        self._planes = (latent, rope, scale)
        self._flat = None
        self._check()

    def _check(self) -> None:
        latent, rope, scale = self._planes
        if latent.dtype not in (torch.bfloat16, torch.float8_e4m3fn) or rope.dtype != torch.bfloat16:
            raise TypeError("latent must be bfloat16 or float8_e4m3fn, rope bfloat16")
        if latent.dim() != 3 or latent.shape[2] != 512 or latent.stride(2) != 1:
            raise ValueError(f"latent must be [pages, page_size, 512] with a contiguous last dimension, got "
                             f"{tuple(latent.shape)}")
        pages, page_size, _ = latent.shape
        if pages < 1 or not (page_size in (16, 32) or (page_size > 0 and page_size % 64 == 0)):
            raise ValueError(f"page_size must be 16, 32 or a multiple of 64, got {pages} pages of {page_size}")
        if pages * page_size >= 2 ** 31:
            raise ValueError(f"{pages} pages of {page_size} rows: a cache holds at most 2^31 - 1 rows")
        if tuple(rope.shape) != (pages, page_size, 64) or rope.stride(2) != 1:
            raise ValueError(f"rope must be {(pages, page_size, 64)} with a contiguous last dimension, got "
                             f"{tuple(rope.shape)}")
        if (scale is None) != (latent.dtype == torch.bfloat16):
            raise ValueError("an 8-bit cache has a scale plane, a bfloat16 cache has none")
        if scale is not None and (scale.dtype != torch.float32 or tuple(scale.shape) != (pages, page_size)):
            raise ValueError(f"scale must be float32 {(pages, page_size)}")
        for name, t in (("rope", rope), ("scale", scale)):
            if t is not None and t.device != latent.device:
                raise ValueError(f"{name} is on {t.device}, latent on {latent.device}")

    @property
    def flat(self) -> tuple:
        """The fields of ``pith_latent_cache``, in order, of the planes as they are now."""
        latent, rope, scale = self._planes
        flat = self._flat
        if flat is None or latent.data_ptr() != flat[0] or rope.data_ptr() != flat[1] \
                or scale is not None and scale.data_ptr() != flat[2]:  # the first call, or a plane has moved
            self._check()
            for t in self._planes:
                if t is not None:
                    end = t.storage_offset() + 1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride()))
                    if t.untyped_storage().nbytes() < end * t.element_size():
                        raise RuntimeError("the memory of a plane of the latent cache has been released")
            flat = self._flat = (latent.data_ptr(), rope.data_ptr(), 0 if scale is None else scale.data_ptr(),
                                 _lib.DTYPE_BF16 if scale is None else _lib.DTYPE_E4M3, *latent.shape[:2],
                                 *latent.stride()[:2], *rope.stride()[:2], *(scale.stride() if scale is not None else (0, 0)))
        return flat

    @classmethod
    def allocate(cls, num_pages: int, page_size: int = 64, dtype: torch.dtype = torch.bfloat16, device="cuda"):
        """A cache of zeroed planes; ``dtype`` bfloat16 (1152 bytes a token) or float8_e4m3fn (644)."""
        scale = torch.ones((num_pages, page_size), dtype=torch.float32, device=device) \
            if dtype == torch.float8_e4m3fn else None
        return cls(torch.zeros((num_pages, page_size, 512), dtype=dtype, device=device),
                   torch.zeros((num_pages, page_size, 64), dtype=torch.bfloat16, device=device), scale)

    @property
    def latent(self) -> torch.Tensor:
        return self._planes[0]

    @property
    def rope(self) -> torch.Tensor:
        return self._planes[1]

    @property
    def scale(self) -> torch.Tensor | None:
        return self._planes[2]

    @property
    def requires_grad(self) -> bool:
        latent, rope, scale = self._planes
        return latent.requires_grad or rope.requires_grad or (scale is not None and scale.requires_grad)

    @property
    def num_pages(self) -> int:
        return self.latent.shape[0]

    @property
    def page_size(self) -> int:
        return self.latent.shape[1]


# What a traced call becomes (``torch.compile``): ``torch.library`` custom ops with fake kernels, as the library's other CP = 1
# operators. An eager call goes to the kernels directly; through an op it would cost the host several times as much.
@torch.library.custom_op("pithtrain_b200::latent_cache_write", mutates_args=("latent", "rope", "scale"))
def latent_cache_write_op(latent: torch.Tensor, rope: torch.Tensor, scale: Optional[torch.Tensor], slots: torch.Tensor,
                          compressed_kv: torch.Tensor, k_pe: torch.Tensor, norm_weight: torch.Tensor, cos: torch.Tensor,
                          sin: torch.Tensor, eps: float, position_ids: Optional[torch.Tensor]) -> None:
    kernels.latent_write(LatentCache(latent, rope, scale), slots, compressed_kv, k_pe, norm_weight, cos, sin, eps, position_ids)


@latent_cache_write_op.register_fake
def _(latent, rope, scale, slots, compressed_kv, k_pe, norm_weight, cos, sin, eps, position_ids):
    return None


@torch.library.custom_op("pithtrain_b200::latent_cache_read", mutates_args=())
def latent_cache_read_op(latent: torch.Tensor, rope: torch.Tensor, scale: Optional[torch.Tensor],
                         slots: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    return kernels.latent_read(LatentCache(latent, rope, scale), slots)


@latent_cache_read_op.register_fake
def _(latent, rope, scale, slots):
    return rope.new_empty((*slots.shape, 512)), rope.new_empty((*slots.shape, 64))


@torch.library.custom_op("pithtrain_b200::latent_attention", mutates_args=())
def latent_attention_op(query: torch.Tensor, latent: torch.Tensor, rope: torch.Tensor, scale: Optional[torch.Tensor],
                        block_table: torch.Tensor, seq_lens: torch.Tensor, softmax_scale: float,
                        query_lens: Optional[torch.Tensor], tree_mask: Optional[torch.Tensor],
                        return_lse: bool) -> Tuple[torch.Tensor, torch.Tensor]:
    """(out, lse); an empty tensor in the place of an LSE that was not asked for."""
    out, lse = kernels.latent_attn(query, LatentCache(latent, rope, scale), block_table, seq_lens, softmax_scale, query_lens,
                                   tree_mask, return_lse)
    return out, lse if return_lse else query.new_empty(0, dtype=torch.float32)


@latent_attention_op.register_fake
def _(query, latent, rope, scale, block_table, seq_lens, softmax_scale, query_lens, tree_mask, return_lse):
    b, s, h, _ = query.shape
    return query.new_empty((b, s, h, 512)), query.new_empty((b, h, s) if return_lse else 0, dtype=torch.float32)


@torch.library.custom_op("pithtrain_b200::latent_query", mutates_args=())
def latent_query_op(q: torch.Tensor, kv_b_weight: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
                    position_ids: Optional[torch.Tensor]) -> torch.Tensor:
    return kernels.latent_query(q, kv_b_weight, cos, sin, position_ids)


@latent_query_op.register_fake
def _(q, kv_b_weight, cos, sin, position_ids):
    return q.new_empty((*q.shape[:3], 576))


@torch.library.custom_op("pithtrain_b200::latent_output", mutates_args=())
def latent_output_op(attn: torch.Tensor, kv_b_weight: torch.Tensor) -> torch.Tensor:
    return kernels.latent_output(attn, kv_b_weight)


@latent_output_op.register_fake
def _(attn, kv_b_weight):
    return attn.new_empty((*attn.shape[:3], 128))


def latent_cache_write(cache: LatentCache, slots: torch.Tensor, compressed_kv: torch.Tensor, k_pe: torch.Tensor,
                       norm_weight: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, eps: float,
                       position_ids: torch.Tensor | None = None) -> None:
    """Normalises (RMSNorm), rotates and stores new tokens: compressed_kv ``[B,S,512]`` and k_pe ``[B,S,64]`` or
    ``[B,S,1,64]`` bf16 are the two parts of ``kv_a_proj_with_mqa``'s output (views are fine), ``norm_weight`` / ``eps``
    those of ``kv_a_layernorm``; slots int64 ``[B,S]``, negative for tokens that are not to be stored. The slots of one
    call have to differ, as the indices of ``torch.Tensor.index_put_``.

    cos / sin (bf16 or fp32): tables ``[rows, 64]`` with ``position_ids`` int64 ``[B or 1, S]``, or ``[B or 1, S, 64]``
    already gathered. fp32 arithmetic, one rounding to the cache's type; an 8-bit row gets the least power of two as its
    scale with which no value passes 448.
    """
    if torch.is_grad_enabled() and (compressed_kv.requires_grad or k_pe.requires_grad or norm_weight.requires_grad or
                                    cos.requires_grad or sin.requires_grad or cache.requires_grad) \
            or forward_ad._current_level >= 0:
        _refuse_gradients("latent_cache_write", compressed_kv, k_pe, norm_weight, cos, sin, *cache._planes)
    if _is_compiling():
        latent_cache_write_op(*cache._planes, slots, compressed_kv, k_pe, norm_weight, cos, sin, eps, position_ids)
    else:
        kernels.latent_write(cache, slots, compressed_kv, k_pe, norm_weight, cos, sin, eps, position_ids)


def latent_cache_read(cache: LatentCache, slots: torch.Tensor):
    """Rows of the cache as bf16, ``(latent [*slots.shape, 512], k_pe [*slots.shape, 64])``: what the expanded form of a
    prompt's next chunk takes for its cached prefix (``kv_b_proj(latent)``; ``k_pe`` is rotated already). Negative slots
    give zeros. Rows that ``latent_cache_write`` stored in 8 bits are exact in bf16."""
    if torch.is_grad_enabled() and cache.requires_grad or forward_ad._current_level >= 0:
        _refuse_gradients("latent_cache_read", *cache._planes)
    if _is_compiling():
        return latent_cache_read_op(*cache._planes, slots)
    return kernels.latent_read(cache, slots)


def latent_attention(query: torch.Tensor, cache: LatentCache, block_table: torch.Tensor, seq_lens: torch.Tensor,
                     softmax_scale: float, *, query_lens: torch.Tensor | None = None,
                     tree_mask: torch.Tensor | None = None, return_lse: bool = False):
    """Attention of new tokens over the cached latent vectors, absorbed form: query ``[B,S,H,576]`` bf16
    (``latent_query``; strided views are fine) -> ``[B,S,H,512]`` bf16, the weighted means of the latent vectors, for
    ``latent_output``. The new tokens' own rows have been written to the cache before.

    * ``block_table`` int32 ``[B, pages]``: the pages of each sequence in order; entries behind its last key are not read.
    * ``seq_lens`` int32 ``[B]``: keys of a sequence, its new tokens included. 0 is a sequence without keys.
    * ``query_lens`` int32 ``[B]``: how many of the S tokens a sequence has (a padded batch); default all. Rows behind
      them give 0.
    * default mask: causal, the new tokens being the last ones of the sequence. ``tree_mask`` bool ``[B,S,S]``: new token i
      sees the whole prefix and the new tokens j with ``tree_mask[b, i, j]`` (a tree of drafted tokens: its ancestors
      and itself).
    * ``return_lse``: also the log2-domain LSE, fp32 ``[B,H,S]`` (-inf for a row that sees no key), the convention of
      this library's other operators.

    Lengths and tables are read on the device: the call can be captured once and replayed with other contents. Results repeat bit
    for bit for the same inputs. They depend on the other sequences of the batch through where a context is cut for the SMs:
    softmax weights are rounded relative to a running maximum of each part, to 8 significant bits (half a step: 2^-8 of a weight),
    in an 8-bit cache to steps of 2^-17 of the largest at least, upwards or downwards key by key so that sums are kept. Row sums
    and the LSE take the weights unrounded, in fp32.
    """
    if torch.is_grad_enabled() and (query.requires_grad or cache.requires_grad) or forward_ad._current_level >= 0:
        _refuse_gradients("latent_attention", query, *cache._planes)
    if _is_compiling():
        out, lse = latent_attention_op(query, *cache._planes, block_table, seq_lens, softmax_scale, query_lens, tree_mask,
                                       return_lse)
    else:
        out, lse = kernels.latent_attn(query, cache, block_table, seq_lens, softmax_scale, query_lens, tree_mask, return_lse)
    return (out, lse) if return_lse else out


def latent_query(q: torch.Tensor, kv_b_weight: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
                 position_ids: torch.Tensor | None = None) -> torch.Tensor:
    """The query that ``latent_attention`` takes: q ``[B,S,H,192]`` = ``[q_nope | q_pe]`` bf16 (the projection output,
    viewed per head; strided views are fine if they begin and step in multiples of 16 bytes and repeat nothing) ->
    ``[B,S,H,576]`` bf16, ``q_nope`` times head h's key rows of
    ``kv_b_weight`` ``[H * 256, 512]`` (``kv_b_proj.weight`` as it is), and ``q_pe`` rotated as the cached keys.
    cos / sin / position_ids as in ``latent_cache_write``."""
    if torch.is_grad_enabled() and (q.requires_grad or kv_b_weight.requires_grad or cos.requires_grad or sin.requires_grad) \
            or forward_ad._current_level >= 0:
        _refuse_gradients("latent_query", q, kv_b_weight, cos, sin)
    if _is_compiling():
        return latent_query_op(q, kv_b_weight, cos, sin, position_ids)
    return kernels.latent_query(q, kv_b_weight, cos, sin, position_ids)


def latent_output(attn: torch.Tensor, kv_b_weight: torch.Tensor) -> torch.Tensor:
    """``latent_attention``'s result ``[B,S,H,512]`` times head h's value rows of ``kv_b_weight``: ``[B,S,H,128]`` bf16,
    contiguous, which the layer views as ``[B,S,H * 128]`` for ``o_proj``."""
    if torch.is_grad_enabled() and (attn.requires_grad or kv_b_weight.requires_grad) or forward_ad._current_level >= 0:
        _refuse_gradients("latent_output", attn, kv_b_weight)
    if _is_compiling():
        return latent_output_op(attn, kv_b_weight)
    return kernels.latent_output(attn, kv_b_weight)
