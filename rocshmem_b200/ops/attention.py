"""Operators around attention for training and serving: norms of query and key heads with the position rotation, a paged
cache that can quantise what is written into it, attention of one new token over that cache, and the join of partial
results of caches that lie on several PEs.

* :func:`qk_norm_rope`: RMS norm of every head and rotation by position in one pass, differentiable;
* :class:`KvCache`, :func:`kv_cache_write`, :func:`kv_cache_read`: pages of keys and values in 16 bits or as e4m3 with
  one fp32 factor for each token and head;
* :func:`paged_attention`: one new token for each sequence against its pages;
* :func:`attention_join`: partial results of parts of a cache made into one
  (:class:`rocshmem_b200.parallel.context.ContextParallelDecode` uses it over a team).

All tensors are CUDA tensors on one device. ``stream`` (a ``torch.cuda.Stream`` or a raw handle; the current stream by
default) is the stream that the kernels, new outputs and workspaces belong to; the caller orders it after the work that
made the inputs. No call synchronises, and every call can be captured into a CUDA graph. The reference has no
attention code; its nearest building blocks are the put and collective calls that move a sequence's parts
(``src/ipc/context_ipc_tmpl_device.hpp:282-359``).
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional, Tuple

import torch

from .. import _native
from .. import runtime as rt

E4M3 = torch.float8_e4m3fn
E4M3_MAX = 448.0


# ---- streams ---------------------------------------------------------------------------------------------------------

class _On:
    """Makes ``stream`` current on the device of ``tensors``, whose memory is kept until the stream is done with it."""

    def __init__(self, stream, *tensors):
        device = tensors[0].device
        if device.type != "cuda":
            raise ValueError("tensors must be on a CUDA device")
        if isinstance(stream, torch.cuda.Stream):
            if stream.device != device:
                raise ValueError(f"the stream is on {stream.device}, the tensors are on {device}")
            own = stream
        else:
            default = torch.cuda.default_stream(device)
            handle = int(stream)
            own = default if handle in (default.cuda_stream, 1) else torch.cuda.ExternalStream(handle, device=device)
        self._inner = torch.cuda.stream(own)
        if own.cuda_stream != torch.cuda.current_stream(device).cuda_stream:
            for t in tensors:
                if t is not None and t.is_cuda and t.numel():
                    t.record_stream(own)

    def __enter__(self):
        return self._inner.__enter__()

    def __exit__(self, *args):
        return self._inner.__exit__(*args)


# ---- norm and rotation -----------------------------------------------------------------------------------------------

def rope_table(num_positions: int, rotary_dim: int, base: float = 10000.0, device=None,
               frequencies: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The table ``[num_positions, rotary_dim]`` fp32 that :func:`qk_norm_rope` reads: row ``p`` holds the cosines and
    then the sines of ``p * frequency_i``, ``i < rotary_dim / 2``. ``frequencies`` (scaled ones, for instance) default
    to ``base ** (-2 i / rotary_dim)``. Angles are computed in 64 bits: those of far positions keep no digits in 32. The
    table lies on ``device``, by default where the frequencies do."""
    if rotary_dim % 2 or rotary_dim < 2 or num_positions < 1:
        raise ValueError("rope_table: rotary_dim must be even, num_positions positive")
    if frequencies is not None and device is None:
        device = frequencies.device
    if frequencies is None:
        frequencies = base ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64, device=device) / rotary_dim)
    if tuple(frequencies.shape) != (rotary_dim // 2,):
        raise ValueError(f"rope_table: frequencies must be [{rotary_dim // 2}]")
    angle = torch.arange(num_positions, dtype=torch.float64, device=device)[:, None] * frequencies.to(device).double()
    return torch.cat([angle.cos(), angle.sin()], dim=1).float()


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, q_weight: torch.Tensor, k_weight: torch.Tensor,
                 positions: torch.Tensor, table: torch.Tensor, eps: float = 1e-6, interleaved: bool = False,
                 stream=None) -> Tuple[torch.Tensor, torch.Tensor]:
    """RMS norm of every head of ``q [T, Hq, D]`` and ``k [T, Hk, D]`` with weights ``[D]``, then the rotation of the
    first ``R`` elements by the token's position, in one pass: ``(q', k')``, contiguous.

    bf16, fp16 or fp32; sums, norm and rotation in fp32, rounded once. ``D`` is a multiple of 8 up to 256. Rows may be
    strided (views of a fused projection) as long as each is contiguous and 16-byte aligned. The weights have the rows'
    type or fp32. ``table [positions, R]`` is :func:`rope_table`'s, ``R`` a multiple of 16. Pairs are ``(i, i + R /
    2)``, or with ``interleaved`` ``(2 i, 2 i + 1)``. ``positions [T]`` int32 or int64: a negative one marks padding,
    whose rows become zeros and have no gradient; one past the table makes its token's rows NaN.

    Differentiable once (``create_graph`` and forward-mode derivatives are refused) with respect to ``q``, ``k`` and
    both weights; the weights' gradients are the same in every run. A ``table`` that requires a gradient is refused. A
    backward pass can be captured into a CUDA graph with its forward pass; while an eager graph of the same leaves is
    alive, the captured forward pass is refused."""
    if stream is not None:
        with _On(stream, q, k, q_weight, k_weight, positions, table):
            return qk_norm_rope(q, k, q_weight, k_weight, positions, table, eps, interleaved)
    return _native.load_attention().qk_norm_rope(q, k, q_weight, k_weight, positions, table, eps, interleaved)


# ---- the paged cache -------------------------------------------------------------------------------------------------

@dataclass(frozen=True, eq=False)
class KvCache:
    """Keys and values of many sequences in pages: ``k``, ``v`` ``[pages, kv_heads, page_size, head_dim]`` in bf16, fp16
    or e4m3; for e4m3 with ``k_scale``, ``v_scale [pages, kv_heads, page_size]`` fp32, the factor of each row. The page
    size is a power of two. A token's slot is ``page * page_size + offset``."""
    k: torch.Tensor
    v: torch.Tensor
    k_scale: Optional[torch.Tensor] = None
    v_scale: Optional[torch.Tensor] = None

    def __post_init__(self):
        object.__setattr__(self, "_cache", _native.load_attention().Cache(self.k, self.v, self.k_scale, self.v_scale))

    def __reduce__(self):
        return KvCache, (self.k, self.v, self.k_scale, self.v_scale)

    @classmethod
    def allocate(cls, num_pages: int, page_size: int, kv_heads: int, head_dim: int, dtype: torch.dtype = torch.bfloat16,
                 device=None, symmetric: bool = False) -> "KvCache":
        """A cache of zeros on ``device`` (default: the current CUDA device). ``symmetric``: on the symmetric heap, so
        that other PEs can put pages into it (collective; give it back with :meth:`free`)."""
        shape = (num_pages, kv_heads, page_size, head_dim)
        if symmetric:
            def zeros(shape, dtype):
                return rt.zeros(shape, torch.uint8).view(dtype) if dtype == E4M3 else rt.zeros(shape, dtype)
        else:
            device = torch.device("cuda") if device is None else device

            def zeros(shape, dtype):
                return torch.zeros(shape, dtype=dtype, device=device)
        if dtype != E4M3:
            return cls(zeros(shape, dtype), zeros(shape, dtype))
        return cls(zeros(shape, dtype), zeros(shape, dtype), zeros(shape[:3], torch.float32),
                   zeros(shape[:3], torch.float32))

    def free(self) -> None:
        """Collective: give a symmetric cache's memory back to the heap."""
        if self.k.is_cuda:
            torch.cuda.synchronize(self.k.device)
        rt.free_all([t for t in (self.k, self.v, self.k_scale, self.v_scale) if t is not None])

    @property
    def num_pages(self) -> int:
        """Pages of the cache."""
        return self.k.shape[0]

    @property
    def page_size(self) -> int:
        """Tokens a page."""
        return self.k.shape[2]

    @property
    def kv_heads(self) -> int:
        """Key and value heads."""
        return self.k.shape[1]

    @property
    def head_dim(self) -> int:
        """Elements a head."""
        return self.k.shape[3]

    def _tensors(self):
        return (self.k, self.v) if self.k_scale is None else (self.k, self.v, self.k_scale, self.v_scale)


def token_slots(block_table: torch.Tensor, sequences: torch.Tensor, positions: torch.Tensor,
                page_size: int) -> torch.Tensor:
    """Slots (int64) of tokens: token ``i`` is position ``positions[i]`` of sequence ``sequences[i]``, whose pages are
    row ``sequences[i]`` of ``block_table``. -1 for a sequence that the table does not have, a negative position, one
    past the table or one without a page. Plain PyTorch, any device, no synchronisation."""
    at, row = positions.long(), sequences.long()
    if block_table.numel() == 0:
        return torch.full_like(at, -1)
    # Clamped, an index is one of the table's; where that changed it, there is no slot.
    at_in, row_in = at.clamp(0, block_table.shape[1] * page_size - 1), row.clamp(0, block_table.shape[0] - 1)
    page = block_table[row_in, at_in // page_size].long()
    return torch.where((at == at_in) & (row == row_in) & (page >= 0), page * page_size + at % page_size, -1)


def kv_cache_write(cache: KvCache, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, stream=None) -> None:
    """Writes ``k``, ``v [T, kv_heads, head_dim]`` (bf16, fp16 or fp32; rows may be strided as in :func:`qk_norm_rope`)
    into the slots ``[T]`` (int32 or int64). Slots outside the cache, negative ones among them, are skipped: padding.
    The others have to differ from one another. Neither the inputs nor the cache's own tensors may share memory with
    another tensor of the cache (a cache whose keys are its values can be read, but not written).

    A 16-bit cache takes the values rounded to its type. In an e4m3 cache a row with the largest magnitude ``m`` becomes
    codes ``x * 448 / m`` with the factor ``m / 448``; a row that holds a NaN or an infinity reads back as NaN."""
    if stream is not None:
        with _On(stream, k, v, slots, *cache._tensors()):
            return kv_cache_write(cache, k, v, slots)
    _native.load_attention().kv_cache_write(cache._cache, k, v, slots)


def kv_cache_read(cache: KvCache, slots: torch.Tensor, dtype: torch.dtype = torch.bfloat16,
                  stream=None) -> Tuple[torch.Tensor, torch.Tensor]:
    """The keys and values of slots ``[T]`` (int32 or int64), each ``[T, kv_heads, head_dim]`` in bf16, fp16 or fp32
    (codes times factors in fp32, rounded once). Slots outside the cache give zeros."""
    if stream is not None:
        with _On(stream, slots, *cache._tensors()):
            return kv_cache_read(cache, slots, dtype)
    return _native.load_attention().kv_cache_read(cache._cache, slots, dtype)


# ---- attention over the cache -------------------------------------------------------------------------------------

def paged_attention(q: torch.Tensor, cache: KvCache, block_table: torch.Tensor, lengths: torch.Tensor,
                    scale: Optional[float] = None, softcap: float = 0.0, window: int = 0,
                    out: Optional[torch.Tensor] = None, lse: Optional[torch.Tensor] = None, return_lse: bool = False,
                    stream=None):
    """Attention of one new token for each sequence: ``q [B, H, D]`` against the first ``lengths[b]`` tokens of sequence
    ``b``, which lie in the pages ``block_table[b]``. Returns ``out [B, H, D]``, with ``return_lse`` ``(out, lse)``.

    ``q`` is bf16 or fp16 and of the cache's type, or either for an e4m3 cache; ``D`` is 64, 96, 128 or 256; ``H`` a
    multiple of the cache's heads, whose groups share a key head. Scores are ``scale * q.k`` (default ``D ** -0.5``),
    with ``softcap`` > 0 ``softcap * tanh(scale * q.k / softcap)``; ``window`` > 0 leaves the last ``window`` tokens.
    ``scale`` and ``softcap`` lie between 1e-30 and 1e30.
    Sums and softmax are fp32. ``out`` may be given, in q's type or fp32, and ``lse [B, H]`` fp32, the natural logarithm
    of the sum of the scores' exponentials; neither may share memory with an input. ``block_table [B, pages]`` and
    ``lengths [B]`` are int32 on the device.

    The kernel is chosen by the block table's width (or the window), the most that the lengths on the device can be: a
    batch of short sequences, and a captured graph of one, is faster with the table cut to the pages that it can need
    (``block_table[:, :n]``): 4 sequences of up to 300 tokens 8.3 us on the device, with a table 16 or 256 times as wide
    10.3; 16 of up to 64 tokens 6.3 and 10.0.

    Sums are fp32 and hold up to 2^14 times a value: results are finite as long as the magnitudes of a sequence's values
    add up to less than 1e34.

    Lengths are taken between 0 and the table's end. Tokens in a page that is no page of the cache are not seen. A
    sequence that sees nothing has zeros and an lse of -inf. Rows that are not seen may hold anything, NaN included; an
    infinity or NaN in a row that is seen makes the results of its heads NaN, except a score of -inf, which counts for
    nothing."""
    if stream is not None:
        with _On(stream, q, block_table, lengths, *cache._tensors(), out, lse):
            return paged_attention(q, cache, block_table, lengths, scale, softcap, window, out, lse, return_lse)
    both = _native.load_attention().paged_attention(q, cache._cache, block_table, lengths, scale, softcap, window, out,
                                                    lse, return_lse)
    return both if return_lse else both[0]


def attention_join(outs: torch.Tensor, lses: torch.Tensor, dtype: Optional[torch.dtype] = None,
                   out: Optional[torch.Tensor] = None, stream=None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Joins attention results over disjoint parts of a cache: ``outs [n, B, H, D]`` (bf16, fp16 or fp32) with ``lses
    [n, B, H]`` fp32, as :func:`paged_attention` returns them for each part. Returns ``(out [B, H, D], lse [B, H])``:
    the parts' sum weighted by ``exp(lse)``. Every part must be contiguous; the parts may lie apart. ``dtype`` of the
    result defaults to that of ``out`` if given, else of ``outs``. A part with an lse of -inf does not count, whatever
    its ``outs`` hold."""
    if stream is not None:
        with _On(stream, outs, lses, out):
            return attention_join(outs, lses, dtype, out)
    return _native.load_attention().attention_join(outs, lses, dtype, out)


# ---- references (plain PyTorch, any device) -------------------------------------------------------------------------

def ref_norm_rope(x: torch.Tensor, weight: torch.Tensor, positions: torch.Tensor, table: torch.Tensor,
                  eps: float = 1e-6, interleaved: bool = False) -> torch.Tensor:
    """PyTorch reference of :func:`qk_norm_rope` for one of the two tensors, in 64 bits, differentiable."""
    R = table.shape[1]
    x = x.double()
    y = x * (x.square().mean(dim=-1, keepdim=True) + eps).rsqrt() * weight.double()
    at = positions.long().clamp(0, table.shape[0] - 1)
    c, s = (a[:, None] for a in table.double()[at].chunk(2, dim=1))
    if interleaved:
        a, b = y[..., 0:R:2], y[..., 1:R:2]
        turned = torch.stack([a * c - b * s, b * c + a * s], dim=-1).flatten(-2)
    else:
        a, b = y[..., :R // 2], y[..., R // 2:R]
        turned = torch.cat([a * c - b * s, b * c + a * s], dim=-1)
    y = torch.cat([turned, y[..., R:]], dim=-1)
    p = positions.long()[:, None, None]
    return torch.where(p < 0, 0.0, torch.where(p >= table.shape[0], float("nan"), y))


def ref_quantize_rows(x: torch.Tensor):
    """PyTorch reference of the cache's quantisation: ``(e4m3 codes, fp32 factors)`` of the last dimension's rows."""
    x = x.float()
    m = x.abs().amax(dim=-1)
    m = torch.where(m.isfinite(), m.clamp(min=2.0 ** -110), float("nan"))
    # A division by hand: `448.0 / m` is computed as the reciprocal times 448, two roundings instead of one.
    codes = (x * torch.div(torch.full_like(m, E4M3_MAX), m)[..., None]).clamp(-E4M3_MAX, E4M3_MAX).to(E4M3)
    return codes, m * (1.0 / E4M3_MAX)


def ref_paged_attention(q: torch.Tensor, cache: KvCache, block_table: torch.Tensor, lengths: torch.Tensor,
                        scale: Optional[float] = None, softcap: float = 0.0, window: int = 0):
    """PyTorch reference of :func:`paged_attention` in 64 bits, sequence by sequence: ``(out, lse)``. The CPU backend's
    form of the operator too."""
    _native.load_attention().check_paged(q, cache._cache, block_table, lengths, scale, softcap, window)
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    B, H, D = q.shape
    K, P = cache.kv_heads, cache.page_size
    out = torch.zeros((B, H, D), dtype=torch.float64, device=q.device)
    lse = torch.full((B, H), float("-inf"), dtype=torch.float64, device=q.device)
    for b, n in enumerate(lengths.tolist()):
        n = min(max(n, 0), block_table.shape[1] * P)
        pos = torch.arange(max(0, n - window) if window else 0, n, device=q.device)
        page = block_table[b, pos // P].long()
        seen = (page >= 0) & (page < cache.num_pages)
        page, offset = page[seen], (pos % P)[seen]
        if page.numel() == 0:
            continue

        def rows(x, factor):
            y = x.view(torch.uint8)[page, :, offset].view(x.dtype).float().double() if factor is not None else \
                x[page, :, offset].double()
            return y if factor is None else y * factor[page, :, offset].double()[..., None]

        k, v = rows(cache.k, cache.k_scale), rows(cache.v, cache.v_scale)   # [n, K, D]
        s = torch.einsum("kgd,nkd->kgn", q[b].double().view(K, H // K, D), k) * scale
        if softcap:
            s = softcap * torch.tanh(s / softcap)
        lse[b] = torch.logsumexp(s, dim=-1).view(H)
        out[b] = torch.einsum("kgn,nkd->kgd", torch.softmax(s, dim=-1), v).reshape(H, D)
    return out, lse


def ref_attention_join(outs: torch.Tensor, lses: torch.Tensor):
    """PyTorch reference of :func:`attention_join` in 64 bits. The CPU backend's form of the operator too."""
    l = lses.double()
    top = l.amax(dim=0)
    w = torch.exp(l - torch.where(top == float("-inf"), 0.0, top))
    total = w.sum(dim=0)
    out = torch.where(w[..., None] > 0, outs.double() * w[..., None], 0.0).sum(dim=0)
    out = out / torch.where(total > 0, total, 1.0)[..., None]
    return out, torch.where(total > 0, top + total.clamp(min=1e-300).log(), float("-inf"))
