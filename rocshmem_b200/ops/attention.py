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

from .. import runtime as rt

E4M3 = torch.float8_e4m3fn
E4M3_MAX = 448.0
# Codes of the native launchers (attention_kernels.hpp).
_CODE = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2, E4M3: 3}
_HALF = (torch.bfloat16, torch.float16)
_FLOAT = (torch.bfloat16, torch.float16, torch.float32)
HEAD_DIMS = (64, 96, 128, 256)


# ---- arguments, devices and streams ---------------------------------------------------------------------------------

def _rows(t: torch.Tensor, name: str, heads: Optional[int] = None, dim: Optional[int] = None):
    """Strides of dimensions 0 and 1 of ``t [tokens, heads, dim]``, whose rows the kernels read 16 bytes at a time."""
    if t.dim() != 3 or (heads is not None and t.shape[1] != heads) or (dim is not None and t.shape[2] != dim):
        raise ValueError(f"{name} must be [tokens, {heads or 'heads'}, {dim or 'dim'}], got {tuple(t.shape)}")
    s0, s1, s2 = t.stride()
    vec = 16 // t.element_size()
    n0, n1, _ = t.shape
    s0, s1 = (s0 if n0 > 1 else 0), (s1 if n1 > 1 else 0)
    if s2 != 1 or s0 % vec or s1 % vec or t.data_ptr() % 16:
        raise ValueError(f"{name}: rows must be contiguous and 16-byte aligned (strides {tuple(t.stride())})")
    return s0, s1


def _index(t: torch.Tensor, name: str, count: int) -> int:
    """1 for 64-bit, 0 for 32-bit whole numbers."""
    if t.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"{name} must be int32 or int64")
    if tuple(t.shape) != (count,) or not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous [{count}]")
    return 1 if t.dtype == torch.int64 else 0


def _no_grad(what: str, *tensors) -> None:
    if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
        raise ValueError(f"{what} has no backward pass: call it under torch.no_grad(), or detach its inputs")


def _on_one_device(what: str, *tensors) -> torch.device:
    device = tensors[0].device
    if device.type != "cuda":
        raise ValueError(f"{what}: tensors must be on a CUDA device")
    for t in tensors:
        if t is not None and t.device != device:
            raise ValueError(f"{what}: tensors are on {device} and {t.device}")
    return device


class _Place:
    """Makes `device` and `stream` current, and keeps the inputs' memory until the stream is done with it."""

    def __init__(self, stream, device: torch.device, tensors):
        if stream is None:
            self._inner = torch.cuda.device(device)
            return
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
                if t is not None and t.numel():
                    t.record_stream(own)

    def __enter__(self):
        return self._inner.__enter__()

    def __exit__(self, *args):
        return self._inner.__exit__(*args)


def _elsewhere(stream, device: torch.device) -> bool:
    return stream is not None or torch.cuda.current_device() != device.index


def _here() -> int:
    return torch.cuda.current_stream().cuda_stream


# ---- norm and rotation ------------------------------------------------------------------------------------------------

def rope_table(num_positions: int, rotary_dim: int, base: float = 10000.0, device=None,
               frequencies: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The table ``[num_positions, rotary_dim]`` fp32 that :func:`qk_norm_rope` reads: row ``p`` holds the cosines and
    then the sines of ``p * frequency_i``, ``i < rotary_dim / 2``. ``frequencies`` (scaled ones, for instance) default
    to ``base ** (-2 i / rotary_dim)``. Angles are computed in 64 bits: those of far positions keep no digits in 32."""
    if rotary_dim % 2 or rotary_dim < 2 or num_positions < 1:
        raise ValueError("rope_table: rotary_dim must be even, num_positions positive")
    if frequencies is None:
        frequencies = base ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64, device=device) / rotary_dim)
    if tuple(frequencies.shape) != (rotary_dim // 2,):
        raise ValueError(f"rope_table: frequencies must be [{rotary_dim // 2}]")
    angle = torch.arange(num_positions, dtype=torch.float64, device=device)[:, None] * frequencies.to(device).double()
    return torch.cat([angle.cos(), angle.sin()], dim=1).float()


def _norm_rope_args(q, k, q_weight, k_weight, positions, table, eps, interleaved, strides, wide):
    return (q.data_ptr(), k.data_ptr(), *strides, q_weight.data_ptr(), k_weight.data_ptr(), positions.data_ptr(),
            table.data_ptr(), q.shape[0], q.shape[1], k.shape[1], q.shape[2], table.shape[1], table.shape[0], eps,
            int(interleaved), _CODE[q.dtype], _CODE[q_weight.dtype], wide)


def _norm_rope(args, q, k) -> Tuple[torch.Tensor, torch.Tensor]:
    q_out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    k_out = torch.empty(k.shape, dtype=k.dtype, device=k.device)
    rt._C().qk_norm_rope(args, q_out.data_ptr(), k_out.data_ptr(), _here())
    return q_out, k_out


class _NormRope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, positions, table, eps, interleaved, strides, wide):
        ctx.save_for_backward(q, k, q_weight, k_weight, positions, table)
        ctx.options = (eps, interleaved, strides, wide)
        return _norm_rope(_norm_rope_args(q, k, q_weight, k_weight, positions, table, *ctx.options), q, k)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, gq, gk):
        q, k, q_weight, k_weight, positions, table = ctx.saved_tensors
        # Gradients come in any layout (an expanded one behind a sum, for instance); the kernel reads plain rows.
        gq, gk = (g.contiguous() if g.data_ptr() % 16 == 0 else g.clone(memory_format=torch.contiguous_format)
                  for g in (gq, gk))
        dq, dk = torch.empty(q.shape, dtype=q.dtype, device=q.device), torch.empty(k.shape, dtype=k.dtype, device=k.device)
        dwq, dwk = torch.empty_like(q_weight), torch.empty_like(k_weight)
        C = rt._C()
        workspace = torch.empty(C.qk_norm_rope_workspace(q.shape[2]), dtype=torch.float32, device=q.device)
        C.qk_norm_rope_backward(_norm_rope_args(q, k, q_weight, k_weight, positions, table, *ctx.options),
                                gq.data_ptr(), gk.data_ptr(), dq.data_ptr(), dk.data_ptr(), dwq.data_ptr(), dwk.data_ptr(),
                                workspace.data_ptr(), _here())
        return dq, dk, dwq, dwk, None, None, None, None, None, None


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, q_weight: torch.Tensor, k_weight: torch.Tensor,
                 positions: torch.Tensor, table: torch.Tensor, eps: float = 1e-6, interleaved: bool = False,
                 stream=None) -> Tuple[torch.Tensor, torch.Tensor]:
    """RMS norm of every head of ``q [T, Hq, D]`` and ``k [T, Hk, D]`` with weights ``[D]``, then the rotation of the
    first ``R`` elements by the token's position, in one pass: ``(q', k')``, contiguous.

    bf16, fp16 or fp32; sums, norm and rotation in fp32, rounded once. ``D`` is a multiple of 8 up to 256. Rows may be
    strided (views of a fused projection) as long as each is contiguous and 16-byte aligned. The weights have the rows'
    type or fp32. ``table [positions, R]`` is :func:`rope_table`'s, ``R`` a multiple of 16. Pairs are ``(i, i + R / 2)``, or with ``interleaved``
    ``(2 i, 2 i + 1)``. ``positions [T]`` int32 or int64: a negative one marks padding, whose rows become zeros and have no
    gradient; one past the table makes its token's rows NaN.

    Differentiable once with respect to ``q``, ``k`` and both weights; the weights' gradients are the same in every run."""
    if q.dtype not in _FLOAT or k.dtype != q.dtype:
        raise TypeError(f"q and k must both be bf16, fp16 or fp32, got {q.dtype} and {k.dtype}")
    q_strides = _rows(q, "q")
    T, Hq, D = q.shape
    k_strides = _rows(k, "k", dim=D)
    if k.shape[0] != T or Hq < 1 or k.shape[1] < 1:
        raise ValueError(f"q and k must have the same tokens and at least one head, got {tuple(q.shape)} and {tuple(k.shape)}")
    if D % 8 or not 8 <= D <= 256:
        raise ValueError(f"the head dimension must be a multiple of 8 up to 256, got {D}")
    for w, name in ((q_weight, "q_weight"), (k_weight, "k_weight")):
        if w.dtype not in (q.dtype, torch.float32) or w.dtype != q_weight.dtype:
            raise TypeError(f"{name} must be {q.dtype} or fp32, both weights the same")
        if tuple(w.shape) != (D,) or not w.is_contiguous() or w.data_ptr() % 16:
            raise ValueError(f"{name} must be contiguous [{D}], 16-byte aligned")
    if table.dtype != torch.float32 or table.dim() != 2 or not table.is_contiguous() or table.data_ptr() % 16:
        raise ValueError("table must be contiguous fp32 [positions, rotary], 16-byte aligned")
    R = table.shape[1]
    if R % 16 or not 16 <= R <= D or table.shape[0] < 1:
        raise ValueError(f"the table's rows must have a multiple of 16 elements up to {D}, got {tuple(table.shape)}")
    wide = _index(positions, "positions", T)
    inputs = (q, k, q_weight, k_weight, positions, table)
    device = _on_one_device("qk_norm_rope", *inputs)

    def call():
        options = (float(eps), bool(interleaved), q_strides + k_strides, wide)
        if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or q_weight.requires_grad or k_weight.requires_grad):
            return _NormRope.apply(*inputs, *options)
        return _norm_rope(_norm_rope_args(*inputs, *options), q, k)

    if _elsewhere(stream, device):
        with _Place(stream, device, inputs):
            return call()
    return call()


# ---- the paged cache --------------------------------------------------------------------------------------------------

@dataclass(frozen=True)
class KvCache:
    """Keys and values of many sequences in pages: ``k``, ``v`` ``[pages, kv_heads, page_size, head_dim]`` in bf16, fp16
    or e4m3; for e4m3 with ``k_scale``, ``v_scale [pages, kv_heads, page_size]`` fp32, the factor of each row. The page
    size is a power of two. A token's slot is ``page * page_size + offset``."""
    k: torch.Tensor
    v: torch.Tensor
    k_scale: Optional[torch.Tensor] = None
    v_scale: Optional[torch.Tensor] = None

    def __post_init__(self):
        k, v = self.k, self.v
        shape = k.shape
        if k.dim() != 4 or v.shape != shape or k.dtype != v.dtype or k.dtype not in (*_HALF, E4M3):
            raise ValueError("KvCache: k and v must both be [pages, kv_heads, page_size, head_dim] in bf16, fp16 or e4m3")
        if shape[2] & (shape[2] - 1) or not 1 <= shape[2] <= 1 << 20:
            raise ValueError(f"KvCache: the page size must be a power of two up to 2^20, got {shape[2]}")
        if shape[1] < 1 or shape[3] % 8 or not 8 <= shape[3] <= 256:
            raise ValueError("KvCache: at least one head, head_dim a multiple of 8 up to 256")
        if k.dtype == E4M3:
            tensors = (k, v, self.k_scale, self.v_scale)
            for s in tensors[2:]:
                if s is None or s.dtype != torch.float32 or s.shape != shape[:3]:
                    raise ValueError("KvCache: e4m3 needs k_scale and v_scale, fp32 [pages, kv_heads, page_size]")
        else:
            tensors = (k, v)
            if self.k_scale is not None or self.v_scale is not None:
                raise ValueError("KvCache: only e4m3 caches have scales")
        for t in tensors:
            if not t.is_contiguous() or t.data_ptr() % 16 or t.device != k.device:
                raise ValueError("KvCache: tensors must be contiguous, 16-byte aligned and on one device")

    @classmethod
    def allocate(cls, num_pages: int, page_size: int, kv_heads: int, head_dim: int, dtype: torch.dtype = torch.bfloat16,
                 device=None, symmetric: bool = False) -> "KvCache":
        """A cache of zeros on ``device`` (default: the current CUDA device). ``symmetric``: on the symmetric heap, so that
        other PEs can put pages into it (collective; give it back with :meth:`free`)."""
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
        return cls(zeros(shape, dtype), zeros(shape, dtype), zeros(shape[:3], torch.float32), zeros(shape[:3], torch.float32))

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

    def _args(self):
        k = self.k
        pages, heads, size, dim = k.shape
        scales = (0, 0) if self.k_scale is None else (self.k_scale.data_ptr(), self.v_scale.data_ptr())
        return (k.data_ptr(), self.v.data_ptr(), *scales, pages, heads, size.bit_length() - 1, dim, _CODE[k.dtype])


def token_slots(block_table: torch.Tensor, sequences: torch.Tensor, positions: torch.Tensor, page_size: int) -> torch.Tensor:
    """Slots (int64) of tokens: token ``i`` is position ``positions[i]`` of sequence ``sequences[i]``, whose pages are row
    ``sequences[i]`` of ``block_table``. -1 for a negative position, one past the table or one without a page. Plain PyTorch,
    any device, no synchronisation."""
    at = positions.long()
    known = (at >= 0) & (at < block_table.shape[1] * page_size)
    if block_table.shape[1] == 0:
        return torch.full_like(at, -1)
    page = block_table[sequences.long(), torch.where(known, at, 0) // page_size].long()
    return torch.where(known & (page >= 0), page * page_size + at % page_size, -1)


def kv_cache_write(cache: KvCache, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, stream=None) -> None:
    """Writes ``k``, ``v [T, kv_heads, head_dim]`` (bf16, fp16 or fp32; rows may be strided as in :func:`qk_norm_rope`) into
    the slots ``[T]`` (int32 or int64). Slots outside the cache, negative ones among them, are skipped: padding. The
    others have to differ from one another.

    A 16-bit cache takes the values rounded to its type. In an e4m3 cache a row with the largest magnitude ``m`` becomes
    codes ``x * 448 / m`` with the factor ``m / 448``; a row that holds a NaN or an infinity reads back as NaN."""
    if k.dtype not in _FLOAT or v.dtype != k.dtype:
        raise TypeError(f"k and v must both be bf16, fp16 or fp32, got {k.dtype} and {v.dtype}")
    strides = _rows(k, "k", cache.kv_heads, cache.head_dim) + _rows(v, "v", cache.kv_heads, cache.head_dim)
    if v.shape[0] != k.shape[0]:
        raise ValueError(f"k and v must have the same tokens, got {k.shape[0]} and {v.shape[0]}")
    wide = _index(slots, "slots", k.shape[0])
    _no_grad("kv_cache_write", k, v)
    inputs = (k, v, slots, *cache._tensors())
    device = _on_one_device("kv_cache_write", *inputs)

    def call():
        rt._C().kv_cache_write(cache._args(), k.data_ptr(), v.data_ptr(), *strides, slots.data_ptr(), wide, k.shape[0],
                               _CODE[k.dtype], _here())

    if _elsewhere(stream, device):
        with _Place(stream, device, inputs):
            return call()
    return call()


def kv_cache_read(cache: KvCache, slots: torch.Tensor, dtype: torch.dtype = torch.bfloat16,
                  stream=None) -> Tuple[torch.Tensor, torch.Tensor]:
    """The keys and values of slots ``[T]`` (int32 or int64), each ``[T, kv_heads, head_dim]`` in bf16, fp16 or fp32 (codes
    times factors in fp32, rounded once). Slots outside the cache give zeros."""
    if dtype not in _FLOAT:
        raise TypeError(f"dtype must be bf16, fp16 or fp32, got {dtype}")
    if slots.dim() != 1:
        raise ValueError("slots must be [T]")
    T = slots.shape[0]
    wide = _index(slots, "slots", T)
    inputs = (slots, *cache._tensors())
    device = _on_one_device("kv_cache_read", *inputs)

    def call():
        k = torch.empty((T, cache.kv_heads, cache.head_dim), dtype=dtype, device=device)
        v = torch.empty_like(k)
        rt._C().kv_cache_read(cache._args(), k.data_ptr(), v.data_ptr(), slots.data_ptr(), wide, T, _CODE[dtype], _here())
        return k, v

    if _elsewhere(stream, device):
        with _Place(stream, device, inputs):
            return call()
    return call()


# ---- attention over the cache -------------------------------------------------------------------------------------

def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether the address ranges of two tensors meet."""
    def span(t):
        last = sum((n - 1) * s for n, s in zip(t.shape, t.stride()))
        return t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size()
    if a.numel() == 0 or b.numel() == 0:
        return False
    (a0, a1), (b0, b1) = span(a), span(b)
    return a0 < b1 and b0 < a1


def _result(t: torch.Tensor, name: str, shape, dtypes, inputs) -> None:
    if tuple(t.shape) != shape or t.dtype not in dtypes or not t.is_contiguous() or t.data_ptr() % 16:
        raise ValueError(f"{name} must be a contiguous, 16-byte aligned {list(shape)} tensor of {' or '.join(map(str, dtypes))}")
    if any(_overlap(t, x) for x in inputs if x is not None):
        raise ValueError(f"{name} shares memory with an input")


def _check_paged(q, cache, block_table, lengths, scale, softcap, window):
    """Checks what does not depend on a device; returns q's strides."""
    if q.dtype not in _HALF or (cache.k.dtype != E4M3 and cache.k.dtype != q.dtype):
        raise TypeError(f"q must be bf16 or fp16, and of the cache's type unless that is e4m3: got {q.dtype} and {cache.k.dtype}")
    strides = _rows(q, "q", dim=cache.head_dim)
    B, H, D = q.shape
    if H < 1 or H % cache.kv_heads:
        raise ValueError(f"the {H} query heads must be a multiple of the cache's {cache.kv_heads}")
    if D not in HEAD_DIMS:
        raise ValueError(f"paged_attention: the head dimension must be one of {HEAD_DIMS}, got {D}")
    if block_table.dtype != torch.int32 or lengths.dtype != torch.int32:
        raise TypeError("block_table and lengths must be int32")
    if block_table.dim() != 2 or block_table.shape[0] != B or (block_table.shape[1] > 1 and block_table.stride(1) != 1):
        raise ValueError(f"block_table must be [{B}, pages] with contiguous rows")
    if tuple(lengths.shape) != (B,) or not lengths.is_contiguous():
        raise ValueError(f"lengths must be contiguous [{B}]")
    if not scale > 0 or softcap < 0 or window < 0 or window != int(window):
        raise ValueError("scale must be positive, softcap and window not negative")
    return strides


def paged_attention(q: torch.Tensor, cache: KvCache, block_table: torch.Tensor, lengths: torch.Tensor,
                    scale: Optional[float] = None, softcap: float = 0.0, window: int = 0,
                    out: Optional[torch.Tensor] = None, lse: Optional[torch.Tensor] = None, return_lse: bool = False,
                    stream=None):
    """Attention of one new token for each sequence: ``q [B, H, D]`` against the first ``lengths[b]`` tokens of sequence
    ``b``, which lie in the pages ``block_table[b]``. Returns ``out [B, H, D]``, with ``return_lse`` ``(out, lse)``.

    ``q`` is bf16 or fp16 and of the cache's type, or either for an e4m3 cache; ``D`` is 64, 96, 128 or 256; ``H`` a multiple of the cache's
    heads, whose groups share a key head. Scores are ``scale * q.k`` (default ``D ** -0.5``), with ``softcap`` > 0
    ``softcap * tanh(scale * q.k / softcap)``; ``window`` > 0 leaves the last ``window`` tokens. Sums and softmax are fp32. ``out`` may be given,
    in q's type or fp32, and ``lse [B, H]`` fp32, the natural logarithm of the sum of the scores' exponentials; neither may share
    memory with an input. ``block_table [B, pages]`` and ``lengths [B]`` are int32 on the device.

    Lengths are taken between 0 and the table's end. Tokens in a page that is no page of the cache are not seen. A sequence that sees
    nothing has zeros and an lse of -inf. Rows that are not seen may hold anything, NaN included."""
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    strides = _check_paged(q, cache, block_table, lengths, scale, softcap, window)
    B, H, D = q.shape
    inputs = (q, block_table, lengths, *cache._tensors())
    if out is not None:
        _result(out, "out", (B, H, D), (q.dtype, torch.float32), (*inputs, lse))
    if lse is not None:
        _result(lse, "lse", (B, H), (torch.float32,), inputs)
    _no_grad("paged_attention", q)
    device = _on_one_device("paged_attention", *inputs, out, lse)

    def call():
        o = torch.empty((B, H, D), dtype=q.dtype, device=device) if out is None else out
        s = torch.empty((B, H), dtype=torch.float32, device=device) if lse is None and return_lse else lse
        C = rt._C()
        args = cache._args()
        size = C.paged_attention_workspace(args, B, H)
        workspace = torch.empty(size, dtype=torch.uint8, device=device)
        C.paged_attention(args, q.data_ptr(), *strides, block_table.data_ptr(), block_table.stride(0), lengths.data_ptr(),
                          B, H, block_table.shape[1], int(window), scale, softcap, _CODE[q.dtype], _CODE[o.dtype],
                          o.data_ptr(), 0 if s is None else s.data_ptr(), workspace.data_ptr(), size, _here())
        return (o, s) if return_lse else o

    if _elsewhere(stream, device):
        with _Place(stream, device, (*inputs, out, lse)):
            return call()
    return call()


def attention_join(outs: torch.Tensor, lses: torch.Tensor, dtype: Optional[torch.dtype] = None,
                   out: Optional[torch.Tensor] = None, stream=None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Joins attention results over disjoint parts of a cache: ``outs [n, B, H, D]`` (bf16, fp16 or fp32) with ``lses
    [n, B, H]`` fp32, as :func:`paged_attention` returns them for each part. Returns ``(out [B, H, D], lse [B, H])``: the parts'
    sum weighted by ``exp(lse)``. Every part must be contiguous; the parts may lie apart. ``dtype`` of the result defaults to that
    of ``out`` if given, else of ``outs``. A part with an lse of -inf does not count, whatever its ``outs`` hold."""
    if outs.dtype not in _FLOAT or lses.dtype != torch.float32:
        raise TypeError("outs must be bf16, fp16 or fp32, lses fp32")
    if outs.dim() != 4 or tuple(lses.shape) != tuple(outs.shape[:3]) or outs.shape[0] < 1:
        raise ValueError(f"outs must be [n, B, H, D] and lses [n, B, H], got {tuple(outs.shape)} and {tuple(lses.shape)}")
    n, B, H, D = outs.shape
    if D % 8 or not 8 <= D <= 256:
        raise ValueError(f"the head dimension must be a multiple of 8 up to 256, got {D}")
    if not outs[0].is_contiguous() or not lses[0].is_contiguous():
        raise ValueError("attention_join: every part must be contiguous")
    if outs.data_ptr() % 16 or (n > 1 and outs.stride(0) * outs.element_size() % 16):
        raise ValueError("attention_join: every part of outs must be 16-byte aligned")
    dtype = (outs.dtype if out is None else out.dtype) if dtype is None else dtype
    if dtype not in _FLOAT:
        raise TypeError(f"dtype must be bf16, fp16 or fp32, got {dtype}")
    if out is not None:
        _result(out, "out", (B, H, D), (dtype,), (outs, lses))
    _no_grad("attention_join", outs, lses)
    device = _on_one_device("attention_join", outs, lses, out)

    def call():
        o = torch.empty((B, H, D), dtype=dtype, device=device) if out is None else out
        lse = torch.empty((B, H), dtype=torch.float32, device=device)
        rt._C().attention_join(outs.data_ptr(), lses.data_ptr(), outs.stride(0), lses.stride(0), n, B * H, D,
                               _CODE[outs.dtype], _CODE[dtype], o.data_ptr(), lse.data_ptr(), _here())
        return o, lse

    if _elsewhere(stream, device):
        with _Place(stream, device, (outs, lses, out)):
            return call()
    return call()


# ---- references (plain PyTorch, any device) -------------------------------------------------------------------------

def ref_norm_rope(x: torch.Tensor, weight: torch.Tensor, positions: torch.Tensor, table: torch.Tensor, eps: float = 1e-6,
                  interleaved: bool = False) -> torch.Tensor:
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
    """PyTorch reference of :func:`paged_attention` in 64 bits, sequence by sequence: ``(out, lse)``. The CPU backend's form
    of the operator too."""
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    _check_paged(q, cache, block_table, lengths, scale, softcap, window)
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
    out = torch.where(w[..., None] > 0, outs.double() * w[..., None], 0.0).sum(dim=0) / torch.where(total > 0, total, 1.0)[..., None]
    return out, torch.where(total > 0, top + total.clamp(min=1e-300).log(), float("-inf"))
