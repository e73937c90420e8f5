"""Decoding with a cache that is spread over a team: the counterpart, for one new token, of the sequence-sharded
prefill of :mod:`rocshmem_b200.parallel.ring`.

Every member keeps the keys and values of some of a sequence's tokens (after ring attention, those of its own part of
the prompt; the new tokens go to any one member) in a paged cache of its own. For a step every member computes the
attention of the same queries over its tokens, the partial results and their log-sum-exps are gathered, and every member
joins them:

    step = ContextParallelDecode(max_batch=64, heads=32, head_dim=128)
    out = step(q, cache, block_table, lengths)      # cache, block_table and lengths: this member's part

The reference has no attention code; the exchange is its all-gather (``fcollect``,
``src/ipc/context_ipc_tmpl_device.hpp:503-531``). On GPUs a step is one attention call, one all-gather kernel and one
join on the current stream; on the CPU backend the same in plain PyTorch over the host-blocking all-gather. """
from __future__ import annotations

from typing import Optional

import torch
import torch.autograd.forward_ad as fwd

from .. import runtime as rt
from ..ops import attention
from ..ops import collectives as coll


class ContextParallelDecode:
    """Symmetric buffers for the partial results of one (team, batch, heads) combination; collective to create, to call
    and to destroy. A team of one needs none and calls :func:`rocshmem_b200.ops.attention.paged_attention` directly."""

    def __init__(self, max_batch: int, heads: int, head_dim: int, team: Optional[rt.Team] = None):
        if rt.n_local_pes() != 1:
            raise RuntimeError("ContextParallelDecode needs one PE per process")
        if max_batch < 1 or heads < 1:
            raise ValueError("max_batch and heads must be positive")
        self.team = team or rt.team_world()
        self.n, self.max_batch, self.heads, self.head_dim = self.team.n_pes(), max_batch, heads, head_dim
        self.mine = self.all = None
        if self.n > 1:
            words = self._words(max_batch)
            self.mine = rt.zeros(words, torch.float32)
            self.all = rt.zeros(self.n * words, torch.float32)

    def destroy(self) -> None:
        """Collective: give the buffers back to the heap."""
        if self.mine is not None:
            if rt.is_cuda():
                torch.cuda.synchronize()
            rt.free_all([self.mine, self.all])
        self.mine = self.all = None

    def _words(self, batch: int) -> int:
        """fp32 words of a member's partial result: the outputs, their log-sum-exps, whole 16 bytes."""
        words = batch * self.heads * (self.head_dim + 1)
        return words + -words % 4

    def _views(self, words: torch.Tensor, parts: int, batch: int):
        """The outputs ``[parts, batch, heads, head_dim]`` and log-sum-exps ``[parts, batch, heads]`` in a buffer."""
        rows = batch * self.heads
        blocks = words[:parts * self._words(batch)].view(parts, -1)
        return (blocks[:, :rows * self.head_dim].view(parts, batch, self.heads, self.head_dim),
                blocks[:, rows * self.head_dim:rows * (self.head_dim + 1)].view(parts, batch, self.heads))

    def __call__(self, q: torch.Tensor, cache: attention.KvCache, block_table: torch.Tensor, lengths: torch.Tensor,
                 scale: Optional[float] = None, softcap: float = 0.0) -> torch.Tensor:
        """``q [B, heads, head_dim]``, the same on every member; ``cache``, ``block_table [B, pages]`` and ``lengths
        [B]`` describe this member's part and may be empty (a length of zero). Returns the attention over all members'
        tokens ``[B, heads, head_dim]`` in q's type, the same bits on every member. Arguments as in
        :func:`rocshmem_b200.ops.attention.paged_attention`. There is no sliding window: a member does not know which
        positions of the whole sequence its tokens have, and a block table can leave out whole pages only, while a
        window's edge mostly lies inside one. A ``q`` with a derivative is refused."""
        if q.dim() != 3 or q.shape[1:] != (self.heads, self.head_dim) or q.shape[0] > self.max_batch:
            raise ValueError(f"q must be [batch <= {self.max_batch}, {self.heads}, {self.head_dim}], "
                             f"got {tuple(q.shape)}")
        if q.shape[0] == 0:
            return torch.empty_like(q)
        cuda = rt.is_cuda()
        if not cuda:
            # What paged_attention refuses on GPUs; the reference that stands in for it would let autograd into the
            # symmetric buffers.
            if torch.is_grad_enabled() and q.requires_grad:
                raise ValueError("ContextParallelDecode has no backward pass: call it under torch.no_grad(), or detach "
                                 "q")
            if fwd.unpack_dual(q).tangent is not None:
                raise ValueError("ContextParallelDecode has no forward-mode derivative: pass the primal of q")
        if self.n == 1:
            if cuda:
                return attention.paged_attention(q, cache, block_table, lengths, scale=scale, softcap=softcap)
            out = attention.ref_paged_attention(q, cache, block_table, lengths, scale=scale, softcap=softcap)[0]
            return out.to(q.dtype)
        if self.mine is None:
            raise RuntimeError("ContextParallelDecode was destroyed")
        B = q.shape[0]
        words = self._words(B)
        out, lse = (t[0] for t in self._views(self.mine, 1, B))
        mine, everyone = self.mine[:words], self.all[:self.n * words]
        if cuda:
            attention.paged_attention(q, cache, block_table, lengths, scale=scale, softcap=softcap, out=out, lse=lse)
            # The collective's entry barrier keeps a member's parts from being overwritten while it still joins them.
            coll.fcollect_async(everyone, mine, team=self.team)
            return attention.attention_join(*self._views(everyone, self.n, B), dtype=q.dtype)[0]
        o, l = attention.ref_paged_attention(q, cache, block_table, lengths, scale=scale, softcap=softcap)
        out.copy_(o)
        lse.copy_(l)
        if coll.fcollect(everyone, mine, self.team) != rt.SUCCESS:
            raise RuntimeError("all-gather of the partial results failed")
        joined = attention.ref_attention_join(*self._views(everyone, self.n, B))[0].to(q.dtype)
        if self.team.sync() != rt.SUCCESS:   # nobody gathers anew while a member still reads its parts
            raise RuntimeError("synchronisation after the join failed")
        return joined
