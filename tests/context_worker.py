"""One PE of the sequence-sharded decode test (started by test_context_decode.py): the cache of a batch is spread over
the members, some of which hold nothing of a sequence; every member's result is the attention over all tokens."""
import os

import torch

import rocshmem_b200 as shm
from rocshmem_b200.ops import attention as at
from rocshmem_b200.parallel.context import ContextParallelDecode


def main() -> None:
    backend = os.environ.get("ROCSHMEM_TEST_BACKEND", "host")
    shm.init(heap_size="64M", backend=backend, timeout_s=60)
    me, n, dev = shm.my_pe(), shm.n_pes(), shm.device()
    g = torch.Generator().manual_seed(23)                       # everybody can rebuild the whole problem for the check
    B, H, K, D, P = 4, 6, 2, 64, 16
    lengths = [70, 1, 0, 129]
    used_before = shm.heap_info()["used"]
    step = ContextParallelDecode(B + 1, H, D)
    for case, (dtype, softcap) in enumerate([(torch.bfloat16, 0.0), (torch.float8_e4m3fn, 20.0)]):
        whole = at.KvCache.allocate(64, P, K, D, dtype, device="cpu")
        if dtype == torch.bfloat16:
            whole.k.copy_(torch.randn(whole.k.shape, generator=g))
            whole.v.copy_(torch.randn(whole.v.shape, generator=g))
        else:
            for codes, factors in ((whole.k, whole.k_scale), (whole.v, whole.v_scale)):
                codes.copy_((torch.randn(codes.shape, generator=g) * 100).clamp(-448, 448).to(dtype))
                factors.copy_(torch.rand(factors.shape, generator=g) / 100 + 1e-3)
        table = torch.randperm(64, generator=g)[:B * 9].view(B, 9).int()
        q = torch.randn(B, H, D, generator=g).to(torch.bfloat16)
        want, _ = at.ref_paged_attention(q, whole, table, torch.tensor(lengths, dtype=torch.int32), softcap=softcap)
        # Whole pages are dealt to the members in turn; a member's pages lie in a cache of its own.
        mine = at.KvCache.allocate(40, P, K, D, dtype, device=dev)
        own_table = torch.full((B, 9), -1, dtype=torch.int32)
        own_lengths = torch.zeros(B, dtype=torch.int32)
        used = 0
        for b, length in enumerate(lengths):
            held = [i for i in range((length + P - 1) // P) if (i + b) % n == me]
            for j, i in enumerate(held):
                for a, c in zip(whole._tensors(), mine._tensors()):
                    c[used] = a[int(table[b, i])].to(dev)
                own_table[b, j] = used
                used += 1
                own_lengths[b] += min(P, length - i * P)
        for _ in range(3):
            out = step(q.to(dev), mine, own_table.to(dev), own_lengths.to(dev), softcap=softcap)
            # One rounding to bf16 of the result, fp32 or better before it (on GPUs: sums of at most 129 rows).
            off = (out.cpu().double() - want).abs()
            assert (off <= want.abs() * 2.0 ** -8 + 2.0 ** -12).all(), float(off.max())
        assert out.shape == q.shape and out.dtype == q.dtype
        few = step(q[:1].to(dev), mine, own_table[:1].to(dev), own_lengths[:1].to(dev), softcap=softcap)
        assert torch.equal(few[0], out[0])
        assert step(q[:0].to(dev), mine, own_table[:0].to(dev), own_lengths[:0].to(dev)).shape == (0, H, D)
        seen = [torch.zeros_like(out.cpu()) for _ in range(n)]
        buf = shm.zeros((n,) + tuple(out.shape), torch.bfloat16)
        src = shm.zeros(tuple(out.shape), torch.bfloat16)
        src.copy_(out)
        if shm.is_cuda():
            torch.cuda.synchronize()
        from rocshmem_b200.ops import collectives as coll
        assert coll.fcollect(buf, src) == shm.SUCCESS
        seen = buf.cpu()
        assert all(torch.equal(seen[i], out.cpu()) for i in range(n)), "the same bits on every member"
        shm.free_all([buf, src])
    for bad in (torch.zeros(B + 2, H, D), torch.zeros(B, H + 1, D), torch.zeros(B, H, D + 8)):
        try:
            step(bad.to(torch.bfloat16).to(dev), mine, own_table.to(dev), own_lengths.to(dev))
            raise AssertionError("accepted a query of another shape")
        except ValueError:
            pass
    step.destroy()
    assert shm.heap_info()["used"] == used_before
    shm.barrier_all()
    shm.finalize()


if __name__ == "__main__":
    main()
