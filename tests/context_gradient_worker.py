"""One PE of the test that decoding over a team refuses queries with a derivative (started by
test_context_arguments.py)."""
import torch
import torch.autograd.forward_ad as fwd

import rocshmem_b200 as shm
from rocshmem_b200.ops import attention as at
from rocshmem_b200.parallel.context import ContextParallelDecode


def main() -> None:
    shm.init(heap_size="16M", backend="host", timeout_s=60)
    step = ContextParallelDecode(2, 4, 64)
    g = torch.Generator().manual_seed(7 + shm.my_pe())
    cache = at.KvCache.allocate(4, 16, 2, 64, torch.bfloat16, device="cpu")
    cache.k.copy_(torch.randn(cache.k.shape, generator=g))
    cache.v.copy_(torch.randn(cache.v.shape, generator=g))
    args = (cache, torch.tensor([[0, 1], [2, 3]], dtype=torch.int32), torch.tensor([20, 5], dtype=torch.int32))
    q = torch.randn(2, 4, 64, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)
    want = step(q, *args)

    def refused(x, match):
        try:
            step(x, *args)
        except ValueError as e:
            assert match in str(e), e
        else:
            raise AssertionError(f"accepted a query with a derivative ({match})")

    refused(q.clone().requires_grad_(), "no backward pass")
    with fwd.dual_level():
        refused(fwd.make_dual(q.clone(), torch.ones_like(q)), "no forward-mode derivative")
        assert torch.equal(step(q, *args), want)
    with torch.no_grad():
        assert torch.equal(step(q.clone().requires_grad_(), *args), want)
    # The buffers are nobody's result: a call after the refusals is what it was before them.
    again = step(q, *args)
    assert torch.equal(again, want) and not again.requires_grad
    assert step.mine is None or not (step.mine.requires_grad or step.all.requires_grad)
    step.destroy()
    shm.barrier_all()
    shm.finalize()


if __name__ == "__main__":
    main()
