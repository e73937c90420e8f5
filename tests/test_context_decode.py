"""Decoding over a cache that is spread over a team (rocshmem_b200.parallel.context): several processes on the CPU
backend, one process on a GPU, several GPUs where there are any."""
import os
import subprocess
import sys

import pytest
import torch

from mp_util import HERE, ROOT, assert_all_ok, free_port


def run(world, backend):
    port, procs = free_port(), []
    for rank in range(world):
        env = dict(os.environ, RANK=str(rank), WORLD_SIZE=str(world), LOCAL_RANK=str(rank), MASTER_ADDR="127.0.0.1",
                   MASTER_PORT=str(port), ROCSHMEM_TEST_BACKEND=backend, NCCL_NVLS_ENABLE="0",
                   PYTHONPATH=ROOT + os.pathsep + HERE + os.pathsep + os.environ.get("PYTHONPATH", ""))
        procs.append(subprocess.Popen([sys.executable, os.path.join(HERE, "context_worker.py")], env=env,
                                      stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True))
    results = []
    for p in procs:
        try:
            out, _ = p.communicate(timeout=240)
        except subprocess.TimeoutExpired:
            p.kill()
            out = p.communicate()[0] + "\n[killed: timeout]"
        results.append((p.returncode, out))
    assert_all_ok(results)


@pytest.mark.parametrize("world", [1, 2, 3])
def test_members_join_their_parts_on_the_cpu_backend(world):
    run(world, "host")


@pytest.mark.gpu
def test_one_member_on_a_gpu():
    run(1, "cuda")


@pytest.mark.gpu
@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs at least two GPUs")
def test_members_join_their_parts_on_gpus():
    run(2, "cuda")


@pytest.mark.gpu
def test_parts_in_one_buffer_join_to_the_whole():
    """What the members of a team of three do between the collectives, with one process's buffer in place of the
    gathered one: each part is written where the all-gather would put it."""
    from rocshmem_b200.ops import attention as at
    from rocshmem_b200.parallel.context import ContextParallelDecode
    step = ContextParallelDecode.__new__(ContextParallelDecode)
    step.heads, step.head_dim = 6, 96
    B, H, D, n = 3, 6, 96, 3
    g = torch.Generator(device="cuda").manual_seed(1)
    cache = at.KvCache.allocate(30, 32, 2, D, torch.bfloat16)
    cache.k.normal_(generator=g)
    cache.v.normal_(generator=g)
    table = torch.randperm(30, generator=g, device="cuda")[:B * 9].view(B, 9).int()
    lengths = torch.tensor([250, 3 * 32, 20], dtype=torch.int32, device="cuda")
    q = torch.randn(B, H, D, generator=g, device="cuda").to(torch.bfloat16)
    gathered = torch.full((n * step._words(B) + 5,), float("nan"), device="cuda")
    assert step._words(B) % 4 == 0 and step._words(B) >= B * H * (D + 1)
    outs, lses = step._views(gathered, n, B)
    for p in range(n):
        own = (lengths - p * 3 * 32).clamp(0, 3 * 32)
        at.paged_attention(q, cache, table[:, 3 * p:3 * p + 3], own, out=outs[p], lse=lses[p])
    out, lse = at.attention_join(outs, lses, dtype=torch.bfloat16)
    want, want_lse = at.ref_paged_attention(q, cache, table, lengths)
    # One rounding to bf16; probabilities in two bf16 parts, 2^-16 of the values' magnitudes (at most 5), and fp32 sums.
    assert ((out.double() - want).abs() <= want.abs() * 2.0 ** -8 + 5 * 2.0 ** -12).all()
    # A score is a sum of 96 products in fp32 (2^-23 each), at most |q| |k| / sqrt(96) = 14 x 14 / 9.8 in all.
    assert ((lse.double() - want_lse).abs() <= 96 * 2.0 ** -23 * 20).all()
    assert gathered[-5:].isnan().all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float8_e4m3fn])
def test_cache_on_the_symmetric_heap(fresh_runtime, dtype):
    from rocshmem_b200.ops import attention as at
    shm = fresh_runtime
    shm.init(n_local=1, heap_size="256M", device=0)
    used = shm.heap_info()["used"]
    cache = at.KvCache.allocate(8, 16, 2, 64, dtype, symmetric=True)
    assert shm.is_symmetric(cache.k) and shm.is_symmetric(cache.v) and (dtype == torch.bfloat16 or shm.is_symmetric(cache.k_scale))
    g = torch.Generator(device="cuda").manual_seed(1)
    k, v = (torch.randn(100, 2, 64, generator=g, device="cuda").to(torch.bfloat16) for _ in range(2))
    slots = torch.arange(100, device="cuda")
    at.kv_cache_write(cache, k, v, slots)
    plain = at.KvCache.allocate(8, 16, 2, 64, dtype)
    at.kv_cache_write(plain, k, v, slots)
    for a, b in zip(at.kv_cache_read(cache, slots), at.kv_cache_read(plain, slots)):
        assert torch.equal(a, b)
    q = torch.randn(2, 4, 64, generator=g, device="cuda").to(torch.bfloat16)
    table = torch.arange(8, device="cuda", dtype=torch.int32).view(2, 4)
    lengths = torch.tensor([64, 30], dtype=torch.int32, device="cuda")
    assert torch.equal(at.paged_attention(q, cache, table, lengths), at.paged_attention(q, plain, table, lengths))
    cache.free()
    assert shm.heap_info()["used"] == used
