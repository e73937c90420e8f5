"""Attention operators without a GPU: refusals of bad arguments (all are made before anything touches a device), the
arithmetic of the split over blocks, helpers and references in plain PyTorch, the sequence-sharded decode over the CPU
backend."""
import os
import shutil
import subprocess

import pytest
import torch

from rocshmem_b200.ops import attention as at

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BF16, F16, F32, E4M3 = torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_split_over_blocks_and_rows_of_pages(tmp_path):
    exe = tmp_path / "plan"
    subprocess.run(["g++", "-std=c++17", "-O1", "-g", "-Wall", "-Werror", "-fsanitize=address,undefined",
                    "-fno-sanitize-recover=all", "-I", os.path.join(ROOT, "rocshmem_b200", "csrc"),
                    os.path.join(ROOT, "tests", "cpp", "attention_plan_unit.cpp"), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0 and out.stdout.strip() == "ok", out.stderr


def norm_rope_args(**over):
    a = dict(q=torch.zeros(3, 4, 64, dtype=BF16), k=torch.zeros(3, 2, 64, dtype=BF16),
        q_weight=torch.ones(64, dtype=BF16),
             k_weight=torch.ones(64, dtype=BF16), positions=torch.zeros(3, dtype=torch.int32), table=torch.zeros(8, 64))
    a.update(over)
    return a


@pytest.mark.parametrize("over,error,match", [
    (dict(q=torch.zeros(3, 4, 64, dtype=torch.float64)), TypeError, "bf16, fp16 or fp32"),
    (dict(k=torch.zeros(3, 2, 64, dtype=F16)), TypeError, "bf16, fp16 or fp32"),
    (dict(q=torch.zeros(3, 4 * 64, dtype=BF16)), ValueError, "q must be"),
    (dict(k=torch.zeros(3, 2, 32, dtype=BF16)), ValueError, "k must be"),
    (dict(k=torch.zeros(2, 2, 64, dtype=BF16)), ValueError, "same tokens"),
    (dict(q=torch.zeros(3, 4, 128, dtype=BF16)[..., ::2]), ValueError, "rows must be contiguous"),
    (dict(q=torch.zeros(3 * 4 * 64 + 1, dtype=BF16)[1:].view(3, 4, 64)), ValueError, "16-byte aligned"),
    (dict(q=torch.zeros(3, 4, 65, dtype=BF16)[..., :64]), ValueError, "16-byte aligned"),
    (dict(q_weight=torch.ones(64, dtype=F16)), TypeError, "q_weight"),
    (dict(k_weight=torch.ones(64, dtype=F32)), TypeError, "k_weight"),
    (dict(k_weight=torch.ones(32, dtype=BF16)), ValueError, "k_weight"),
    (dict(positions=torch.zeros(3)), TypeError, "positions"),
    (dict(positions=torch.zeros(4, dtype=torch.int32)), ValueError, "positions"),
    (dict(table=torch.zeros(8, 64, dtype=BF16)), ValueError, "table"),
    (dict(table=torch.zeros(8, 128)), ValueError, "multiple of 16"),
    (dict(table=torch.zeros(8, 24)), ValueError, "multiple of 16"),
    (dict(table=torch.zeros(0, 64)), ValueError, "multiple of 16"),
    (dict(), ValueError, "CUDA device"),
])
def test_norm_rope_refusals(over, error, match):
    with pytest.raises(error, match=match):
        at.qk_norm_rope(**norm_rope_args(**over))


def test_norm_rope_refuses_odd_head_dimensions():
    for d in (4, 36, 264):
        with pytest.raises(ValueError):
            at.qk_norm_rope(**norm_rope_args(q=torch.zeros(3, 4, d), k=torch.zeros(3, 2, d), q_weight=torch.ones(d),
                                             k_weight=torch.ones(d)))


def kv(dtype=BF16, pages=4, heads=2, size=16, dim=64):
    return at.KvCache.allocate(pages, size, heads, dim, dtype, device="cpu")


@pytest.mark.parametrize("make", [
    lambda: at.KvCache(torch.zeros(4, 2, 16, 64), torch.zeros(4, 2, 16, 64)),
    lambda: at.KvCache(torch.zeros(4, 2, 16, 64, dtype=BF16), torch.zeros(4, 2, 16, 64, dtype=F16)),
    lambda: at.KvCache(torch.zeros(4, 2, 16, 64, dtype=BF16), torch.zeros(4, 2, 16, 32, dtype=BF16)),
    lambda: at.KvCache(torch.zeros(2, 16, 64, dtype=BF16), torch.zeros(2, 16, 64, dtype=BF16)),
    lambda: kv(size=24),
    lambda: kv(dim=60),
    lambda: kv(dim=264),
    lambda: at.KvCache(torch.zeros(4, 2, 16, 64).to(E4M3), torch.zeros(4, 2, 16, 64).to(E4M3)),
    lambda: at.KvCache(torch.zeros(4, 2, 16, 64).to(E4M3), torch.zeros(4, 2, 16, 64).to(E4M3), torch.ones(4, 2, 8),
        torch.ones(4, 2, 16)),
    lambda: at.KvCache(torch.zeros(4, 2, 16, 64, dtype=BF16), torch.zeros(4, 2, 16, 64, dtype=BF16),
        torch.ones(4, 2, 16), None),
    lambda: at.KvCache(torch.zeros(4, 2, 64, 16, dtype=BF16).transpose(2, 3), torch.zeros(4, 2, 16, 64, dtype=BF16)),
])
def test_cache_refusals(make):
    with pytest.raises(ValueError, match="KvCache"):
        make()


def test_cache_shape_properties_and_frozen():
    c = kv(E4M3, pages=5, heads=3, size=32, dim=96)
    assert (c.num_pages, c.kv_heads, c.page_size, c.head_dim) == (5, 3, 32, 96)
    assert c.k_scale.shape == (5, 3, 32)
    with pytest.raises(Exception):
        c.k = c.v


@pytest.mark.parametrize("over,error,match", [
    (dict(k=torch.zeros(3, 2, 64, dtype=torch.float64)), TypeError, "bf16, fp16 or fp32"),
    (dict(v=torch.zeros(3, 2, 64, dtype=F16)), TypeError, "bf16, fp16 or fp32"),
    (dict(k=torch.zeros(3, 3, 64, dtype=BF16)), ValueError, "k must be"),
    (dict(v=torch.zeros(3, 2, 32, dtype=BF16)), ValueError, "v must be"),
    (dict(v=torch.zeros(2, 2, 64, dtype=BF16)), ValueError, "same tokens"),
    (dict(slots=torch.zeros(3)), TypeError, "slots"),
    (dict(slots=torch.zeros(2, dtype=torch.int64)), ValueError, "slots"),
    (dict(slots=torch.zeros(6, dtype=torch.int64)[::2]), ValueError, "slots"),
    (dict(k=torch.zeros(3, 2, 64, dtype=BF16, requires_grad=True)), ValueError, "no backward"),
    (dict(), ValueError, "CUDA device"),
])
def test_write_refusals(over, error, match):
    a = dict(k=torch.zeros(3, 2, 64, dtype=BF16), v=torch.zeros(3, 2, 64, dtype=BF16),
        slots=torch.zeros(3, dtype=torch.int64))
    a.update(over)
    with pytest.raises(error, match=match):
        at.kv_cache_write(kv(), **a)


def test_read_refusals():
    with pytest.raises(TypeError, match="dtype"):
        at.kv_cache_read(kv(), torch.zeros(3, dtype=torch.int64), dtype=torch.float64)
    with pytest.raises(TypeError, match="slots"):
        at.kv_cache_read(kv(), torch.zeros(3))
    with pytest.raises(ValueError, match="slots"):
        at.kv_cache_read(kv(), torch.zeros(3, 1, dtype=torch.int64))
    with pytest.raises(ValueError, match="CUDA device"):
        at.kv_cache_read(kv(), torch.zeros(3, dtype=torch.int64))


def paged_args(cache=None, **over):
    a = dict(q=torch.zeros(2, 4, 64, dtype=BF16), cache=cache or kv(), block_table=torch.zeros(2, 2, dtype=torch.int32),
             lengths=torch.zeros(2, dtype=torch.int32))
    a.update(over)
    return a


@pytest.mark.parametrize("over,error,match", [
    (dict(q=torch.zeros(2, 4, 64)), TypeError, "bf16 or fp16"),
    (dict(q=torch.zeros(2, 4, 64, dtype=F16)), TypeError, "cache's type"),
    (dict(q=torch.zeros(2, 4, 128, dtype=BF16)), ValueError, "q must be"),
    (dict(q=torch.zeros(2, 3, 64, dtype=BF16)), ValueError, "multiple"),
    (dict(cache=kv(dim=72), q=torch.zeros(2, 4, 72, dtype=BF16)), ValueError, "head dimension"),
    (dict(q=torch.zeros(2, 4, 68, dtype=BF16)[..., :64]), ValueError, "16-byte"),
    (dict(block_table=torch.zeros(2, 2, dtype=torch.int64)), TypeError, "int32"),
    (dict(block_table=torch.zeros(3, 2, dtype=torch.int32)), ValueError, "block_table"),
    (dict(block_table=torch.zeros(2, 2, dtype=torch.int32).t()), ValueError, "block_table"),
    (dict(lengths=torch.zeros(2, dtype=torch.int64)), TypeError, "int32"),
    (dict(lengths=torch.zeros(3, dtype=torch.int32)), ValueError, "lengths"),
    (dict(scale=0.0), ValueError, "scale"),
    (dict(scale=float("nan")), ValueError, "scale"),
    (dict(softcap=-1.0), ValueError, "softcap"),
    (dict(window=-1), ValueError, "window"),
    (dict(out=torch.zeros(2, 4, 64, dtype=F16)), ValueError, "out must"),
    (dict(out=torch.zeros(2, 2, 64, dtype=BF16)), ValueError, "out must"),
    (dict(lse=torch.zeros(2, 4, dtype=BF16)), ValueError, "lse must"),
    (dict(q=torch.zeros(2, 4, 64, dtype=BF16, requires_grad=True)), ValueError, "no backward"),
    (dict(), ValueError, "CUDA device"),
])
def test_paged_attention_refusals(over, error, match):
    with pytest.raises(error, match=match):
        at.paged_attention(**paged_args(**over))


def test_paged_attention_refuses_results_over_its_inputs():
    both = torch.zeros(2, 8, 64, dtype=BF16)
    with pytest.raises(ValueError, match="shares memory"):
        at.paged_attention(**paged_args(q=both[:, :4], out=both.view(-1)[:512].view(2, 4, 64)))
    store = torch.zeros(4 * 2 * 16 * 64, dtype=BF16)
    c = at.KvCache(store.view(4, 2, 16, 64), torch.zeros(4, 2, 16, 64, dtype=BF16))
    with pytest.raises(ValueError, match="shares memory"):
        at.paged_attention(**paged_args(cache=c, out=store[1024:1024 + 512].view(2, 4, 64)))
    with pytest.raises(ValueError, match="shares memory"):
        at.paged_attention(**paged_args(cache=c, lse=store.view(F32)[:8].view(2, 4)))


@pytest.mark.parametrize("outs,lses,kw,error,match", [
    (torch.zeros(2, 3, 4, 64, dtype=torch.float64), torch.zeros(2, 3, 4), {}, TypeError, "outs"),
    (torch.zeros(2, 3, 4, 64), torch.zeros(2, 3, 4, dtype=BF16), {}, TypeError, "lses"),
    (torch.zeros(2, 3, 4, 64), torch.zeros(2, 3, 5), {}, ValueError, "lses"),
    (torch.zeros(0, 3, 4, 64), torch.zeros(0, 3, 4), {}, ValueError, "lses"),
    (torch.zeros(2, 3, 4, 60), torch.zeros(2, 3, 4), {}, ValueError, "head dimension"),
    (torch.zeros(2, 4, 3, 64).transpose(1, 2), torch.zeros(2, 3, 4), {}, ValueError, "contiguous"),
    (torch.zeros(2, 3, 4, 64), torch.zeros(2, 3, 4), {"dtype": E4M3}, TypeError, "dtype"),
    (torch.zeros(2, 3, 4, 64), torch.zeros(2, 3, 4), {"out": torch.zeros(3, 4, 32)}, ValueError, "out must"),
    (torch.zeros(2, 3, 4, 64), torch.zeros(2, 3, 4), {}, ValueError, "CUDA device"),
])
def test_join_refusals(outs, lses, kw, error, match):
    with pytest.raises(error, match=match):
        at.attention_join(outs, lses, **kw)


def test_rope_table_keeps_far_positions():
    t = at.rope_table(1 << 17, 64)
    p, i = 131071, 0
    assert t.shape == (1 << 17, 64) and t.dtype == F32
    assert abs(float(t[p, i]) - float(torch.tensor(float(p), dtype=torch.float64).cos())) < 1e-7
    scaled = at.rope_table(16, 32, frequencies=torch.full((16,), 0.5))
    assert torch.allclose(scaled[3, 16:], torch.full((16,), 1.5).sin())
    for bad in ((16, 31), (0, 32)):
        with pytest.raises(ValueError):
            at.rope_table(*bad)


def test_token_slots():
    table = torch.tensor([[4, 2, -1], [0, 7, 1]], dtype=torch.int32)
    seq = torch.tensor([0, 0, 0, 1, 1, 0])
    pos = torch.tensor([0, 17, 32, 47, 48, -1])
    assert at.token_slots(table, seq, pos, 16).tolist() == [64, 33, -1, 31, -1, -1]
    assert at.token_slots(table[:, :0], seq, pos, 16).tolist() == [-1] * 6


def test_references_agree_with_each_other():
    """The parts of a cache joined are the attention over all of it; the quantised form is near the plain one."""
    g = torch.Generator().manual_seed(1)
    c = kv(pages=6, heads=2, size=16, dim=64)
    c.k.copy_(torch.randn(c.k.shape, generator=g))
    c.v.copy_(torch.randn(c.v.shape, generator=g))
    q = torch.randn(1, 6, 64, generator=g).to(BF16)
    table = torch.tensor([[5, 0, 3, 1]], dtype=torch.int32)
    whole, lse = at.ref_paged_attention(q, c, table, torch.tensor([53], dtype=torch.int32))
    parts = [at.ref_paged_attention(q, c, table[:, i:j], torch.tensor([n], dtype=torch.int32))
             for i, j, n in ((0, 2, 32), (2, 4, 21), (1, 2, 0))]
    out, l = at.ref_attention_join(torch.stack([p[0] for p in parts]), torch.stack([p[1] for p in parts]))
    assert torch.allclose(out, whole, atol=1e-12) and torch.allclose(l, lse, atol=1e-12)
    codes, factors = at.ref_quantize_rows(c.k)
    # Half a step of e4m3 is 2^-4 of a value and more below 2^-6, where steps are 2^-9: 2^-10 in units of the factor.
    near = codes.float() * factors[..., None]
    bound = c.k.float().abs() * 2 ** -4 + factors[..., None] * 2 ** -10
    assert bool(((near - c.k.float()).abs() <= bound * (1 + 1e-6)).all())
