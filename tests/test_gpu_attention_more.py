"""Attention operators on a GPU, beside test_gpu_attention.py: tensors that are written in place, the range of sums."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F32, E4M3 = torch.bfloat16, torch.float32, torch.float8_e4m3fn


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape, dtype=F32, scale=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


# ---- tensors that are written in place ------------------------------------------------------------------------------

def small_call(cache_dtype=BF16):
    from rocshmem_b200.ops import attention as at
    g = gen(1)
    c = at.KvCache.allocate(4, 16, 2, 64, cache_dtype)
    k, v, q = (randn(g, 3, 2, 64, dtype=BF16) for _ in range(3))
    at.kv_cache_write(c, k, v, torch.arange(3, device="cuda"))
    table = torch.arange(3, dtype=torch.int32, device="cuda")[:, None].contiguous()
    lengths = torch.tensor([3, 0, 1], dtype=torch.int32, device="cuda")
    return at, c, k, v, q, table, lengths


@pytest.mark.parametrize("cache", [BF16, E4M3])
def test_autograd_sees_what_a_cache_write_changes(cache):
    """A product saves the cache's values (or factors) for its backward pass; after a write that pass is refused."""
    at, c, k, v, *_ = small_call(cache)
    for i, kept in enumerate((c.k, c.v) if cache == BF16 else (c.k_scale, c.v_scale)):
        x = torch.ones(kept.shape, device="cuda", dtype=kept.dtype, requires_grad=True)
        product = (x * kept).sum()
        at.kv_cache_write(c, k, v, torch.arange(3, device="cuda"))
        with pytest.raises(RuntimeError, match="inplace operation"):
            product.backward()
        product = (x * kept).sum()
        at.kv_cache_read(c, torch.arange(3, device="cuda"))      # reads change nothing
        product.backward()
        assert torch.equal(x.grad, kept)


def test_autograd_sees_given_results():
    at, c, _, _, q, table, lengths = small_call()
    out, lse = torch.ones(3, 2, 64, dtype=BF16, device="cuda"), torch.ones(3, 2, device="cuda")
    for kept, call in ((out, lambda: at.paged_attention(q, c, table, lengths, out=out)),
                       (lse, lambda: at.paged_attention(q, c, table, lengths, lse=lse)),
                       (out, lambda: at.attention_join(q[None], torch.zeros(1, 3, 2, device="cuda"), out=out))):
        x = torch.ones_like(kept, requires_grad=True)
        product = (x * kept).sum()
        call()
        with pytest.raises(RuntimeError, match="inplace operation"):
            product.backward()


def test_tensors_made_in_inference_mode_are_written_inside_and_outside_of_it():
    """They have no version to advance."""
    with torch.inference_mode():
        at, c, k, v, q, table, lengths = small_call()
        out, lse = torch.zeros(3, 2, 64, dtype=BF16, device="cuda"), torch.zeros(3, 2, device="cuda")
        want = at.paged_attention(q, c, table, lengths)
        at.paged_attention(q, c, table, lengths, out=out, lse=lse)
        assert torch.equal(out, want)
    at.kv_cache_write(c, k, v, torch.arange(3, device="cuda"))
    at.paged_attention(q, c, table, lengths, out=out, lse=lse)
    joined, _ = at.attention_join(out[None], lse[None], out=torch.empty_like(out))
    assert torch.equal(out, want) and torch.equal(joined, want)


# ---- the range of sums ----------------------------------------------------------------------------------------------

@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("cache", [BF16, E4M3])
def test_values_whose_magnitudes_add_up_to_1e34(cache, wide):
    """The largest that the documentation allows, in one launch and in two (partial results hold up to 2^14 times a
    sum), with equal and with different weights. The bound: one rounding to bf16, and fp32 sums of 300 terms."""
    from rocshmem_b200.ops import attention as at
    g, n, D = gen(3), 300, 128
    c = at.KvCache.allocate(19, 16, 1, D, cache)
    size = 0.99e34 / n
    signs = torch.randint(0, 2, c.v.shape, generator=g, device="cuda") * 2.0 - 1.0
    if cache == E4M3:
        c.k.copy_(randn(g, *c.k.shape).to(E4M3))
        c.v.copy_((signs * 448).to(E4M3))
        c.k_scale.fill_(1.0)
        c.v_scale.fill_(size / 448)
    else:
        c.k.copy_(randn(g, *c.k.shape))
        c.v.copy_(signs * size)
    table = torch.full((1, 200 if wide else 19), -1, dtype=torch.int32, device="cuda")
    table[0, :19] = torch.randperm(19, generator=g, device="cuda")
    lengths = torch.tensor([n], dtype=torch.int32, device="cuda")
    for q in (torch.zeros(1, 4, D, dtype=BF16, device="cuda"), randn(g, 1, 4, D, dtype=BF16)):
        out = at.paged_attention(q, c, table, lengths)
        want, _ = at.ref_paged_attention(q, c, table, lengths)
        assert out.isfinite().all()
        assert ((out.double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -13 * size).all()


# ---- derivatives of the backward pass -------------------------------------------------------------------------------

def test_gradients_with_a_derivative_of_their_own_are_refused():
    """A backward pass whose incoming gradient has a tangent (its result would have none), and one under vmap. The
    engine turns the refusals into a RuntimeError, as it does that of a second derivative."""
    import torch.autograd.forward_ad as fwd
    from rocshmem_b200.ops import attention as at
    g = gen(2)
    leaves = [randn(g, 5, 2, 64).requires_grad_(), randn(g, 5, 1, 64).requires_grad_()]
    w, positions = torch.ones(64, device="cuda"), torch.arange(5, device="cuda")
    table = at.rope_table(8, 64, device="cuda")
    out = at.qk_norm_rope(*leaves, w, w, positions, table)
    grads = [randn(g, *x.shape) for x in out]
    plain = torch.autograd.grad(out, leaves, grads, retain_graph=True)
    with fwd.dual_level():
        with pytest.raises(RuntimeError, match="no forward-mode derivative"):
            torch.autograd.grad(out, leaves, [grads[0], fwd.make_dual(grads[1], grads[1])], retain_graph=True)
        within = torch.autograd.grad(out, leaves, grads, retain_graph=True)
    with pytest.raises(RuntimeError, match="torch.func transform"):
        torch.autograd.grad(out, leaves, [torch.stack([x, x]) for x in grads], retain_graph=True, is_grads_batched=True)
    again = torch.autograd.grad(out, leaves, grads)
    assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(plain, within, again))
