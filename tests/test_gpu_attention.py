"""Attention operators on a GPU against plain PyTorch in 64 bits.

Tolerances, with u the half step of the result's type (eps / 2) and 2^-23 for one fp32 operation (tensor cores
truncate):

* norm and rotation: the result's rounding, and fp32 sums of D squares, each at most D / 8 + 8 additions deep in a lane and
  across lanes: (D / 8 + 16) 2^-23 of the magnitudes that enter an element;
* attention: the result's rounding; probabilities rounded to the cache's type (2^-8 or, in fp16, 2^-11) on the sum of
  p |v|; scores are sums of D products in fp32, off by at most d = D 2^-23 of the sum of |q k| scale, which changes a
  probability by d and the normalisation by as much, and the exponential by 2^-21;
* join: the result's rounding and (n + 16) 2^-23 of the sum of w |o|.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F16, F32, E4M3 = torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn
HALF_STEP = {t: torch.finfo(t).eps / 2 for t in (BF16, F16, F32)}
ONE = 2.0 ** -23


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape, dtype=F32, scale=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def near(got, want, tolerance, what=""):
    got = got.double()
    assert got.shape == want.shape
    assert torch.equal(got.isnan(), want.isnan()), f"{what}: NaN in other places"
    fine = want.isfinite()
    assert torch.equal(got[~fine & ~want.isnan()], want[~fine & ~want.isnan()]), f"{what}: infinities"
    off = (got - want).abs()[fine]
    allowed = tolerance[fine] if torch.is_tensor(tolerance) else torch.full_like(off, tolerance)
    worst = (off / allowed.clamp(min=1e-300)).max().item() if off.numel() else 0.0
    assert worst <= 1.0, f"{what}: off by {worst:.3g} times the tolerance"


# ---- norm and rotation --------------------------------------------------------------------------------------------

def norm_rope_case(T, Hq, Hk, D, R, dtype, weight, interleaved, fused, seed, positions=777):
    from rocshmem_b200.ops import attention as at
    g = gen(seed)
    if fused:
        whole = randn(g, T, Hq + 2 * Hk, D, dtype=dtype)
        q, k = whole[:, :Hq], whole[:, Hq:Hq + Hk]
    else:
        q, k = randn(g, T, Hq, D, dtype=dtype), randn(g, T, Hk, D, dtype=dtype)
    wq, wk = (randn(g, D, scale=0.3).add(1.0).to(weight) for _ in range(2))
    pos = torch.randint(0, positions, (T,), generator=g, device="cuda", dtype=torch.int32)
    return at, q, k, wq, wk, pos, at.rope_table(positions, R, device="cuda")


def norm_rope_tolerance(x, w, pos, table, interleaved, dtype, want):
    """The result's half step and the fp32 part: two elements enter each rotated one."""
    x = x.detach().double()
    D = x.shape[-1]
    n = (x * (x.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * w.detach().double()).abs()
    both = n.clone()
    R = table.shape[1]
    if interleaved:
        pair = n[..., :R].unflatten(-1, (R // 2, 2)).sum(-1)
        both[..., :R] = pair.repeat_interleave(2, -1)
    else:
        pair = n[..., :R // 2] + n[..., R // 2:R]
        both[..., :R] = torch.cat([pair, pair], -1)
    smallest = torch.finfo(dtype).tiny * torch.finfo(dtype).eps
    return HALF_STEP[dtype] * want.abs().nan_to_num() + (D / 8 + 16) * ONE * both + smallest


@pytest.mark.parametrize("T,Hq,Hk,D,R,dtype,weight,interleaved,fused", [
    (1, 1, 1, 64, 64, BF16, BF16, False, False),
    (1, 8, 1, 128, 128, BF16, F32, False, True),
    (5, 5, 3, 128, 64, F16, F16, True, True),
    (67, 32, 8, 128, 128, BF16, BF16, False, True),
    (700, 32, 8, 128, 128, BF16, BF16, False, True),       # four rows a group
    (700, 7, 2, 96, 96, F32, F32, False, False),
    (333, 24, 8, 96, 48, F16, F32, True, False),
    (130, 3, 1, 256, 256, BF16, F32, False, True),
    (129, 4, 4, 256, 32, F32, F32, True, True),
    (33, 2, 2, 16, 16, BF16, BF16, False, False),
    (9, 2, 1, 80, 80, F16, F16, False, False),
    (9, 2, 1, 200, 176, BF16, BF16, False, False),
])
def test_norm_rope_and_gradients(T, Hq, Hk, D, R, dtype, weight, interleaved, fused):
    at, q, k, wq, wk, pos, table = norm_rope_case(T, Hq, Hk, D, R, dtype, weight, interleaved, fused, seed=T + D)
    if T > 4:
        pos[T // 2] = -1
        pos[-1] = -7
    leaves = [t.detach().requires_grad_() for t in (q, k, wq, wk)]
    got = at.qk_norm_rope(*leaves, pos, table, interleaved=interleaved)
    grads = [randn(gen(3 + i), *x.shape, dtype=dtype) for i, x in enumerate(got)]
    back = torch.autograd.grad(got, leaves, grads)
    with torch.no_grad():
        plain = at.qk_norm_rope(*leaves, pos, table, interleaved=interleaved)
    assert torch.equal(plain[0], got[0]) and torch.equal(plain[1], got[1])
    for i, (x, w) in enumerate(((q, wq), (k, wk))):
        xd, wd = x.detach().double().requires_grad_(), w.detach().double().requires_grad_()
        want = at.ref_norm_rope(xd, wd, pos, table, interleaved=interleaved)
        near(got[i], want.detach(), norm_rope_tolerance(x, w, pos, table, interleaved, dtype, want.detach()), "output")
        dx, dw = torch.autograd.grad(want, (xd, wd), grads[i].double())
        # dx = r (a - n mean(a n)): the magnitudes of both terms, a at most |w| times the pair of gradients.
        live = (pos >= 0).double()[:, None, None]
        r = (xd.detach().square().mean(-1, keepdim=True) + 1e-6).rsqrt()
        n = xd.detach() * r
        g2 = grads[i].double().abs()
        a = (g2 + torch.cat([g2[..., :R].roll(R // 2, -1) if not interleaved else
                             g2[..., :R].unflatten(-1, (R // 2, 2)).flip(-1).flatten(-2), g2[..., R:]], -1)) * live
        aw = a * wd.detach().abs()
        size = r * (aw + n.abs() * (aw * n.abs()).mean(-1, keepdim=True))
        smallest = torch.finfo(dtype).tiny * torch.finfo(dtype).eps
        near(back[i], dx, HALF_STEP[dtype] * dx.abs() + (D / 4 + 32) * ONE * size + smallest, "input gradient")
        # A sum of T x H terms in fp32; a term itself is a few operations off.
        terms = (a * n.abs()).sum(dim=(0, 1))
        near(back[2 + i], dw, HALF_STEP[weight] * dw.abs() + (T * x.shape[1] + D / 8 + 64) * ONE * terms,
            "weight gradient")


def test_norm_rope_gradient_against_differences():
    """The slope of L = sum of g q' + g' k' along a random direction, from two forward passes: central differences are
    off by h^2 / 6 of the third derivative (a few units for rows of norm 1) and 2^-22 / h of the terms; 1e-3 of the
    terms covers both at h = 2^-6."""
    at, q, k, wq, wk, pos, table = norm_rope_case(40, 4, 2, 64, 64, F32, F32, False, False, seed=5)
    leaves = [t.requires_grad_() for t in (q, k, wq, wk)]
    got = at.qk_norm_rope(*leaves, pos, table)
    g = [randn(gen(7 + i), *x.shape) for i, x in enumerate(got)]
    back = torch.autograd.grad(got, leaves, g)
    h = 2.0 ** -6
    for i, (leaf, d) in enumerate(zip(leaves, back)):
        way = randn(gen(11 + i), *leaf.shape)

        def value(sign):
            at_ = [t.detach() + sign * h * way if t is leaf else t.detach() for t in leaves]
            return [x.double() * gi.double() for x, gi in zip(at.qk_norm_rope(*at_, pos, table), g)]

        hi, lo = value(1.0), value(-1.0)
        slope = sum((a - b).sum() for a, b in zip(hi, lo)) / (2 * h)
        size = sum(a.abs().sum() for a in hi)
        assert abs(float(slope - (d.double() * way.double()).sum())) <= 1e-3 * float(size)


def test_norm_rope_positions():
    """Both integer types; padding is zeros with no gradient, even where its gradient is NaN; past the table is NaN."""
    at, q, k, wq, wk, pos, table = norm_rope_case(6, 2, 1, 64, 32, BF16, BF16, False, False, seed=2, positions=50)
    pos[0], pos[1], pos[2], pos[3] = 49, 50, -1, 2 ** 31 - 1
    a = at.qk_norm_rope(q, k, wq, wk, pos, table)
    b = at.qk_norm_rope(q, k, wq, wk, pos.long(), table)
    for x, y in zip(a, b):
        assert torch.equal(x.nan_to_num(7.0), y.nan_to_num(7.0))
        assert x[1].isnan().all() and x[3].isnan().all() and (x[2] == 0).all() and x[[0, 4, 5]].isfinite().all()
    far = pos.long()
    far[3] = 2 ** 40
    assert at.qk_norm_rope(q, k, wq, wk, far, table)[0][3].isnan().all()
    pos[1] = pos[3] = -5
    leaves = [t.detach().requires_grad_() for t in (q, k, wq, wk)]
    out = at.qk_norm_rope(*leaves, pos, table)
    g = [torch.ones_like(x) for x in out]
    g[0][2] = float("nan")
    back = torch.autograd.grad(out, leaves, g)
    assert all(x.isfinite().all() for x in back) and (back[0][2] == 0).all()


def test_norm_rope_gradients_of_expanded_and_shared_inputs():
    """One key head expanded to four, one weight for both, the gradient of a sum (expanded, stride 0)."""
    at, q, k, wq, _, pos, table = norm_rope_case(20, 4, 1, 64, 64, F32, F32, False, False, seed=9)
    leaves = [t.detach().requires_grad_() for t in (q, k, wq)]
    q1, k1 = at.qk_norm_rope(leaves[0], leaves[1].expand(-1, 4, -1), leaves[2], leaves[2], pos, table)
    (q1.sum() + k1.sum()).backward()
    wide = [t.detach().double().requires_grad_() for t in (q, k, wq)]
    rq = at.ref_norm_rope(wide[0], wide[2], pos, table)
    rk = at.ref_norm_rope(wide[1].expand(-1, 4, -1), wide[2], pos, table)
    (rq.sum() + rk.sum()).backward()
    for a, b in zip(leaves, wide):
        # Every element takes part in at most 160 rows' sums of terms of size one.
        near(a.grad, b.grad, 256 * 160 * ONE)
    only_k = at.qk_norm_rope(leaves[0], leaves[1], leaves[2], leaves[2], pos, table)[1]
    dq, dk = torch.autograd.grad(only_k.sum(), leaves[:2])
    assert (dq == 0).all() and dk.isfinite().all()


def test_norm_rope_empty_and_repeatable():
    at, q, k, wq, wk, pos, table = norm_rope_case(0, 4, 2, 128, 128, BF16, F32, False, False, seed=1)
    leaves = [t.detach().requires_grad_() for t in (q, k, wq, wk)]
    out = at.qk_norm_rope(*leaves, pos, table)
    back = torch.autograd.grad(out, leaves, [torch.empty_like(x) for x in out])
    assert out[0].shape == (0, 4, 128) and (back[2] == 0).all() and (back[3] == 0).all()
    at, q, k, wq, wk, pos, table = norm_rope_case(3000, 8, 2, 128, 128, BF16, F32, False, False, seed=1)
    leaves = [t.detach().requires_grad_() for t in (q, k, wq, wk)]
    out = at.qk_norm_rope(*leaves, pos, table)
    g = [torch.ones_like(x) for x in out]
    first = torch.autograd.grad(out, leaves, g, retain_graph=True)
    again = torch.autograd.grad(out, leaves, g)
    assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_norm_rope_refuses_a_second_derivative():
    at, q, k, wq, wk, pos, table = norm_rope_case(5, 2, 1, 64, 64, F32, F32, False, False, seed=2)
    leaves = [t.detach().requires_grad_() for t in (q, k, wq, wk)]
    out = at.qk_norm_rope(*leaves, pos, table)
    with pytest.raises(RuntimeError, match="differentiated once"):
        torch.autograd.grad(out, leaves, [torch.ones_like(x) for x in out], create_graph=True)
    out = at.qk_norm_rope(*leaves, pos, table)
    torch.autograd.backward(out, [torch.ones_like(x) for x in out])
    assert all(t.grad is not None and t.grad.shape == t.shape for t in leaves)
    frozen = at.qk_norm_rope(leaves[0].detach(), leaves[1].detach(), leaves[2], wk.detach(), pos, table)
    assert torch.equal(torch.autograd.grad(frozen[0].sum() + frozen[1].sum(), leaves[2])[0], leaves[2].grad)


# ---- the cache --------------------------------------------------------------------------------------------------

def random_cache(g, pages, size, heads, dim, dtype):
    from rocshmem_b200.ops import attention as at
    c = at.KvCache.allocate(pages, size, heads, dim, dtype)
    if dtype == E4M3:
        for codes, factors in ((c.k, c.k_scale), (c.v, c.v_scale)):
            codes.copy_(randn(g, *codes.shape, scale=120.0).clamp(-448, 448).to(E4M3))
            factors.copy_((torch.rand(factors.shape, generator=g, device="cuda") + 0.2) / 120)
    else:
        c.k.copy_(randn(g, *c.k.shape))
        c.v.copy_(randn(g, *c.v.shape))
    return c


def bytes_of(t):
    return t.view(torch.uint8) if t.dtype == E4M3 else t


@pytest.mark.parametrize("T,heads,dim,size,dtype,cache,wide,fused", [
    (1, 1, 64, 16, BF16, BF16, True, False),
    (1, 2, 128, 1, BF16, E4M3, False, True),
    (5, 3, 96, 32, F16, E4M3, True, False),
    (67, 8, 128, 16, BF16, E4M3, True, True),
    (300, 4, 256, 64, F32, E4M3, False, False),
    (300, 4, 64, 128, F16, F16, True, True),
    (1500, 8, 128, 16, F32, BF16, False, True),
    (2500, 8, 128, 64, BF16, E4M3, True, True),          # four rows a group
    (40, 2, 40, 8, BF16, F16, True, False),
    (40, 2, 8, 8, F16, E4M3, True, False),
])
def test_cache_write_and_read(T, heads, dim, size, dtype, cache, wide, fused):
    from rocshmem_b200.ops import attention as at
    g = gen(T + dim)
    pages = (T + size - 1) // size + 2
    c = random_cache(g, pages, size, heads, dim, cache)
    before = [t.clone() for t in c._tensors()]
    both = randn(g, T, 2 * heads, dim, dtype=dtype)
    k, v = (both[:, :heads], both[:, heads:]) if fused else (both[:, :heads].contiguous(), both[:, heads:].contiguous())
    if T > 4:
        k[1, 0] = 0.0                                     # a row of zeros
        k[2, 0] *= 2.0 ** -20
        v[2, 0, :] = torch.finfo(dtype).tiny              # tiny rows
    slots = torch.randperm(pages * size, generator=g, device="cuda")[:T]
    if T > 8:
        slots[3], slots[4], slots[5] = -1, pages * size, 2 ** 31 - 1
    if not wide:
        slots = slots.int()
    at.kv_cache_write(c, k, v, slots)
    ok = (slots >= 0) & (slots < pages * size)
    s = slots[ok].long()
    for i, x in enumerate((k, v)):
        want = before[i].clone()
        if cache == E4M3:
            codes, factors = at.ref_quantize_rows(x[ok])
            bytes_of(want)[s // size, :, s % size] = bytes_of(codes)
            before[2 + i][s // size, :, s % size] = factors
            assert torch.equal(c._tensors()[2 + i], before[2 + i]), "factors"
        else:
            want[s // size, :, s % size] = x[ok].to(cache)
        assert torch.equal(bytes_of(c._tensors()[i]), bytes_of(want)), "values, and slots that were not written"
    for out_dtype in (BF16, F16, F32):
        got = at.kv_cache_read(c, slots, dtype=out_dtype)
        for i, x in enumerate(got):
            assert (x[~ok] == 0).all()
            rows = c._tensors()[i].float()[s // size, :, s % size]
            if cache == E4M3:
                rows = rows * c._tensors()[2 + i][s // size, :, s % size][..., None]
            assert torch.equal(x[ok], rows.to(out_dtype))


def test_cache_quantisation_error_and_rows_that_are_not_finite():
    from rocshmem_b200.ops import attention as at
    g = gen(4)
    c = at.KvCache.allocate(2, 16, 2, 128, E4M3)
    k, v = randn(g, 20, 2, 128, dtype=BF16), randn(g, 20, 2, 128, dtype=BF16)
    k[3, 1, 5], k[4, 0, 127], v[7, 0, 0] = float("nan"), float("inf"), float("-inf")
    slots = torch.arange(20, device="cuda")
    at.kv_cache_write(c, k, v, slots)
    rk, rv = at.kv_cache_read(c, slots, dtype=F32)
    for x, r in ((k, rk), (v, rv)):
        bad = ~x.isfinite().all(-1)
        assert r[bad].isnan().all() and r[~bad].isfinite().all()
        x, r = x[~bad].double(), r[~bad].double()
        # Half a step of e4m3 is 2^-4 of a value, below 2^-6 half of 2^-9; codes are values times 448 / largest.
        unit = x.abs().amax(-1, keepdim=True) / 448
        assert ((x - r).abs() <= (x.abs() * 2 ** -4 + unit * 2 ** -10) * (1 + 2 ** -20)).all()


def test_cache_empty_calls():
    from rocshmem_b200.ops import attention as at
    c = at.KvCache.allocate(2, 16, 2, 64, E4M3)
    none = torch.empty(0, 2, 64, dtype=BF16, device="cuda")
    at.kv_cache_write(c, none, none, torch.empty(0, dtype=torch.int64, device="cuda"))
    k, v = at.kv_cache_read(c, torch.empty(0, dtype=torch.int32, device="cuda"))
    assert k.shape == v.shape == (0, 2, 64)
    empty = at.KvCache.allocate(0, 16, 2, 64, BF16)
    one = torch.ones(1, 2, 64, dtype=BF16, device="cuda")
    at.kv_cache_write(empty, one, one, torch.zeros(1, dtype=torch.int64, device="cuda"))
    assert (at.kv_cache_read(empty, torch.zeros(1, dtype=torch.int64, device="cuda"))[0] == 0).all()


# ---- attention over the cache -------------------------------------------------------------------------------------

def paged_case(lengths, H, K, D, size, dtype, cache, seed, extra_pages=1, poison=True):
    """A cache in which everything that no sequence sees is NaN (codes 0x7f, factors NaN)."""
    g = gen(seed)
    B = len(lengths)
    per = max(1, max((n + size - 1) // size for n in lengths)) + extra_pages
    pages = B * per + 3
    c = random_cache(g, pages, size, K, D, cache)
    table = torch.randperm(pages, generator=g, device="cuda")[:B * per].view(B, per).int()
    ln = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    if poison:
        used = torch.zeros(pages * size, dtype=torch.bool, device="cuda")
        pos = torch.arange(per * size, device="cuda")
        for b in range(B):
            p = pos[:max(0, lengths[b])]
            used[table[b, p // size].long() * size + p % size] = True
        gone = ~used.view(pages, 1, size).expand(pages, K, size)
        for x in c._tensors():
            if x.dtype == E4M3:
                x.view(torch.uint8)[gone] = 0x7f
            else:
                x[gone] = float("nan")
    q = randn(g, B, H, D, dtype=dtype, scale=1.5)
    return c, q, table, ln


def check_paged(at, c, q, table, ln, out, lse, softcap=0.0, window=0, scale=None, what=""):
    want, want_lse = at.ref_paged_attention(q, c, table, ln, scale=scale, softcap=softcap, window=window)
    D = q.shape[2]
    f = D ** -0.5 if scale is None else scale

    def absolute(x, factor):
        if factor is None:
            return at.KvCache(x.nan_to_num().abs(), x.nan_to_num().abs())
        a = (x.view(torch.uint8) & 0x7f).view(E4M3)
        return at.KvCache(a, a, factor, factor)

    # Sum of p |v| with the same probabilities: the values' magnitudes in the place of the values.
    mags = at.KvCache(c.k, absolute(c.v, c.v_scale).v, c.k_scale, c.v_scale)
    sum_pv, _ = at.ref_paged_attention(q, mags, table, ln, scale=scale, softcap=softcap, window=window)
    # The largest sum of |q k| scale that a sequence's rows can have: norms.
    kn = c.k.float().nan_to_num().double() if c.k_scale is None else \
        c.k.float().nan_to_num().double() * c.k_scale.double().nan_to_num()[..., None]
    most = kn.square().sum(-1).max().sqrt()
    d = D * ONE * q.double().square().sum(-1).sqrt() * most * f + 2.0 ** -21          # [B, H]
    p_step = HALF_STEP[BF16] if c.k.dtype == BF16 else HALF_STEP[F16]
    u = HALF_STEP[out.dtype]
    smallest = torch.finfo(out.dtype).tiny * torch.finfo(out.dtype).eps
    near(out, want, u * want.abs() + (p_step + 2 * d[..., None] + 32 * ONE) * sum_pv + smallest, what + " out")
    if lse is not None:
        near(lse, want_lse, d + 8 * ONE * want_lse.abs().nan_to_num(posinf=0.0), what + " lse")


LENGTHS = [1, 0, 17, 300, 64, 16, 15, 129, 63, 65, 128, 33]


@pytest.mark.parametrize("dtype,cache", [(BF16, BF16), (F16, F16), (BF16, E4M3), (F16, E4M3)])
@pytest.mark.parametrize("D", [64, 96, 128, 256])
@pytest.mark.parametrize("H,K,size", [(4, 4, 16), (16, 2, 32), (10, 1, 128), (48, 2, 1)])
def test_paged_attention_lengths_and_groups(dtype, cache, D, H, K, size):
    from rocshmem_b200.ops import attention as at
    c, q, table, ln = paged_case(LENGTHS, H, K, D, size, dtype, cache, seed=D + H)
    out, lse = at.paged_attention(q, c, table, ln, return_lse=True)
    assert out.dtype == dtype and (out[1] == 0).all() and (lse[1] == -math.inf).all()
    check_paged(at, c, q, table, ln, out, lse)


@pytest.mark.parametrize("dtype,cache", [(BF16, BF16), (F16, F16), (BF16, E4M3)])
@pytest.mark.parametrize("lengths,H,K,D", [([20011], 4, 1, 128), ([9000, 3, 0, 40000], 16, 2, 64),
                                           ([5003, 5003], 32, 2, 128), ([7777], 12, 12, 96), ([6007, 1], 8, 1, 256)])
def test_paged_attention_split_over_long_caches(dtype, cache, lengths, H, K, D):
    from rocshmem_b200.ops import attention as at
    c, q, table, ln = paged_case(lengths, H, K, D, 16, dtype, cache, seed=len(lengths) + D)
    out, lse = at.paged_attention(q, c, table, ln, return_lse=True)
    check_paged(at, c, q, table, ln, out, lse)
    again, lse2 = at.paged_attention(q, c, table, ln, return_lse=True)
    assert torch.equal(out, again) and torch.equal(lse, lse2), "results do not depend on the blocks' order"


def test_paged_attention_many_sequences():
    """More sequences than the threads of a block, most of them short or empty."""
    from rocshmem_b200.ops import attention as at
    g = torch.Generator().manual_seed(3)
    lengths = [int(n) for n in torch.randint(-1, 40, (700,), generator=g)]
    lengths[350] = 900
    c, q, table, ln = paged_case(lengths, 6, 3, 64, 16, BF16, BF16, seed=8, extra_pages=0)
    out, lse = at.paged_attention(q, c, table, ln, return_lse=True)
    check_paged(at, c, q, table, ln, out, lse)


@pytest.mark.parametrize("softcap,window,scale", [(30.0, 0, None), (0.0, 1, None), (0.0, 100, 0.2), (5.0, 257, 1.0),
                                                  (0.0, 10 ** 6, None)])
@pytest.mark.parametrize("cache", [F16, E4M3])
def test_paged_attention_caps_and_windows(softcap, window, scale, cache):
    from rocshmem_b200.ops import attention as at
    c, q, table, ln = paged_case([1, 50, 99, 100, 101, 700, 4001], 8, 2, 128, 32, F16, cache, seed=6)
    out, lse = at.paged_attention(q, c, table, ln, scale=scale, softcap=softcap, window=window, return_lse=True)
    check_paged(at, c, q, table, ln, out, lse, softcap, window, scale)


def test_paged_attention_does_not_see_bad_pages_or_bad_lengths():
    from rocshmem_b200.ops import attention as at
    for cache in (BF16, E4M3):
        c, q, table, ln = paged_case([200, 200, 90, 64, 10], 8, 2, 128, 16, BF16, cache, seed=2, extra_pages=0,
            poison=False)
        table[0, 2], table[0, 5], table[1, :] = -1, c.num_pages, 2 ** 31 - 1
        table[2, 0] = -2 ** 31
        ln[2], ln[3], ln[4] = 10 ** 6, -5, 2 ** 31 - 1
        out, lse = at.paged_attention(q, c, table, ln, return_lse=True)
        assert (out[1] == 0).all() and (lse[1] == -math.inf).all() and (out[3] == 0).all()
        check_paged(at, c, q, table, ln, out, lse)
    none = torch.empty(5, 0, dtype=torch.int32, device="cuda")
    out, lse = at.paged_attention(q, c, none, ln, return_lse=True)
    assert (out == 0).all() and (lse == -math.inf).all()
    empty = at.paged_attention(q[:0], c, table[:0], ln[:0])
    assert empty.shape == (0, 8, 128)


def test_paged_attention_strides_and_given_results():
    from rocshmem_b200.ops import attention as at
    c, q, table, ln = paged_case([130, 3, 77], 8, 2, 64, 16, F16, F16, seed=12)
    want, want_lse = at.paged_attention(q, c, table, ln, return_lse=True)
    wide_q = torch.full((3, 12, 64), float("nan"), dtype=F16, device="cuda")
    wide_q[:, 2:10] = q
    wide_table = torch.full((3, 40), -9, dtype=torch.int32, device="cuda")
    wide_table[:, :table.shape[1]] = table
    out = torch.full((5, 8, 64), 3.0, dtype=F16, device="cuda")
    lse = torch.full((5, 8), 3.0, device="cuda")
    got = at.paged_attention(wide_q[:, 2:10], c, wide_table[:, :table.shape[1]], ln, out=out[1:4], lse=lse[1:4])
    assert got.data_ptr() == out[1:4].data_ptr()
    assert torch.equal(out[1:4], want) and torch.equal(lse[1:4], want_lse)
    assert (out[[0, 4]] == 3).all() and (lse[[0, 4]] == 3).all()
    exact = torch.empty(3, 8, 64, dtype=F32, device="cuda")
    at.paged_attention(q, c, table, ln, out=exact)
    assert torch.equal(exact.to(F16), want)
    assert not torch.equal(exact, want.float())


def test_paged_attention_extreme_values():
    """Queries and factors far from one, keys and values of the type's largest, scores of -inf, infinities and NaN that
    are seen."""
    from rocshmem_b200.ops import attention as at
    c, q, table, ln = paged_case([40, 300], 8, 2, 128, 16, BF16, E4M3, seed=3, poison=False)
    c.k_scale.mul_(1e-30)
    c.v_scale.mul_(1e-25)
    big = (q.float() * 1e30).to(BF16)
    out, lse = at.paged_attention(big, c, table, ln, return_lse=True)
    check_paged(at, c, big, table, ln, out, lse, what="small factors")
    c.k_scale.mul_(1e30)
    c.v_scale.mul_(1e25 * 3e4)
    out, lse = at.paged_attention(q, c, table, ln, return_lse=True)
    check_paged(at, c, q, table, ln, out, lse, what="large values")
    small = (q.float() * 2.0 ** -126).to(BF16)
    out, lse = at.paged_attention(small, c, table, ln, return_lse=True)
    check_paged(at, c, small, table, ln, out, lse, what="small queries")
    zero = torch.zeros_like(q)
    out, lse = at.paged_attention(zero, c, table, ln, return_lse=True)
    check_paged(at, c, zero, table, ln, out, lse, what="zero queries")

    c, q, table, ln = paged_case([40, 300], 8, 2, 128, 16, BF16, BF16, seed=4, poison=False)
    q = q.abs() + 0.1
    c.k[table[1, 3].long()] = -math.inf                        # scores of -inf: keys that count for nothing
    out, lse = at.paged_attention(q, c, table, ln, return_lse=True)
    keep = table.clone()
    keep[1, 3] = -1
    want, want_lse = at.paged_attention(q, c, keep, ln, return_lse=True)
    assert torch.equal(out, want) and torch.equal(lse, want_lse)
    c.k[table[0, 0].long(), 1] = math.nan                      # one key head of one sequence
    out, lse = at.paged_attention(q, c, table, ln, return_lse=True)
    assert out[0, 4:].isnan().all() and out[0, :4].isfinite().all() and torch.equal(out[1], want[1])
    assert lse[0, 4:].isnan().all()


def test_paged_attention_on_another_stream_and_in_a_graph():
    """A graph replayed with other contents; two graphs and an eager call have workspaces of their own."""
    from rocshmem_b200.ops import attention as at
    cases = [paged_case(l, 8, 2, 128, 16, BF16, E4M3, seed=s) for l, s in (([3000, 17, 0], 1), ([5, 900, 2500], 2))]
    want = [at.paged_attention(q, c, t, n, return_lse=True) for c, q, t, n in cases]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for stream in (side, side.cuda_stream):
        c, q, t, n = cases[0]
        got = at.paged_attention(q, c, t, n, return_lse=True, stream=stream)
        side.synchronize()
        assert torch.equal(got[0], want[0][0]) and torch.equal(got[1], want[0][1])
    graphs = []
    for c, q, t, n in cases:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            res = at.paged_attention(q, c, t, n, return_lse=True)
        graphs.append((g, res))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(5):
        for (g, _), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    eager = at.paged_attention(cases[1][1], cases[1][0], cases[1][2], cases[1][3])
    torch.cuda.synchronize()
    assert torch.equal(eager, want[1][0])
    for (_, res), w in zip(graphs, want):
        assert torch.equal(res[0], w[0]) and torch.equal(res[1], w[1])
    c, q, t, n = cases[0]
    n.copy_(torch.tensor([100, 2990, 1], dtype=torch.int32))   # the replay reads lengths from the device
    t[1] = t[0]
    graphs[0][0].replay()
    torch.cuda.synchronize()
    now = at.paged_attention(q, c, t, n, return_lse=True)
    # The third sequence now sees a row that it did not write, NaN: the same bits, NaN included.
    for a, b in zip(graphs[0][1], now):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    assert now[0][:2].isfinite().all() and now[0][2].isnan().all()


def test_streams_are_refused_or_followed():
    from rocshmem_b200.ops import attention as at
    side = torch.cuda.Stream()
    g = gen(1)
    x = randn(g, 40, 3, 64, dtype=BF16)
    w = torch.ones(64, dtype=BF16, device="cuda")
    pos, table = torch.arange(40, device="cuda"), at.rope_table(64, 64, device="cuda")
    c = at.KvCache.allocate(4, 16, 1, 64, E4M3)
    side.wait_stream(torch.cuda.current_stream())
    q, k = at.qk_norm_rope(x[:, :2], x[:, 2:], w, w, pos, table, stream=side)
    at.kv_cache_write(c, k, k, pos, stream=side)
    rk, _ = at.kv_cache_read(c, pos, stream=side)
    o, l = at.attention_join(q[None], torch.zeros(1, 40, 2, device="cuda"), stream=side)
    side.synchronize()
    q2, k2 = at.qk_norm_rope(x[:, :2], x[:, 2:], w, w, pos, table)
    assert torch.equal(q, q2) and torch.equal(k, k2) and torch.equal(o, q)
    codes, factors = at.ref_quantize_rows(k2)
    assert torch.equal(rk, (codes.float() * factors[..., None]).to(BF16))


# ---- join ------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("n,B,H,D,dtype,out_dtype",
    [(1, 1, 1, 64, F32, BF16), (2, 3, 8, 128, F32, BF16), (3, 70, 5, 96, BF16, F32),
                                                      (8, 33, 16, 256, F32, F16), (17, 2, 2, 8, F16, F16), (9, 5, 7,
                                                          200, BF16, BF16)])
def test_attention_join(n, B, H, D, dtype, out_dtype):
    from rocshmem_b200.ops import attention as at
    g = gen(n * D)
    outs, lses = randn(g, n, B, H, D, dtype=dtype), randn(g, n, B, H, scale=3.0)
    if n > 1:
        lses[0, 0, 0] = -math.inf
        outs[0, 0, 0] = math.nan                  # a part that has seen nothing does not count
        lses[1] += 200.0                          # exponentials far outside fp32's range
        lses[:, -1, -1] = -math.inf               # nobody has seen anything
    out, lse = at.attention_join(outs, lses, dtype=out_dtype)
    want, want_lse = at.ref_attention_join(outs, lses)
    mags, _ = at.ref_attention_join(outs.abs(), lses)
    assert out.dtype == out_dtype
    smallest = torch.finfo(out_dtype).tiny * torch.finfo(out_dtype).eps
    near(out, want, HALF_STEP[out_dtype] * want.abs() + (n + 16) * ONE * mags + smallest, "out")
    near(lse, want_lse, (n + 16) * ONE * (1 + want_lse.abs().nan_to_num(posinf=0.0)), "lse")


def test_attention_join_of_parts_that_lie_apart_and_of_nan():
    from rocshmem_b200.ops import attention as at
    g = gen(5)
    B, H, D, n = 4, 6, 64, 3
    block = B * H * D + B * H
    block += -block % 4
    store = randn(g, n, block)
    outs, lses = store[:, :B * H * D].view(n, B, H, D), store[:, B * H * D:B * H * D + B * H].view(n, B, H)
    target = torch.empty(B, H, D, dtype=BF16, device="cuda")
    out, lse = at.attention_join(outs, lses, out=target)
    plain, plain_lse = at.attention_join(outs.contiguous(), lses.contiguous(), dtype=BF16)
    assert out.data_ptr() == target.data_ptr() and torch.equal(out, plain) and torch.equal(lse, plain_lse)
    lses[1, 2, 3] = math.nan
    out, lse = at.attention_join(outs, lses)
    assert out[2, 3].isnan().all() and lse[2, 3].isnan() and int(lse.isnan().sum()) == 1
    with pytest.raises(ValueError, match="shares memory"):
        at.attention_join(outs, lses, out=outs[0])


# ---- a decode step of a layer -----------------------------------------------------------------------------------

@pytest.mark.parametrize("cache,size", [(BF16, 16), (E4M3, 32)])
def test_prefill_then_decode_steps(cache, size):
    """Prompts are normed, rotated and written, then tokens are added one by one; each step's result is the attention
    over all rows so far, as the cache holds them. The cache of one sequence split over two joins to the same."""
    from rocshmem_b200.ops import attention as at
    g = gen(31)
    B, H, K, D = 3, 8, 2, 128
    prompts, steps, pages = [40, 1, 130], 3, 40
    table = torch.randperm(pages, generator=g, device="cuda")[:B * 10].view(B, 10).int()
    c = at.KvCache.allocate(pages, size, K, D, cache)
    rope = at.rope_table(512, D, device="cuda")
    wq, wk = (randn(g, D, scale=0.2).add(1.0).to(BF16) for _ in range(2))

    def project(positions, sequences):
        qkv = randn(g, len(positions), H + 2 * K, D, dtype=BF16)
        q, k = at.qk_norm_rope(qkv[:, :H], qkv[:, H:H + K], wq, wk, positions, rope)
        at.kv_cache_write(c, k, qkv[:, H + K:], at.token_slots(table, sequences, positions, size))
        return q, k, qkv[:, H + K:]

    seq = torch.tensor([b for b, n in enumerate(prompts) for _ in range(n)], device="cuda")
    pos = torch.tensor([i for n in prompts for i in range(n)], device="cuda")
    _, k0, v0 = project(pos, seq)
    if cache == BF16:
        rk, rv = at.kv_cache_read(c, at.token_slots(table, seq, pos, size))
        assert torch.equal(rk, k0) and torch.equal(rv, v0)
    lengths = torch.tensor(prompts, dtype=torch.int32, device="cuda")
    for _ in range(steps):
        q, _, _ = project(lengths.clone(), torch.arange(B, device="cuda"))
        lengths += 1
        out, lse = at.paged_attention(q, c, table, lengths, return_lse=True)
        check_paged(at, c, q, table, lengths, out, lse)
        half = 2 * size
        first = at.paged_attention(q, c, table[:, :2].contiguous(), lengths.clamp(max=half), return_lse=True,
                                   out=torch.empty(B, H, D, device="cuda"))
        rest = at.paged_attention(q, c, table[:, 2:], (lengths - half).clamp(min=0), return_lse=True,
                                  out=torch.empty(B, H, D, device="cuda"))
        joined, lse2 = at.attention_join(torch.stack([first[0], rest[0]]), torch.stack([first[1], rest[1]]), dtype=BF16)
        check_paged(at, c, q, table, lengths, joined, lse2)


# ---- captures, far offsets, odd but allowed arguments ---------------------------------------------------------------

def test_norm_rope_training_step_in_a_graph():
    """Forward and backward captured together and replayed on new contents; refused while an eager graph of the same
    leaves is alive."""
    at, q, k, wq, wk, pos, table = norm_rope_case(200, 4, 2, 128, 128, BF16, F32, False, False, seed=8)
    leaves = [t.detach().clone().requires_grad_() for t in (q, k, wq, wk)]
    grads = [randn(gen(20 + i), *t.shape, dtype=BF16) for i, t in enumerate((q, k))]

    def step():
        out = at.qk_norm_rope(*leaves, pos, table)
        return out, torch.autograd.grad(out, leaves, grads)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, back = step()
    out = [x.detach() for x in out]
    with torch.no_grad():
        leaves[0].copy_(randn(gen(31), 200, 4, 128, dtype=BF16))
        leaves[3].mul_(0.5)
    graph.replay()
    torch.cuda.synchronize()
    got = [x.clone() for x in (*out, *back)]
    fresh = [t.detach().clone().requires_grad_() for t in leaves]
    want = at.qk_norm_rope(*fresh, pos, table)
    want = [x.detach() for x in want] + list(torch.autograd.grad(want, fresh, grads))
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    new = [t.detach().clone().requires_grad_() for t in (q, k, wq, wk)]
    alive = at.qk_norm_rope(*new, pos, table)
    with pytest.raises(RuntimeError, match="alive"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            at.qk_norm_rope(*new, pos, table)
    torch.cuda.synchronize()
    assert torch.autograd.grad(alive, new, grads)[0].isfinite().all()


@pytest.mark.parametrize("cache", [BF16, E4M3])
def test_rows_behind_four_gigabytes(cache):
    """Rows whose offset in bytes does not fit 32 bits: written, read back and attended to."""
    from rocshmem_b200.ops import attention as at
    D, size, K = 256, 64, 4
    pages = (9 << 30) // (2 if cache == BF16 else 1) // (K * size * D) // 2 + 3
    c = at.KvCache.allocate(pages, size, K, D, cache)
    assert c.k.numel() * c.k.element_size() > 1 << 32
    g = gen(3)
    n = 150
    k, v = randn(g, n, K, D, dtype=BF16), randn(g, n, K, D, dtype=BF16)
    table = torch.tensor([[pages - 1, 0, pages - 2]], dtype=torch.int32, device="cuda")
    pos = torch.arange(n, device="cuda")
    slots = at.token_slots(table, torch.zeros_like(pos), pos, size)
    at.kv_cache_write(c, k, v, slots)
    small = at.KvCache.allocate(3, size, K, D, cache)
    near_table = torch.tensor([[2, 0, 1]], dtype=torch.int32, device="cuda")
    at.kv_cache_write(small, k, v, at.token_slots(near_table, torch.zeros_like(pos), pos, size))
    for a, b in zip(at.kv_cache_read(c, slots),
        at.kv_cache_read(small, at.token_slots(near_table, torch.zeros_like(pos), pos, size))):
        assert torch.equal(a, b) and (cache == E4M3 or torch.equal(a, k) or torch.equal(a, v))
    q = randn(g, 1, 8, D, dtype=BF16)
    ln = torch.tensor([n], dtype=torch.int32, device="cuda")
    assert torch.equal(at.paged_attention(q, c, table, ln), at.paged_attention(q, small, near_table, ln))


def test_caches_without_pages_and_factors_below_zero():
    from rocshmem_b200.ops import attention as at
    q = randn(gen(1), 2, 4, 64, dtype=BF16)
    for dtype in (BF16, E4M3):
        empty = at.KvCache.allocate(0, 16, 2, 64, dtype)
        out, lse = at.paged_attention(q, empty, torch.zeros(2, 3, dtype=torch.int32, device="cuda"),
                                      torch.full((2,), 40, dtype=torch.int32, device="cuda"), return_lse=True)
        assert (out == 0).all() and (lse == -math.inf).all()
    c, q, table, ln = paged_case([40, 129], 8, 2, 128, 16, BF16, E4M3, seed=3, poison=False)
    c.k_scale[:, :, ::3] *= -1
    c.v_scale[:, 1:] *= -40.0
    out, lse = at.paged_attention(q, c, table, ln, return_lse=True)
    mags = at.KvCache(c.k, c.v, c.k_scale, c.v_scale.abs())
    want, want_lse = at.ref_paged_attention(q, c, table, ln)
    a = (mags.v.view(torch.uint8) & 0x7f).view(E4M3)
    sum_pv, _ = at.ref_paged_attention(q, at.KvCache(c.k, a, c.k_scale, mags.v_scale), table, ln)
    near(out, want, HALF_STEP[BF16] * want.abs() + 2.0 ** -11 * sum_pv, "out")


def test_expanded_queries_and_caches_that_are_copied():
    import copy
    import pickle
    from rocshmem_b200.ops import attention as at
    c, q, table, ln = paged_case([40, 129, 3], 8, 2, 64, 16, BF16, BF16, seed=3, poison=False)
    one = q[:1].expand(3, -1, -1)
    want = at.paged_attention(one.contiguous(), c, table, ln)
    assert torch.equal(at.paged_attention(one, c, table, ln), want)
    for other in (copy.copy(c), copy.deepcopy(c), pickle.loads(pickle.dumps(c))):
        assert torch.equal(at.paged_attention(one, other, table, ln), want)
    assert c != copy.copy(c) and c == c
    with pytest.raises(ValueError, match="gradient"):
        at.KvCache(torch.zeros(2, 2, 16, 64, dtype=BF16, device="cuda", requires_grad=True),
            torch.zeros(2, 2, 16, 64, dtype=BF16, device="cuda"))


@pytest.mark.parametrize("cache", [BF16, E4M3])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("B,K,H,pages", [(1, 1, 1, 1), (2, 2, 12, 7), (37, 4, 16, 20), (37, 4, 16, 33), (149, 1, 8,
    5), (5, 1, 40, 16)])
def test_paged_attention_one_launch_and_two(cache, D, B, K, H, pages):
    """Calls on both sides of the rule that chooses between a block for each pair and shares of all tiles."""
    from rocshmem_b200.ops import attention as at
    g = torch.Generator().manual_seed(B + pages)
    lengths = [int(n) for n in torch.randint(0, 32 * pages + 1, (B,), generator=g)]
    lengths[B // 2] = 32 * pages
    c, q, table, ln = paged_case(lengths, H, K, D, 32, BF16, cache, seed=pages, extra_pages=0)
    out, lse = at.paged_attention(q, c, table, ln, return_lse=True)
    check_paged(at, c, q, table, ln, out, lse)
    exact = torch.empty(q.shape, device="cuda")
    at.paged_attention(q, c, table, ln, out=exact)
    assert torch.equal(exact.to(BF16), out)
