"""Attention operators against 64 bits with bounds as narrow as their arithmetic: a probability that enters the second
product with one rounding to 16 bits, or a token whose part of a weight's gradient is lost, is outside of them. That
the bounds notice both is shown on the CPU, with the mistake in the oracle.

E = 2^-24 is the rounding of one fp32 operation, relative to its result.

Paged attention, fp32 results. Queries, keys, factors of keys and the scale are small multiples of powers of two, so
that a score q.k is exact. The score in base 2 then has the rounding of log2(e) and of one product (2 E of it), the
subtraction of the maximum one (E of score and maximum; fp16 and e4m3: the maximum is 14 less), its power of two 2^-22
(4 E). A running result is multiplied by a power of two at every tile of 16 keys at most and at every part that is
joined, each with 6 E; every tile adds to the sum of a lane (4 E, and 8 for the lanes). A weight is off by the sum of
these, the normalised result by that of the weights and that of their sum. A matrix instruction adds 17 numbers, each
cut off at E of the largest, two for a tile (34 E). In two parts a probability is off by 2^-17 of it in bf16: the rest
of the first rounding is less than 2^-8 of its power of two, and 8 bits of it are kept; 2^-23 in fp16, and what is
below the smallest number, 2^-25 where the largest probability is 2^14. A one-part probability would be off by up to
2^-8 or 2^-11.

Weight gradients. A term g n has two roundings from the rotation, 11 from the norm (10 positive additions count half
under the root, 4 for the reciprocal root, 2 products) and is 16 E off at most; sums have one rounding for each
addition on the longest path: two rows a round and lane group, the groups of a block, a 32nd of the blocks, 5 within a
warp."""
import math

import pytest
import torch

from rocshmem_b200.ops import attention as at

BF16, F16, F32, E4M3 = torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn
E = 2.0 ** -24


# ---- paged attention ------------------------------------------------------------------------------------------------

LENGTHS = [1, 2, 3, 5, 9, 15, 16, 17, 33, 40]
MODES = [(BF16, BF16), (F16, F16), (BF16, E4M3), (F16, E4M3)]


class Case:
    """Contents on the CPU: rows of every sequence in order, in the cache's types."""

    def __init__(self, dtype, cache, heads, kv_heads, dim, seed):
        g = torch.Generator().manual_seed(seed)
        B, n = len(LENGTHS), max(LENGTHS)
        self.dtype, self.cache, self.scale = dtype, cache, 2.0 ** -round(math.log2(dim) / 2 + 0.25)
        self.q = (torch.randint(-4, 5, (B, heads, dim), generator=g) / 4).to(dtype)
        k = torch.randint(-6, 7, (B, n, kv_heads, dim), generator=g) / 4
        v = torch.randn(B, n, kv_heads, dim, generator=g)
        if cache == E4M3:
            self.k, self.v = k.to(E4M3), (v * 100).clamp(-448, 448).to(E4M3)
            self.k_scale = 2.0 ** torch.randint(-1, 2, (B, n, kv_heads), generator=g).float()
            self.v_scale = (torch.rand(B, n, kv_heads, generator=g) + 0.2) / 100
        else:
            self.k, self.v, self.k_scale, self.v_scale = k.to(cache), v.to(cache), None, None
        assert torch.equal(self.k.float(), k)

    def exact(self, weigh=None):
        """out, lse, the sum of p |v|, the largest |score| of each sequence and head, in 64 bits; with ``weigh`` the
        probabilities (the largest of them 1, and the values' factors) pass through it on their way to the product."""
        q = self.q.double()
        k, v = self.k.float().double(), self.v.float().double()
        factor = torch.ones(v.shape[:3], dtype=torch.float64)
        if self.k_scale is not None:
            k, factor = k * self.k_scale.double()[..., None], self.v_scale.double()
        B, H, D = q.shape
        K = k.shape[2]
        s = torch.einsum("bkgd,bnkd->bkgn", q.view(B, K, H // K, D), k) * self.scale
        seen = torch.arange(k.shape[1])[None] < torch.tensor(LENGTHS)[:, None]
        s = torch.where(seen[:, None, None], s, -math.inf)
        top = s.amax(-1, keepdim=True)
        p = (s - top).exp()
        total = p.sum(-1, keepdim=True)
        w = p * factor.transpose(1, 2)[:, :, None] if weigh is None else weigh(p, factor.transpose(1, 2)[:, :, None])
        out = torch.einsum("bkgn,bnkd->bkgd", w / total, v).reshape(B, H, D)
        size = torch.einsum("bkgn,bnkd->bkgd", p * factor.transpose(1, 2)[:, :, None] / total, v.abs()).reshape(B, H, D)
        most = torch.where(seen[:, None, None], s, 0.0).abs().amax(-1).reshape(B, H)
        return out, (top + total.log()).reshape(B, H), size, most

    def bounds(self, out, lse, size, most):
        """How far out and lse may be off."""
        bf16 = self.cache == BF16
        shift = 0 if bf16 else 14
        tiles = torch.tensor([(n + 15) // 16 for n in LENGTHS], dtype=torch.float64)[:, None]
        s2 = most * math.log2(math.e)
        weight = math.log(2) * (2 * s2 + 2 * s2 + shift) + 4 + 6 * (2 * tiles + 8) + 4 * tiles + 8 + 4
        part = 2.0 ** -17 if bf16 else 2.0 ** -23
        lost = 0.0 if bf16 else max(LENGTHS) * 2.0 ** -39 * float(self.v.float().abs().max()) * (
            1.0 if self.v_scale is None else 2 * float(self.v_scale.max()))
        bound = (part + ((2 * weight + 34 * tiles) * E)[..., None]) * size + E * out.abs() + lost
        return bound, (weight + 4 * (most + shift + math.log(max(LENGTHS)) + lse.abs())) * E


def cases():
    return [pytest.param(dtype, cache, H, K, D, id=f"{dtype}-{cache}-{H}-{K}-{D}".replace("torch.", ""))
            for dtype, cache in MODES for H, K, D in ((8, 2, 64), (16, 1, 64), (5, 5, 96), (8, 2, 128), (12, 1, 128),
                                                      (4, 1, 256))]


@pytest.mark.parametrize("dtype,cache,H,K,D", cases())
def test_the_bound_notices_probabilities_of_one_part(dtype, cache, H, K, D):
    c = Case(dtype, cache, H, K, D, seed=D + H)
    out, lse, size, most = c.exact()
    bound, _ = c.bounds(out, lse, size, most)

    def one_part(p, factor):
        if cache == BF16:
            return p.to(BF16).double() * factor
        unit = 2.0 ** math.ceil(math.log2(float(factor.max()))) if cache == E4M3 else 1.0
        return (p * 2.0 ** 14 * factor / unit).to(F16).double() * unit * 2.0 ** -14

    wrong = c.exact(one_part)[0]
    assert float(((wrong - out).abs() / bound).max()) > 2.0
    assert (bound[0] <= 2.0 ** -14 * size[0] + 2.0 ** -24 * out[0].abs()).all(), "as narrow as the text above says"


@pytest.mark.gpu
@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("dtype,cache,H,K,D", cases())
def test_paged_attention_in_fp32_results(dtype, cache, H, K, D, wide):
    """A block table as wide as the lengths need (one launch) and one for a thousand tokens more (two)."""
    c = Case(dtype, cache, H, K, D, seed=D + H)
    B, P = len(LENGTHS), 16
    per = (max(LENGTHS) + P - 1) // P
    kv = at.KvCache.allocate(B * per, P, K, D, cache, device="cuda")
    g = torch.Generator().manual_seed(1)
    pages = torch.randperm(B * per, generator=g).view(B, per)
    whole = torch.full((B, per + (100 if wide else 0)), -1, dtype=torch.int32)
    whole[:, :per] = pages
    for to, x in ((kv.k, c.k), (kv.v, c.v), (kv.k_scale, c.k_scale), (kv.v_scale, c.v_scale)):
        if x is None:
            continue
        raw = x.view(torch.uint8) if x.dtype == E4M3 else x
        rows = torch.zeros((B, per * P) + tuple(raw.shape[2:]), dtype=raw.dtype)
        rows[:, :raw.shape[1]] = raw
        rows = rows.view((B, per, P) + tuple(raw.shape[2:])).transpose(2, 3).contiguous().cuda()
        (to.view(torch.uint8) if x.dtype == E4M3 else to)[pages.cuda()] = rows
    out, lse = torch.empty(B, H, D, device="cuda"), torch.empty(B, H, device="cuda")
    at.paged_attention(c.q.cuda(), kv, whole.cuda(), torch.tensor(LENGTHS, dtype=torch.int32, device="cuda"),
                       scale=c.scale, out=out, lse=lse)
    want, want_lse, size, most = c.exact()
    bound, bound_lse = c.bounds(want, want_lse, size, most)
    worst = float(((out.cpu().double() - want).abs() / bound).max())
    assert worst <= 1.0, f"off by {worst:.3g} times the bound"
    worst = float(((lse.cpu().double() - want_lse).abs() / bound_lse).max())
    assert worst <= 1.0, f"lse off by {worst:.3g} times the bound"


# ---- weight gradients of norm and rotation --------------------------------------------------------------------------

SHAPES = [
    (700, 32, 8, 128, 128, BF16, F32, False),      # two rounds of the blocks
    (9000, 8, 2, 64, 64, BF16, F32, False),        # four
    (3000, 5, 3, 256, 64, F16, F32, True),         # five, an odd number of heads
    (2500, 7, 1, 96, 96, F32, F32, True),
    (700, 32, 8, 128, 128, BF16, BF16, False),
]


def gradient_case(T, Hq, Hk, D, R, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    x = [torch.randn(T, H, D, generator=g).to(dtype) for H in (Hq, Hk)]
    grads = [torch.randn(T, H, D, generator=g).to(dtype) for H in (Hq, Hk)]
    positions = torch.randint(0, 777, (T,), generator=g, dtype=torch.int32)
    positions[T // 3] = -1
    return x, grads, positions, at.rope_table(777, R)


def terms(x, g, positions, table, interleaved):
    """The terms of a weight's gradient, [T, H, D], and their magnitudes, in 64 bits."""
    x, g, R = x.double(), g.double(), table.shape[1]
    live = (positions >= 0).double()[:, None, None]
    n = x * (x.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * live
    c, s = (a[:, None] for a in table.double()[positions.long().clamp(min=0)].chunk(2, dim=1))
    first = torch.arange(R // 2) * (2 if interleaved else 1)
    second = first + (1 if interleaved else R // 2)
    back, size = g.clone(), g.abs()
    back[..., first] = g[..., first] * c + g[..., second] * s
    back[..., second] = g[..., second] * c - g[..., first] * s
    size[..., first] = (g[..., first] * c).abs() + (g[..., second] * s).abs()
    size[..., second] = (g[..., second] * c).abs() + (g[..., first] * s).abs()
    return back * n, size * n.abs()


def longest_path(T, heads, other, D, sms):
    """Additions behind one another in the gradient of the weight of `heads`, beside `other` of the other kind."""
    lanes = 8 if D <= 64 else 16 if D <= 128 else 32
    groups = 256 // lanes
    items, rest = T * ((heads + 1) // 2), T * ((other + 1) // 2)
    blocks = max(2, min(3 * sms, (items + rest + groups - 1) // groups))
    own = max(1, items * blocks // (items + rest) - 1)
    rounds = (items + own * groups - 1) // (own * groups)
    return 2 * rounds + groups + (blocks + 31) // 32 + 5


def gradient_bound(want, size, path, weight):
    return torch.finfo(weight).eps / 2 * want.abs() + (path + 16) * E * size.sum(dim=(0, 1))


@pytest.mark.parametrize("T,Hq,Hk,D,R,dtype,weight,interleaved", SHAPES)
def test_the_bound_notices_one_lost_token(T, Hq, Hk, D, R, dtype, weight, interleaved):
    x, grads, positions, table = gradient_case(T, Hq, Hk, D, R, dtype, seed=T + D)
    for i, (heads, other) in enumerate(((Hq, Hk), (Hk, Hq))):
        t, size = terms(x[i], grads[i], positions, table, interleaved)
        want = t.sum(dim=(0, 1))
        bound = gradient_bound(want, size, longest_path(T, heads, other, D, 148), weight)
        for lost in (0, T // 2, T - 1):
            off = (t[lost].sum(dim=0).abs() / bound).max()
            assert float(off) > (2.0 if weight == F32 else 1.0), "a token"
        if weight == F32:
            assert float((t[T - 1, heads - 1].abs() / bound).max()) > 2.0, "a row"


@pytest.mark.gpu
@pytest.mark.parametrize("T,Hq,Hk,D,R,dtype,weight,interleaved", SHAPES)
def test_weight_gradients(T, Hq, Hk, D, R, dtype, weight, interleaved):
    x, grads, positions, table = gradient_case(T, Hq, Hk, D, R, dtype, seed=T + D)
    g = torch.Generator().manual_seed(3)
    w = [(torch.randn(D, generator=g) * 0.3 + 1).to(weight).cuda().requires_grad_() for _ in range(2)]
    out = at.qk_norm_rope(x[0].cuda(), x[1].cuda(), w[0], w[1], positions.cuda(), table.cuda(), interleaved=interleaved)
    back = torch.autograd.grad(out, w, [t.cuda() for t in grads])
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    for i, (heads, other) in enumerate(((Hq, Hk), (Hk, Hq))):
        t, size = terms(x[i], grads[i], positions, table, interleaved)
        want = t.sum(dim=(0, 1))
        bound = gradient_bound(want, size, longest_path(T, heads, other, D, sms), weight)
        worst = float(((back[i].cpu().double() - want).abs() / bound).max())
        assert worst <= 1.0, f"off by {worst:.3g} times the bound"
