"""Attention operators without a GPU: calls that would drop a derivative, write over what somebody else keeps, or mean
something else than they say. All are refused before anything touches a device, so CPU tensors show it: what passes
every check ends with the refusal of the CPU device."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

from rocshmem_b200.ops import attention as at

BF16, F16, F32, E4M3 = torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn


def zeros(*shape, dtype=BF16, **kw):
    return torch.zeros(*shape, dtype=dtype, **kw)


def cache(dtype=BF16, pages=4, heads=2, size=16, dim=64):
    return at.KvCache.allocate(pages, size, heads, dim, dtype, device="cpu")


def norm_rope(**over):
    a = dict(q=zeros(3, 4, 64, dtype=F32), k=zeros(3, 2, 64, dtype=F32), q_weight=torch.ones(64),
             k_weight=torch.ones(64), positions=torch.zeros(3, dtype=torch.int32), table=torch.zeros(8, 64))
    a.update(over)
    return at.qk_norm_rope(**a)


def write(c=None, **over):
    a = dict(k=zeros(3, 2, 64), v=zeros(3, 2, 64), slots=torch.arange(3))
    a.update(over)
    return at.kv_cache_write(c or cache(), **a)


def attend(c=None, **over):
    a = dict(q=zeros(2, 4, 64), block_table=torch.zeros(2, 2, dtype=torch.int32),
             lengths=torch.zeros(2, dtype=torch.int32))
    a.update(over)
    return at.paged_attention(cache=c or cache(), **a)


def join(**over):
    a = dict(outs=torch.zeros(2, 3, 4, 64), lses=torch.zeros(2, 3, 4))
    a.update(over)
    return at.attention_join(**a)


# ---- forward-mode derivatives ---------------------------------------------------------------------------------------

def dual(x):
    return fwd.make_dual(x, torch.ones_like(x))


@pytest.mark.parametrize("call", [
    lambda: norm_rope(q=dual(zeros(3, 4, 64, dtype=F32))),
    lambda: norm_rope(k=dual(zeros(3, 2, 64, dtype=F32))),
    lambda: norm_rope(q_weight=dual(torch.ones(64))),
    lambda: norm_rope(k_weight=dual(torch.ones(64))),
    lambda: norm_rope(table=dual(torch.zeros(8, 64))),
    lambda: write(k=dual(zeros(3, 2, 64))),
    lambda: write(v=dual(zeros(3, 2, 64))),
    lambda: at.KvCache(dual(zeros(4, 2, 16, 64)), zeros(4, 2, 16, 64)),
    lambda: at.KvCache(zeros(4, 2, 16, 64, dtype=E4M3), zeros(4, 2, 16, 64, dtype=E4M3), torch.ones(4, 2, 16),
                       dual(torch.ones(4, 2, 16))),
    lambda: attend(q=dual(zeros(2, 4, 64))),
    lambda: attend(out=dual(zeros(2, 4, 64))),
    lambda: attend(lse=dual(torch.zeros(2, 4))),
    lambda: join(outs=dual(torch.zeros(2, 3, 4, 64))),
    lambda: join(lses=dual(torch.zeros(2, 3, 4))),
    lambda: join(out=dual(torch.zeros(3, 4, 64))),
])
def test_dual_tensors_are_refused(call):
    with fwd.dual_level():
        with pytest.raises(ValueError, match="no forward-mode derivative"):
            call()


def test_primals_within_a_dual_level_pass():
    with fwd.dual_level():
        for call in (norm_rope, write, attend, join):
            with pytest.raises(ValueError, match="CUDA device"):
                call()
        q = fwd.unpack_dual(dual(zeros(2, 4, 64))).primal
        with pytest.raises(ValueError, match="CUDA device"):
            attend(q=q)


# ---- torch.func transforms ------------------------------------------------------------------------------------------

@pytest.mark.parametrize("call", [
    lambda: torch.func.vmap(lambda q: norm_rope(q=q))(zeros(2, 3, 4, 64, dtype=F32)),
    lambda: torch.func.grad(lambda q: norm_rope(q=q)[0].sum())(zeros(3, 4, 64, dtype=F32)),
    lambda: torch.func.jvp(lambda t: norm_rope(table=t)[0], (torch.zeros(8, 64),), (torch.ones(8, 64),)),
    lambda: torch.func.functionalize(lambda w: norm_rope(q_weight=w)[0])(torch.ones(64)),
    lambda: torch.func.vmap(lambda k: write(k=k) or k)(zeros(2, 3, 2, 64)),
    lambda: torch.func.vmap(lambda at_: at.kv_cache_read(cache(), at_)[0])(torch.zeros(2, 3, dtype=torch.int64)),
    lambda: torch.func.vmap(lambda k: at.KvCache(k, zeros(4, 2, 16, 64)) and k)(zeros(2, 4, 2, 16, 64)),
    lambda: torch.func.vmap(lambda q: attend(q=q))(zeros(3, 2, 4, 64)),
    lambda: torch.func.grad(lambda q: attend(q=q).float().sum())(zeros(2, 4, 64)),
    lambda: torch.func.vmap(lambda out: attend(out=out))(zeros(3, 2, 4, 64)),
    lambda: torch.func.vmap(lambda n: attend(lengths=n))(torch.zeros(3, 2, dtype=torch.int32)),
    lambda: torch.func.vmap(lambda outs: join(outs=outs)[0])(torch.zeros(5, 2, 3, 4, 64)),
    lambda: torch.func.jvp(lambda l: join(lses=l)[1], (torch.zeros(2, 3, 4),), (torch.ones(2, 3, 4),)),
])
def test_transforms_are_refused_by_the_operators_themselves(call):
    with pytest.raises(ValueError, match="torch.func transform"):
        call()


# ---- gradients that no operator computes ----------------------------------------------------------------------------

@pytest.mark.parametrize("leaves", [False, True])
def test_a_table_that_requires_a_gradient_is_refused(leaves):
    """Alone its gradient would be cut off, beside trained inputs undefined: frequencies that never train."""
    frequencies = torch.full((32,), 0.5, requires_grad=True)
    table = at.rope_table(8, 64, frequencies=frequencies)
    assert table.requires_grad
    q = zeros(3, 4, 64, dtype=F32, requires_grad=leaves)
    with pytest.raises(ValueError, match="gradient for its table"):
        norm_rope(q=q, table=table)
    for fine in (lambda: norm_rope(q=q, table=table.detach()), torch.no_grad()(lambda: norm_rope(q=q, table=table))):
        with pytest.raises(ValueError, match="CUDA device"):
            fine()


@pytest.mark.parametrize("which", ["k_scale", "v_scale"])
def test_factors_that_require_a_gradient_are_refused(which):
    """At construction, and at a call where they came to require one later."""
    c = cache(E4M3)
    parts = dict(k=c.k, v=c.v, k_scale=c.k_scale, v_scale=c.v_scale)
    parts[which] = torch.zeros(4, 2, 16, requires_grad=True)
    with pytest.raises(ValueError, match="cannot require a gradient"):
        at.KvCache(**parts)
    getattr(c, which).requires_grad_()
    for call in (write, attend, lambda c: at.kv_cache_read(c, torch.arange(3))):
        with pytest.raises(ValueError, match="cannot require a gradient"):
            call(c)


@pytest.mark.parametrize("call", [
    lambda: attend(out=zeros(2, 4, 64, requires_grad=True)),
    lambda: attend(out=zeros(2, 4, 64, requires_grad=True) * 2),
    lambda: attend(lse=torch.zeros(2, 4, requires_grad=True)),
    lambda: join(out=torch.zeros(3, 4, 64, requires_grad=True)),
])
def test_given_results_that_require_a_gradient_are_refused(call):
    """A result written over a tensor that autograd follows would leave the graph with another tensor's gradient."""
    with pytest.raises(ValueError, match="no backward pass"):
        call()
    with torch.no_grad(), pytest.raises(ValueError, match="CUDA device"):
        call()


# ---- shared memory --------------------------------------------------------------------------------------------------

def test_writes_into_tensors_that_share_memory_are_refused():
    """Keys and values of one call would be written to the same rows by different threads, in no order."""
    one = zeros(5, 2, 16, 64)
    codes, factors = zeros(4, 2, 16, 64, dtype=E4M3), [torch.ones(4, 2, 16) for _ in range(2)]
    shared = [at.KvCache(one[:4], one[:4]), at.KvCache(one[:4], one[1:]),
              at.KvCache(codes, codes, *factors),
              at.KvCache(codes, codes.clone(), factors[0], factors[0]),
              at.KvCache(codes, codes.clone(), codes.view(F32).view(-1)[:128].view(4, 2, 16), factors[0])]
    for c in shared:
        with pytest.raises(ValueError, match="share memory with one another"):
            write(c)
        with pytest.raises(ValueError, match="CUDA device"):       # read they may be
            at.kv_cache_read(c, torch.arange(3))
    c = cache()
    rows = c.k.view(-1)[:3 * 2 * 64].view(3, 2, 64)
    for over in (dict(k=rows), dict(v=rows), dict(slots=c.v.view(torch.int64).view(-1)[:3])):
        with pytest.raises(ValueError, match="shares memory with the cache"):
            write(c, **over)
    apart = at.KvCache(one[:2], one[2:4])
    with pytest.raises(ValueError, match="CUDA device"):
        write(apart)


# ---- numbers that are another number in the kernels' type -----------------------------------------------------------

@pytest.mark.parametrize("over", [dict(softcap=1e-50), dict(softcap=1e-40), dict(softcap=1e-31), dict(scale=1e-50),
                                  dict(scale=1e-40), dict(softcap=1e31), dict(scale=float("inf"))])
def test_scales_and_caps_out_of_range_are_refused(over):
    """A cap that becomes zero in 32 bits was no cap."""
    with pytest.raises(ValueError, match="scale"):
        attend(**over)
    for fine in (dict(softcap=1e-30), dict(scale=1e-30), dict(softcap=0.0), dict(softcap=9e29), dict(scale=9e29)):
        with pytest.raises(ValueError, match="CUDA device"):
            attend(**fine)


@pytest.mark.parametrize("eps", [-1e-6, float("nan"), float("inf"), -float("inf"), 1e39, 1e-50, 5e-324])
def test_eps_out_of_range_is_refused(eps):
    """One below zero or NaN gives NaN; one that becomes zero in 32 bits makes rows of zeros NaN, which have a norm."""
    with pytest.raises(ValueError, match="eps"):
        norm_rope(eps=eps)
    for fine in (0.0, 0, 1e-45, 1e-6, 1e-3, 3e38):
        with pytest.raises(ValueError, match="CUDA device"):
            norm_rope(eps=fine)


# ---- slots ----------------------------------------------------------------------------------------------------------

def test_slots_of_sequences_that_the_table_does_not_have():
    """A negative sequence (padding of a batch) is not the last one counted from the end, whose tokens a write would
    replace, and one past the table is no index out of range, which on a GPU ends the process."""
    table = torch.tensor([[4, 2, -1], [0, 7, 1]], dtype=torch.int32)
    seq = torch.tensor([-1, -2, 2, 2 ** 31 - 1, 0, 1, -2 ** 31])
    pos = torch.tensor([0, 17, 0, 5, 17, 33, 0])
    for s, p in ((seq, pos), (seq.int(), pos.int())):
        got = at.token_slots(table, s, p, 16)
        assert got.dtype == torch.int64 and got.tolist() == [-1, -1, -1, -1, 33, 17, -1]
    assert at.token_slots(table[:0], seq, pos, 16).tolist() == [-1] * 7
    assert at.token_slots(table, seq[:0], pos[:0], 16).tolist() == []


# ---- the table of angles --------------------------------------------------------------------------------------------

def test_a_table_lies_where_its_frequencies_do():
    """Without a device of its own (here one without memory stands for the GPU)."""
    f = torch.full((16,), 0.5)
    assert at.rope_table(8, 32, frequencies=f.to("meta")).device.type == "meta"
    assert at.rope_table(8, 32, frequencies=f).device.type == "cpu"
    assert at.rope_table(8, 32, frequencies=f, device="meta").device.type == "meta"
    assert at.rope_table(8, 32).device.type == "cpu" and at.rope_table(8, 32, device="meta").device.type == "meta"
