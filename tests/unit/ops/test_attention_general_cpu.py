"""The PyTorch paths of ``attention_fwd`` / ``attention_bwd`` against the definition in 64 bits
and against differences, and what the operator refuses."""

import math

import pytest
import torch

from nanofed_amd.core.exceptions import DeviceError
from nanofed_amd.ops import attention as A
from nanofed_amd.ops import library
from tests import transformer_oracles as oracle

F64 = torch.float64


def rand(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed), dtype=F64)


def case(B, Tq, Tk, H, Hk, D):
    return rand(B, Tq, H, D, seed=1), rand(B, Tk, Hk, D, seed=2), rand(B, Tk, Hk, D, seed=3), rand(B, Tq, H, D, seed=4)


def ints(*x):
    return torch.tensor(x, dtype=torch.int32)


CASES = [
    (2, 7, 7, 2, 2, 8, dict()),
    (2, 5, 9, 4, 2, 16, dict(p=0.3, seed=11, step=5)),
    (1, 9, 5, 2, 1, 8, dict(p=0.1, seed=(1 << 64) - 1, step=(1 << 32) - 1)),  # four queries see nothing
    (3, 6, 6, 2, 1, 8, dict(q_lengths=ints(0, 6, 3), k_lengths=ints(0, 6, 3), p=0.2, first_batch=7)),
    (2, 4, 6, 2, 2, 8, dict(causal=False, k_lengths=ints(0, 9), scale=0.7)),
    (1, 1, 1, 1, 1, 8, dict()),
]


@pytest.mark.parametrize("B,Tq,Tk,H,Hk,D,how", CASES)
def test_against_the_definition_and_differences(B, Tq, Tk, H, Hk, D, how):
    q, k, v, dout = case(B, Tq, Tk, H, Hk, D)
    mine = {**how, "dropout": how.get("p", 0.0)}
    mine.pop("p", None)
    want = oracle.attention(q, k, v, dout, **how)
    out, lse = A.attention_fwd(q, k, v, lse=torch.empty(B, H, Tq), **mine)
    dq, dk, dv = torch.full_like(q, math.nan), torch.full_like(k, math.nan), torch.full_like(v, math.nan)
    A.attention_bwd(q, k, v, out, lse, dout, dq, dk, dv, **mine)
    # the oracle's scale is a 64-bit number, the operator's a 32-bit one
    for name, x in (("out", out), ("lse", lse), ("dq", dq), ("dk", dk), ("dv", dv)):
        fine = torch.isfinite(want[name][0])
        assert torch.equal(x.double()[~fine], want[name][0][~fine])
        torch.testing.assert_close(x.double()[fine], want[name][0][fine], rtol=2e-6, atol=2e-6)

    def loss(q, k, v):
        return float((A.attention_fwd(q, k, v, lse=torch.empty(B, H, Tq), **mine)[0] * dout).sum())

    step = 1e-6
    for which, grad in enumerate((dq, dk, dv)):
        direction = rand(*grad.shape, seed=9)
        at = [q, k, v]
        hi, lo = list(at), list(at)
        hi[which], lo[which] = at[which] + step * direction, at[which] - step * direction
        # central difference: off by step^2 times the third derivative, and 1e-15 / step
        assert (loss(*hi) - loss(*lo)) / (2 * step) == pytest.approx(float((grad * direction).sum()), abs=1e-5, rel=1e-5)


def test_what_lies_behind_the_lengths_does_not_matter():
    q, k, v, dout = case(2, 6, 6, 2, 1, 8)
    n = ints(4, 0)
    ref = None
    for junk in (0.0, math.nan, math.inf):
        x = [t.clone() for t in (q, k, v, dout)]
        for t in x:
            t[0, 4:] = junk
            t[1] = junk
        how = dict(q_lengths=n, k_lengths=n, dropout=0.2, seed=3)
        out, lse = A.attention_fwd(*x[:3], lse=torch.empty(2, 2, 6), **how)
        g = [torch.empty_like(t) for t in x[:3]]
        A.attention_bwd(*x[:3], out, lse, x[3], *g, **how)
        got = [out, lse, *g]
        assert all(bool((t[1] == 0).all()) for t in (out, *g)) and bool((lse[1] == -math.inf).all())
        ref = ref or got
        assert all(torch.equal(a, b) for a, b in zip(ref, got))


def test_masks_of_a_batch_done_in_parts_are_those_of_the_whole():
    q, k, v, _ = case(4, 5, 5, 2, 2, 8)
    whole, _ = A.attention_fwd(q, k, v, lse=torch.empty(4, 2, 5), dropout=0.4, seed=8, step=2)
    for b in (0, 1, 3):
        part, _ = A.attention_fwd(q[b:b + 1], k[b:b + 1], v[b:b + 1], lse=torch.empty(1, 2, 5), dropout=0.4,
                                  seed=8, step=torch.tensor([2]), first_batch=b)
        assert torch.equal(part[0], whole[b])


def test_no_keys_and_no_queries():
    q, k, v, dout = case(2, 3, 4, 2, 2, 8)
    out, lse = A.attention_fwd(q, k[:, :0], v[:, :0], lse=torch.empty(2, 2, 3))
    assert bool((out == 0).all()) and bool((lse == -math.inf).all())
    dq, dk = torch.ones_like(q), torch.ones_like(k[:, :0])
    A.attention_bwd(q, k[:, :0], v[:, :0], out, lse, dout, dq, dk, dk.clone())
    assert bool((dq == 0).all())
    out, _ = A.attention_fwd(q[:, :0], k, v)
    assert out.shape == (2, 0, 2, 8)
    dk, dv = torch.ones_like(k), torch.ones_like(v)
    A.attention_bwd(q[:, :0], k, v, out, torch.empty(2, 2, 0), out, q[:, :0].clone(), dk, dv)
    assert bool((dk == 0).all()) and bool((dv == 0).all())


def test_refusals():
    bf = torch.bfloat16
    q, k = torch.zeros(2, 4, 4, 16, dtype=bf), torch.zeros(2, 6, 2, 16, dtype=bf)
    ok = dict(seed=1)
    bad = [
        (dict(dropout=1.0), "in \\[0, 1\\)"), (dict(dropout=-0.1), "in \\[0, 1\\)"),
        (dict(dropout=0.999), "round below 1"), (dict(dropout=math.nan), "in \\[0, 1\\)"),
        (dict(seed=-1), "seed"), (dict(seed=1 << 64), "seed"), (dict(step=1 << 32), "step"), (dict(step=-1), "step"),
        (dict(step=torch.zeros(2, dtype=torch.int64)), "step"), (dict(step=torch.zeros(1)), "step"),
        (dict(scale=0.0), "scale"), (dict(scale=math.inf), "scale"), (dict(first_batch=-1), "first_batch"),
        (dict(k_lengths=torch.zeros(2, dtype=torch.int64)), "k_lengths"),
        (dict(q_lengths=torch.zeros(3, dtype=torch.int32)), "q_lengths"),
        (dict(out=torch.zeros(2, 4, 4, 16)), "out"), (dict(out=torch.zeros(2, 4, 2, 16, dtype=bf)), "out"),
        (dict(out=torch.zeros(1, 4, 4, 16, dtype=bf).expand(2, 4, 4, 16)), "expanded"),
        (dict(lse=torch.zeros(2, 4, 4, dtype=bf)), "lse"), (dict(lse=torch.zeros(2, 4, 5)), "lse"),
    ]
    for how, match in bad:
        with pytest.raises(DeviceError, match=match):
            A.attention_fwd(q, k, k, **{**ok, **how})
    with pytest.raises(DeviceError, match="share"):
        A.attention_fwd(q, k.new_zeros(2, 6, 3, 16), k.new_zeros(2, 6, 3, 16))
    with pytest.raises(DeviceError, match="head dimension"):
        A.attention_fwd(q[..., :12], k[..., :12], k[..., :12])
    with pytest.raises(DeviceError, match="head dimension"):
        A.attention_fwd(q.new_zeros(1, 1, 1, 136), q.new_zeros(1, 1, 1, 136), q.new_zeros(1, 1, 1, 136))
    with pytest.raises(DeviceError, match="v must be"):
        A.attention_fwd(q, k, k[:, :5])
    with pytest.raises(DeviceError, match="columns"):
        A.attention_fwd(q.transpose(2, 3).contiguous().transpose(2, 3), k, k)
    with pytest.raises(DeviceError, match="\\[batch"):
        A.attention_fwd(q[0], k, k)
    with pytest.raises(DeviceError, match="bfloat16 or float16"):
        A.attention_fwd(q.to(torch.int32), k, k)
    out, lse = A.attention_fwd(q, k, k)
    with pytest.raises(DeviceError, match="dk must be"):
        A.attention_bwd(q, k, k, out, lse, out, q.clone(), q.clone(), k.clone())
    with pytest.raises(DeviceError, match="dq is written"):
        A.attention_bwd(q, k, k, out, lse, out, q[:1].clone().expand_as(q), k.clone(), k.clone())


def test_argument_block_mirrors_the_kernels():
    assert A._PACK.size == library.hip_lib().nf_attention_args_size()


def test_launcher_refuses_what_the_kernels_cannot_take():
    """The C entry itself, with addresses that are never followed: every refusal comes before a
    launch."""
    fn = A._fn("nf_attention")

    def code(type_=1, backward=0, B=1, Tq=1, Tk=1, H=2, Hk=1, D=64, scale=1.0, limit=0, v=(4096, 8, 8, 8),
             q=4096, lse=4096, dv=4096, delta=4096):
        a = A._Args()
        a.B, a.Tq, a.Tk, a.H, a.Hk, a.D, a.scale, a.limit, a.up = B, Tq, Tk, H, Hk, D, scale, limit, 1.0
        a.causal = a.seed = a.step_at = a.step = a.first_head = a.qlen = a.klen = 0
        some = (4096, 8, 8, 8)
        a.q, a.k, a.v = (q, 8, 8, 8), some, v
        return fn(a.pack(lse, some, some, some, some, (dv, 8, 8, 8), delta), type_, backward, None)

    assert code(B=0) == -1 and code(Tk=0) == -1 and code(Hk=0) == -1 and code(H=3, Hk=2) == -1
    assert code(D=12) == -1 and code(D=136) == -1 and code(limit=256) == -1 and code(scale=0.0) == -1
    assert code(scale=math.nan) == -1 and code(type_=0) == -1
    assert code(Tq=(1 << 22) + 1) == -3 and code(B=1 << 23) == -3
    assert code(q=4104) == -2 and code(lse=0) == -2 and code(v=(4096, 0, 4, 0)) == -2
    assert code(v=(4096, 0, 1 << 24, 0)) == -2
    assert code(backward=1, delta=0) == -2 and code(backward=1, dv=0) == -2
    assert code(Tk=4096) == -2  # many keys for one query, and no scratch for the parts
