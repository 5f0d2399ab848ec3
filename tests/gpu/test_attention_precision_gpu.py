"""How far the gfx950 attention kernels are from the definition in 64 bits, in units of what rounding the
exact result once leaves (root mean squares, so that no bound per element can hide a lost correction).

Independent roundings add in squares: results whose operands P and dS were rounded to the same type are
sqrt(2) = 1.42 times as far off as rounded results at most, so up to 1.5 is right for them."""

import math

import pytest
import torch

from nanofed_amd.ops import attention as A
from tests import transformer_oracles as oracle

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, FP = torch.bfloat16, torch.float16
TWO_ROUNDINGS = 1.5


def rand(*shape, seed, dtype, scale=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype)


def inputs(B, Tq, Tk, H, Hk, D, dtype, dout=1.0, q=1.0, k=1.0):
    return (rand(B, Tq, H, D, seed=1, dtype=dtype, scale=q), rand(B, Tk, Hk, D, seed=2, dtype=dtype, scale=k),
            rand(B, Tk, Hk, D, seed=3, dtype=dtype), rand(B, Tq, H, D, seed=4, dtype=dtype, scale=dout))


def run(q, k, v, dout=None, p=0.0, **how):
    q, k, v = (t.to(DEV) for t in (q, k, v))
    out, lse = A.attention_fwd(q, k, v, dropout=p, **how)
    got = {"out": out}
    if dout is not None:
        got.update({n: torch.full_like(t, math.nan) for n, t in (("dq", q), ("dk", k), ("dv", v))})
        A.attention_bwd(q, k, v, out, lse, dout.to(DEV), got["dq"], got["dk"], got["dv"], dropout=p, **how)
    return got


def off(got, want):
    """Error over that of rounding the exact value once."""
    want, got = want.double(), got.cpu()
    rounded = (want.to(got.dtype).double() - want).square().mean().sqrt()
    return float((got.double() - want).square().mean().sqrt() / rounded)


def check(x, most, p=0.0, names=("dq", "dk", "dv"), **how):
    want = oracle.attention(*x, p=p, **how)
    got = run(*x, p=p, **how)
    ratios = {n: round(off(got[n], want[n][0]), 3) for n in names}
    assert all(r <= most for r in ratios.values()), ratios
    return got


# -- half has the exponents 2^-24 .. 2^15 only ------------------------------------------------------
@pytest.mark.parametrize("dout", [1e2, 1.0, 1e-2, 1e-3, 1e-4, 1e-5])
@pytest.mark.parametrize("D,p", [(64, 0.0), (128, 0.1)])
def test_half_gradients_of_any_size_against_many_keys(dout, D, p):
    check(inputs(1, 2048, 2048, 2, 1, D, FP, dout=dout), TWO_ROUNDINGS, p=p, seed=3)


@pytest.mark.parametrize("T", [33, 300])
@pytest.mark.parametrize("dout", [1e2, 1e-4])
def test_half_gradients_of_short_sequences(T, dout):
    check(inputs(2, T, T, 2, 2, 64, FP, dout=dout), TWO_ROUNDINGS)


def test_half_gradients_of_rows_of_different_sizes():
    """Each query's gradient is as exact as if the others were not there."""
    q, k, v, dout = inputs(1, 512, 512, 1, 1, 64, FP)
    size = 10.0 ** torch.linspace(2, -4, 512)[torch.randperm(512, generator=torch.Generator().manual_seed(1))]
    x = (q, k, v, (dout * size.view(1, -1, 1, 1)).to(FP))
    want, got = oracle.attention(*x), run(*x)
    for name in ("dq", "dk", "dv"):
        assert off(got[name], want[name][0]) <= TWO_ROUNDINGS, name
    small = size < 1e-2  # (their errors vanish in the mean of all rows)
    assert off(got["dq"][:, small], want["dq"][0][:, small]) <= TWO_ROUNDINGS


def test_half_gradients_whose_factors_pass_the_type_though_they_do_not():
    """dS reaches 10^5, dQ and dK stay below 10^3."""
    q, k, v, dout = inputs(1, 300, 300, 1, 1, 64, FP, dout=8e3, q=0.01, k=0.01)
    got = check((q, k, v * 8, dout), TWO_ROUNDINGS)
    assert all(bool(torch.isfinite(t).all()) for t in got.values())


def test_half_value_gradients_of_small_probabilities():
    """20000 keys: probabilities of 5e-5, below the smallest normal half."""
    check(inputs(1, 256, 20000, 1, 1, 64, FP), TWO_ROUNDINGS, causal=False)


def test_half_gradients_beside_a_row_that_is_not_finite():
    """An infinite gradient of one query leaves the other queries' alone, and the keys behind its tile."""
    q, k, v, dout = inputs(1, 200, 200, 1, 1, 64, FP, dout=1e-4)
    want = oracle.attention(q, k, v, dout)
    bad = dout.clone()
    bad[0, 10] = math.inf
    got = run(q, k, v, bad)
    assert not bool(torch.isfinite(got["dq"][:, 10]).all())
    rows = torch.arange(200) != 10
    assert off(got["dq"][:, rows.to(DEV)], want["dq"][0][:, rows]) <= TWO_ROUNDINGS
    for name in ("dk", "dv"):  # (query 10 sees keys 0 .. 10)
        assert off(got[name][:, 64:], want[name][0][:, 64:]) <= TWO_ROUNDINGS, name


@pytest.mark.parametrize("dtype", [FP, BF])
@pytest.mark.parametrize("Tq,D", [(40, 8), (1, 8), (40, 128)])
def test_many_small_probabilities_behind_a_large_one(dtype, Tq, D):
    """2^20 keys that each have e^-18 of the first one's weight have 1.6 % of it together."""
    n, big = 1 << 20, 18.0
    q, k = torch.zeros(1, Tq, 1, D, dtype=dtype, device=DEV), torch.zeros(1, n, 1, D, dtype=dtype, device=DEV)
    v = torch.ones(1, n, 1, D, dtype=dtype, device=DEV)
    q[..., 0], k[0, 0, 0, 0], v[0, 0] = 1.0, big, 0.0
    out, lse = A.attention_fwd(q, k, v, scale=1.0, causal=False)
    tail = (n - 1) * math.exp(-big)
    # equal terms round alike: one rounding of P, one of the result, and 2^16 additions (16 keys each) in fp32
    bound = 2 * oracle.UNIT[dtype] + 2.0**16 * 2.0**-24
    assert float((out.double() / (tail / (1 + tail)) - 1).abs().max()) <= bound
    # the sum of the probabilities is about 1 from the first key on, and each of 2^15 additions (32 keys) to it is
    # off by up to 2^-24 of that, alike again
    assert float((lse.double() - (big + math.log1p(tail))).abs().max()) <= big * 2.0**-22 + 2.0**15 * 2.0**-24 * (1 + tail)


# -- which roundings are undone ---------------------------------------------------------------------
ONE_ROUNDING = 1.1  # (sums in fp32 and what is left of the two roundings come on top)


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("B,T,H,Hk,D", [(1, 64, 1, 1, 64), (2, 33, 2, 2, 128), (40, 64, 12, 12, 64), (300, 9, 8, 2, 64)])
@pytest.mark.parametrize("p", [0.0, 0.2])
def test_gradients_of_short_sequences_are_off_by_one_rounding(dtype, B, T, H, Hk, D, p):
    check(inputs(B, T, T, H, Hk, D, dtype), ONE_ROUNDING, p=p, seed=4)


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("B,T,H,Hk,D", [(1, 65, 2, 2, 64), (2, 129, 4, 1, 64), (1, 700, 1, 1, 64), (3, 300, 2, 2, 128)])
def test_longer_sequences_are_off_by_two_roundings(dtype, B, T, H, Hk, D):
    check(inputs(B, T, T, H, Hk, D, dtype), TWO_ROUNDINGS, names=("out", "dq", "dk", "dv"))


@pytest.mark.parametrize("dtype,D", [(BF, 64), (FP, 64), (BF, 128)])
@pytest.mark.parametrize("B,Tq,Tk,H,Hk", [(1, 1, 700, 1, 1), (1, 1, 77, 4, 4), (9, 2, 2050, 8, 1), (3, 4, 900, 8, 2), (2, 16, 300, 3, 3)])
def test_up_to_16_rows_that_share_keys_are_off_by_one_rounding(dtype, D, B, Tq, Tk, H, Hk):
    check(inputs(B, Tq, Tk, H, Hk, D, dtype)[:3], ONE_ROUNDING, names=("out",))


@pytest.mark.parametrize("B,Tq,Tk,H,Hk", [(2, 17, 700, 4, 4), (2, 5, 1500, 8, 1), (2, 32, 1024, 4, 2)])
def test_more_rows_are_off_by_two_roundings(B, Tq, Tk, H, Hk):
    check(inputs(B, Tq, Tk, H, Hk, 64, BF)[:3], TWO_ROUNDINGS, names=("out",))


@pytest.mark.parametrize("T,most", [(64, ONE_ROUNDING), (200, TWO_ROUNDINGS)])
@pytest.mark.parametrize("dtype", [BF, FP])
def test_gradients_where_the_rounding_of_the_output_counts(T, most, dtype):
    """Values with a common offset make an output whose rounding, were D = rowsum(dO * O) left as it is, would
    outweigh the other two."""
    q, k, v, dout = inputs(1, T, T, 2, 2, 64, dtype)
    check((q, k, (v.float() + 64).to(dtype), dout), most, names=("dq", "dk"))


@pytest.mark.parametrize("T", [7, 64, 128])
def test_a_sequence_has_the_same_bits_whatever_shares_its_launch(T):
    B, H, D = 96, 12, 64
    x = [t.to(DEV) for t in inputs(B, T, T, H, H, D, BF)]
    whole = run(*x[:3], x[3], p=0.1, seed=3, step=2)
    for b in (0, 41, 95):
        alone = run(*(t[b:b + 1] for t in x[:3]), x[3][b:b + 1], p=0.1, seed=3, step=2, first_batch=b)
        assert all(torch.equal(alone[n][0], whole[n][b]) for n in whole), b


def test_a_token_has_the_same_bits_whatever_shares_its_launch():
    B, Tk, H, D = 96, 120, 12, 64
    q, k, v, _ = (t.to(DEV) for t in inputs(B, 1, Tk, H, H, D, BF))
    whole = run(q, k, v)["out"]
    for b in (0, 41, 95):
        assert torch.equal(run(q[b:b + 1], k[b:b + 1], v[b:b + 1])["out"][0], whole[b]), b


# -- half: what the factors must not depend on --------------------------------------------------------
@pytest.mark.parametrize("Tq,Tk,D,p", [(90, 90, 64, 0.2), (300, 300, 128, 0.0), (64, 50, 64, 0.0), (600, 200, 64, 0.1)])
def test_half_gradients_do_not_depend_on_what_lies_behind_the_lengths(Tq, Tk, D, p):
    q, k, v, dout = inputs(3, Tq, Tk, 2, 1, D, FP, dout=1e-3)
    nq, nk = [Tq // 2, 0, Tq], [Tk // 2, 0, Tk]
    how = dict(q_lengths=torch.tensor(nq, dtype=torch.int32, device=DEV),
               k_lengths=torch.tensor(nk, dtype=torch.int32, device=DEV), p=p, seed=6)
    ref = None
    for junk in (0.0, math.nan, math.inf, 6e4):
        x = [t.clone() for t in (q, k, v, dout)]
        for b in range(3):
            x[0][b, nq[b]:], x[3][b, nq[b]:] = junk, junk
            x[1][b, nk[b]:], x[2][b, nk[b]:] = junk, junk
        got = run(*x[:3], x[3], **how)
        ref = ref or got
        assert all(torch.equal(got[n], ref[n]) for n in got), junk
    assert all(bool((ref[n][1] == 0).all()) for n in ref)


def test_half_gradients_of_nothing_and_of_the_largest_and_smallest_values():
    q, k, v, dout = inputs(2, 150, 150, 2, 2, 64, FP)
    none = run(q, k, v, dout * 0)
    assert all(bool((none[n] == 0).all()) for n in ("dq", "dk", "dv"))
    # the largest half where the gradients fit all the same, the smallest where they are steps of 2^-24 themselves
    check((q * 2**-12, k * 2**-12, v, dout.sign() * 65504), TWO_ROUNDINGS, names=("dq", "dk"))
    check((q, k, v * 64, dout.sign() * 2**-24), TWO_ROUNDINGS)


def test_half_gradients_in_two_graphs_that_are_replayed_in_turn():
    x = [[t.to(DEV) for t in inputs(2, 330, 330, 4, 2, 64, FP, dout=s)] for s in (1e-4, 1e2)]

    def make(q, k, v, _):
        return [torch.empty_like(q), torch.empty(2, 4, 330, device=DEV), torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)]

    def go(x, b):
        A.attention_fwd(*x[:3], b[0], b[1], dropout=0.1, seed=2)
        A.attention_bwd(*x[:3], b[0], b[1], x[3], *b[2:], dropout=0.1, seed=2)

    eager, bufs, graphs = [make(*y) for y in x], [make(*y) for y in x], [torch.cuda.CUDAGraph() for _ in x]
    for y, b in zip(x, eager):
        go(y, b)
    torch.cuda.synchronize()
    for y, b, graph in zip(x, bufs, graphs):
        with torch.cuda.graph(graph):
            go(y, b)
    for _ in range(3):
        for b in bufs:
            for t in b:
                t.zero_()
        for graph in graphs:
            graph.replay()
        make(*x[0])
        torch.cuda.synchronize()
        for b, e in zip(bufs, eager):
            assert all(torch.equal(s, t) for s, t in zip(b, e))
