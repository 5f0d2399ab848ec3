"""gfx950 attention kernels of any length and layout against the definition in 64 bits."""

import math

import pytest
import torch

from nanofed_amd.core.exceptions import DeviceError
from nanofed_amd.ops import attention as A
from tests import transformer_oracles as oracle

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, FP = torch.bfloat16, torch.float16


def rand(*shape, seed=0, dtype=BF, scale=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype)


def ints(x):
    return None if x is None else torch.tensor(x, dtype=torch.int32)


def check(q, k, v, dout, dtype, q_lengths=None, k_lengths=None, p=0.0, grads=None, backward=True, **how):
    want = oracle.attention(q, k, v, dout if backward else None, p=p, q_lengths=q_lengths, k_lengths=k_lengths,
                            unit=oracle.UNIT[dtype], least=oracle.LEAST[dtype], **how)
    d = [t.to(DEV) if not isinstance(t, tuple) else t for t in (q, k, v, dout)]
    mine = dict(how, dropout=p, q_lengths=ints(q_lengths), k_lengths=ints(k_lengths))
    for n in ("q_lengths", "k_lengths"):
        mine[n] = mine[n].to(DEV) if mine[n] is not None else None
    B, Tq, H, D = q.shape
    out = torch.full((B, Tq, H, D), math.nan, dtype=dtype, device=DEV)
    lse = torch.full((B, H, Tq), math.nan, device=DEV)
    A.attention_fwd(*d[:3], out, lse, **mine)
    got = {"out": out, "lse": lse}
    if backward:
        g = [torch.full(t.shape, math.nan, dtype=dtype, device=DEV) for t in (q, k, v)]
        A.attention_bwd(*d[:3], out, lse, d[3], *g, **mine)
        got.update(dq=g[0], dk=g[1], dv=g[2])
    for name, x in got.items():
        oracle.within(name, x, *want[name])
    return got


def inputs(B, Tq, Tk, H, Hk, D, dtype):
    return (rand(B, Tq, H, D, seed=1, dtype=dtype), rand(B, Tk, Hk, D, seed=2, dtype=dtype),
            rand(B, Tk, Hk, D, seed=3, dtype=dtype), rand(B, Tq, H, D, seed=4, dtype=dtype))


@pytest.mark.parametrize("T", [1, 2, 31, 32, 33, 64, 65, 127, 128, 129, 200])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("p", [0.0, 0.3])
def test_self_attention_of_any_length(T, D, p):
    check(*inputs(2, T, T, 2, 2, D, BF), BF, p=p, seed=5, step=9)


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("D", [8, 32, 40, 64, 72, 80, 120, 128])
def test_head_dimensions(dtype, D):
    check(*inputs(1, 70, 70, 3, 1, D, dtype), dtype, p=0.1, seed=1)


@pytest.mark.parametrize("H,Hk", [(4, 4), (4, 2), (6, 1), (8, 1)])
@pytest.mark.parametrize("p", [0.0, 0.5])
def test_shared_key_heads(H, Hk, p):
    check(*inputs(2, 97, 97, H, Hk, 64, BF), BF, p=p, seed=3, step=1)


@pytest.mark.parametrize("Tq,Tk", [(1, 1), (1, 77), (1, 513), (3, 400), (5, 64), (40, 200), (200, 40), (130, 1), (33, 32)])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("p", [0.0, 0.2])
def test_other_numbers_of_queries_and_keys(Tq, Tk, causal, p):
    # more queries than keys: the first ones see nothing
    check(*inputs(2, Tq, Tk, 4, 2, 64, BF), BF, causal=causal, p=p, seed=8)


@pytest.mark.parametrize("dtype,D", [(BF, 64), (FP, 128)])
@pytest.mark.parametrize("causal", [True, False])
def test_lengths_of_each_sequence(dtype, D, causal):
    n = [0, 1, 64, 150, 129, 33]
    check(*inputs(6, 150, 150, 2, 1, D, dtype), dtype, q_lengths=n, k_lengths=n, p=0.2, causal=causal, seed=2)
    # a cache longer than the queries; more queries than keys; lengths outside [0, T]
    check(*inputs(6, 20, 150, 2, 1, D, dtype), dtype, q_lengths=[20, 0, 5, 25, 7, 20], k_lengths=[150, 9, 0, 200, 3, 64],
          p=0.2, causal=causal, seed=2)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("q_lengths,k_lengths", [([700, 130, 3, 0], [700, 130, 3, 0]), ([5, 700, 260, 64], [512, 300, 260, 129]),
                                                 (None, None)])
def test_gradients_of_keys_that_many_queries_share(D, causal, q_lengths, k_lengths):
    """Long and short sums over the queries of eight heads in one launch."""
    check(*inputs(4, 700, 512 if k_lengths and k_lengths[0] == 512 else 700, 8, 1, D, BF), BF, q_lengths=q_lengths,
          k_lengths=k_lengths, causal=causal, p=0.1, seed=6)


@pytest.mark.parametrize("Tq,Tk,H,Hk", [(1, 700, 4, 4), (1, 2050, 8, 1), (2, 333, 12, 3), (5, 90, 6, 1)])
@pytest.mark.parametrize("D", [64, 128])
def test_few_queries_against_a_cache(Tq, Tk, H, Hk, D):
    keys = [Tk, 1, Tk // 2 + 1, 0]
    check(*inputs(4, Tq, Tk, H, Hk, D, BF), BF, q_lengths=[min(Tq, n) for n in keys], k_lengths=keys, backward=False)


@pytest.mark.parametrize("Tq,Tk,H,Hk", [(5, 700, 8, 1), (5, 1030, 14, 2), (32, 1024, 8, 1), (33, 1100, 1, 1), (9, 1500, 28, 1), (1, 1200, 160, 2)])
@pytest.mark.parametrize("causal,dtype,D", [(True, BF, 64), (False, FP, 128)])
def test_few_queries_of_many_heads_against_a_cache(Tq, Tk, H, Hk, causal, dtype, D):
    check(*inputs(3, Tq, Tk, H, Hk, D, dtype), dtype, q_lengths=[Tq, Tq // 2, Tq], k_lengths=[Tk, Tk // 3, 1],
          causal=causal, backward=False)


@pytest.mark.parametrize("B,T,H,D", [(16, 260, 20, 64), (9, 300, 12, 128), (1, 1100, 2, 64), (1, 1061, 2, 128), (2, 513, 1, 40)])
@pytest.mark.parametrize("causal,p", [(True, 0.1), (False, 0.0)])
def test_many_and_few_tiles_of_queries(B, T, H, D, causal, p):
    check(*inputs(B, T, T, H, H, D, FP), FP, causal=causal, p=p, seed=2)


@pytest.mark.parametrize("D", [64, 128])
def test_few_long_sequences_of_different_lengths(D):
    check(*inputs(3, 600, 900, 2, 1, D, BF), BF, q_lengths=[600, 0, 333], k_lengths=[700, 900, 130], p=0.2, seed=4)


def test_scores_far_apart_and_equal():
    q, k, v, dout = inputs(1, 96, 96, 2, 2, 64, BF)
    check(q * 8, k * 4, v, dout, BF, p=0.1)          # near one-hot rows
    check(q * 0, k, v, dout, BF, p=0.1)              # uniform rows
    check(q, k, v, dout, BF, scale=0.5)


def test_strided_views_and_neighbours_left_alone():
    B, T, H, D = 2, 75, 3, 64
    qkv = rand(B, T, 3, H, D, seed=7)
    dout = rand(B, T, H, D, seed=8)
    want = check(*qkv.unbind(2), dout, BF, p=0.1, seed=4)
    # packed gradients, q | k | v and a fourth part that nobody may touch
    dev, grad = qkv.to(DEV), torch.full((B, T, 4, H, D), 7.0, dtype=BF, device=DEV)
    A.attention_bwd(*dev.unbind(2), want["out"], want["lse"], dout.to(DEV), *grad.unbind(2)[:3], dropout=0.1, seed=4)
    for i, n in enumerate(("dq", "dk", "dv")):
        assert torch.equal(grad[:, :, i], want[n])
    assert bool((grad[:, :, 3] == 7.0).all())
    # heads before rows, and an output row in a wider matrix
    q, k, v = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in dev.unbind(2))
    wide = torch.full((B, T, H + 1, D), 7.0, dtype=BF, device=DEV)
    A.attention_fwd(q, k, v, wide[:, :, :H], want["lse"].clone(), dropout=0.1, seed=4)
    assert torch.equal(wide[:, :, :H], want["out"]) and bool((wide[:, :, H] == 7.0).all())
    # keys and values shared by the batch (expanded)
    k1, v1 = k[:1].expand_as(k), v[:1].expand_as(v)
    a, _ = A.attention_fwd(q, k1, v1)
    b, _ = A.attention_fwd(q, k1.contiguous(), v1.contiguous())
    assert torch.equal(a, b)


@pytest.mark.parametrize("Tq,D,p", [(90, 64, 0.2), (90, 128, 0.0), (1, 64, 0.0)])
def test_what_lies_behind_the_lengths_does_not_matter(Tq, D, p):
    B, Tk = 3, 90
    q, k, v, dout = inputs(B, Tq, Tk, 2, 1, D, BF)
    nk, nq = [70, 0, 90], [min(Tq, 70), 0, Tq]
    ref = None
    for junk in (0.0, math.nan, math.inf):
        x = [t.clone() for t in (q, k, v, dout)]
        for b in range(B):
            x[0][b, nq[b]:], x[3][b, nq[b]:] = junk, junk
            x[1][b, nk[b]:], x[2][b, nk[b]:] = junk, junk
        x = [t.to(DEV) for t in x]
        how = dict(q_lengths=ints(nq).to(DEV), k_lengths=ints(nk).to(DEV), dropout=p, seed=6)
        out, lse = A.attention_fwd(*x[:3], **how)
        g = [torch.full_like(t, math.nan) for t in x[:3]]
        A.attention_bwd(*x[:3], out, lse, x[3], *g, **how)
        got = [out, lse, *g]
        ref = ref or got
        assert all(torch.equal(a, b) for a, b in zip(ref, got)), junk
    assert bool((ref[0][1] == 0).all()) and bool((ref[1][1] == -math.inf).all())


def test_a_long_cache_beyond_32_bit_offsets():
    # 5.4 GB of keys in rows 16 KB apart: offsets pass 2^31 elements
    rows, pitch, D = 330_000, 8192, 64
    store = torch.zeros(rows, pitch, dtype=BF, device=DEV)
    T = rows - 5
    k = store[:T, :D].view(1, T, 1, D)
    v = store[:T, D:2 * D].view(1, T, 1, D)
    k[0, -1, 0, 0] = 40.0
    v[0, -1, 0] = torch.arange(D, device=DEV).to(BF)
    v[0, 0, 0] = 5.0
    q = torch.zeros(1, 1, 1, D, dtype=BF, device=DEV)
    q[..., 0] = 8.0
    out, lse = A.attention_fwd(q, k, v)  # score of the last key: 40; the others: 0
    w = math.exp(40.0)
    assert float(lse) == pytest.approx(math.log(w + T - 1), rel=1e-6)
    torch.testing.assert_close(out[0, 0, 0].float(), torch.arange(D, device=DEV).float(), rtol=2**-7, atol=1e-3)


def test_repeatable_and_step_in_memory_in_a_graph():
    B, T, H, D = 2, 140, 4, 64
    q, k, v, dout = (t.to(DEV) for t in inputs(B, T, T, H, 2, D, BF))
    step = torch.zeros(1, dtype=torch.int64, device=DEV)

    def make():
        out, lse = torch.empty_like(q), torch.empty(B, H, T, device=DEV)
        return [out, lse, torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)]

    def go(bufs, s):
        A.attention_fwd(q, k, v, bufs[0], bufs[1], dropout=0.25, seed=21, step=s)
        A.attention_bwd(q, k, v, bufs[0], bufs[1], dout, *bufs[2:], dropout=0.25, seed=21, step=s)

    eager = {}
    for n in (0, 1, 7):
        eager[n] = make()
        go(eager[n], n)
        again = make()
        go(again, n)
        assert all(torch.equal(a, b) for a, b in zip(eager[n], again))
    assert not torch.equal(eager[0][0], eager[1][0])
    bufs, two = make(), make()
    graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        go(bufs, step)
    with torch.cuda.graph(other):
        go(two, 7)
    for n in (0, 7, 1, 0):
        step.fill_(n)
        graph.replay()
        other.replay()
        make()  # eager allocations between the replays
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(bufs, eager[n])), n
        assert all(torch.equal(a, b) for a, b in zip(two, eager[7])), n


def test_two_streams_at_once():
    q, k, v, _ = (t.to(DEV) for t in inputs(2, 1, 3000, 8, 2, 64, BF))
    q2 = q * 0.5
    want = [A.attention_fwd(x, k, v)[0] for x in (q, q2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, (s, x) in enumerate(zip(streams, (q, q2))):
            with torch.cuda.stream(s):
                got[i].append(A.attention_fwd(x, k, v)[0])
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in got[i])


def test_refusals_of_device_tensors():
    q = torch.zeros(1, 8, 2, 64, dtype=BF, device=DEV)
    flat = torch.zeros(8 * 128 + 8, dtype=BF, device=DEV)
    with pytest.raises(DeviceError, match="16 bytes"):
        A.attention_fwd(flat[4:4 + 1024].view(1, 8, 2, 64), q, q)
    with pytest.raises(DeviceError, match="16 bytes"):
        A.attention_fwd(q, torch.zeros(1, 8, 2, 68, dtype=BF, device=DEV)[..., :64], q)
    with pytest.raises(DeviceError, match="k must be"):
        A.attention_fwd(q, q.cpu(), q)
    with pytest.raises(DeviceError, match="bfloat16 or float16"):
        A.attention_fwd(q.float(), q.float(), q.float())
    with pytest.raises(DeviceError, match="k_lengths"):
        A.attention_fwd(q, q, q, k_lengths=torch.zeros(1, dtype=torch.int32))
