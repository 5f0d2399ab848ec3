"""gfx950 kernels of ``ops.dropout`` and ``ops.embedding`` against the definitions in 64 bits."""

import math

import pytest
import torch

from nanofed_amd.ops import dropout as D
from nanofed_amd.ops import embedding as E
from tests import transformer_oracles as oracle

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32


def rand(*shape, seed=0, dtype=F32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


@pytest.mark.parametrize("dtype", [F32, BF, FP])
@pytest.mark.parametrize("shape", [(1, 1), (1, 7), (3, 8), (5, 13), (1, 4099), (64, 768), (3, 5, 17)])
@pytest.mark.parametrize("p,first", [(0.1, 0), (0.5, 3), (0.0, 0), (0.9, (1 << 35) + 5)])
def test_dropout(dtype, shape, p, first):
    x, res = rand(*shape, seed=1, dtype=dtype), rand(*shape, seed=2, dtype=dtype)
    f = oracle.row_factor(x.numel(), p, 77, 3, first).view(shape)
    u, e, least = oracle.UNIT[dtype], oracle.E32, oracle.LEAST[dtype]
    how = dict(seed=77, step=3, first=first)
    a = x.double() * f
    y = D.dropout_fwd(x.to(DEV), p, **how)
    oracle.within("out", y, a, (u + 2 * e) * a.abs() + least)
    y = D.dropout_fwd(x.to(DEV), p, residual=res.to(DEV), **how)
    want = a + res.double()
    oracle.within("residual", y, want, u * want.abs() + 3 * e * a.abs() + e * want.abs() + least)
    y = D.dropout_bwd(res.to(DEV), p, out=(g := res.to(DEV)), **how)
    want = res.double() * f
    oracle.within("gradient", g, want, (u + 2 * e) * want.abs() + least)
    assert y is g


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("C", [5, 16, 33, 768])
def test_dropout_of_strided_rows_in_place_and_neighbours(dtype, C):
    R = 37
    wide, res = rand(R, C + 3, seed=1, dtype=dtype).to(DEV), rand(R, C, seed=2, dtype=dtype).to(DEV)
    x = wide[:, 1:C + 1]
    want = D.dropout_fwd(x.contiguous(), 0.3, seed=9, residual=res)
    assert torch.equal(D.dropout_fwd(x, 0.3, seed=9, residual=res), want)
    out = torch.full((R, C + 5), 7.0, dtype=dtype, device=DEV)
    D.dropout_fwd(x, 0.3, seed=9, residual=res, out=out[:, 2:C + 2])
    assert torch.equal(out[:, 2:C + 2], want)
    assert bool((out[:, :2] == 7).all()) and bool((out[:, C + 2:] == 7).all())
    edge = wide.clone()
    D.dropout_fwd(x, 0.3, seed=9, residual=res, out=x)
    assert torch.equal(x, want) and torch.equal(wide[:, 0], edge[:, 0]) and torch.equal(wide[:, C + 1:], edge[:, C + 1:])
    D.dropout_fwd(edge[:, 1:C + 1], 0.3, seed=9, residual=res, out=res)
    assert torch.equal(res, want)


def test_dropped_infinities_and_nans_are_zero():
    x = torch.tensor([math.nan, math.inf, -math.inf] * 64, device=DEV)
    y = D.dropout_fwd(x, 0.5, seed=1).cpu()
    kept = oracle.row_factor(x.numel(), 0.5, 1, 0) > 0
    assert bool((y[~kept] == 0).all()) and not bool(torch.isfinite(y[kept]).any())


def test_dropout_parts_steps_and_graph():
    n = 100_003
    x = rand(n, seed=1, dtype=BF).to(DEV)
    step = torch.zeros(1, dtype=torch.int64, device=DEV)
    eager = [D.dropout_fwd(x, 0.2, seed=4, step=i) for i in range(4)]
    parts = torch.cat([D.dropout_fwd(x[a:b], 0.2, seed=4, step=2, first=a) for a, b in ((0, 13), (13, 4099), (4099, n))])
    assert torch.equal(parts, eager[2])
    out = torch.empty_like(x)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        D.dropout_fwd(x, 0.2, seed=4, step=step, out=out)
        step.add_(1)
    for i in range(4):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager[i])


def embed_case(B, T, V, C, dtype, tokens, how, padding=None, accumulate=False, grad=None, given=False):
    how = dict(how)
    grad = grad or dtype
    table, pos, dout = rand(V, C, seed=2, dtype=dtype), rand(T + 1, C, seed=3, dtype=dtype), rand(B, T, C, seed=4, dtype=dtype)
    old = rand(V, C, seed=5, dtype=grad)
    dtable, dpos = old.to(DEV), torch.full((T + 1, C), 7.0, dtype=grad, device=DEV)
    tok = tokens.to(DEV)
    out = E.embedding_fwd(tok, table.to(DEV), positions=pos.to(DEV), **how)
    order = E.token_order(tok, V, padding) if given else None
    E.embedding_bwd(tok, dout.to(DEV), dtable, dpositions=dpos, padding_idx=padding, accumulate=accumulate, order=order, **how)
    scale = how.get("scale", 1.0)
    f = oracle.row_factor(B * T * C, how.get("dropout", 0.0), how.get("seed", 0), how.get("step", 0), how.get("first", 0)).view(B, T, C)
    inside = (tokens >= 0) & (tokens < V)
    x = torch.where(inside[..., None], table.double()[tokens.clamp(0, V - 1)] * scale, 0.0)
    want = (x + pos[:T].double()) * f
    e = oracle.E32
    oracle.within("out", out, want, oracle.UNIT[dtype] * want.abs() + 4 * e * (x.abs() + pos[:T].double().abs()) * f + oracle.LEAST[dtype])
    u = oracle.UNIT[grad]
    d = dout.double() * f
    oracle.within("dpositions", dpos[:T], d.sum(0), u * d.sum(0).abs() + e * (B + 2) * d.abs().sum(0) + oracle.LEAST[grad])
    assert bool((dpos[T:] == 7.0).all())
    has = inside & (tokens != (padding if padding is not None else -5))
    g, size = torch.zeros(V, C, dtype=torch.float64), torch.zeros(V, C, dtype=torch.float64)
    count = torch.zeros(V, 1, dtype=torch.float64)
    g.index_add_(0, tokens[has], d[has] * scale)
    size.index_add_(0, tokens[has], d[has].abs() * scale)
    count.index_add_(0, tokens[has], torch.ones(int(has.sum()), 1, dtype=torch.float64))
    want = g + old.double() if accumulate else g
    oracle.within("dtable", dtable, want, u * want.abs() + e * (count + 4) * (size + old.double().abs() * accumulate) + oracle.LEAST[grad])
    if accumulate:
        absent = count[:, 0] == 0
        assert torch.equal(dtable.cpu()[absent], old[absent])
    return dtable


def uniform(B, T, V, outside=0):
    return torch.randint(-outside, V + outside, (B, T), generator=torch.Generator().manual_seed(1))


@pytest.mark.parametrize("dtype", [F32, BF, FP])
@pytest.mark.parametrize("B,T,V,C", [(1, 1, 1, 1), (1, 3, 2, 8), (2, 33, 211, 64), (3, 50, 40, 65), (2, 7, 5000, 768), (1, 300, 9, 1030)])
@pytest.mark.parametrize("how", [dict(), dict(scale=2.5, dropout=0.2, seed=5, step=1, first=24)])
def test_embedding(dtype, B, T, V, C, how):
    embed_case(B, T, V, C, dtype, uniform(B, T, V, outside=1), how)


@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("grad", [BF, F32])
def test_embedding_padding_accumulation_and_given_order(accumulate, grad):
    B, T, V, C = 3, 41, 100, 72
    tokens = uniform(B, T, V)
    tokens[:, 20:] = 99
    embed_case(B, T, V, C, BF, tokens, dict(dropout=0.1, seed=2), padding=99, accumulate=accumulate, grad=grad)
    embed_case(B, T, V, C, BF, tokens, dict(dropout=0.1, seed=2), padding=99, accumulate=accumulate, grad=grad, given=True)
    embed_case(B, T, V, C, BF, torch.full_like(tokens, 99), dict(), padding=99, accumulate=accumulate, grad=grad)


@pytest.mark.parametrize("B,T", [(4, 1024), (9, 1000), (20, 1000)])
@pytest.mark.parametrize("kind", ["one", "two", "zipf", "uniform"])
def test_embedding_gradient_of_frequent_tokens(B, T, kind):
    V, C = 3000, 40
    g = torch.Generator().manual_seed(3)
    if kind == "one":
        tokens = torch.full((B, T), 1234)
    elif kind == "two":
        tokens = torch.where(torch.rand(B, T, generator=g) < 0.01, 7, 2999)
    elif kind == "zipf":
        tokens = torch.multinomial(torch.arange(1, V + 1).float() ** -1.0, B * T, replacement=True, generator=g).view(B, T)
    else:
        tokens = uniform(B, T, V)
    a = embed_case(B, T, V, C, F32, tokens, dict(dropout=0.1, seed=1))
    b = embed_case(B, T, V, C, F32, tokens, dict(dropout=0.1, seed=1))
    assert torch.equal(a, b)  # no atomics: the same bits


@pytest.mark.parametrize("R", [1, 2, 255, 256, 257, 4096, 5000, 8191, 20_000, 65_536])
@pytest.mark.parametrize("V", [1, 200, 50_257, 1 << 20])
def test_token_order(R, V):
    tokens = torch.randint(-2, V + 2, (R,), generator=torch.Generator().manual_seed(R + V))
    key, order = E.token_order(tokens.to(DEV), V, padding_idx=V // 2)
    want_key, want_order = E.token_order(tokens, V, padding_idx=V // 2)
    assert torch.equal(key.cpu(), want_key) and torch.equal(order.cpu(), want_order)


@pytest.mark.parametrize("R,V", [(32_768, 1 << 16), (100_001, (1 << 24) + 5), (300_000, 3)])
def test_token_order_of_many_and_large_tokens(R, V):
    """Tiles of several rounds, one to four digits."""
    test_token_order(R, V)


def test_embedding_step_in_a_graph():
    B, T, V, C = 4, 600, 500, 128
    tok, table = uniform(B, T, V).to(DEV), rand(V, C, seed=1, dtype=BF).to(DEV)
    pos, dout = rand(T, C, seed=2, dtype=BF).to(DEV), rand(B, T, C, seed=3, dtype=BF).to(DEV)
    step = torch.zeros(1, dtype=torch.int64, device=DEV)

    def make():
        return torch.empty(B, T, C, dtype=BF, device=DEV), torch.empty_like(table), torch.empty_like(pos)

    def go(bufs, s):
        E.embedding_fwd(tok, table, bufs[0], positions=pos, dropout=0.1, seed=3, step=s)
        E.embedding_bwd(tok, dout, bufs[1], dpositions=bufs[2], dropout=0.1, seed=3, step=s)

    eager = []
    for i in range(3):
        eager.append(make())
        go(eager[i], i)
    bufs = make()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        go(bufs, step)
    for i in (0, 2, 1, 2):
        step.fill_(i)
        graph.replay()
        make()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(bufs, eager[i]))
