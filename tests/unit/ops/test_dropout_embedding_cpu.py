"""The PyTorch paths of ``ops.dropout`` and ``ops.embedding`` against the definitions in 64 bits,
and what the operators refuse."""

import math

import pytest
import torch

from nanofed_amd.core.exceptions import DeviceError
from nanofed_amd.ops import dropout as D
from nanofed_amd.ops import embedding as E
from nanofed_amd.ops import library
from tests import transformer_oracles as oracle

BF = torch.bfloat16


def rand(*shape, seed=0, dtype=torch.float32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


@pytest.mark.parametrize("dtype", [torch.float32, BF, torch.float16])
@pytest.mark.parametrize("shape,p,first", [((3, 7), 0.5, 0), ((1, 1), 0.1, 5), ((5, 16), 0.0, 0), ((2, 3, 5), 0.9, 3),
                                           ((4, 9), 0.25, (1 << 35) + 6)])
def test_dropout(dtype, shape, p, first):
    x, res = rand(*shape, seed=1, dtype=dtype), rand(*shape, seed=2, dtype=dtype)
    f = oracle.row_factor(x.numel(), p, 77, 3, first).view(shape)
    u = oracle.UNIT[dtype]
    y = D.dropout_fwd(x, p, seed=77, step=3, first=first)
    want = x.double() * f
    oracle.within("out", y, want, (u + 2 * oracle.E32) * want.abs() + oracle.LEAST[dtype])
    y = D.dropout_fwd(x, p, seed=77, step=torch.tensor([3]), residual=res, first=first)
    want = want + res.double()
    oracle.within("residual", y, want, u * want.abs() + 3 * oracle.E32 * (x.double() * f).abs() + oracle.E32 * want.abs() + oracle.LEAST[dtype])
    assert torch.equal(D.dropout_bwd(res, p, seed=77, step=3, first=first), D.dropout_fwd(res, p, seed=77, step=3, first=first))


def test_dropout_share_scale_and_independence():
    n = 1 << 16
    x = torch.ones(n)
    y = D.dropout_fwd(x, 0.1, seed=5)
    share = float((y != 0).float().mean())
    keep = 1 - round(0.1 * 65536) / 65536
    assert abs(share - keep) < 5 * math.sqrt(keep * (1 - keep) / n)
    assert torch.allclose(y[y != 0], torch.tensor(1 / keep))
    other = D.dropout_fwd(x, 0.1, seed=5, step=1)
    both = float(((y != 0) & (other != 0)).float().mean())
    assert abs(both - keep * keep) < 5 * math.sqrt(keep * keep * (1 - keep * keep) / n)
    parts = torch.cat([D.dropout_fwd(x[a:b], 0.1, seed=5, first=a) for a, b in ((0, 13), (13, 4099), (4099, n))])
    assert torch.equal(parts, y)


def test_dropped_values_are_zero_whatever_they_were():
    x = torch.tensor([math.nan, math.inf, -math.inf] * 64)
    y = D.dropout_fwd(x, 0.5, seed=1)
    kept = oracle.row_factor(x.numel(), 0.5, 1, 0) > 0
    assert bool((y[~kept] == 0).all()) and not bool(torch.isfinite(y[kept]).any())


def test_dropout_refusals():
    x = torch.zeros(4, 8)
    for how, match in [(dict(p=1.0), "in \\[0, 1\\)"), (dict(p=0.999999), "round below 1"), (dict(seed=-2), "seed"),
                       (dict(step=-1), "step"), (dict(first=-1), "first"), (dict(residual=x.to(BF)), "residual"),
                       (dict(residual=x[:3]), "residual"), (dict(out=x.T), "out")]:
        with pytest.raises(DeviceError, match=match):
            D.dropout_fwd(x, **{"p": 0.5, "seed": 1, **how})
    with pytest.raises(DeviceError, match="float32, bfloat16"):
        D.dropout_fwd(x.long(), 0.5, seed=1)


@pytest.mark.parametrize("B,T,V,C,how", [
    (2, 5, 11, 8, dict()), (3, 4, 7, 5, dict(scale=2.5, dropout=0.3, seed=9, step=4)), (1, 1, 1, 1, dict()),
    (2, 6, 9, 16, dict(padding_idx=3, dropout=0.1, seed=1, first=1000)),
])
@pytest.mark.parametrize("dtype", [torch.float32, BF])
@pytest.mark.parametrize("accumulate", [False, True])
def test_embedding(B, T, V, C, how, dtype, accumulate):
    how = dict(how)
    padding = how.pop("padding_idx", None)
    tokens = torch.randint(-1, V + 1, (B, T), generator=torch.Generator().manual_seed(1))  # some outside
    table, pos, dout = rand(V, C, seed=2, dtype=dtype), rand(T + 2, C, seed=3, dtype=dtype), rand(B, T, C, seed=4, dtype=dtype)
    old = rand(V, C, seed=5, dtype=dtype)
    dtable, dpos = old.clone(), torch.full((T + 2, C), 7.0, dtype=dtype)
    out = E.embedding_fwd(tokens, table, positions=pos, **how)
    E.embedding_bwd(tokens, dout, dtable, dpositions=dpos, padding_idx=padding, accumulate=accumulate, **how)
    scale = how.get("scale", 1.0)
    f = oracle.row_factor(B * T * C, how.get("dropout", 0.0), how.get("seed", 0), how.get("step", 0), how.get("first", 0)).view(B, T, C)
    inside = (tokens >= 0) & (tokens < V)
    x = torch.where(inside[..., None], table.double()[tokens.clamp(0, V - 1)] * scale, 0.0)
    want = (x + pos[:T].double()) * f
    u, e = oracle.UNIT[dtype], oracle.E32
    oracle.within("out", out, want, u * want.abs() + 4 * e * (x.abs() + pos[:T].double().abs()) * f)
    d = dout.double() * f
    oracle.within("dpositions", dpos[:T], d.sum(0), u * d.sum(0).abs() + e * (B + 2) * d.abs().sum(0))
    assert bool((dpos[T:] == 7.0).all())
    has = inside & (tokens != (padding if padding is not None else -5))
    g, size = torch.zeros(V, C, dtype=torch.float64), torch.zeros(V, C, dtype=torch.float64)
    g.index_add_(0, tokens[has], d[has] * scale)
    size.index_add_(0, tokens[has], d[has].abs() * scale)
    want = g + old.double() if accumulate else g
    oracle.within("dtable", dtable, want, u * want.abs() + e * (B * T + 4) * (size + old.double().abs() * accumulate))
    if accumulate:
        absent = torch.ones(V, dtype=torch.bool)
        absent[tokens[has]] = False
        assert torch.equal(dtable[absent], old[absent])


def test_token_order_is_stable_and_puts_what_has_no_gradient_last():
    tokens = torch.tensor([[5, 2, 9, 2], [-1, 5, 3, 2]])
    key, order = E.token_order(tokens, 9, padding_idx=3)
    assert key.tolist() == [2, 2, 2, 5, 5, 9, 9, 9] and order.tolist() == [1, 3, 7, 0, 5, 2, 4, 6]
    assert key.dtype == order.dtype == torch.int32


def test_no_tokens():
    dt = torch.ones(3, 4)
    E.embedding_bwd(torch.zeros(2, 0, dtype=torch.int64), torch.zeros(2, 0, 4), dt, accumulate=True)
    assert bool((dt == 1).all())
    E.embedding_bwd(torch.zeros(2, 0, dtype=torch.int64), torch.zeros(2, 0, 4), dt)
    assert bool((dt == 0).all())
    assert E.embedding_fwd(torch.zeros(0, dtype=torch.int64), dt).shape == (0, 4)


def test_embedding_refusals():
    tok, table, dout = torch.zeros(2, 3, dtype=torch.int64), torch.zeros(5, 4), torch.zeros(2, 3, 4)
    for how, match in [(dict(tokens=tok.int()), "int64"), (dict(tokens=tok[None]), "\\[T\\]"), (dict(table=table.long()), "float matrix"),
                       (dict(positions=table[:2]), "at least 3 rows"), (dict(positions=torch.zeros(3, 5)), "positions"),
                       (dict(out=torch.zeros(2, 3, 5)), "rows of 4"), (dict(out=torch.zeros(2, 3, 4, dtype=BF)), "out"),
                       (dict(dropout=1.0), "in \\[0, 1\\)"), (dict(first=-1), "first")]:
        with pytest.raises(DeviceError, match=match):
            E.embedding_fwd(**{"tokens": tok, "table": table, **how})
    for how, match in [(dict(dtable=table.to(BF)), "dtable"), (dict(dout=dout[:1]), "dout"), (dict(padding_idx=5), "padding"),
                       (dict(padding_idx=-1), "padding"), (dict(dpositions=torch.zeros(3, 4, dtype=BF)), "dpositions"),
                       (dict(order=(torch.zeros(6), torch.zeros(6))), "key"), (dict(dropout=math.nan), "in \\[0, 1\\)")]:
        with pytest.raises(DeviceError, match=match):
            E.embedding_bwd(**{"tokens": tok, "dout": dout, "dtable": table, **how})


def test_argument_blocks_have_the_kernels_layout():
    lib = library.hip_lib()
    assert D._ARGS.size == lib.nf_dropout_args_size()
    assert E._ARGS.size == lib.nf_embedding_args_size()


def test_places_beyond_62_bits_are_refused():
    x, tokens, table = torch.zeros(8), torch.zeros(2, dtype=torch.int64), torch.zeros(3, 8)
    for first in (-1, 1 << 62):
        with pytest.raises(DeviceError, match="first"):
            D.dropout_fwd(x, 0.5, seed=1, first=first)
        with pytest.raises(DeviceError, match="first"):
            E.embedding_fwd(tokens, table, first=first)
        with pytest.raises(DeviceError, match="first"):
            E.embedding_bwd(tokens, torch.zeros(2, 8), table, first=first)
