"""Few queries against the caches of many sequences: more of them than a wave looks at together, lengths of 0 on
both sides of that, and launches that do not cut the keys."""

import math

import pytest
import torch

from nanofed_amd.ops import attention as A

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, FP = torch.bfloat16, torch.float16


def reference(q, k, v, q_lengths, k_lengths):
    """Output and log-sum-exp in 64 bits (causal: the last query sees every key)."""
    B, Tq, H, D = q.shape
    Tk, Hk = k.shape[1:3]
    q, k, v = (t.double().transpose(1, 2) for t in (q, k, v))
    k, v = (t.repeat_interleave(H // Hk, 1) for t in (k, v))
    i, j = torch.arange(Tq, device=DEV).view(1, Tq, 1), torch.arange(Tk, device=DEV).view(1, 1, Tk)
    m, n = q_lengths.view(B, 1, 1), k_lengths.view(B, 1, 1)
    seen = ((i < m) & (j < n) & (j <= i + n - m)).unsqueeze(1)
    s = (q @ k.transpose(-1, -2).contiguous() * D**-0.5).masked_fill(~seen, -math.inf)
    lse = torch.logsumexp(s, -1)
    p = torch.exp(s - lse.masked_fill(lse == -math.inf, 0.0).unsqueeze(-1)).masked_fill(~seen, 0.0)
    return (p @ v).transpose(1, 2), lse


def check(B, Tq, Tk, H, Hk, D, dtype, most, full=False):
    g = torch.Generator(device=DEV).manual_seed(B + Tk)
    q, k, v = (torch.randn(B, t, h, D, generator=g, device=DEV).to(dtype) for t, h in ((Tq, H), (Tk, Hk), (Tk, Hk)))
    keys = torch.randint(1, Tk + 1, (B,), generator=g, device=DEV, dtype=torch.int32)
    for b in (0, 3, 62, 63, 64, 65, B - 2):  # empty ones on both sides of each border
        if b < B:
            keys[b] = 0
    keys[B - 1] = Tk
    if full:
        keys.fill_(Tk)
    rows = keys.clamp(max=Tq)
    out, lse = torch.full_like(q, math.nan), torch.full((B, H, Tq), math.nan, device=DEV)
    A.attention_fwd(q, k, v, out, lse, q_lengths=None if full else rows, k_lengths=None if full else keys)
    want, sums = reference(q, k, v, rows, keys)
    there = torch.isfinite(sums)
    assert torch.equal(lse == -math.inf, ~there) and bool((out.transpose(1, 2)[~there] == 0).all())
    # scores of D products in fp32 (below 2^5 in all), their exponentials and sums
    assert float((lse.double() - sums)[there].abs().max()) <= (2 * (D + 8) * 2**5 + 2 * Tk + 16) * 2.0**-24
    rounded = (want.to(dtype).double() - want).square().mean().sqrt()
    assert float((out.double() - want).square().mean().sqrt() / rounded) <= most
    top = want.abs().amax((1, 2, 3), keepdim=True)  # (no sequence may hide among the others)
    assert float(((out.double() - want).abs() / top.clamp(min=1e-30)).max()) <= 8 * torch.finfo(dtype).eps


@pytest.mark.parametrize("B,Hk", [(64, 1), (65, 1), (130, 2), (130, 3), (511, 1), (255, 2)])
@pytest.mark.parametrize("Tq,group,Tk", [(1, 1, 300), (2, 4, 517), (1, 1, 129)])
def test_keys_of_many_sequences_cut_on_the_device(B, Hk, Tq, group, Tk):
    check(B, Tq, Tk, Hk * group, Hk, 64, BF, 1.1)


@pytest.mark.parametrize("dtype,D", [(FP, 128), (BF, 40)])
def test_keys_of_many_sequences_in_other_types(dtype, D):
    check(130, 1, 700, 4, 2, D, dtype, 1.1)
    check(70, 5, 1100, 16, 2, D, dtype, 1.5)  # two tiles of rows


@pytest.mark.parametrize("B,Hk", [(512, 1), (300, 2)])
@pytest.mark.parametrize("full", [False, True])
def test_keys_of_more_sequences_than_are_cut(B, Hk, full):
    check(B, 1, 200, 4 * Hk, Hk, 64, BF, 1.1, full)


@pytest.mark.parametrize("B,Tq,H,Hk", [(260, 1, 64, 1), (130, 2, 64, 1), (64, 2, 32, 1)])
@pytest.mark.parametrize("full", [False, True])
def test_several_tiles_of_rows_with_and_without_cuts(B, Tq, H, Hk, full):
    check(B, Tq, 1030, H, Hk, 64, BF, 1.5, full)
