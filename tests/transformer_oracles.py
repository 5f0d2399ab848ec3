"""Plain implementations in 64 bits of the transformer operators with dropout, for the CPU tests
of the PyTorch paths and the GPU tests of the kernels, with the error bounds that the tests
compare against.

A rounding to a type is off by at most ``eps / 2`` of the value.  What the kernels round: the
probabilities and their gradients once on their way into a matrix product, and every output once;
sums run in fp32.
"""

import math

import numpy as np
import torch

UNIT = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.bfloat16, torch.float16)}
E32 = 2.0**-24
# half the distance of neighbours below the smallest normal number (half: 2^-24 apart from 0 to
# 2^-14): there a rounding is off by up to this, however small the value
LEAST = {t: torch.finfo(t).tiny * torch.finfo(t).eps / 2 for t in UNIT}


def philox(counter, seed):
    """Words ``[..., 4]`` (uint32) of the 7-round Philox4x32 blocks with the given counter words."""
    x, y, z, w = (np.asarray(a, dtype=np.uint64) for a in counter)
    k, l, cut, half = seed % 2**32, seed // 2**32, np.uint64(2**32 - 1), np.uint64(32)
    for _ in range(7):
        p, q = x * np.uint64(0xD2511F53), z * np.uint64(0xCD9E8D57)
        x, y, z, w = (q >> half) ^ y ^ np.uint64(k), q & cut, (p >> half) ^ w ^ np.uint64(l), p & cut
        k, l = (k + 0x9E3779B9) % 2**32, (l + 0xBB67AE85) % 2**32
    return np.stack(np.broadcast_arrays(x, y, z, w), -1).astype("<u4")


def row_factor(n, p, seed, step, first=0):
    """What elements ``first .. first + n - 1`` of a flattened tensor are multiplied by."""
    e = np.arange(first, first + n, dtype=np.uint64)
    b = e >> np.uint64(3)
    w = philox((b & np.uint64(2**32 - 1), b >> np.uint64(32), 0 * b, 0 * b + np.uint64(step)), seed)
    at = (e % np.uint64(8)).astype(int)
    halves = w.view("<u2").reshape(n, 8)[np.arange(n), at]
    cut = round(p * 65536)
    return torch.from_numpy((halves >= cut) * (65536 / (65536 - cut)))


def pair_factor(B, H, Tq, Tk, p, seed, step, first_batch=0):
    """What the probabilities ``[B, H, Tq, Tk]`` are multiplied by."""
    bh, i, j = np.meshgrid(np.arange(first_batch * H, (first_batch + B) * H), np.arange(Tq),
                           np.arange(Tk), indexing="ij")
    w = philox((j >> 2, i >> 2, bh, 0 * bh + step), seed)
    word = np.take_along_axis(w, (i & 3)[..., None], -1)[..., 0]
    byte = (word >> (8 * (j & 3)).astype(np.uint32)) & np.uint32(255)
    cut = round(p * 256)
    return torch.from_numpy((byte >= cut) * (256 / (256 - cut))).view(B, H, Tq, Tk)


def _lengths(t, B, T):
    return [T] * B if t is None else [min(max(int(x), 0), T) for x in t]


def attention(q, k, v, dout=None, *, causal=True, scale=None, q_lengths=None, k_lengths=None, p=0.0,
              seed=0, step=0, first_batch=0, unit=0.0, least=0.0):
    """``{name: (value, bound)}`` of out, lse and (with ``dout``) dq, dk, dv.  ``unit``: half a step
    of the type the kernel rounds to, ``least``: half its smallest step (subnormal values)."""
    B, Tq, H, D = q.shape
    Tk, Hk = k.shape[1], k.shape[2]
    G = H // Hk
    scale = D**-0.5 if scale is None else scale
    f = pair_factor(B, H, Tq, Tk, p, seed, step, first_batch)
    shapes = {"out": q.shape, "lse": (B, H, Tq), "dq": q.shape, "dk": k.shape, "dv": k.shape}
    got = {n: [torch.zeros(s, dtype=torch.float64) for _ in range(2)] for n, s in shapes.items()}
    got["lse"][0].fill_(-math.inf)
    nq, nk = _lengths(q_lengths, B, Tq), _lengths(k_lengths, B, Tk)
    for b in range(B):
        m, n = nq[b], nk[b]
        for h in range(H):
            Q, K, V = q[b, :m, h].double(), k[b, :n, h // G].double(), v[b, :n, h // G].double()
            seen = torch.ones(m, n, dtype=torch.bool)
            if causal:
                seen = torch.arange(n) <= torch.arange(m)[:, None] + (n - m)
            if not seen.any():
                continue
            S = (Q @ K.T * scale).masked_fill(~seen, -math.inf)
            lse = torch.logsumexp(S, 1)
            P = torch.where(seen, torch.exp(S - lse.masked_fill(lse == -math.inf, 0)[:, None]), 0.0)
            F = f[b, h, :m, :n]
            A = P * F
            O = A @ V
            # fp32: D products per score, the exponent, the sum of the row
            big = float((Q.abs() @ K.abs().T).max()) * scale
            ep = E32 * (2 * (D + 8) * big + 2 * n + 16)
            to = (unit + ep) * (A @ V.abs()) + least * (F @ V.abs()) + unit * O.abs() + least
            got["out"][0][b, :m, h], got["out"][1][b, :m, h] = O, to
            got["lse"][0][b, h, :m] = lse
            got["lse"][1][b, h, :m] = ep + 4 * E32 * lse.abs().nan_to_num(0.0, 0.0, 0.0)
            if dout is None:
                continue
            dO = dout[b, :m, h].double()
            dP = dO @ V.T * F
            delta = (dO * O).sum(1, keepdim=True)
            dS = P * (dP - delta)
            tdelta = (dO.abs() * (to + unit * O.abs())).sum(1, keepdim=True) + E32 * D * (dO * O).abs().sum(1, keepdim=True)
            tS = (unit + ep) * dS.abs() + P * (ep * (dP.abs() + delta.abs()) + tdelta
                                              + E32 * (D + 2) * (dO.abs() @ V.abs().T) * F) + least * seen
            tA = (unit + ep) * A + least * F * seen
            for name, x, tx, at in (("dq", dS @ K, tS @ K.abs(), h), ("dk", dS.T @ Q, tS.T @ Q.abs(), h // G),
                                    ("dv", A.T @ dO, tA.T @ dO.abs(), h // G)):
                up = 1.0 if name == "dv" else scale
                rows = m if name == "dq" else n
                got[name][0][b, :rows, at] += x * up
                got[name][1][b, :rows, at] += tx * up + E32 * (m + n) * (x * up).abs()
    for name in ("dq", "dk", "dv"):
        got[name][1] += unit * got[name][0].abs() + least
    return {n: tuple(x) for n, x in got.items() if dout is not None or n in ("out", "lse")}


def within(name, value, want, bound):
    """Asserts ``|value - want| <= bound`` everywhere, non-finite values equal."""
    value = value.detach().double().cpu()
    fine = torch.isfinite(want)
    assert torch.equal(value[~fine], want[~fine]), f"{name}: non-finite values differ"
    off = (value - want).abs()[fine] - 1.001 * bound[fine]
    assert torch.isfinite(value[fine]).all(), f"{name}: not finite"
    assert not off.numel() or float(off.max()) <= 0, \
        f"{name}: {float(off.max()):.3g} beyond the bound at {int(off.argmax())} of {off.numel()}"
