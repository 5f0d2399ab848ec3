"""Attention for the GPT-2 configuration.

``causal_attention_fwd`` / ``_bwd``: causal self-attention on the packed ``[B*T, 3C]`` q|k|v layout
(csrc/hip/attention.hip: MFMA flash attention, head dimension 64, lengths that are multiples of 128).

``attention_fwd`` / ``attention_bwd`` (csrc/hip/attention_general.hip): any length from one token
on, strided ``[B, T, H, D]`` operands, shared key heads, head dimensions up to 128, a length per
sequence, and dropped probabilities whose mask is a function of (seed, step, place) and never
stored.

Device tensors run the gfx950 kernels; CPU tensors run PyTorch's
``scaled_dot_product_attention`` in fp32 (and autograd for the backward),
which is also the oracle of the kernel tests.  The reference has no attention
layer; this serves the GPT-2 configuration of the benchmark suite.
"""

from __future__ import annotations

import struct
from ctypes import c_int, c_long, c_void_p
from functools import lru_cache

import torch
import torch.nn.functional as F

from nanofed_amd.core.exceptions import DeviceError

from . import library
from .dropout import check_key, limit_of, philox_words, refuse_recording

P, I, L = c_void_p, c_int, c_long
_SIGS = {
    "nf_attn_seq_multiple": ([], I),
    "nf_attn_fwd": ([P, P, P, I, I, I, P], I),
    "nf_attn_bwd": ([P, P, P, P, P, P, I, I, I, P], I),
    "nf_attn_set_split": ([I], None),
    "nf_attention_args_size": ([], I),
    "nf_attention_fwd_floats": ([P], L),
    "nf_attention_bwd_floats": ([P], L),
    "nf_attention": ([P, I, I, P], I),
}
_fns: dict[str, object] = {}
HEAD_DIM = 64


def _fn(name: str):
    fn = _fns.get(name)
    if fn is None:
        argtypes, restype = _SIGS[name]
        fn = library.declare(name, argtypes, restype)
        _fns[name] = fn
    return fn


def symbols() -> list[str]:
    return sorted(_SIGS)


def _p(t: torch.Tensor) -> c_void_p:
    return c_void_p(t.data_ptr())


def _check(qkv: torch.Tensor, batch: int, seq: int, heads: int) -> int:
    C = heads * HEAD_DIM
    if qkv.dtype != torch.bfloat16 or not qkv.is_contiguous():
        raise DeviceError("qkv must be a contiguous bf16 matrix")
    if tuple(qkv.shape) != (batch * seq, 3 * C):
        raise DeviceError(f"qkv must be [{batch * seq}, {3 * C}], got {tuple(qkv.shape)}")
    if qkv.device.type == "cuda":
        mult = int(_fn("nf_attn_seq_multiple")())
        if seq % mult:
            raise DeviceError(f"sequence length {seq} is not a multiple of {mult}")
    return C


def set_forward_split(groups: int) -> None:
    """Wave groups (1, 2 or 4) that share one 128-query tile in the forward
    kernel, each taking every ``groups``-th key stage (tuning hook)."""
    if groups not in (1, 2, 4):
        raise DeviceError("the forward split must be 1, 2 or 4")
    _fn("nf_attn_set_split")(groups)


def backward_scratch(batch: int, heads: int, seq: int, device: torch.device) -> torch.Tensor:
    return torch.empty(batch * heads * seq, dtype=torch.float32, device=device)


def _split(qkv: torch.Tensor, batch: int, seq: int, heads: int):
    q, k, v = qkv.float().view(batch, seq, 3, heads, HEAD_DIM).unbind(2)
    return q.transpose(1, 2), k.transpose(1, 2), v.transpose(1, 2)


def causal_attention_fwd(qkv: torch.Tensor, out: torch.Tensor, lse: torch.Tensor, batch: int,
                         seq: int, heads: int) -> None:
    """``out[B*T, C] = softmax(q k^T / 8 + causal mask) v`` per head;
    ``lse[B, H, T]`` receives the log-sum-exp of every score row."""
    C = _check(qkv, batch, seq, heads)
    if qkv.device.type == "cuda":
        library.check(_fn("nf_attn_fwd")(_p(qkv), _p(out), _p(lse), batch, seq, heads,
                                         library.stream_ptr(qkv.device)), "attn_fwd")
        return
    q, k, v = _split(qkv, batch, seq, heads)
    scores = (q @ k.transpose(-1, -2)) * HEAD_DIM**-0.5
    mask = torch.ones(seq, seq, dtype=torch.bool).tril()
    scores = scores.masked_fill(~mask, float("-inf"))
    lse.view(batch, heads, seq).copy_(torch.logsumexp(scores, -1))
    y = torch.softmax(scores, -1) @ v
    out.copy_(y.transpose(1, 2).reshape(batch * seq, C).to(torch.bfloat16))


def causal_attention_bwd(qkv: torch.Tensor, out: torch.Tensor, lse: torch.Tensor,
                         dout: torch.Tensor, dqkv: torch.Tensor, scratch: torch.Tensor,
                         batch: int, seq: int, heads: int) -> None:
    """``dqkv`` (same packed layout as ``qkv``, fully overwritten) from ``dout``."""
    C = _check(qkv, batch, seq, heads)
    if qkv.device.type == "cuda":
        library.check(_fn("nf_attn_bwd")(_p(qkv), _p(out), _p(lse), _p(dout), _p(dqkv),
                                         _p(scratch), batch, seq, heads,
                                         library.stream_ptr(qkv.device)), "attn_bwd")
        return
    with torch.enable_grad():
        leaf = qkv.float().detach().requires_grad_(True)
        q, k, v = leaf.view(batch, seq, 3, heads, HEAD_DIM).unbind(2)
        y = F.scaled_dot_product_attention(q.transpose(1, 2), k.transpose(1, 2),
                                           v.transpose(1, 2), is_causal=True)
        y = y.transpose(1, 2).reshape(batch * seq, C)
        (g,) = torch.autograd.grad(y, leaf, dout.float())
    dqkv.copy_(g.to(torch.bfloat16))


# ---------------------------------------------------------------------------
# any length, layout and head grouping

MAX_HEAD_DIM = 128
_TYPES = {torch.bfloat16: 1, torch.float16: 2}

# ``AttnArgs`` of csrc/hip/attention_general.hip: q k v out dout dq dk dv, each an address and the
# distances between sequences, rows and heads; addresses of lse, delta, the lengths and the step in
# memory; seed and first head, sizes, scale and factor of what is kept, threshold and step, scratch
_PACK = struct.Struct("@" + "P3q" * 8 + "5P2Q7i2f2IP2i0q")
_NONE = (0, 0, 0, 0)


class _Args:
    """What both directions share, checked."""

    __slots__ = ("B", "Tq", "Tk", "H", "Hk", "D", "causal", "scale", "limit", "up", "seed", "step_at",
                 "step", "first_head", "q", "k", "v", "qlen", "klen")

    def pack(self, lse: int, out: tuple, dout=_NONE, dq=_NONE, dk=_NONE, dv=_NONE, delta: int = 0,
             parts: int = 0) -> bytes:
        return _PACK.pack(
            *self.q, *self.k, *self.v, *out, *dout, *dq, *dk, *dv, lse, delta, self.qlen, self.klen,
            self.step_at, self.seed, self.first_head, self.B, self.Tq, self.Tk, self.H, self.Hk, self.D,
            self.causal, self.scale, self.up, self.limit, self.step, parts, 0, 0)


@lru_cache(maxsize=1024)
def _scratch_floats(backward: bool, B: int, Tq: int, Tk: int, H: int, Hk: int, D: int, limit: int) -> int:
    sizes = _PACK.pack(*_NONE * 8, 0, 0, 0, 0, 0, 0, 0, B, Tq, Tk, H, Hk, D, 0, 1.0, 1.0, limit, 0, 0, 0, 0)
    return _fn("nf_attention_bwd_floats" if backward else "nf_attention_fwd_floats")(sizes)


def _operand(t: torch.Tensor, name: str, shape: tuple, dtype: torch.dtype, dev: torch.device,
             written: bool) -> tuple:
    """Checks a ``[B, T, heads, D]`` operand; its address and the distances between its sequences,
    rows and heads."""
    if t.dtype is not dtype or t.device != dev:
        raise DeviceError(f"attention: {name} must be {dtype} on {dev}, got {t.dtype} on {t.device}")
    if t.shape != shape:
        raise DeviceError(f"attention: {name} must be {list(shape)}, got {list(t.shape)}")
    at = t.data_ptr()
    b, s, h, d = t.stride()
    if d == 1 and not (at & 15 or (b | s | h) & 7) and b and s and h and s < 1 << 24:
        return at, b, s, h
    # lengths of one have any distance, and distances of 0 are fine to read
    strides = [0 if n == 1 else x for n, x in zip(shape, (b, s, h))]
    if shape[3] > 1 and d != 1:
        raise DeviceError(f"attention: the columns of {name} must be contiguous")
    if t.is_cuda and (at & 15 or any(x & 7 for x in strides)):
        raise DeviceError(f"attention: rows of {name} must start at multiples of 16 bytes")
    if strides[1] >= 1 << 24:
        raise DeviceError(f"attention: rows of {name} must be less than 2^24 elements apart")
    if written and any(n > 1 and x == 0 for n, x in zip(shape, strides)):
        raise DeviceError(f"attention: {name} is written and must not be expanded")
    return (at, *strides)


def _lengths(t: torch.Tensor | None, name: str, like: torch.Tensor) -> int:
    if t is None:
        return 0
    if t.dtype != torch.int32 or not t.is_contiguous() or t.shape != like.shape[:1] or t.device != like.device:
        raise DeviceError(f"attention: {name} must be {like.shape[0]} contiguous int32 on {like.device}")
    return t.data_ptr()


def _arguments(q, k, v, causal, scale, q_lengths, k_lengths, dropout, seed, step, first_batch) -> _Args:
    if q.dim() != 4 or k.dim() != 4:
        raise DeviceError("attention: q, k and v are [batch, length, heads, head dimension]")
    if q.dtype not in _TYPES and not (q.device.type == "cpu" and q.dtype in (torch.float32, torch.float64)):
        raise DeviceError(f"attention: bfloat16 or float16, got {q.dtype}")
    a = _Args()
    shape = q.shape
    a.B, a.Tq, a.H, a.D = B, Tq, H, D = shape
    _, a.Tk, a.Hk, _ = k.shape
    Tk, Hk = a.Tk, a.Hk
    if Hk == 0 or H % Hk:
        raise DeviceError(f"attention: {H} query heads do not share {Hk} key heads evenly")
    if not 0 < D <= MAX_HEAD_DIM or D % 8:
        raise DeviceError(f"attention: the head dimension must be a multiple of 8 up to {MAX_HEAD_DIM}, got {D}")
    if max(Tq, Tk) > 1 << 22 or B * H > 1 << 23:
        raise DeviceError("attention: lengths go up to 2^22, batch * heads up to 2^23")
    a.scale = scale = D**-0.5 if scale is None else float(scale)
    if not 0.0 < scale < float("inf"):
        raise DeviceError("attention: the scale must be positive")
    a.limit = limit_of(dropout, 8, "attention") if dropout else 0
    a.up = 256 / (256 - a.limit)
    dtype, dev = q.dtype, q.device
    check_key(seed, step, dev, "attention")
    a.seed = seed
    a.step_at, a.step = (step.data_ptr(), 0) if isinstance(step, torch.Tensor) else (0, step)
    if not 0 <= first_batch or (first_batch + B) * H > 1 << 32:
        raise DeviceError("attention: first_batch must not be negative, nor (first_batch + batch) * heads pass 2^32")
    a.first_head = first_batch * H
    a.causal = bool(causal)
    shared = (B, Tk, Hk, D)
    a.q = _operand(q, "q", shape, dtype, dev, False)
    a.k = _operand(k, "k", shared, dtype, dev, False)
    a.v = _operand(v, "v", shared, dtype, dev, False)
    a.qlen, a.klen = _lengths(q_lengths, "q_lengths", q), _lengths(k_lengths, "k_lengths", q)
    return a


def _check_lse(lse: torch.Tensor, a: _Args, dev: torch.device) -> None:
    if (lse.dtype is not torch.float32 or not lse.is_contiguous() or lse.device != dev
            or lse.shape != (a.B, a.H, a.Tq)):
        raise DeviceError(f"attention: lse must be contiguous float32 [{a.B}, {a.H}, {a.Tq}] on {dev}")


def attention_fwd(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, out: torch.Tensor | None = None,
                  lse: torch.Tensor | None = None, *, causal: bool = True, scale: float | None = None,
                  q_lengths: torch.Tensor | None = None, k_lengths: torch.Tensor | None = None,
                  dropout: float = 0.0, seed: int = 0, step: "int | torch.Tensor" = 0,
                  first_batch: int = 0) -> tuple[torch.Tensor, torch.Tensor]:
    """``out = drop(softmax(scale q k^T)) v`` per head and the log-sum-exp of every score row;
    returns ``(out, lse)``.

    ``q`` ``[B, Tq, H, D]``, ``k`` / ``v`` ``[B, Tk, Hk, D]``: bfloat16 or float16 with contiguous
    columns, the other distances free (multiples of 8 elements, 16-byte aligned: views of a packed
    projection or of a longer cache do).  Query head h reads key head ``h // (H // Hk)``.  ``D`` is a
    multiple of 8 up to 128; ``scale`` is ``D ** -0.5`` by default.

    ``q_lengths`` / ``k_lengths`` (int32 ``[B]`` on the device, taken to ``[0, T]``): sequence b has
    that many queries and keys, right-padded; what lies behind them is not used and may hold
    anything.  With ``causal`` the last query sees every key: key j is seen by query i where
    ``j <= i + keys - queries`` (equal numbers: the usual triangle; one query: all of the cache).
    Queries behind the length and queries that see no key give 0 and a log-sum-exp of -inf.  A
    non-finite value that some query sees may spread to other queries of its sequence.  ``out`` and
    ``lse`` must not overlap what is read.  Not recorded by autograd: a tensor that requires a gradient
    is refused while gradients are enabled.

    ``dropout`` (taken to a multiple of 1 / 256: 0.1 is 0.1016; less than 1 / 512 is refused): each
    probability is dropped with it, what stays is scaled by the inverse of the share that stays.  The mask is a function of ``seed``, ``step`` (a
    number, or one int64 on the device that the kernel reads when it runs) and of the sequence, head,
    query and key: probability (i, j) of head h of sequence b takes byte ``j & 3`` of word ``i & 3`` of
    the Philox4x32-7 block with counter ``(j >> 2, i >> 2, (first_batch + b) H + h, step)``."""
    a = _arguments(q, k, v, causal, scale, q_lengths, k_lengths, dropout, seed, step, first_batch)
    refuse_recording("attention", q, k, v, out, lse)
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    if lse is None:
        lse = q.new_empty((a.B, a.H, a.Tq), dtype=torch.float32)
    dev = q.device
    to = _operand(out, "out", q.shape, q.dtype, dev, True)
    _check_lse(lse, a, dev)
    if a.B == 0 or a.Tq == 0:
        return out, lse
    if a.Tk == 0:
        out.zero_()
        lse.fill_(float("-inf"))
        return out, lse
    if not q.is_cuda:
        prob, kept, sums = _probabilities(a, q, k, q_lengths, k_lengths, step)
        lse.copy_(sums)
        y = (prob * kept) @ _shared(a, v, k_lengths)
        out.copy_(y.transpose(1, 2))
        return out, lse
    # (scratch of its own for every call: the allocator hands it on in stream order, and a captured
    # call's belongs to its graph)
    floats = _scratch_floats(False, a.B, a.Tq, a.Tk, a.H, a.Hk, a.D, a.limit)
    parts = q.new_empty(floats, dtype=torch.float32) if floats else None
    packed = a.pack(lse.data_ptr(), to, parts=parts.data_ptr() if floats else 0)
    with library.on_device(dev):
        library.check(_fn("nf_attention")(packed, _TYPES[q.dtype], 0, library.stream_ptr(dev)), "attention_fwd")
    return out, lse


def attention_bwd(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, out: torch.Tensor,
                  lse: torch.Tensor, dout: torch.Tensor, dq: torch.Tensor, dk: torch.Tensor,
                  dv: torch.Tensor, *, causal: bool = True, scale: float | None = None,
                  q_lengths: torch.Tensor | None = None, k_lengths: torch.Tensor | None = None,
                  dropout: float = 0.0, seed: int = 0, step: "int | torch.Tensor" = 0,
                  first_batch: int = 0) -> None:
    """Gradients of ``attention_fwd`` (called with the same arguments) from ``dout``: ``dq``, ``dk``,
    ``dv`` are written everywhere, with 0 behind the lengths.  The probabilities are computed again
    from ``lse`` and the mask from its counter; a key head's gradient is summed over the query heads
    that share it in a fixed order, without atomics.  With float16 operands ``dout`` may be of any size
    (no loss scaling is needed): the factors inside take the exponent that fits them.  ``dq``, ``dk``,
    ``dv`` must not overlap what is read."""
    a = _arguments(q, k, v, causal, scale, q_lengths, k_lengths, dropout, seed, step, first_batch)
    refuse_recording("attention", q, k, v, out, lse, dout, dq, dk, dv)
    shape, shared, dtype, dev = q.shape, k.shape, q.dtype, q.device
    operands = (_operand(out, "out", shape, dtype, dev, False), _operand(dout, "dout", shape, dtype, dev, False),
                _operand(dq, "dq", shape, dtype, dev, True), _operand(dk, "dk", shared, dtype, dev, True),
                _operand(dv, "dv", shared, dtype, dev, True))
    _check_lse(lse, a, dev)
    if a.B == 0 or a.Tq == 0 or a.Tk == 0:
        for t in (dq, dk, dv):
            t.zero_()
        return
    if not q.is_cuda:
        prob, kept, _ = _probabilities(a, q, k, q_lengths, k_lengths, step)
        rows = _valid(a, q_lengths, a.Tq).view(a.B, 1, a.Tq, 1)
        qf = _masked(q, rows)
        do, o = _masked(dout, rows), _masked(out, rows)
        kf, vf = _shared(a, k, k_lengths), _shared(a, v, k_lengths)
        gv = (prob * kept).transpose(-1, -2) @ do
        ds = prob * (do @ vf.transpose(-1, -2) * kept - (do * o).sum(-1, keepdim=True)) * a.scale
        dq.copy_((ds @ kf).transpose(1, 2))
        for t, g in ((dk, ds.transpose(-1, -2) @ qf), (dv, gv)):
            t.copy_(g.view(a.B, a.Hk, a.H // a.Hk, a.Tk, a.D).sum(2).transpose(1, 2))
        return
    scratch = q.new_empty(_scratch_floats(True, a.B, a.Tq, a.Tk, a.H, a.Hk, a.D, a.limit), dtype=torch.float32)
    packed = a.pack(lse.data_ptr(), *operands, delta=scratch.data_ptr())
    with library.on_device(dev):
        library.check(_fn("nf_attention")(packed, _TYPES[dtype], 1, library.stream_ptr(dev)), "attention_bwd")


def _valid(a: _Args, lengths: torch.Tensor | None, T: int) -> torch.Tensor:
    n = torch.full((a.B,), T) if lengths is None else lengths.clamp(0, T).long()
    return torch.arange(T) < n[:, None]


def _masked(t: torch.Tensor, rows: torch.Tensor) -> torch.Tensor:
    """``[B, heads, T, D]`` in fp32 (double stays), rows that are not there as zeros."""
    x = t if t.dtype == torch.float64 else t.float()
    return torch.where(rows, x.transpose(1, 2), torch.zeros((), dtype=x.dtype))


def _shared(a: _Args, t: torch.Tensor, lengths: torch.Tensor | None) -> torch.Tensor:
    x = _masked(t, _valid(a, lengths, a.Tk).view(a.B, 1, a.Tk, 1))
    return x.repeat_interleave(a.H // a.Hk, 1)


def _probabilities(a: _Args, q, k, q_lengths, k_lengths, step):
    """CPU: (probabilities, what each is multiplied by, log-sum-exp), ``[B, H, Tq, Tk]``."""
    rows, keys = _valid(a, q_lengths, a.Tq), _valid(a, k_lengths, a.Tk)
    seen = rows[:, :, None] & keys[:, None, :]
    if a.causal:
        off = (keys.sum(1) - rows.sum(1))[:, None, None]
        seen = seen & (torch.arange(a.Tk) <= torch.arange(a.Tq)[:, None] + off)
    qf = _masked(q, rows.view(a.B, 1, a.Tq, 1))
    scores = (qf @ _shared(a, k, k_lengths).transpose(-1, -2)) * a.scale
    scores = scores.masked_fill(~seen[:, None], float("-inf"))
    sums = torch.logsumexp(scores, -1)
    prob = torch.exp(scores - sums.masked_fill(sums == float("-inf"), 0.0)[..., None])
    return prob, kept_pairs(a, step).to(prob.dtype) * a.up if a.limit else 1.0, sums


def kept_pairs(a: _Args, step: "int | torch.Tensor") -> torch.Tensor:
    """Whether each probability ``[B, H, Tq, Tk]`` is kept (CPU)."""
    nq, nk = (a.Tq + 3) // 4, (a.Tk + 3) // 4
    heads = (a.first_head + torch.arange(a.B * a.H).view(-1, 1, 1)) & 0xFFFFFFFF
    w = philox_words(a.seed, step, torch.arange(nk), torch.arange(nq).view(-1, 1), heads)
    b = w.transpose(2, 3).unsqueeze(-1) >> torch.tensor([0, 8, 16, 24]) & 0xFF
    return (b >= a.limit).reshape(a.B, a.H, nq * 4, nk * 4)[:, :, : a.Tq, : a.Tk]
