"""Embedding lookup with scaling, positions and dropout, and its gradient by sorted tokens
(csrc/hip/embedding_ops.hip).

    x[b, t]  = drop(scale * table[tokens[b, t]] + positions[t])
    dtable   = scale * sum of drop'(dout) over the places of each token
    dpos[t]  = sum over b of drop'(dout[b, t])

Tables are float32, bfloat16 or float16; sums run in fp32 in a fixed order (the places of a token
in ascending order), without atomics.  The dropout mask is that of ``ops.dropout`` on the
flattened output.  A token outside the table looks up zeros and gets no gradient.

Device tensors go to the gfx950 kernels; CPU tensors run the same arithmetic in PyTorch.  The
reference has no sequence model; this serves the GPT-2 configuration of the benchmark suite.
"""

from __future__ import annotations

import struct
from ctypes import c_char_p, c_int, c_long, c_void_p
from functools import lru_cache

import torch

from nanofed_amd.core.exceptions import DeviceError

from . import library
from .dropout import FLOAT_TYPES, check_first, check_key, kept_rows, limit_of, refuse_recording, step_args

P, L, I, ARGS = c_void_p, c_long, c_int, c_char_p
_SIGS = {
    "nf_embedding_fwd": ([ARGS, P], I),
    "nf_token_order_words": ([L], L),
    "nf_token_order": ([P, P, P, P, L, L, L, P], I),
    "nf_embedding_bwd_words": ([L, L, I], L),
    "nf_embedding_bwd": ([ARGS, P], I),
    "nf_embedding_args_size": ([], I),
}
_ARGS = struct.Struct("@8P6qQd2I4i")  # EmbeddingArgs of csrc/hip/embedding_ops.hip
_fns: dict[str, object] = {}


def _fn(name: str):
    fn = _fns.get(name)
    if fn is None:
        argtypes, restype = _SIGS[name]
        fn = library.declare(name, argtypes, restype)
        _fns[name] = fn
    return fn


def symbols() -> list[str]:
    return sorted(_SIGS)


def _address(t: torch.Tensor | None) -> int:
    return 0 if t is None else t.data_ptr()


@lru_cache(maxsize=256)
def _bwd_words(rows: int, columns: int, ordered: bool) -> int:
    return _fn("nf_embedding_bwd_words")(rows, columns, ordered)


def _need(t: torch.Tensor, shape: tuple, dtypes, device: torch.device, name: str) -> None:
    if t.dtype not in dtypes or t.device != device or not t.is_contiguous():
        raise DeviceError(f"embedding: {name} must be contiguous {' or '.join(map(str, dtypes))} on "
                          f"{device}, got {t.dtype} on {t.device}")
    if t.shape != shape:
        raise DeviceError(f"embedding: {name} must be {list(shape)}, got {list(t.shape)}")


def _tokens(tokens: torch.Tensor, device: torch.device) -> tuple[int, int]:
    if tokens.dtype != torch.int64 or not tokens.is_contiguous() or tokens.device != device:
        raise DeviceError(f"embedding: tokens must be contiguous int64 on {device}")
    if tokens.dim() not in (1, 2):
        raise DeviceError("embedding: tokens must be [T] or [B, T]")
    return (1, tokens.shape[0]) if tokens.dim() == 1 else (tokens.shape[0], tokens.shape[1])


def embedding_fwd(tokens: torch.Tensor, table: torch.Tensor, out: torch.Tensor | None = None, *,
                  positions: torch.Tensor | None = None, scale: float = 1.0, dropout: float = 0.0,
                  seed: int = 0, step: "int | torch.Tensor" = 0, first: int = 0) -> torch.Tensor:
    """``drop(scale * table[tokens] + positions[t])`` for ``tokens`` ``[T]`` or ``[B, T]``;
    ``positions`` (optional) has at least T rows.  ``dropout``, ``seed``, ``step``, ``first``: as
    in ``ops.dropout``.  Not recorded by autograd."""
    if table.dim() != 2 or table.dtype not in FLOAT_TYPES or not table.is_contiguous():
        raise DeviceError("embedding: the table must be a contiguous float matrix")
    dev, (V, C) = table.device, table.shape
    B, T = _tokens(tokens, dev)
    limit = limit_of(dropout, 16, "embedding")
    check_key(seed, step, dev, "embedding")
    check_first(first, "embedding")
    refuse_recording("embedding", table, positions, out)
    if positions is not None:
        if positions.dim() != 2 or positions.shape[0] < T:
            raise DeviceError(f"embedding: positions must have at least {T} rows")
        _need(positions, (positions.shape[0], C), (table.dtype,), dev, "positions")
    if out is None:
        out = table.new_empty((*tokens.shape, C))
    elif out.numel() != B * T * C or out.shape[-1] != C:
        raise DeviceError(f"embedding: out must hold {B * T} rows of {C}")
    else:
        _need(out, out.shape, (table.dtype,), dev, "out")
    if B * T * C == 0:
        return out
    if V == 0:
        raise DeviceError("embedding: the table has no rows")
    if dev.type != "cuda":
        x = _looked_up(tokens, table) * scale
        if positions is not None:
            x = x + positions[:T].float()
        if limit:
            kept = kept_rows(x.numel(), limit, seed, step, first, dev).view(x.shape)
            x = torch.where(kept, x * (65536 / (65536 - limit)), 0.0)
        out.copy_(x.view(out.shape))
        return out
    at, number = step_args(step)
    args = _ARGS.pack(tokens.data_ptr(), table.data_ptr(), _address(positions), out.data_ptr(), 0, 0, 0, at,
                      -1, B, T, V, C, first, seed, scale, limit, number, FLOAT_TYPES[table.dtype], 0, 0, 0)
    with library.on_device(dev):
        library.check(_fn("nf_embedding_fwd")(args, library.stream_ptr(dev)), "embedding_fwd")
    return out


def _looked_up(tokens: torch.Tensor, table: torch.Tensor) -> torch.Tensor:
    inside = (tokens >= 0) & (tokens < table.shape[0])
    return torch.where(inside.unsqueeze(-1), table[torch.where(inside, tokens, 0)].float(), 0.0)


def _padding(padding_idx: int | None, vocab: int) -> int:
    if padding_idx is not None and not 0 <= padding_idx < vocab:
        raise DeviceError(f"embedding: the padding token must be in [0, {vocab}), got {padding_idx}")
    return -1 if padding_idx is None else int(padding_idx)


def token_order(tokens: torch.Tensor, vocab: int, padding_idx: int | None = None
                ) -> tuple[torch.Tensor, torch.Tensor]:
    """``(key, order)``, both int32 ``[R]``: the flattened tokens in ascending order and the places
    they come from, equal tokens in the order of their places.  Tokens without a gradient (outside
    ``[0, vocab)``, or ``padding_idx``) have the key ``vocab`` and come last."""
    if tokens.dtype != torch.int64 or not tokens.is_contiguous():
        raise DeviceError("embedding: tokens must be contiguous int64")
    if not 0 < vocab < 1 << 31 or tokens.numel() >= 1 << 31:
        raise DeviceError("embedding: the vocabulary and the number of tokens must be below 2^31")
    dev, R = tokens.device, tokens.numel()
    padding = _padding(padding_idx, vocab)
    if dev.type != "cuda":
        flat = tokens.reshape(-1)
        flat = torch.where((flat < 0) | (flat >= vocab) | (flat == padding), vocab, flat)
        key, order = torch.sort(flat, stable=True)
        return key.to(torch.int32), order.to(torch.int32)
    key, order = torch.empty(2, R, dtype=torch.int32, device=dev).unbind(0)
    if R:
        words = _fn("nf_token_order_words")(R)
        scratch = torch.empty(words, dtype=torch.int32, device=dev) if words else None
        with library.on_device(dev):
            library.check(_fn("nf_token_order")(tokens.data_ptr(), key.data_ptr(), order.data_ptr(),
                                                scratch.data_ptr() if words else None, R, vocab, padding, library.stream_ptr(dev)), "token_order")
    return key, order


def embedding_bwd(tokens: torch.Tensor, dout: torch.Tensor, dtable: torch.Tensor, *,
                  dpositions: torch.Tensor | None = None, scale: float = 1.0,
                  padding_idx: int | None = None, accumulate: bool = False, dropout: float = 0.0,
                  seed: int = 0, step: "int | torch.Tensor" = 0, first: int = 0,
                  order: tuple[torch.Tensor, torch.Tensor] | None = None) -> None:
    """Gradients of ``embedding_fwd`` from ``dout`` (rows of the output).

    ``dtable`` is written everywhere (rows of absent tokens become 0); with ``accumulate`` the
    gradient is added to what is there, and rows of absent tokens are left alone.  ``dpositions``
    (optional): its first T rows are written.  Both have the type of ``dout``, or float32.
    ``padding_idx``: this token's row gets no gradient.  ``order``: what ``token_order`` returned
    for these tokens (with the same vocabulary and padding), if the caller has it already."""
    if dtable.dim() != 2 or dout.dtype not in FLOAT_TYPES:
        raise DeviceError("embedding: dtable must be a matrix, dout float32, bfloat16 or float16")
    dev, (V, C) = dout.device, dtable.shape
    B, T = _tokens(tokens, dev)
    R = B * T
    padding = _padding(padding_idx, V)
    limit = limit_of(dropout, 16, "embedding")
    check_key(seed, step, dev, "embedding")
    check_first(first, "embedding")
    refuse_recording("embedding", dout, dtable, dpositions)
    if dout.numel() != R * C or (dout.numel() and dout.shape[-1] != C) or not dout.is_contiguous():
        raise DeviceError(f"embedding: dout must be {R} contiguous rows of {C}")
    _need(dtable, (V, C), (dout.dtype, torch.float32), dev, "dtable")
    if dpositions is not None:
        if dpositions.dim() != 2 or dpositions.shape[0] < T:
            raise DeviceError(f"embedding: dpositions must have at least {T} rows")
        _need(dpositions, (dpositions.shape[0], C), (dtable.dtype,), dev, "dpositions")
    if order is not None:
        for t, name in zip(order, ("key", "order")):
            _need(t, (R,), (torch.int32,), dev, name)
    if R == 0 or C == 0:
        if not accumulate:
            dtable.zero_()
        if dpositions is not None:
            dpositions[:T].zero_()
        return
    if V == 0:
        raise DeviceError("embedding: the table has no rows")
    if dev.type != "cuda":
        d = dout.reshape(B, T, C).float()
        if limit:
            kept = kept_rows(d.numel(), limit, seed, step, first, dev).view(d.shape)
            d = torch.where(kept, d * (65536 / (65536 - limit)), 0.0)
        if dpositions is not None:
            dpositions[:T].copy_(d.sum(0))
        flat = tokens.reshape(-1)
        has = (flat >= 0) & (flat < V) & (flat != padding)
        acc = torch.zeros(V, C).index_add_(0, flat[has], d.view(R, C)[has]) * scale
        if accumulate:
            seen = torch.zeros(V, dtype=torch.bool)
            seen[flat[has]] = True
            dtable.copy_(torch.where(seen[:, None], dtable.float() + acc, dtable.float()))
        else:
            dtable.copy_(acc)
        return
    key, rows = order if order is not None else (None, None)
    at, number = step_args(step)
    # (scratch of its own for every call: the allocator hands it on in stream order, and a captured
    # call's belongs to its graph)
    scratch = dout.new_empty(_bwd_words(R, C, order is not None), dtype=torch.float32)
    args = _ARGS.pack(tokens.data_ptr(), dout.data_ptr(), _address(dpositions), dtable.data_ptr(), _address(key),
                      _address(rows), scratch.data_ptr(), at, padding, B, T, V, C, first, seed, scale, limit, number,
                      FLOAT_TYPES[dout.dtype], FLOAT_TYPES[dtable.dtype], bool(accumulate), 0)
    with library.on_device(dev):
        library.check(_fn("nf_embedding_bwd")(args, library.stream_ptr(dev)), "embedding_bwd")
