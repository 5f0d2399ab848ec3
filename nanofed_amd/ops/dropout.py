"""Dropout whose mask is never stored (csrc/hip/dropout_ops.hip).

Whether a value is kept is a function of ``(seed, step, place)``: the backward pass (and a replay
of a captured step, with the step number read from device memory) draws the mask of the forward
pass again instead of reading it.  The generator is Philox4x32 with 7 rounds; the key is ``seed``
and element ``e`` of the flattened tensor (counted from ``first``) takes the 16-bit half ``e & 1``
of word ``(e >> 1) & 3`` of the block with counter ``(e >> 3, 0, step)``.  It is kept where the
half is at least ``round(65536 p)``, i.e. ``p`` is taken to a multiple of 2^-16, and what is kept
is scaled by the exact inverse of the share that is kept.  A dropped value is 0 whatever it was.

Device tensors go to the gfx950 kernel; CPU tensors run the same arithmetic in PyTorch, which is
also what the kernel tests compare against.  The reference applies ``F.dropout`` to its one network
(nanofed/models/mnist.py:22,26); this serves the GPT-2 configuration of the benchmark suite.
"""

from __future__ import annotations

import hashlib
import struct
from ctypes import c_char_p, c_int, c_void_p

import torch

from nanofed_amd.core.exceptions import DeviceError

from . import library

_SIGS = {
    "nf_dropout_args_size": ([], c_int),
    "nf_dropout": ([c_char_p, c_void_p], c_int),
}
_ARGS = struct.Struct("@4P6qQ2I2i")  # DropoutArgs of csrc/hip/dropout_ops.hip
_fns: dict[str, object] = {}

FLOAT_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def _fn(name: str):
    fn = _fns.get(name)
    if fn is None:
        argtypes, restype = _SIGS[name]
        fn = library.declare(name, argtypes, restype)
        _fns[name] = fn
    return fn


def symbols() -> list[str]:
    return sorted(_SIGS)


def site_seed(seed: int, *site) -> int:
    """A 64-bit seed for one place of a model (layer, kind of dropout) under a run's seed: places
    with different names draw independent masks."""
    text = "|".join(str(x) for x in (seed, *site))
    return int.from_bytes(hashlib.sha256(text.encode()).digest()[:8], "little")


# -- the generator ------------------------------------------------------------------------
def limit_of(p: float, bits: int, what: str) -> int:
    """The threshold ``round(2^bits p)`` of a dropout probability; one that is not 0 but would be taken
    to 0 is refused."""
    limit = round(p * (1 << bits)) if 0.0 <= p < 1.0 else 1 << bits
    if limit >= 1 << bits:
        raise DeviceError(f"{what}: the dropout probability must be in [0, 1) and round below 1 "
                          f"at {bits} bits, got {p}")
    if limit == 0 and p > 0.0:
        raise DeviceError(f"{what}: the dropout probability is taken to a multiple of 2^-{bits}, {p} would drop nothing")
    return limit


def check_key(seed: int, step: "int | torch.Tensor", device: torch.device, what: str) -> None:
    if not 0 <= seed < 1 << 64:
        raise DeviceError(f"{what}: the seed must be a 64-bit unsigned number")
    if isinstance(step, torch.Tensor):
        if step.dtype != torch.int64 or step.numel() != 1 or step.device != device:
            raise DeviceError(f"{what}: a step in memory is one int64 on the tensors' device")
    elif not 0 <= step < 1 << 32:
        raise DeviceError(f"{what}: the step must be a 32-bit unsigned number")


def step_args(step: "int | torch.Tensor") -> tuple[int, int]:
    """(address of the step in device memory or 0, its value when it is a plain number)."""
    if isinstance(step, torch.Tensor):
        return step.data_ptr(), 0
    return 0, step


def refuse_recording(what: str, *tensors: "torch.Tensor | None") -> None:
    """Raises for a tensor that autograd would follow: the kernels' results are not recorded, so its
    gradient would be lost without a word."""
    if not torch.is_grad_enabled():
        return
    for t in tensors:
        if t is not None and t.requires_grad:
            raise DeviceError(f"{what}: autograd does not record this operator: call it under torch.no_grad() (its "
                              "gradient is an operator of its own), or give it detached tensors")


def check_first(first: int, what: str) -> None:
    if not 0 <= first < 1 << 62:
        raise DeviceError(f"{what}: first must not be negative (nor pass 2^62)")


def philox_words(seed: int, step: "int | torch.Tensor", c0: torch.Tensor, c1: torch.Tensor,
                 c2: torch.Tensor) -> torch.Tensor:
    """The four 32-bit words ``[..., 4]`` (as int64) of the blocks with counter words
    ``(c0, c1, c2, step)``: the arithmetic of ``philox4x32_7`` in csrc/common/philox.h."""
    low = 0xFFFFFFFF
    k0, k1 = seed & low, seed >> 32
    c3 = torch.as_tensor(step, device=c0.device).reshape(()) & low
    x, y, z, w = torch.broadcast_tensors(c0, c1, c2, c3)
    for _ in range(7):
        a, b = x * 0xD2511F53, z * 0xCD9E8D57  # 64-bit products; the high halves survive the wrap
        x, y, z, w = (b >> 32) & low ^ y ^ k0, b & low, (a >> 32) & low ^ w ^ k1, a & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    return torch.stack([x, y, z, w], -1)


def kept_rows(n: int, limit: int, seed: int, step: "int | torch.Tensor", first: int,
              device: torch.device) -> torch.Tensor:
    """Whether each of ``n`` flattened elements from ``first`` on is kept."""
    block = torch.arange(first >> 3, (first + n + 7) >> 3, device=device)
    zero = torch.zeros_like(block)
    w = philox_words(seed, step, block & 0xFFFFFFFF, block >> 32, zero)
    halves = torch.stack([w & 0xFFFF, w >> 16], -1).reshape(-1)
    return halves[first & 7 : (first & 7) + n] >= limit


# -- the operator -------------------------------------------------------------------------
def dropout_fwd(x: torch.Tensor, p: float, *, seed: int, step: "int | torch.Tensor" = 0,
                residual: torch.Tensor | None = None, out: torch.Tensor | None = None,
                first: int = 0) -> torch.Tensor:
    """``out = dropout(x) (+ residual)`` for float32, bfloat16 or float16 tensors, computed in
    fp32 and rounded once.

    Tensors are contiguous, or two-dimensional with contiguous columns (the places of the mask
    are those of the contiguous tensor).  ``out`` may be ``x`` or ``residual``; without it a
    contiguous tensor is made.  ``step``: a number, or one int64 on the device that the kernel
    reads when it runs.  ``first``: the place of the first element, so that a tensor can be done
    in parts.  Not recorded by autograd (a tensor that requires a gradient is refused while gradients
    are enabled)."""
    limit = limit_of(p, 16, "dropout")
    if x.dtype not in FLOAT_TYPES:
        raise DeviceError(f"dropout: float32, bfloat16 or float16, got {x.dtype}")
    check_first(first, "dropout")
    check_key(seed, step, x.device, "dropout")
    refuse_recording("dropout", x, residual, out)
    if out is None:
        out = torch.empty_like(x, memory_format=torch.contiguous_format)
    for t, name in ((residual, "residual"), (out, "out")):
        if t is not None and (t.shape != x.shape or t.dtype != x.dtype or t.device != x.device):
            raise DeviceError(f"dropout: {name} must have the shape, type and device of x")
    if x.device.type != "cuda":
        y = x.float()
        if limit:
            kept = kept_rows(x.numel(), limit, seed, step, first, x.device).view(x.shape)
            y = torch.where(kept, y * (65536 / (65536 - limit)), 0.0)
        out.copy_(y if residual is None else y + residual.float())
        return out
    if x.numel() == 0:
        return out
    R, C, ld, ldr, ldo = 1, x.numel(), 0, 0, 0
    if not (x.is_contiguous() and out.is_contiguous() and (residual is None or residual.is_contiguous())):
        # some tensor has rows apart: all are walked by rows
        for t, name in ((x, "x"), (out, "out"), (residual, "residual")):
            if t is not None and (t.dim() != 2 or t.stride(1) != 1 or t.stride(0) < t.shape[1]):
                raise DeviceError(f"dropout: {name} must be contiguous, or rows of contiguous columns")
        (R, C), ld, ldo = x.shape, x.stride(0), out.stride(0)
        ldr = residual.stride(0) if residual is not None else 0
    at, number = step_args(step)
    args = _ARGS.pack(x.data_ptr(), 0 if residual is None else residual.data_ptr(), out.data_ptr(), at,
                      R, C, ld, ldr, ldo, first, seed, limit, number, FLOAT_TYPES[x.dtype], 0)
    dev = x.device
    with library.on_device(dev):
        library.check(_fn("nf_dropout")(args, library.stream_ptr(dev)), "dropout")
    return out


def dropout_bwd(dout: torch.Tensor, p: float, *, seed: int, step: "int | torch.Tensor" = 0,
                out: torch.Tensor | None = None, first: int = 0) -> torch.Tensor:
    """Gradient of ``dropout_fwd`` with respect to ``x`` (that of the residual is ``dout``): the
    same mask and scale on ``dout``."""
    return dropout_fwd(dout, p, seed=seed, step=step, out=out, first=first)
