"""Rotary position embedding from positions, on an MI355X.

The rotary prologue of ``rope.py`` takes cos / sin tables of the whole head in
the half layout, as transformers makes them.  Here the kernel is given the
positions and the frequencies and computes the angles itself: the half or the
interleaved layout, the whole head or its first columns, frequencies scaled
for contexts longer than the model was trained on, and no table (1 million
positions of 128 columns would be 512 MiB).  ``fa_rotary`` reads q and k once
and writes them once; its backward is the same kernel with negative angles.

    rotary = RotaryPositions(64, base=500000.0,
                             scaling={"type": "yarn", "factor": 8, "original_length": 8192})
    q_out, k_out = apply_rotary_positions(q, k, positions, rotary)

Semantics per row x (one (b, s, head)) at position p, pair j of R / 2:
    a' = m (a cos(p f_j) - b sin(p f_j)),   b' = m (b cos(p f_j) + a sin(p f_j))
with (a, b) = x[j], x[R/2 + j] (half) or x[2j], x[2j + 1] (interleaved), the
columns from R on unchanged, in fp32, rounded once.

The reference has no counterpart: it leaves rotary embeddings to transformers
(flash_attn_volta/patch_hf.py:177, :291-303, :462).
"""
from __future__ import annotations

import ctypes
import math
from fractions import Fraction

import torch

from . import _capi, _runtime
from .autograd import _compiling, _cpp, _transforms_active
from .forward import (FlashAttnArgumentError, _DTYPES, _kernel_ready, _on_device, _require,
                      _stream_ptr, kernel_strides)

__all__ = ["RotaryPositions", "apply_rotary_positions", "rotary_forward", "rotary_backward"]

# 2^64 / (2 pi) in units of 2^-80 (2 pi to 50 digits): a step is exact to 2^-64
# turns whatever the frequency
_TURN = round(Fraction(1 << 144) / Fraction("6.28318530717958647692528676655900576839433879875021"))


def _step(f: float) -> int:
    """f / (2 pi) turns a position, mod 1 in units of 2^-64, as an int64."""
    n, d = f.as_integer_ratio()
    s = ((n * _TURN // d + (1 << 79)) >> 80) % (1 << 64)
    return s - (1 << 64) if s >> 63 else s


def _number(scaling: dict, name: str, default=None) -> float:
    v = scaling.get(name, default)
    _require(isinstance(v, (int, float)) and not isinstance(v, bool) and math.isfinite(v) and v > 0,
             lambda: f"scaling[{name!r}] must be a positive number, got {v!r}")
    return float(v)


def _plain_frequencies(R: int, base: float) -> list:
    return [base ** (-2.0 * j / R) for j in range(R // 2)]


def _scaled_frequencies(R: int, base: float, scaling: dict | None):
    """(R / 2 frequencies in radians a position, m)."""
    if scaling is None:
        return _plain_frequencies(R, base), 1.0
    _require(isinstance(scaling, dict), lambda: f"scaling must be a dict or None, got {scaling!r}")
    kind = scaling.get("type")
    known = {"linear": {"factor"}, "ntk": {"factor"},
             "yarn": {"factor", "original_length", "beta_fast", "beta_slow", "attention_factor"},
             "wavelength": {"factor", "original_length", "low", "high"},
             "factors": {"factors", "attention_factor"}}
    _require(kind in known, lambda: f"scaling type {kind!r} is none of {sorted(known)}")
    extra = set(scaling) - known[kind] - {"type"}
    _require(not extra, lambda: f"scaling type {kind!r} takes no {sorted(extra)}")
    if kind == "factors":
        f, factors = _plain_frequencies(R, base), scaling.get("factors")
        _require(isinstance(factors, (list, tuple)) and len(factors) == R // 2,
                 lambda: f"scaling['factors'] must be {R // 2} numbers")
        for i in range(len(factors)):
            _number({"factors": factors[i]}, "factors")
        return ([x / float(y) for x, y in zip(f, factors)],
                _number(scaling, "attention_factor", 1.0))
    factor = _number(scaling, "factor")
    if kind == "ntk":
        # the base grown so that the slowest pair turns `factor` times slower
        return _plain_frequencies(R, base * factor ** (R / max(R - 2, 1))), 1.0
    f = _plain_frequencies(R, base)
    if kind == "linear":
        return [x / factor for x in f], 1.0
    length = _number(scaling, "original_length")
    if kind == "yarn":
        # Pairs that turn over beta_fast times in the original length keep
        # their frequency, those under beta_slow turns get it divided, a
        # ramp over the pairs' numbers in between.
        _require(base > 1.0, lambda: f"yarn scaling needs a base over 1, got {base}")
        lo, hi = (R * math.log(length / (2 * math.pi * turns)) / (2 * math.log(base))
                  for turns in (_number(scaling, "beta_fast", 32.0),
                                _number(scaling, "beta_slow", 1.0)))
        lo, hi = max(math.floor(lo), 0), min(math.ceil(hi), R - 1)
        ramp = [min(max((j - lo) / max(hi - lo, 1e-3), 0.0), 1.0) for j in range(R // 2)]
        m = _number(scaling, "attention_factor",
                    0.1 * math.log(factor) + 1.0 if factor > 1.0 else 1.0)
        return [x / factor * r + x * (1.0 - r) for x, r in zip(f, ramp)], m
    # wavelength: pairs with more than `high` turns in the original length
    # keep their frequency, those with fewer than `low` get it divided,
    # linear in the number of turns in between
    low, high = _number(scaling, "low"), _number(scaling, "high")
    _require(high > low, lambda: f"scaling['high'] must be over scaling['low'], got {high} {low}")
    out = []
    for x in f:
        s = min(max((length * x / (2 * math.pi) - low) / (high - low), 0.0), 1.0)
        out.append((1.0 - s) * x / factor + s * x)
    return out, 1.0


class RotaryPositions:
    """The frequencies of a model's rotary embedding, laid out once.

    Args:
        rotary_dim: R, the columns that are rotated (the first of a head), even.
        base: f_j = base^(-2j / R).
        interleaved: pairs (2j, 2j + 1) instead of (j, R/2 + j).
        scaling: None, or a dict with a "type":
            "linear": factor -- every frequency divided;
            "ntk": factor -- the base times factor^(R / (R - 2));
            "yarn": factor, original_length, beta_fast = 32, beta_slow = 1,
                attention_factor = 0.1 ln(factor) + 1 (the m above);
            "wavelength": factor, original_length, low, high (turns);
            "factors": factors -- R / 2 divisors, attention_factor = 1.
        device: where q and k are.

    Attributes: rotary_dim, interleaved, attention_factor, frequencies (R / 2
    floats, radians a position), steps (the device tensor the kernels read).
    """

    __slots__ = ("_args", "_frequencies")

    def __init__(self, rotary_dim: int, base: float = 10000.0, *, interleaved: bool = False,
                 scaling: dict | None = None, device="cuda"):
        _require(isinstance(rotary_dim, int) and 2 <= rotary_dim <= 256 and rotary_dim % 2 == 0,
                 lambda: f"rotary_dim must be an even number from 2 to 256, got {rotary_dim!r}")
        _require(isinstance(base, (int, float)) and math.isfinite(base) and base > 0,
                 lambda: f"base must be a positive number, got {base!r}")
        try:
            self._frequencies, factor = _scaled_frequencies(rotary_dim, float(base), scaling)
        except OverflowError:
            self._frequencies, factor = [math.inf], 1.0
        _require(all(map(math.isfinite, self._frequencies)),
                 lambda: f"base {base!r} and this scaling give frequencies that are not finite")
        _require(factor <= torch.finfo(torch.float32).max,
                 lambda: f"attention_factor {factor!r} is over fp32's largest number")
        steps = torch.tensor([_step(f) for f in self._frequencies], dtype=torch.int64, device=device)
        # (fixed: the kernels read rotary_dim / 2 steps)
        self._args = (steps, factor, rotary_dim, _capi.FA_ROTARY_INTERLEAVED if interleaved else 0)

    steps = property(lambda self: self._args[0])
    attention_factor = property(lambda self: self._args[1])
    rotary_dim = property(lambda self: self._args[2])
    interleaved = property(lambda self: bool(self._args[3]))
    frequencies = property(lambda self: list(self._frequencies))
    _flags = property(lambda self: self._args[3])

    def __repr__(self):
        return (f"RotaryPositions(rotary_dim={self.rotary_dim}, interleaved={self.interleaved}, "
                f"attention_factor={self.attention_factor:g}, device={self.steps.device})")


def _check(q, k, rotary):
    _require(isinstance(rotary, RotaryPositions),
             lambda: f"rotary must be a RotaryPositions, got {type(rotary).__name__}")
    _require(q.is_cuda and (k is None or k.is_cuda), "q and k must be on the GPU")
    _require(k is None or q.device == k.device, "q and k must be on one device")
    _require(rotary.steps.device == q.device,
             lambda: f"rotary is on {rotary.steps.device}, q on {q.device}")
    _require(q.dtype in _DTYPES and (k is None or q.dtype == k.dtype),
             lambda: f"fp16 or bf16 only, q and k alike (got {q.dtype}, {getattr(k, 'dtype', None)})")
    _require(q.dim() == 4 and (k is None or k.dim() == 4),
             "expected (B, S, H, D) tensors")
    _require(k is None or (q.shape[:2] == k.shape[:2] and q.shape[3] == k.shape[3]),
             lambda: f"q {tuple(q.shape)} and k {tuple(k.shape)} differ outside the head dimension")
    D = q.shape[3]
    _require(D % 8 == 0 and 8 <= D <= 256,
             lambda: f"unsupported head_dim {D} (a multiple of 8, at most 256)")
    _require(rotary.rotary_dim <= D,
             lambda: f"rotary_dim {rotary.rotary_dim} is over the head_dim {D}")


def _positions(t, B: int, S: int, device):
    """positions as (1 or B, S) int32 or int64 on the device."""
    _require(isinstance(t, torch.Tensor) and t.dtype in (torch.int32, torch.int64),
             "positions must be an int32 or int64 tensor")
    if t.dim() == 1:
        t = t.unsqueeze(0)
    _require(t.dim() == 2 and t.shape[1] == S and t.shape[0] in (1, B),
             lambda: f"positions must be (B or 1, S) = (.., {S}) or ({S},), got {tuple(t.shape)}")
    _require(t.device == device, lambda: f"positions must be on {device}")
    return t


def _launch(q, k, positions, rotary, inverse):
    """(q, k) rotated; the arguments are checked."""
    B, S, H, D = q.shape
    Hk = 0 if k is None else k.shape[2]
    q_out = torch.empty((B, S, H, D), dtype=q.dtype, device=q.device)
    k_out = None if k is None else torch.empty((B, S, Hk, D), dtype=q.dtype, device=q.device)
    if B * S == 0 or H + Hk == 0:
        return q_out, k_out
    if H == 0:                               # the C ABI's first tensor is not empty
        return q_out, _launch(k, None, positions, rotary, inverse)[0]
    q = _kernel_ready(q)
    if Hk:
        k = _kernel_ready(k)
    flags = rotary._flags | (_capi.FA_ROTARY_INVERSE if inverse else 0)
    if positions.dtype == torch.int64:
        flags |= _capi.FA_ROTARY_POS64
    pst = (ctypes.c_int64 * 2)(0 if positions.shape[0] == 1 else positions.stride(0),
                               positions.stride(1))
    lib = _capi.load()
    with _on_device(q.device):
        rc = lib.fa_rotary(
            q.data_ptr(), k.data_ptr() if Hk else None, q_out.data_ptr(),
            k_out.data_ptr() if Hk else None, rotary.steps.data_ptr(), rotary.attention_factor,
            rotary.rotary_dim, flags, positions.data_ptr(), pst, B, S, H, Hk, D,
            kernel_strides(q), kernel_strides(k) if Hk else None, kernel_strides(q_out),
            kernel_strides(k_out) if Hk else None, _DTYPES[q.dtype], _stream_ptr(q.device))
    _capi.check(rc, "fa_rotary")
    return q_out, k_out


def rotary_forward(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor,
                   rotary: RotaryPositions):
    """(q_out, k_out), contiguous, in q's dtype (k_out None without k): see
    apply_rotary_positions.  No autograd."""
    _check(q, k, rotary)
    return _launch(q, k, _positions(positions, q.shape[0], q.shape[1], q.device), rotary, False)


def rotary_backward(dq_out: torch.Tensor, dk_out: torch.Tensor | None, positions: torch.Tensor,
                    rotary: RotaryPositions):
    """(dq, dk): the gradients of rotary_forward's q and k from those of its
    outputs."""
    _check(dq_out, dk_out, rotary)
    return _launch(dq_out, dk_out,
                   _positions(positions, dq_out.shape[0], dq_out.shape[1], dq_out.device), rotary,
                   True)


class _RotaryFn(torch.autograd.Function):
    """The rotation, or with `inverse` its gradient: each is the other's, so
    gradients of gradients work too."""

    @staticmethod
    def forward(ctx, q, k, positions, rotary, inverse):
        ctx.save_for_backward(positions)
        ctx.rotary, ctx.inverse, ctx.dtype = rotary, inverse, q.dtype
        return _launch(q, k, positions, rotary, inverse)

    @staticmethod
    def backward(ctx, g_q, g_k):
        positions, = ctx.saved_tensors
        need_q, need_k = ctx.needs_input_grad[:2]
        # a side that needs no gradient is not rotated
        sides = [g.to(ctx.dtype) for n, g in ((need_q, g_q), (need_k, g_k))
                 if n and g is not None]
        if not sides:
            return None, None, None, None, None
        run = _RotaryFn.apply if torch.is_grad_enabled() else _launch
        got = run(sides[0], sides[1] if len(sides) > 1 else None, positions, ctx.rotary,
                  not ctx.inverse)
        if len(sides) > 1:
            return got[0], got[1], None, None, None
        return (got[0], None, None, None, None) if need_q and g_q is not None \
            else (None, got[0], None, None, None)


def apply_rotary_positions(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor,
                           rotary: RotaryPositions):
    """Autograd-aware rotation of q and k by their positions (no counterpart in
    the reference, which calls transformers' apply_rotary_pos_emb,
    patch_hf.py:177, :462).

    Args:
        q: (B, S, H, D), k: (B, S, Hk, D) or None, fp16 or bf16 on the GPU, D a
            multiple of 8 up to 256, any strides with unit D stride (others
            are copied).
        positions: (B or 1, S) or (S,) int32 or int64 on the GPU; any values.
        rotary: the frequencies (RotaryPositions), on q's device.

    Returns:
        (q_out, k_out): contiguous (B, S, H, D) / (B, S, Hk, D) in q's dtype
        (k_out None without k).  Gradients flow to q and k.
    """
    if _cpp is not None and isinstance(rotary, RotaryPositions) and not _transforms_active() \
            and not _compiling() and all(isinstance(t, torch.Tensor) for t in (q, positions)) \
            and (k is None or isinstance(k, torch.Tensor)):
        out = _cpp.rotary(q, k, positions, *rotary._args)
        if out is not None:
            return out
    _check(q, k, rotary)
    positions = _positions(positions, q.shape[0], q.shape[1], q.device)
    if not (torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad))):
        return _launch(q, k, positions, rotary, False)
    if _cpp is not None and not _compiling() and _runtime.capturing():
        for t in (q, k):
            _require(t is None or not _cpp.held_on_another_stream(t),
                     "an autograd graph of q or k, made on another stream, is alive: a "
                     "backward pass cannot be captured beside it; drop its outputs first")
    return _RotaryFn.apply(q, k, positions, rotary, False)
