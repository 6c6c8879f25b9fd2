"""Rotary positions with a position per token: the arithmetic of
engine.py:140-157 for tokens that are not one slice of a table, in both
layouts, for part of the head, and scaled for long contexts.

``Rotary(head_dim, theta)(q, k, positions)`` returns the rotated (q, k).  The
angle position * frequency is taken in 64-bit fixed point on the device, so no
table is kept and far positions lose nothing; cosines, sines and products are
fp64, rounded to fp32 and then to the type of q and k.
"""
from __future__ import annotations

import ctypes
import math

import torch

from . import _lib

TWO_PI_E50 = 628318530717958647692528676655900576839433879875021   # 2 pi 10^50
LAYOUTS = ("half", "interleaved")
# the keys that each kind of scaling takes
SCALINGS = {
    "linear": ("factor",),
    "ntk": ("factor",),
    "wavelength": ("factor", "original_len", "low_factor", "high_factor"),
    "yarn": ("factor", "original_len", "beta_fast", "beta_slow"),
}


def rotary_frequencies(rotary_dim: int, theta: float, scaling: dict | None = None) -> tuple[list[float], float]:
    """(radians per position of each pair, magnitude).

    Without scaling pair j turns by theta^(-2 j / rotary_dim) a position
    (engine.py:128-137).  ``scaling`` is a dict with a ``type``:

    linear      every frequency over ``factor``
    ntk         theta times factor^(rotary_dim / (rotary_dim - 2)): the fastest
                pair stays, the slowest is slowed by ``factor``
    wavelength  pairs that turn less than ``low_factor`` times over
                ``original_len`` positions are slowed by ``factor``, those that
                turn more than ``high_factor`` times stay, linear between
    yarn        pairs are slowed by ``factor`` from the one that turns
                ``beta_slow`` times over ``original_len`` positions on, stay up
                to the one that turns ``beta_fast`` times, linear in j between;
                the rotated values grow by 0.1 ln(factor) + 1; a factor of at
                least 1, and ``beta_fast`` no less than ``beta_slow``
    """
    theta = float(theta)
    if not (math.isfinite(theta) and theta > 1.0):
        raise ValueError(f"theta {theta}: a number above 1")
    magnitude = 1.0
    s = dict(scaling) if scaling else None
    if s is not None:
        kind = s.pop("type", None)
        if kind not in SCALINGS:
            raise ValueError(f"rotary scaling {kind!r}: one of {', '.join(SCALINGS)}")
        if set(s) != set(SCALINGS[kind]):
            raise ValueError(f"rotary scaling {kind!r} takes {', '.join(SCALINGS[kind])}, got {', '.join(sorted(s))}")
        if not all(math.isfinite(v) and v > 0 for v in s.values()):
            raise ValueError(f"rotary scaling {kind!r}: positive numbers, got {s}")
        if kind == "ntk":
            if rotary_dim <= 2:
                raise ValueError("rotary scaling 'ntk' needs more than one pair")
            theta *= s["factor"] ** (rotary_dim / (rotary_dim - 2))
        if kind == "yarn" and s["factor"] < 1:
            raise ValueError("rotary scaling 'yarn' lengthens contexts: a factor of at least 1")
        if kind == "yarn" and s["beta_fast"] < s["beta_slow"]:
            raise ValueError("rotary scaling 'yarn': beta_fast below beta_slow")
        if kind == "wavelength" and s["high_factor"] <= s["low_factor"]:
            raise ValueError("rotary scaling 'wavelength': high_factor above low_factor")
    f = [theta ** (-2.0 * j / rotary_dim) for j in range(rotary_dim // 2)]
    if s is None:
        return f, magnitude
    if kind == "linear":
        f = [x / s["factor"] for x in f]
    elif kind == "wavelength":
        lo, hi = s["low_factor"], s["high_factor"]
        keep = [min(max((s["original_len"] * x / (2 * math.pi) - lo) / (hi - lo), 0.0), 1.0) for x in f]
        f = [x * k + x / s["factor"] * (1 - k) for x, k in zip(f, keep)]
    elif kind == "yarn":
        def pair(turns):   # the place in the rotated dims that turns so often over original_len positions
            return rotary_dim * math.log(s["original_len"] / (turns * 2 * math.pi)) / (2 * math.log(theta))
        lo, hi = max(math.floor(pair(s["beta_fast"])), 0), min(math.ceil(pair(s["beta_slow"])), rotary_dim - 1)
        slow = [min(max((j - lo) / max(hi - lo, 0.001), 0.0), 1.0) for j in range(rotary_dim // 2)]
        f = [x * (1 - k) + x / s["factor"] * k for x, k in zip(f, slow)]
        magnitude = 0.1 * math.log(s["factor"]) + 1.0
    return f, magnitude


class Rotary:
    """Rotary positions of heads of ``head_dim``: the first ``rotary_dim`` dims
    (all by default) in pairs (j, j + rotary_dim / 2) (``layout="half"``, the
    reference's) or (2 j, 2 j + 1) (``"interleaved"``); the others are copied.
    ``scaling`` as in ``rotary_frequencies``."""

    def __init__(self, head_dim: int, theta: float, rotary_dim: int | None = None, layout: str = "half",
                 scaling: dict | None = None, device="cuda"):
        self.head_dim = int(head_dim)
        self.rotary_dim = self.head_dim if rotary_dim is None else int(rotary_dim)
        if self.head_dim < 2 or self.head_dim > 256 or self.head_dim % 2:
            raise ValueError(f"head_dim {head_dim}: even, 2 to 256")
        if self.rotary_dim < 2 or self.rotary_dim > self.head_dim or self.rotary_dim % 2:
            raise ValueError(f"rotary_dim {rotary_dim}: even, 2 to head_dim {self.head_dim}")
        if layout not in LAYOUTS:
            raise ValueError(f"layout {layout!r}: one of {', '.join(LAYOUTS)}")
        self.layout = layout
        freq, self.magnitude = rotary_frequencies(self.rotary_dim, theta, scaling)
        # whole turns in 2^-64 a position, to the nearest: 2^64 x / (2 pi) of the exact x
        turns = [((n << 65) * 10 ** 50 // (d * TWO_PI_E50) + 1 >> 1) % 2 ** 64
                 for n, d in (x.as_integer_ratio() for x in freq)]
        self.device = _lib.gpu(device)
        # 64-bit patterns; torch's unsigned type has few operations
        self.freq = torch.tensor([t - 2 ** 64 if t >= 2 ** 63 else t for t in turns], dtype=torch.int64,
                                 device=self.device)
        self._struct = _lib.Rotary(self.head_dim, self.rotary_dim, int(layout == "interleaved"), self.magnitude,
                                   self.freq.data_ptr())
        self._ref = ctypes.byref(self._struct)

    def _rows(self, x: torch.Tensor, what: str):
        shape = x.shape
        if len(shape) != 3 or shape[2] != self.head_dim:
            raise ValueError(f"{what}: (tokens, heads, {self.head_dim}), got {tuple(shape)}")
        if x.dtype not in (torch.float16, torch.bfloat16):
            raise TypeError(f"{what}: float16 or bfloat16, got {x.dtype}")
        if x.device != self.device:
            raise ValueError(f"{what} on {x.device}, the rotary frequencies on {self.device}")
        return _lib.heads(x, shape[1])

    def _output(self, out, x: torch.Tensor, what: str, zeros: bool = False) -> torch.Tensor:
        if out is None:
            return (torch.zeros_like if zeros else torch.empty_like)(x, memory_format=torch.contiguous_format)
        if out.shape != x.shape or out.dtype != x.dtype or out.device != x.device or not out.is_contiguous():
            raise ValueError(f"{what} must be a contiguous tensor like its input")
        return out

    def __call__(self, q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor, q_out=None, k_out=None):
        """(q, k) rotated: q (tokens, n_q, head_dim), k (tokens, n_kv, head_dim)
        or None, fp16 or bf16, any strides; positions (tokens) int32.  q_out and
        k_out: contiguous outputs, which may be the inputs themselves.  A token
        at a negative position is left out: its rows of these are not written,
        those of new outputs are 0."""
        q, hq = self._rows(q, "q")
        N = q.shape[0]
        hk = _lib.Heads()
        if k is not None:
            k, hk = self._rows(k, "k")
            if k.shape[0] != N or k.dtype != q.dtype:
                raise ValueError(f"k {tuple(k.shape)} {k.dtype} beside q {tuple(q.shape)} {q.dtype}")
        if positions.shape != (N,) or positions.dtype != torch.int32 or positions.device != self.device:
            raise ValueError(f"positions: ({N},) int32 on {self.device}, got {tuple(positions.shape)} "
                             f"{positions.dtype} on {positions.device}")
        new = q_out is None and (k is None or k_out is None)
        qo = self._output(q_out, q, "q_out", not new)
        ko = None if k is None else self._output(k_out, k, "k_out", not new)
        for x, o in ((q, qo), (k, ko)):
            if x is not None and o.data_ptr() == x.data_ptr() and not x.is_contiguous():
                raise ValueError("an output that is its own input must be contiguous")
        L = _lib.load_library()
        with _lib.on_device(self.device) as stream:
            _lib.check(L.oi2_rotary_apply(
                self._ref, _lib.dtype_code(q.dtype) | (_lib.ZERO_LEFT_OUT if new else 0), N, positions.contiguous().data_ptr(),
                ctypes.byref(hq), qo.data_ptr(),
                ctypes.byref(hk), _lib.ptr(ko),
                stream))
        return qo, ko
