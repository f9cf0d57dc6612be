"""Rotary positions of a layer's queries and keys (sbsa_rotary).

The sparse layer takes Q and K before and after the rotary embedding (the reference's host
model makes both in its ``_project_qkv``, semblo/vllm_plugin/qwen3_5_model.py:135-189).
``RotaryEmbedding`` makes the rotated ones from those before, in one launch:

    rotary = RotaryEmbedding(256, rotary_dim=64, base=1e7, sections=(11, 11, 10))
    q_post, k_post = rotary(positions, q_pre, k_pre)

Angles are exact at any position: a pair's frequency is kept as a 64-bit fraction of a turn
per position, so that no table over positions is held and none is read.
"""
from __future__ import annotations

import math
from fractions import Fraction

import torch

from . import _lib


def _corrected_dim(turns: float, rotary_dim: int, base: float, length: float) -> float:
    """The (fractional) pair index whose pair makes ``turns`` turns over ``length`` positions."""
    return rotary_dim * math.log(length / (turns * 2 * math.pi)) / (2 * math.log(base))


def rotary_frequencies(rotary_dim: int, base: float = 10000.0, scaling: dict | None = None) -> tuple[list[float], float]:
    """Radians per position of each pair, and the gain on the rotated values.

    ``scaling`` (for contexts longer than the trained one) is a dict of ``kind`` and ``factor``:
      linear   every frequency over the factor
      ntk      the base times factor^(r / (r - 2)): the slowest pair over the factor, the fastest as it was
      yarn     by the turns a pair makes over ``original_length``: over ``beta_fast`` (32) it keeps its
               frequency, under ``beta_slow`` (1) it goes over the factor, a ramp in the pair's index between;
               the gain is ``gain``, or 0.1 ln(factor) + 1
      banded   the same between ``high_factor`` (4) and ``low_factor`` (1) turns, a ramp in the turns
    """
    sc = dict(scaling or {})
    kind = sc.pop("kind", None)
    known = {None: (), "linear": ("factor",), "ntk": ("factor",),
             "yarn": ("factor", "original_length", "beta_fast", "beta_slow", "gain"),
             "banded": ("factor", "original_length", "low_factor", "high_factor")}
    if kind not in known:
        raise ValueError(f"unknown rotary scaling {kind!r}: one of linear, ntk, yarn, banded")
    extra = set(sc) - set(known[kind])
    if extra:
        raise ValueError(f"rotary scaling {kind!r} takes no {sorted(extra)}")
    factor = float(sc.get("factor", 1.0))
    if kind is not None and not (math.isfinite(factor) and factor > 0):
        raise ValueError("rotary scaling needs a positive factor")
    if not (math.isfinite(base) and base > 1):
        raise ValueError("the rotary base is a number above 1")
    r = rotary_dim
    if kind == "ntk":
        base = base * factor ** (r / max(r - 2, 1))
    freq = [base ** (-2.0 * i / r) for i in range(r // 2)]
    if kind in (None, "ntk"):
        return freq, 1.0
    if kind == "linear":
        return [f / factor for f in freq], 1.0
    length = float(sc.get("original_length", 0))
    if not length > 0:
        raise ValueError(f"rotary scaling {kind!r} needs the trained original_length")
    if kind == "banded":
        low, high = float(sc.get("low_factor", 1.0)), float(sc.get("high_factor", 4.0))
        if not high > low:
            raise ValueError("rotary scaling 'banded' needs high_factor above low_factor")
        own = [min(1.0, max(0.0, (length * f / (2 * math.pi) - low) / (high - low))) for f in freq]
        return [f * (w + (1 - w) / factor) for f, w in zip(freq, own)], 1.0
    low = max(math.floor(_corrected_dim(float(sc.get("beta_fast", 32.0)), r, base, length)), 0)
    high = min(math.ceil(_corrected_dim(float(sc.get("beta_slow", 1.0)), r, base, length)), r - 1)
    ramp = [min(1.0, max(0.0, (i - low) / max(high - low, 0.001))) for i in range(r // 2)]
    gain = float(sc.get("gain", 0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0))
    if not (math.isfinite(gain) and gain > 0):
        raise ValueError("the rotary gain is a positive number")
    return [f * (1 - w) + f / factor * w for f, w in zip(freq, ramp)], gain


def section_axes(sections, pairs: int, interleaved: bool = False) -> list[int]:
    """Each pair's axis for positions on several axes (M-RoPE): ``sections`` pairs of each axis one
    after another, or dealt out in turn (axis i takes pairs i, i + 3, ... until it has its own;
    the rest go to axis 0)."""
    sections = [int(n) for n in sections]
    if not 1 <= len(sections) <= 255 or min(sections) < 0 or sum(sections) != pairs:
        raise ValueError(f"sections {sections} must add up to the {pairs} rotated pairs")
    if not interleaved:
        return [a for a, n in enumerate(sections) for _ in range(n)]
    axes = [0] * pairs
    for a, n in enumerate(sections):
        if a:
            for i in range(a, min(pairs, a + n * len(sections)), len(sections)):
                axes[i] = a
    return axes


class RotaryEmbedding:
    """The rotary embedding of one model's heads.

    ``head_dim`` up to 512, of which the first ``rotary_dim`` (even; all by default) turn; ``interleaved``: pairs are
    neighbours (2i, 2i + 1) instead of (i, i + rotary_dim / 2).  ``scaling``: ``rotary_frequencies``.
    ``sections``: positions then come as a grid [axes, T], and each pair takes its angle from one axis
    (``section_axes``; ``sections_interleaved`` deals the pairs out in turn).
    """

    def __init__(self, head_dim: int, *, rotary_dim: int | None = None, base: float = 10000.0,
                 interleaved: bool = False, scaling: dict | None = None, sections=None,
                 sections_interleaved: bool = False) -> None:
        rotary_dim = head_dim if rotary_dim is None else int(rotary_dim)
        if not (2 <= rotary_dim <= head_dim <= 512) or rotary_dim % 2:
            raise ValueError(f"rotary_dim {rotary_dim} must be even, within a head of {head_dim} (at most 512)")
        self.head_dim, self.rotary_dim, self.interleaved = int(head_dim), rotary_dim, bool(interleaved)
        self.frequencies, self.gain = rotary_frequencies(rotary_dim, float(base), scaling)
        # radians to turns (the quotient by 2 pi, in 64 bits), then to 2^-64 turns
        turns = [int(Fraction(f / (2 * math.pi)) * 2 ** 64) % 2 ** 64 for f in self.frequencies]
        self._turns = torch.tensor([t - 2 ** 64 if t >= 2 ** 63 else t for t in turns], dtype=torch.int64)
        self.num_axes = 1 if sections is None else len(tuple(sections))
        self._axes = None if sections is None else torch.tensor(
            section_axes(sections, rotary_dim // 2, sections_interleaved), dtype=torch.uint8)
        self._on: dict = {}

    def _tables(self, q: torch.Tensor):
        """(turns, axes, their addresses) on q's device."""
        tables = self._on.get(q.get_device())
        if tables is None:
            turns, axes = self._turns.to(q.device), None if self._axes is None else self._axes.to(q.device)
            tables = self._on[q.get_device()] = (turns, axes, turns.data_ptr(), None if axes is None else axes.data_ptr())
        return tables

    def _rows(self, x: torch.Tensor, what: str, tokens: int):
        """(heads, token stride, head stride) of a call's queries or keys."""
        shape, stride = x.shape, x.stride()
        if len(shape) != 3 or shape[0] != tokens or shape[2] != self.head_dim:
            raise ValueError(f"{what} must be [{tokens}, heads, {self.head_dim}], got {list(x.shape)}")
        if x.dtype is not torch.bfloat16 or stride[2] != 1:
            raise ValueError(f"{what} must be bfloat16 with a unit inner stride")
        if x.requires_grad and torch.is_grad_enabled():
            raise RuntimeError("the rotary embedding has no backward pass: call it under torch.no_grad()")
        return shape[1], stride[0], stride[1]

    def __call__(self, positions: torch.Tensor, q: torch.Tensor, k: torch.Tensor | None = None, *,
                 out_q: torch.Tensor | None = None, out_k: torch.Tensor | None = None, inverse: bool = False):
        """Rotated copies of ``q`` [T, Hq, D] and ``k`` [T, Hkv, D] (None: of q alone), bfloat16 with any token
        and head strides.  ``positions``: int32 or int64 [T], or the grid [axes, T] where the embedding has sections;
        negative ones too.  ``out_q``, ``out_k``: where to; the inputs themselves rotate in place.
        ``inverse`` rotates back (keys before the embedding from a cache's)."""
        tokens = q.shape[0]
        hq, qst, qsh = self._rows(q, "q", tokens)
        if positions.dtype is not torch.int64 and positions.dtype is not torch.int32:
            raise ValueError("positions must be int32 or int64")
        if positions.shape != ((tokens,) if self._axes is None else (self.num_axes, tokens)):
            raise ValueError(f"positions must be {[tokens] if self._axes is None else [self.num_axes, tokens]}, "
                             f"got {list(positions.shape)}")
        device = q.device
        given = out_q is not None or out_k is not None
        if out_q is None:
            out_q = _lib.rows_like(q)
        else:
            self._output(out_q, q, "out_q")
        ost, osh, _ = out_q.stride()
        if k is None:
            if out_k is not None:
                raise ValueError("out_k without k")
            kv = (None, 0, 0, None, 0, 0, 0)
        else:
            hkv, kst, ksh = self._rows(k, "k", tokens)
            if out_k is None:
                out_k = _lib.rows_like(k)
            else:
                self._output(out_k, k, "out_k")
            okst, oksh, _ = out_k.stride()
            kv = (k.data_ptr(), kst, ksh, out_k.data_ptr(), okst, oksh, hkv)
            if given and (_lib.rows_overlap(out_q, k) or _lib.rows_overlap(out_k, q) or _lib.rows_overlap(out_q, out_k)):
                raise ValueError("an output overlaps the other one, or the other input")
        _lib.require_one_device(q, out_q, positions, k, out_k)
        _, axes, turns_at, axes_at = self._tables(q)
        _lib.call_on(device, "sbsa_rotary", q.data_ptr(), qst, qsh, out_q.data_ptr(), ost, osh, hq, *kv,
                     positions.data_ptr(), positions.element_size(), positions.stride(0) if axes is not None else 0,
                     positions.stride(-1), tokens, self.head_dim, self.rotary_dim, self.interleaved, turns_at,
                     axes_at, self.gain, inverse)
        return out_q if k is None else (out_q, out_k)

    def _output(self, out: torch.Tensor, x: torch.Tensor, what: str) -> None:
        if out.shape != x.shape or out.dtype != x.dtype or out.stride(2) != 1 or not all(out.stride()):
            raise ValueError(f"{what} must have its input's shape and type, a unit inner stride and no stride of 0")
        if out.stride() != x.stride() or out.data_ptr() != x.data_ptr():
            if _lib.overlap(out, x):
                raise ValueError(f"{what} overlaps its input without being it")
