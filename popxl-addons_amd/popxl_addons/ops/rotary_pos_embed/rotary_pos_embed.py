"""Rotary positions on the GPU: queries and keys turned pair by pair by an angle that grows with the position.

For the pair (a, b) number i of a row at position p:  (a, b) -> c (a cos p w_i - b sin p w_i, a sin p w_i + b cos p w_i) with
w_i = base^(-2 i / rotary_dim), stretched or not, and c = 1 or the attention factor of the stretching.  The inverse (the angle's
sign turned, the same factor) is the operator's gradient.
"""
import ctypes
import math

import numpy as np

from popxl_addons import _gq_hip

__all__ = ["RotaryPosEmbed", "rotary_frequencies", "rotary_pos_embed"]

_LAYOUTS = {"interleaved": _gq_hip.GQ_ROTARY_INTERLEAVED, "half": _gq_hip.GQ_ROTARY_HALF}


def rotary_frequencies(rotary_dim, base=10000.0, scaling=None):
    """
    Radians a position of every pair, float64 [rotary_dim / 2], and the factor of the turned values.

    scaling: None, or a dict with "kind" and "factor" s for contexts s times as long as the trained one:
        linear  w / s (positions interpolated)
        ntk     base * s^(r / (r - 2)): the slowest pair is stretched by s, the fastest hardly at all
        yarn    pairs that turn more than beta_fast (32) times in original_length keep w, those that turn less than beta_slow (1)
                times get w / s; in between (turns - beta_slow) / (beta_fast - beta_slow) of w stays, as the paper has it
                (https://arxiv.org/abs/2309.00071): linear in the turns, not in the number of the pair between two corners.  A model
                that was tuned with another ramp needs its own frequencies (RotaryPosEmbed.from_frequencies); factor 0.1 ln s + 1
    """
    if rotary_dim < 2 or rotary_dim % 2 != 0:
        raise ValueError(f"rotary_dim={rotary_dim} must be even and positive")
    if not (math.isfinite(base) and base > 0):
        raise ValueError(f"base={base} must be positive")
    exponent = np.arange(0, rotary_dim, 2, dtype=np.float64) / rotary_dim
    w = float(base) ** -exponent
    if scaling is None:
        return w, 1.0
    known = {"linear": set(), "ntk": set(), "yarn": {"original_length", "beta_fast", "beta_slow"}}
    kind = scaling.get("kind")
    if kind not in known:
        raise ValueError(f"unknown rotary scaling {kind!r}; expected one of {sorted(known)}")
    if set(scaling) - {"kind", "factor"} - known[kind]:
        raise ValueError(f"rotary scaling {kind!r} does not take {sorted(set(scaling) - {'kind', 'factor'} - known[kind])}")
    s = float(scaling.get("factor", 0))
    if not (math.isfinite(s) and s >= 1):
        raise ValueError(f"rotary scaling needs a factor of at least 1, got {scaling.get('factor')!r}")
    if kind == "linear":
        return w / s, 1.0
    if kind == "ntk":
        if rotary_dim == 2:
            raise ValueError("rotary scaling 'ntk' needs a rotary_dim of at least 4")
        return (float(base) * s ** (rotary_dim / (rotary_dim - 2))) ** -exponent, 1.0
    length, fast, slow = scaling.get("original_length", 0), scaling.get("beta_fast", 32.0), scaling.get("beta_slow", 1.0)
    if length <= 0 or fast <= slow:
        raise ValueError("rotary scaling 'yarn' needs an original_length and beta_fast > beta_slow")
    keep = np.clip((length * w / (2 * math.pi) - slow) / (fast - slow), 0.0, 1.0)
    return w / s * (1 - keep) + w * keep, 0.1 * math.log(s) + 1.0


class RotaryPosEmbed:
    """The frequencies of one model, on one device, for `rotary_pos_embed` and `kv_cache_append`.

    layout "interleaved": pair i is elements (2i, 2i + 1); "half": elements (i, i + rotary_dim / 2).  Elements of a head behind
    rotary_dim are left as they are."""

    def __init__(self, rotary_dim, base=10000.0, layout="interleaved", scaling=None, device="cuda"):
        self._adopt(*rotary_frequencies(rotary_dim, base, scaling), layout, device)

    @classmethod
    def from_frequencies(cls, frequencies, factor=1.0, layout="interleaved", device="cuda"):
        """Frequencies that were made elsewhere (host values): radians a position of every pair [rotary_dim / 2], and the factor of the turned
        values."""
        self = cls.__new__(cls)
        frequencies = np.asarray(frequencies)
        if frequencies.ndim != 1 or len(frequencies) == 0 or frequencies.dtype.kind not in "fiu" or not np.isfinite(frequencies).all():
            raise ValueError("RotaryPosEmbed: frequencies must be one finite number for each pair")
        if not math.isfinite(factor):
            raise ValueError(f"RotaryPosEmbed: factor={factor} must be finite")
        self._adopt(frequencies.astype(np.float64), float(factor), layout, device)
        return self

    def _adopt(self, frequencies, factor, layout, device):
        import torch

        if layout not in _LAYOUTS:
            raise ValueError(f"unknown rotary layout {layout!r}; expected one of {sorted(_LAYOUTS)}")
        self.rotary_dim, self.factor, self.layout = 2 * len(frequencies), factor, layout
        if self.rotary_dim > 256:
            raise ValueError(f"rotary_dim={self.rotary_dim} exceeds 256")
        self.turns = torch.from_numpy(frequencies / (2 * math.pi)).to(device)
        self.index = self.turns.get_device()
        self._c = _gq_hip.Rotary(self.turns.data_ptr(), factor, self.rotary_dim, _LAYOUTS[layout])

    @property
    def argument(self):
        """For the C entry points."""
        return ctypes.byref(self._c)


def rotary_pos_embed(t, positions, rotary, inverse=False, out=None):
    """
    Turn the rows of `t` by their positions.

    Args:
        t (torch.Tensor): float16 [tokens, heads, head_dim] on a HIP device, the last axis contiguous: a slice of a fused
            projection's result is read where it lies.  Queries and keys that lie side by side are one call.
        positions (torch.Tensor): int32 [tokens]
        rotary (RotaryPosEmbed): rotary_dim <= head_dim
        inverse (bool): turn back (the gradient of the forward call with respect to t)
        out (torch.Tensor): where the result goes, e.g. `t` itself; a new contiguous tensor if None

    Returns:
        torch.Tensor: `out`.  One rounding to float16.
    """
    import torch

    if t.dim() != 3:
        raise ValueError(f"t must be [tokens, heads, head_dim], got shape {tuple(t.shape)}")
    if not t.is_cuda:
        raise RuntimeError("rotary_pos_embed runs on the GPU only: move the tensors to a HIP device")
    if t.dtype != torch.float16 or (out is not None and out.dtype != torch.float16):
        raise TypeError("rotary_pos_embed: t and out must be float16")
    if positions.dtype != torch.int32:
        raise TypeError(f"rotary_pos_embed: positions must be int32, got {positions.dtype}")
    index, shape = t.get_device(), t.shape
    tokens, heads, head_dim = shape
    if positions.dim() != 1 or positions.shape[0] != tokens:
        raise ValueError(f"positions must have shape ({tokens},), got {tuple(positions.shape)}")
    if positions.get_device() != index or rotary.index != index or (out is not None and out.get_device() != index):
        raise ValueError("t, positions, rotary and out must be on the same device")
    if rotary.rotary_dim > head_dim:
        raise ValueError(f"rotary_dim={rotary.rotary_dim} exceeds the head dimension {head_dim}")
    if out is not None and (out.shape != shape or out.stride(2) != 1):
        raise ValueError("out must have the shape of t and a contiguous last axis")
    if t.stride(2) != 1:
        t = t.contiguous()
    positions = positions.contiguous()
    if out is None:
        out = t.new_empty(shape)
    token_stride, head_stride, _ = t.stride()
    out_token_stride, out_head_stride, _ = out.stride()
    _gq_hip.launch(index, "gq_rotary_f16", t.data_ptr(), token_stride, head_stride, positions.data_ptr(), rotary.argument, inverse,
                   out.data_ptr(), out_token_stride, out_head_stride, tokens, heads, head_dim)
    return out
