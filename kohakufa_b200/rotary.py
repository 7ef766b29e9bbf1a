"""Rotary positions: queries and keys turned by angles that grow with a token's position.

    rotary = Rotary.of(128, base=500000.0)                       # once, e.g. Rotary.of(128, method="yarn_pairs", factor=16, length=4096)
    q, k = apply_rotary(q, k, rotary)                            # training, prompts: tokens 0 .. S - 1
    out = attention(q, k, v, causal=True)

    q, k = apply_rotary(q, k, rotary, positions=positions)       # packed [T, H, D] for attention_varlen, drafted trees, ...

On the way into a cache: ``cache_append_rotary``. There is no table of cosines: angles come from the position itself in fixed point,
off by no more than the position times 2^-52 of the frequency (its division by 2 pi in 64-bit floats) and 2^-65 turns whatever the position, so that nothing has to be
made for a longest length. The reference has no counterpart.
"""

import math

import torch
from torch import Tensor

from kohakufa_b200 import _lib

__all__ = ["Rotary", "apply_rotary", "rotary_frequencies"]

METHODS = ("none", "linear", "base", "ramp", "yarn", "yarn_pairs")


def rotary_frequencies(
    dim: int, base: float = 10000.0, *, method: str = "none", factor: float = 1.0, length: int | None = None, low: float = 1.0,
    high: float = 32.0,
) -> tuple[Tensor, float]:  # fmt: skip
    """Angles per position in radians, float64 ``[dim / 2]`` on the CPU, and the amplitude of cosine and sine, for a head whose ``dim``
    columns are turned: ``f_i = base ** (-2 i / dim)``, and for contexts ``factor`` times as long as the trained ``length``

      * ``"linear"``: ``f_i / factor``;
      * ``"base"``: the base times ``factor ** (dim / (dim - 2))``, which leaves the fastest pair as it is and slows the last one by
        ``factor``;
      * ``"ramp"``: a pair that turns more than ``high`` times over ``length`` keeps its frequency, one that turns less than ``low`` times
        gets ``f_i / factor``, in between in proportion to the turns;
      * ``"yarn"``: the same with an amplitude of ``0.1 ln(factor) + 1`` (1 for a factor below 1);
      * ``"yarn_pairs"``: ``"yarn"`` with a ramp in proportion to the pair's index: the last pair that turns at least ``high`` times and those before it keep their
        frequency, the first that turns at most ``low`` times and those behind it get ``f_i / factor``. Published models of the name were trained and are run
        with this one. The two ramps meet at their ends only: with 128 columns, ``length`` 4096 and ``factor`` 16 a pair between them differs by up to 3 times."""
    if isinstance(dim, bool) or int(dim) != dim or dim < 2 or dim % 2:
        raise ValueError(f"rotary_frequencies: dim {dim}: an even number of columns")
    if method not in METHODS:
        raise ValueError(f"rotary_frequencies: method {method!r}: one of {METHODS}")
    if not (math.isfinite(base) and base > 0 and math.isfinite(factor) and factor > 0):
        raise ValueError(f"rotary_frequencies: base {base}, factor {factor}: positive numbers")
    if method == "base":
        if dim == 2:
            raise ValueError("rotary_frequencies: method 'base' needs more than one pair")
        base = base * factor ** (dim / (dim - 2))
    f = torch.tensor([base ** (-2.0 * i / dim) for i in range(dim // 2)], dtype=torch.float64)
    if method == "linear":
        f = f / factor
    if method in ("ramp", "yarn", "yarn_pairs"):
        if length is None or length < 1:
            raise ValueError(f"rotary_frequencies: method {method!r} needs the trained length")
        if not 0 <= low < high:
            raise ValueError(f"rotary_frequencies: low {low}, high {high}: 0 <= low < high")
        if method == "yarn_pairs":
            first, last = _turning_pairs(dim, base, length, low, high)
            keep = 1.0 - ((torch.arange(dim // 2, dtype=torch.float64) - first) / (last - first)).clamp(0.0, 1.0)
        else:
            keep = ((length * f / (2 * math.pi) - low) / (high - low)).clamp(0.0, 1.0)
        f = keep * f + (1.0 - keep) * f / factor
    return f, (0.1 * math.log(max(factor, 1.0)) + 1.0 if method.startswith("yarn") else 1.0)


def _turning_pairs(dim: int, base: float, length: float, low: float, high: float) -> tuple[float, float]:
    """The index of the last pair that turns at least ``high`` times over ``length`` positions, and of the first that turns at most ``low`` times, whole
    numbers inside ``0 .. dim - 1`` (the bounds that published models were trained with: of columns, not of pairs); apart by something."""
    if base <= 1:
        raise ValueError(f"rotary_frequencies: base {base}: method 'yarn_pairs' needs one above 1")

    def pair(turns: float) -> float:  # length * base ** (-2 pair / dim) = 2 pi turns
        return math.inf if turns == 0 else dim * math.log(length / (2 * math.pi * turns)) / (2 * math.log(base))

    first = max(math.floor(pair(high)), 0)
    last = min(math.ceil(min(pair(low), dim)), dim - 1)
    return first, last if last > first else first + 0.001


class Rotary:
    """The angles of a model's rotary positions, made once and kept on the device.

    ``frequencies``: the angle in radians by which a position turns each pair, a sequence of numbers or a tensor (taken in 64 bits),
    one per pair of columns; a head's columns behind the pairs are left as they are. ``interleaved``: pairs are columns ``2 i`` and ``2 i + 1``,
    else ``i`` and ``i + pairs``. ``amplitude`` multiplies cosines and sines."""

    __slots__ = ("amplitude", "interleaved", "turns")

    def __init__(self, frequencies, *, interleaved: bool = False, amplitude: float = 1.0, device="cuda") -> None:
        f = torch.as_tensor(frequencies, dtype=torch.float64, device="cpu").detach()
        if f.dim() != 1 or not f.numel() or not bool(torch.isfinite(f).all()):
            raise ValueError("Rotary: frequencies is a vector of finite numbers, one per pair of columns")
        if not math.isfinite(amplitude) or not math.isfinite(float(torch.tensor(float(amplitude), dtype=torch.float32))):
            raise ValueError(f"Rotary: amplitude {amplitude}")
        # turns as 64-bit fractions: position * fraction modulo 2^64 is the angle (2 pi is off by 2^-54.5 of itself and the quotient rounded by 2^-53)
        whole = [round(math.fmod(x / (2 * math.pi), 1.0) * 2**64) % 2**64 for x in f.tolist()]
        self.turns = torch.tensor([w - 2**64 if w >= 2**63 else w for w in whole], dtype=torch.int64, device=device)
        self.interleaved, self.amplitude = bool(interleaved), float(amplitude)

    @classmethod
    def of(
        cls, dim: int, base: float = 10000.0, *, method: str = "none", factor: float = 1.0, length: int | None = None, low: float = 1.0,
        high: float = 32.0, interleaved: bool = False, device="cuda",
    ) -> "Rotary":  # fmt: skip
        """The rotary of ``dim`` turned columns with the frequencies and amplitude of ``rotary_frequencies``."""
        f, amplitude = rotary_frequencies(dim, base, method=method, factor=factor, length=length, low=low, high=high)
        return cls(f, interleaved=interleaved, amplitude=amplitude, device=device)

    @property
    def dim(self) -> int:
        """Columns of a head that are turned."""
        return 2 * self.turns.numel()

    def to(self, device) -> "Rotary":
        """The same on another device."""
        other = Rotary.__new__(Rotary)
        other.turns, other.interleaved, other.amplitude = self.turns.to(device), self.interleaved, self.amplitude
        return other


@torch.library.custom_op("kohakufa_b200::rotary", mutates_args=(), device_types="cuda")
def rotary_op(
    x: Tensor, turns: Tensor, positions: Tensor | None, offset: Tensor | None, amplitude: float, interleaved: bool, inverse: bool
) -> Tensor:
    if x.stride(-1) != 1:  # e.g. an expanded gradient
        x = x.contiguous()
    with torch.no_grad():
        return _lib.host().rotary(x, None, turns, positions, offset, amplitude, interleaved, inverse)


@rotary_op.register_fake
def _(x, turns, positions, offset, amplitude, interleaved, inverse):
    if x.dim() == 3:
        return x.new_empty(x.shape)
    batch, heads, tokens, dim = x.shape
    return x.new_empty(batch, tokens, heads, dim).transpose(1, 2)


def _rotary_setup(ctx, inputs, output):
    _, turns, positions, offset, amplitude, interleaved, inverse = inputs
    ctx.save_for_backward(turns, positions, offset)
    ctx.how = (amplitude, interleaved, inverse)


def _rotary_backward(ctx, g):
    turns, positions, offset = ctx.saved_tensors
    amplitude, interleaved, inverse = ctx.how
    return rotary_op(g, turns, positions, offset, amplitude, interleaved, not inverse), None, None, None, None, None, None


rotary_op.register_autograd(_rotary_backward, setup_context=_rotary_setup)


def apply_rotary(
    q: Tensor, k: Tensor | None, rotary: Rotary, *, positions: Tensor | None = None, offset: Tensor | None = None
):
    """``q`` ``[B, H, S, D]`` and ``k`` ``[B, Hkv, S, D]`` (fp16, bf16 or fp32; views of ``[B, S, H, D]`` are usual, any strides with a contiguous last dim; ``D`` up
    to 1024) with their pairs turned by their positions' angles; the columns behind ``rotary.dim`` are copied. With gradients, which
    are the gradients of the outputs turned back.

    Token ``t`` of sequence ``b`` stands at ``positions[b, t]`` (int32 or int64, ``[B, S]``, ``[1, S]`` or ``[S]``; without it at ``t``), and ``offset``
    (int32 ``[B]``, e.g. a cache's lengths) is added to the positions of a sequence. Positions may be negative. Packed sequences ``[T, H, D]`` need
    their positions, ``[T]``.

    Returns new tensors, ``[B, H, S, D]`` laid out as ``[B, S, H, D]`` (packed ones contiguous): ``q, k``, or where ``k`` is None ``q`` alone.
    Sines, cosines and products are fp32, rounded once."""
    if q.dim() == 3 and positions is None:
        raise ValueError("apply_rotary: packed sequences [T, H, D] need positions")
    args = (rotary.turns, positions, offset, rotary.amplitude, rotary.interleaved, False)
    if _lib.plain_eager(q, k, *args[:3]):
        return _lib.host().rotary(q, k, *args)
    if any(t is not None and t.shape[-1] > 1 and t.stride(-1) != 1 for t in (q, k)):  # (the op itself takes any gradient)
        raise ValueError("apply_rotary: q and k need a contiguous last dim")
    if k is None:
        return rotary_op(q, *args)
    if q.dtype != k.dtype:
        raise TypeError("apply_rotary: q and k must be fp16, bf16 or fp32 (both the same)")
    if q.dim() != k.dim() or q.shape[0] != k.shape[0] or q.shape[-1] != k.shape[-1] or (q.dim() == 4 and q.shape[2] != k.shape[2]):
        raise ValueError("apply_rotary: k must have the batch, tokens and head dim of q")
    return rotary_op(q, *args), rotary_op(k, *args)
