"""Rotary positions: half and interleaved pairs, part of each head, frequencies scaled for long contexts.

With angle = position * frequency_i for pair i of the first `2 * len(freqs)` values of a head (pairs (i, i + n/2) for
"half", (2i, 2i + 1) for "interleaved"):

    a' = scale * (a cos - b sin)        b' = scale * (b cos + a sin)

The other values of the head pass through. The gradient turns back by the same angles. Angles are formed in 64 bits
(32 bits lose those of far positions), the rotation is 32-bit arithmetic, the result is rounded once.

`qk_norm_rope` (`ops/rope.py`) fuses the q/k norm with half pairs at unscaled frequencies on a packed projection; this
operator is the rotation alone, for everything that one does not cover. CUDA tensors of bf16, fp16 and fp32 run
`csrc/rotary.cu`; others take `rotary_reference`.
"""
from __future__ import annotations

import math
from dataclasses import dataclass

import torch

from ..kernels import native
from ._util import MAX_ROWS, dtype_code, on_device, refuse_tangents, refuse_twice, stream_of

native.register_signatures({
    "tdllm_rotary": (native.c_int, [native.c_void_p] * 4 + [native.c_int] * 4 + [native.c_ll] * 2 + [native.c_int] * 2
                     + [native.c_float] * 2 + [native.c_void_p]),
})

PAIRS = ("half", "interleaved")


@dataclass(frozen=True)
class RotaryScaling:
    """How the frequencies of a model trained at `original_length` positions are stretched by `factor`.

    kind "linear": every frequency divided by the factor. "ntk": the base theta raised so that the slowest pair is
    stretched by the factor and the fastest not at all. "llama3": pairs that turn at least `high_freq_factor` times over
    the original length keep their frequency, pairs that turn at most `low_freq_factor` times are divided, linear in
    between. "yarn": a linear ramp over the pair index between the pairs that turn `beta_fast` and `beta_slow` times;
    cosine and sine get `attention_factor` (default 0.1 ln(factor) + 1)."""

    kind: str
    factor: float
    original_length: int = 8192
    low_freq_factor: float = 1.0
    high_freq_factor: float = 4.0
    beta_fast: float = 32.0
    beta_slow: float = 1.0
    attention_factor: float | None = None

    def __post_init__(self):
        if self.kind not in ("linear", "ntk", "llama3", "yarn"):
            raise ValueError(f"rotary scaling must be linear, ntk, llama3 or yarn, got {self.kind!r}")
        if not (math.isfinite(self.factor) and self.factor >= 1.0):
            raise ValueError(f"the scaling factor must be >= 1, got {self.factor}")
        if self.original_length < 1:
            raise ValueError("original_length must be positive")
        if self.kind == "llama3" and not 0 < self.low_freq_factor < self.high_freq_factor:
            raise ValueError("llama3 scaling needs 0 < low_freq_factor < high_freq_factor")
        if self.kind == "yarn" and not 0 < self.beta_slow < self.beta_fast:
            raise ValueError("yarn scaling needs 0 < beta_slow < beta_fast")


def rotary_frequencies(part: int, theta: float, scaling: RotaryScaling | None = None,
                       device=None) -> tuple[torch.Tensor, float]:
    """(freqs [part / 2] float32, scale): what `rotary` takes for heads whose first `part` values turn."""
    if part < 2 or part % 2:
        raise ValueError(f"the rotated part must be an even number of values, got {part}")
    i = torch.arange(0, part, 2, dtype=torch.float64)
    base = theta ** (-i / part)
    scale = 1.0
    if scaling is None:
        f = base
    elif scaling.kind == "linear":
        f = base / scaling.factor
    elif scaling.kind == "ntk":
        f = base if part == 2 else (theta * scaling.factor ** (part / (part - 2))) ** (-i / part)
    elif scaling.kind == "llama3":
        turns = scaling.original_length * base / (2 * math.pi)
        keep = ((turns - scaling.low_freq_factor) / (scaling.high_freq_factor - scaling.low_freq_factor)).clamp(0, 1)
        f = base * (keep + (1 - keep) / scaling.factor)
    else:
        at = lambda turns: part * math.log(scaling.original_length / (turns * 2 * math.pi)) / (2 * math.log(theta))  # noqa: E731
        lo, hi = max(math.floor(at(scaling.beta_fast)), 0), min(math.ceil(at(scaling.beta_slow)), part - 1)
        ramp = ((i / 2 - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
        f = base * ((1 - ramp) + ramp / scaling.factor)
        scale = scaling.attention_factor if scaling.attention_factor is not None else 0.1 * math.log(scaling.factor) + 1.0
    return f.to(torch.float32).to(device), float(scale)


def rotary_reference(x, positions, freqs, pairs: str = "half", scale: float = 1.0):
    """The rotation in plain operations: angles in 64 bits, values in 32 (64 for double inputs). Differentiable."""
    n = 2 * freqs.shape[0]
    wide = torch.float64 if x.dtype == torch.float64 else torch.float32
    ang = (positions.double()[:, None] * freqs.double()[None])[:, None]
    cos, sin = (torch.cos(ang) * scale).to(wide), (torch.sin(ang) * scale).to(wide)
    r = x[..., :n].to(wide)
    if pairs == "half":
        a, b = r[..., : n // 2], r[..., n // 2:]
        r = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
    else:
        a, b = r[..., 0::2], r[..., 1::2]
        r = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
    return torch.cat([r.to(x.dtype), x[..., n:]], dim=-1)


def _turn(x, positions, freqs, half: int, scale: float, back: bool):
    rows, H, D = x.shape
    ld_row, ld_head, inner = x.stride()
    if inner != 1:
        x = x.contiguous()
        ld_row, ld_head = H * D, D
    out = torch.empty((rows, H, D), dtype=x.dtype, device=x.device)
    if rows and H:
        with on_device(x):
            native.check(native.lib().tdllm_rotary(
                x.data_ptr(), out.data_ptr(), positions.data_ptr(), freqs.data_ptr(), rows, H, D, 2 * freqs.shape[0], ld_row,
                ld_head, half, dtype_code(x), scale, -1.0 if back else 1.0, stream_of(x)), "rotary")
    return out


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, positions, freqs, half, scale):
        ctx.save_for_backward(positions, freqs)
        ctx.meta = (half, scale)
        return _turn(x, positions, freqs, half, scale, False)

    @staticmethod
    def backward(ctx, dout):
        refuse_twice("rotary")
        positions, freqs = ctx.saved_tensors
        return _turn(dout, positions, freqs, *ctx.meta, True), None, None, None, None


def rotary(x: torch.Tensor, positions: torch.Tensor, freqs: torch.Tensor, *, pairs: str = "half",
           scale: float = 1.0) -> torch.Tensor:
    """x [rows, H, D] (any row and head stride, e.g. the query and key heads of a packed projection) -> [rows, H, D].
    positions [rows] int32 or int64 (within int32), freqs [n / 2] float32 with n <= D (2048 at most in
    the kernel), from `rotary_frequencies` (constants: they get no gradient)."""
    if x.dim() != 3 or positions.shape != x.shape[:1]:
        raise ValueError(f"need x [rows, H, D] and one position per row, got {tuple(x.shape)} and {tuple(positions.shape)}")
    if positions.dtype not in (torch.int32, torch.int64):
        raise ValueError("positions must be int32 or int64")
    if freqs.dim() != 1 or freqs.dtype != torch.float32 or not 1 <= freqs.shape[0] <= x.shape[2] // 2:
        raise ValueError(f"freqs must be a float32 vector of 1 to {x.shape[2] // 2} values")
    if freqs.requires_grad and torch.is_grad_enabled():
        raise ValueError("freqs are constants of the rotation and get no gradient; detach them")
    if pairs not in PAIRS:
        raise ValueError(f"pairs must be one of {PAIRS}, got {pairs!r}")
    if positions.device != x.device or freqs.device != x.device:
        raise ValueError(f"positions and freqs must lie on {x.device}")
    if x.shape[0] > MAX_ROWS:
        raise ValueError(f"rotary takes up to {MAX_ROWS} rows, got {x.shape[0]}")
    if dtype_code(x) is None:
        return rotary_reference(x, positions, freqs, pairs, scale)
    refuse_tangents("rotary", x, freqs)
    if positions.dtype != torch.int32:
        positions = positions.to(torch.int32)
    positions, freqs = positions.contiguous(), freqs.contiguous()
    half = int(pairs == "half")
    if torch.is_grad_enabled() and x.requires_grad:
        return _Rotary.apply(x, positions, freqs, half, float(scale))
    return _turn(x, positions, freqs, half, scale, False)
