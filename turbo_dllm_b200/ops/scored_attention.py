"""Attention with transformed scores: a tanh cap, a bias by distance, document and prefix masks.

Per query row i, key j and head h, with the visibility of a `MaskLayout` (`ops/attention.py`):

    z_ij = scale * q_i . k_j
    z_ij = cap * tanh(z_ij / cap)                          softcap > 0
    z_ij = z_ij - slope_h * |q_pos_i - k_pos_j|            slopes given
    out_i = sum_j softmax_j(z_ij) v_j,   lse_i = log sum_j exp(z_ij)       over the visible j

and backward, with P_ij = exp(z_ij - lse_i) and t_ij = tanh(scale * q_i . k_j / cap):

    dZ_ij = P_ij (dO_i . v_j - dO_i . out_i)               dS_ij = dZ_ij (1 - t_ij^2)
    dq_i = scale * sum_j dS_ij k_j     dk_j = scale * sum_i dS_ij q_i     dv_j = sum_i P_ij dO_i

summed over the query heads that share a KV head. Rows that see no key give out = 0, lse = -inf and no gradient. Query
rows without a visible key and keys that no row sees may hold anything, infinities and NaN included; a value that is not
finite and that some row does see may reach the other rows of its 128-row tile.

A layout's values are those of int32 tensors, noisy groups up to 2^31 - 3 (the codes behind that mark dead keys and padding).

The block-diffusion masks come from `block_diffusion_layout`; `document_layout` gives packed documents (causal, or with
a prefix that is read in both directions). On CUDA bf16 tensors with head width 128 the tcgen05 kernels run
(`csrc/attention_fwd_sm100.cu`, `csrc/attention_bwd_fused_sm100.cu` with the transforms of `csrc/score_mod.cuh`);
everything else takes `scored_attention_reference`. A layout's tile lists and a transform's padded positions are built on
first use and again when one of their tensors has been written to (in every call where the tensors were made in inference
mode, which does not count writes). Writes that torch does not count, those of a replayed graph or of a kernel that was given a
pointer, are told by `layout.changed()` and `transform.changed()`. A captured graph uses the lists that its layout and
transform had then (or builds its own at every replay, if they had none): keep both objects as long as the graph. The form
for few query rows has no lists and follows its tensors. Before a training step is captured, let go of eager autograd graphs
over the same leaves: torch adds into a leaf on the stream of the oldest graph that is alive, which a capture may not use.
"""
from __future__ import annotations

import math
import os
from dataclasses import dataclass, field

import torch

from ..kernels import native
from ._util import on_device, ptr, refuse_tangents, refuse_twice, stream_of
from .attention import TILE, MaskLayout, backward_chunk_tiles, backward_mode

native.register_signatures({
    "tdllm_attn_fwd_scored": (native.c_int, [native.c_void_p] * 6 + [native.c_int] * 4 + [native.c_ll] * 4
                              + [native.c_void_p] * 7 + [native.c_int, native.c_float, native.c_float]
                              + [native.c_void_p] * 4),
    "tdllm_attn_plan_size": (native.c_ll, [native.c_int] * 3 + [native.c_void_p]),
    "tdllm_attn_plan": (native.c_int, [native.c_void_p] * 4 + [native.c_int] * 3 + [native.c_void_p] * 2),
    "tdllm_attn_few_rows_scratch": (native.c_ll, [native.c_int] * 4),
    "tdllm_attn_few_rows": (native.c_int, [native.c_void_p] * 6 + [native.c_int] * 4 + [native.c_ll] * 5
                            + [native.c_void_p] * 4 + [native.c_float] * 2 + [native.c_void_p] * 4),
    "tdllm_attn_bwd_scored": (native.c_int, [native.c_void_p] * 12 + [native.c_int] * 4 + [native.c_ll] * 8
                              + [native.c_void_p] * 7 + [native.c_int, native.c_int, native.c_int, native.c_float,
                                                         native.c_float] + [native.c_void_p] * 4),
})

DEAD_KEY = -(2 ** 31)      # key code that no query row matches
MAX_POSITION = 1 << 24     # distances are taken between positions held as floats
LOG2E = 1.4426950408889634
# caps and scales that 32 bits hold, with their ratio times 2 log2 e and its inverse (a smaller cap would become none there)
CAPS, SCALES = (1e-18, 1e30), (1e-20, 1e18)
# A forward without gradients packs the query heads of a KV head into rows and splits the keys over the GPU (`_few`), instead
# of giving a CTA the whole list of a 128-row query tile, for up to FEW_ROWS query rows, and for as many as one 128-row tile
# of packed rows per SM holds. B200, scores capped, all keys seen, device time in us (split / listed): 32 / 8 heads: 1 row x 20000
# keys 18 / 408, 32 x 32768 38 / 654, 128 x 1024 15 / 27, 512 x 512 15 / 17, 512 x 8192 98 / 170, 1024 x 8192 (two packed tiles
# per SM) 195 / 171; 16 / 8 heads: 1024 x 1024 20 / 28, 1024 x 32768 369 / 659; two key tiles: 200 x 200 17 / 14
FEW_ROWS = 128
SMS = 148
# The backward pass has an item of work per (key tile, chunk of query tiles, KV head). Where the key tiles and heads alone are
# few, shorter chunks make about this many items, 2.5 to each SM. B200, forward and backward in us, one chunk against the
# chunks of this rule: 500 rows, 16 / 8 heads 68 / 50, 2000 rows, 4 / 1 heads 273 / 98, 2000 rows, 16 / 8 heads 191 / 155, 3000
# rows, 16 / 8 heads 276 / 255; from 300 items on one chunk is as good (5000 rows, 16 / 8 heads 533, two chunks 545).
BACKWARD_ITEMS = 370


def _version(t: torch.Tensor) -> int | None:
    """None: a tensor of inference mode, which does not say when it has been written to."""
    return None if t.is_inference() else t._version


def _kept(cache: dict, name: str, sources: tuple, sizes: tuple, build):
    """cache[name] if it was made from these very tensors as they are now and for these sizes, else what `build` makes on their
    device: (tensors, what goes with them). An entry holds its tensors, so that another tensor cannot pass for one of them. What
    is made eagerly is complete on return, so that any stream may use it, and its memory is not given away before those
    streams are done; what is made while a graph is captured belongs to that graph and is not kept, nor is what is made from
    tensors of inference mode. What a capture uses stays with its owner as long as that lives, also when a newer one takes its
    place."""
    like, key = sources[0], (*(_version(t) for t in sources), *sizes, cache.get("changes", 0))
    if None in key:
        return build()
    hit = cache.get(name)
    if hit is not None and (hit[0] != key or any(a is not b for a, b in zip(hit[3], sources))):
        hit = None
    if not like.is_cuda:
        if hit is None:
            cache[name] = hit = (key, build(), None, sources)
        return hit[1]
    capturing = torch.cuda.is_current_stream_capturing()
    if hit is not None:
        if capturing:
            cache.setdefault(name + "_captured", []).append(hit[1])
        elif hit[2] != stream_of(like):
            for t in hit[1][0]:
                t.record_stream(torch.cuda.current_stream(like.device))
        return hit[1]
    made = build()
    if not capturing:
        torch.cuda.current_stream(like.device).synchronize()
        cache[name] = (key, made, stream_of(like), sources)
    return made


@dataclass(frozen=True, eq=False)
class ScoreTransform:
    """What happens to the scores before the softmax.

    softcap: cap of the tanh (1e-18 to 1e30), 0 for none. slopes: [Hq] float32, one slope per query head, with q_pos [nq] and
    k_pos [nk] (int32 or int64, absolute value below 2^24): the distance bias. Slopes are constants: they get no gradient. A
    position beyond the limit is refused; where the host does not see positions, as in calls of few rows, which read them on
    the device, and in captured graphs, rows that meet one get NaN. Scores are 32-bit numbers: a row all of whose keys are far
    away knows them to 2^-24 of slope * distance."""

    softcap: float = 0.0
    slopes: torch.Tensor | None = None
    q_pos: torch.Tensor | None = None
    k_pos: torch.Tensor | None = None
    _cache: dict = field(default_factory=dict, init=False, repr=False)      # (a replaced copy begins with its own)

    def __post_init__(self):
        if not (self.softcap == 0.0 or CAPS[0] <= self.softcap <= CAPS[1]):
            raise ValueError(f"softcap must be 0 or a number from {CAPS[0]} to {CAPS[1]}, got {self.softcap}")
        given = [t is not None for t in (self.slopes, self.q_pos, self.k_pos)]
        if any(given) and not all(given):
            raise ValueError("a distance bias needs slopes, q_pos and k_pos together")
        if self.slopes is None:
            return
        if self.slopes.dim() != 1 or self.slopes.dtype != torch.float32:
            raise ValueError("slopes must be a float32 vector, one value per query head")
        if self.slopes.requires_grad:
            raise ValueError("slopes are constants of the bias and get no gradient; detach them")
        for name, t in (("q_pos", self.q_pos), ("k_pos", self.k_pos)):
            if t.dim() != 1 or t.dtype not in (torch.int32, torch.int64):
                raise ValueError(f"{name} must be a vector of int32 or int64")

    def __getstate__(self):
        """Copies and pickles without what was built."""
        return {**self.__dict__, "_cache": {}}

    def changed(self) -> None:
        """Says that the tensors hold something else now, as `MaskLayout.changed` does."""
        self._cache["changes"] = self._cache.get("changes", 0) + 1

    @property
    def biased(self) -> bool:
        return self.slopes is not None

    def _padded(self, nq_pad: int, nk_pad: int):
        """(slopes * log2 e, q_pos, k_pos) as the kernels read them: floats, positions padded with zeros. Rebuilt when
        one of the tensors has been written to since."""
        return _kept(self._cache, "padded", (self.slopes, self.q_pos, self.k_pos), (nq_pad, nk_pad),
                     lambda: (self._pad(nq_pad, nk_pad),))[0]

    def _pad(self, nq_pad: int, nk_pad: int):
        out = [(self.slopes * LOG2E).contiguous()]
        for t, n in ((self.q_pos, nq_pad), (self.k_pos, nk_pad)):
            f = torch.zeros(n, dtype=torch.float32, device=t.device)
            f[: t.shape[0]] = t
            if t.is_cuda and torch.cuda.is_current_stream_capturing():      # (which may not wait for the device)
                f.masked_fill_(f.abs() >= MAX_POSITION, math.nan)
            elif t.numel() and float(f.abs().max()) >= MAX_POSITION:
                raise ValueError(f"positions of the distance bias must lie between +-{MAX_POSITION}")
            out.append(f)
        return tuple(out)


def document_layout(lengths, *, prefix=None, rows: int | None = None, causal: bool = True, device="cpu") -> MaskLayout:
    """Packed documents: row i of a document sees that document's rows up to itself (all of them when not `causal`), and
    at least the document's first `prefix[d]` rows, so that a prefix is read in both directions. `lengths` are the
    documents' row counts in packing order (zero is allowed); rows behind the last document, up to `rows`, see nothing and
    are seen by nothing."""
    lens = torch.as_tensor(lengths, dtype=torch.int64, device="cpu").reshape(-1)      # (the layout is built there)
    if lens.numel() and int(lens.min()) < 0:
        raise ValueError("document lengths must not be negative")
    pre = torch.zeros_like(lens) if prefix is None else torch.as_tensor(prefix, dtype=torch.int64, device="cpu").reshape(-1)
    if pre.shape != lens.shape or bool((pre < 0).any()) or bool((pre > lens).any()):
        raise ValueError("prefix needs one value per document, between 0 and its length")
    total = int(lens.sum())
    rows = total if rows is None else int(rows)
    if rows < total:
        raise ValueError(f"the documents have {total} rows, more than rows={rows}")
    start = torch.repeat_interleave(lens.cumsum(0) - lens, lens)
    stop = torch.repeat_interleave(lens.cumsum(0), lens)
    first = torch.repeat_interleave(pre, lens)
    at = torch.arange(total, device="cpu")
    hi = torch.maximum(at + 1, start + first) if causal else stop
    pad = rows - total
    z = torch.zeros(pad, dtype=torch.int64, device="cpu")
    grp = torch.zeros(rows, dtype=torch.int64, device="cpu")
    out = [torch.cat([start, z]), torch.cat([hi, z]), grp, torch.cat([at, z + DEAD_KEY])]
    return MaskLayout(*(t.to(torch.int32).to(device) for t in out))


def document_positions(lengths, *, rows: int | None = None, device="cpu") -> torch.Tensor:
    """[rows] int32 positions inside the documents of `document_layout` (0 behind the last one)."""
    lens = torch.as_tensor(lengths, dtype=torch.int64, device="cpu").reshape(-1)
    total = int(lens.sum())
    pos = torch.zeros(total if rows is None else int(rows), dtype=torch.int32, device="cpu")
    pos[:total] = (torch.arange(total, device="cpu") - torch.repeat_interleave(lens.cumsum(0) - lens, lens)).to(torch.int32)
    return pos.to(device)


_PLAN_PARTS = ("q_lo", "q_hi", "q_grp", "k_code", "f_ptr", "f_idx", "f_order", "w_ptr", "w_idx", "w_order")


def _chunk_tiles(nqt: int, nkt: int, Hkv: int) -> int:
    chunk = backward_chunk_tiles()
    chunk = min(chunk, nqt) if chunk > 0 else nqt
    if "TDLLM_ATTN_BWD_CHUNK" not in os.environ:
        pieces = max(1, round(BACKWARD_ITEMS / (nkt * Hkv)))
        chunk = min(chunk, (nqt + pieces - 1) // pieces)
    return chunk


def _plan(layout: MaskLayout, Hkv: int) -> dict:
    """Device pointers of the layout's tile lists (`csrc/attention_plan.cu`) with the buffer they lie in. Kept with the
    layout, and built anew when one of its tensors has been written to or another one assigned."""
    parts = (layout.q_lo, layout.q_hi, layout.q_grp, layout.k_code)
    nqt, nkt = (layout.nq + TILE - 1) // TILE, (layout.nk + TILE - 1) // TILE
    chunk = _chunk_tiles(nqt, nkt, Hkv)
    return _kept(layout._cache, f"scored_{chunk}", parts, (), lambda: _build_plan(layout, chunk, nqt, nkt))[1]


def _build_plan(layout: MaskLayout, chunk: int, nqt: int, nkt: int):
    lib = native.lib()
    nq, nk = layout.nq, layout.nk
    offsets = (native.c_ll * 11)()
    size = lib.tdllm_attn_plan_size(nq, nk, chunk, offsets)
    if size < 0:
        raise native.NativeKernelError(f"{nq} rows x {nk} keys have too many tiles for a plan")
    lo, hi, grp, code = (_int32(t) for t in (layout.q_lo, layout.q_hi, layout.q_grp, layout.k_code))
    buf = torch.empty(size, dtype=torch.int32, device=lo.device)
    native.check(lib.tdllm_attn_plan(ptr(lo), ptr(hi), ptr(grp), ptr(code), nq, nk, chunk, ptr(buf), stream_of(buf)), "attn_plan")
    base = buf.data_ptr()
    plan = {n: base + 4 * offsets[i] for i, n in enumerate(_PLAN_PARTS)}
    plan.update(chunk=chunk, buf=buf, nqt=nqt, nkt=nkt, nq_pad=nqt * TILE, nk_pad=nkt * TILE,
                n_work=(nqt + chunk - 1) // chunk * nkt)
    return (buf,), plan


def scored_attention_reference(q, k, v, layout: MaskLayout, transform: ScoreTransform | None = None,
                               scale: float | None = None):
    """Dense-mask form in fp32 (in 64 bits for double inputs), differentiable. q [nq, Hq, D], k / v [nk, Hkv, D] ->
    (out [nq, Hq, D] in q's dtype, lse [Hq, nq])."""
    nq, Hq, D = q.shape
    G = Hq // k.shape[1]
    scale = scale if scale is not None else 1.0 / math.sqrt(D)
    wide = torch.float64 if q.dtype == torch.float64 else torch.float32
    seen = layout.dense_mask().to(q.device)
    row_live, key_live = seen.any(1), seen.any(0)
    keep = lambda t, live: torch.where(live[:, None, None], t.to(wide), torch.zeros((), dtype=wide, device=t.device))  # noqa: E731
    qf = keep(q, row_live).permute(1, 0, 2)
    kf = keep(k, key_live).permute(1, 0, 2).repeat_interleave(G, dim=0)
    vf = keep(v, key_live).permute(1, 0, 2).repeat_interleave(G, dim=0)
    z = torch.matmul(qf, kf.transpose(1, 2)) * scale
    if transform is not None and transform.softcap:
        z = transform.softcap * torch.tanh(z / transform.softcap)
    if transform is not None and transform.biased:
        far = (transform.q_pos.long()[:, None] - transform.k_pos.long()[None, :]).abs().to(wide)
        z = z - transform.slopes.to(wide)[:, None, None] * far
    z = z.masked_fill(~(seen | ~row_live[:, None]), float("-inf"))      # (rows without a key are taken out below)
    if layout.nk == 0:      # (zeros that hang on the operands, whose gradients are zeros)
        zeros = q.masked_fill(torch.ones((), dtype=torch.bool, device=q.device), 0) + (k.sum() + v.sum())
        return zeros, torch.full((Hq, nq), float("-inf"), dtype=wide, device=q.device)
    lse = torch.logsumexp(z, dim=-1)
    p = torch.where(row_live[None, :, None], torch.exp(z - lse[..., None]), torch.zeros((), dtype=wide, device=q.device))
    out = torch.matmul(p, vf).permute(1, 0, 2)
    return out.to(q.dtype), lse.masked_fill(~row_live[None], float("-inf"))


def _check(q, k, v, layout: MaskLayout, transform: ScoreTransform | None) -> None:
    if q.dim() != 3 or k.dim() != 3 or v.shape != k.shape or k.shape[2] != q.shape[2]:
        raise ValueError(f"need q [nq, Hq, D] and k, v [nk, Hkv, D], got {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    if k.shape[1] == 0 or q.shape[1] == 0 or q.shape[1] % k.shape[1]:
        raise ValueError(f"{q.shape[1]} query heads do not divide over {k.shape[1]} KV heads")
    if not (q.dtype == k.dtype == v.dtype) or not (q.device == k.device == v.device):
        raise ValueError("q, k and v must share dtype and device")
    lo, hi, grp, code = layout.q_lo, layout.q_hi, layout.q_grp, layout.k_code
    rows, dev = lo.shape, q.device
    if rows[0] != q.shape[0] or code.shape[0] != k.shape[0] or hi.shape != rows or grp.shape != rows:
        raise ValueError(f"the layout describes {layout.nq} query rows and {layout.nk} keys, got {q.shape[0]} and {k.shape[0]}")
    if lo.device != dev or hi.device != dev or grp.device != dev or code.device != dev:
        raise ValueError(f"the layout must lie on {q.device}")
    if transform is not None and transform.biased:
        if transform.slopes.shape[0] != q.shape[1]:
            raise ValueError(f"{transform.slopes.shape[0]} slopes for {q.shape[1]} query heads")
        if transform.q_pos.shape[0] != q.shape[0] or transform.k_pos.shape[0] != k.shape[0]:
            raise ValueError("q_pos and k_pos need one position per query row and per key")
        if any(t.device != q.device for t in (transform.slopes, transform.q_pos, transform.k_pos)):
            raise ValueError(f"slopes and positions must lie on {q.device}")


def _operand(t: torch.Tensor) -> torch.Tensor:
    """[n, H, 128] rows the tensor maps can address: packed heads, 16-byte aligned base and row stride."""
    if t.is_contiguous():
        return t if t.data_ptr() % 16 == 0 else t.clone()
    (n, H, D), (row, head, inner) = t.shape, t.stride()
    if inner == 1 and (H == 1 or head == D) and t.data_ptr() % 16 == 0 and (n == 1 or (row % 8 == 0 and row >= H * D)):
        return t
    return t.contiguous()


def _row_stride(t: torch.Tensor) -> int:
    n, H, D = t.shape
    return t.stride(0) if n > 1 else H * D     # (a single row's stride may be anything)


def _mod_args(transform: ScoreTransform | None, L: dict):
    """(softcap, slope2, q_pos, k_pos) of a launch and the tensors behind the pointers."""
    if transform is None:
        return (0.0, None, None, None), ()
    if not transform.biased:
        return (float(transform.softcap), None, None, None), ()
    kept = transform._padded(L["nq_pad"], L["nk_pad"])
    return (float(transform.softcap), *(ptr(t) for t in kept)), kept


def _few(nq: int, nk: int, Hq: int, Hkv: int) -> bool:
    if nq <= FEW_ROWS:
        return True
    G = Hq // Hkv      # (group sizes that do not divide a tile have the form for up to 128 packed rows only)
    return TILE % G == 0 and nk > 2 * TILE and (nq * G + TILE - 1) // TILE * Hkv <= SMS


def _int32_positions(t: torch.Tensor) -> torch.Tensor:
    """(int64 positions that int32 does not hold stay beyond the limit)"""
    return _int32(t.clamp(-MAX_POSITION, MAX_POSITION) if t.dtype == torch.int64 else t)


def _int32(t: torch.Tensor) -> torch.Tensor:
    return t if t.dtype == torch.int32 and t.is_contiguous() else t.to(torch.int32).contiguous()


def _forward_few_rows(q, k, v, layout, transform, scale):
    """(out, lse [Hq, nq]) with the keys split over CTAs. Reads the layout's and the transform's own
    tensors at run time: nothing is built or cached, so a captured graph follows what is written to them."""
    nq, Hq, D = q.shape
    nk, Hkv, _ = k.shape
    lib = native.lib()
    dev = q.device
    out = torch.empty((nq, Hq, D), dtype=q.dtype, device=dev)
    lse = torch.empty((Hq, nq), dtype=torch.float32, device=dev)
    n = lib.tdllm_attn_few_rows_scratch(nq, nk, Hq, Hkv)
    part = torch.empty((n,), dtype=torch.float32, device=dev) if n else None
    meta = [_int32(t) for t in (layout.q_lo, layout.q_hi, layout.q_grp, layout.k_code)]
    bias = (None, None, None)
    if transform is not None and transform.biased:
        bias = [transform.slopes.contiguous(), _int32_positions(transform.q_pos), _int32_positions(transform.k_pos)]
    rc = lib.tdllm_attn_few_rows(
        ptr(q), ptr(k), ptr(v), ptr(out), ptr(lse), ptr(part), nq, nk, Hq, Hkv, _row_stride(q), _row_stride(k),
        _row_stride(v), Hq * D, nq, *[t.data_ptr() for t in meta], float(scale),
        0.0 if transform is None else float(transform.softcap), *[ptr(t) for t in bias], stream_of(q))
    native.check(rc, "attn_few_rows" if part is None else "attn_few_rows_split")
    return out, lse


def _forward(q, k, v, L, mod, scale, for_backward=False):
    """(out, lse [Hq, nq padded to 128], what rounding took from out where a backward pass will want it) by the tile lists
    of `_plan` and the arguments of `_mod_args`."""
    nq, Hq, D = q.shape
    nk, Hkv, _ = k.shape
    out = torch.empty(nq, Hq, D, dtype=q.dtype, device=q.device)
    rest = torch.empty_like(out) if for_backward else None
    lse = torch.empty(Hq, L["nq_pad"], dtype=torch.float32, device=q.device)
    rc = native.lib().tdllm_attn_fwd_scored(
        ptr(q), ptr(k), ptr(v), ptr(out), ptr(rest), ptr(lse), nq, nk, Hq, Hkv, _row_stride(q), _row_stride(k), _row_stride(v),
        out.stride(0), L["q_lo"], L["q_hi"], L["q_grp"], L["k_code"], L["f_ptr"], L["f_idx"], L["f_order"], L["nqt"],
        float(scale), *mod, stream_of(q))
    native.check(rc, "attn_fwd_scored")
    return out, lse, rest


def _backward(q, k, v, out, rest, dout, lse, L, mod, scale):
    nq, Hq, D = q.shape
    nk, Hkv, _ = k.shape
    dev = q.device
    dq, dk, dv = torch.empty(nq, Hq, D, dtype=q.dtype, device=dev), torch.empty_like(k, memory_format=torch.contiguous_format), \
        torch.empty_like(v, memory_format=torch.contiguous_format)
    # row statistics [2, Hq, nq_pad], then the accumulators (allocated per call: two streams, or two captured graphs, must
    # not add into one accumulator)
    stats = 2 * Hq * L["nq_pad"]
    work = torch.empty((stats + L["nq_pad"] * Hq * D + 2 * L["nk_pad"] * Hkv * D,), dtype=torch.float32, device=dev)
    rc = native.lib().tdllm_attn_bwd_scored(
        ptr(q), ptr(k), ptr(v), ptr(out), ptr(rest), ptr(dout), ptr(dq), ptr(dk), ptr(dv), ptr(lse), ptr(work),
        ptr(work) + 4 * stats,
        nq, nk, Hq, Hkv, _row_stride(q), _row_stride(k), _row_stride(v), _row_stride(out), _row_stride(dout),
        dq.stride(0), dk.stride(0), dv.stride(0), L["q_lo"], L["q_hi"], L["q_grp"], L["k_code"], L["w_ptr"], L["w_idx"],
        L["w_order"], L["n_work"], L["nqt"], L["nkt"], float(scale), *mod, stream_of(q))
    native.check(rc, "attn_bwd_scored")
    return dq, dk, dv


class _ScoredAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, layout, transform, scale, want_lse):
        with on_device(q):
            q, k, v = _operand(q), _operand(k), _operand(v)
            # (the backward pass goes by the lists and positions of the forward pass, whatever is written to them since)
            ctx.L = _plan(layout, k.shape[1])
            ctx.mod, ctx.behind_mod = _mod_args(transform, ctx.L)
            out, lse, rest = _forward(q, k, v, ctx.L, ctx.mod, scale, for_backward=True)
        ctx.save_for_backward(q, k, v, out, rest, lse)
        ctx.scale = scale
        ctx.set_materialize_grads(False)
        if not want_lse:
            return out, None
        if lse.shape[1] != q.shape[0]:
            lse = lse[:, : q.shape[0]]
        ctx.mark_non_differentiable(lse)
        return out, lse

    @staticmethod
    def backward(ctx, dout, _dlse):
        refuse_twice("scored attention")
        if dout is None:
            return (None,) * 7
        q, k, v, out, rest, lse = ctx.saved_tensors
        with on_device(q):
            grads = _backward(q, k, v, out, rest, _operand(dout), lse, ctx.L, ctx.mod, ctx.scale)
        return (*(g if need else None for g, need in zip(grads, ctx.needs_input_grad)), None, None, None, None)


def scored_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, layout: MaskLayout,
                     transform: ScoreTransform | None = None, *, scale: float | None = None, return_lse: bool = False):
    """q [nq, Hq, D], k / v [nk, Hkv, D] -> out [nq, Hq, D] (and lse [Hq, nq] float32, without gradient).

    Operands may be views of a packed projection (packed heads, any row stride). Gradients are summed over tiles by
    fp32 adds whose order is not fixed, as in `block_attention`'s one-pass backward."""
    _check(q, k, v, layout, transform)
    scale = scale if scale is not None else 1.0 / math.sqrt(q.shape[-1])
    if not SCALES[0] <= scale <= SCALES[1]:      # (positive: the row maximum is taken before the scale is applied)
        raise ValueError(f"scale must be a number from {SCALES[0]} to {SCALES[1]}, got {scale}")
    if not q.is_cuda or q.dtype != torch.bfloat16:
        out, lse = scored_attention_reference(q, k, v, layout, transform, scale)
        return (out, lse.detach()) if return_lse else out
    if q.shape[2] != 128:
        raise native.NativeKernelError("scored attention on bf16 CUDA tensors is built for head_dim 128 (no silent fallback)")
    refuse_tangents("scored attention", q, k, v, None if transform is None else transform.slopes)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        if backward_mode() == "split":
            raise native.NativeKernelError("scored attention has the one-pass backward only; unset TDLLM_ATTN_BWD=split")
        if q.shape[0] == 0 or k.shape[0] == 0:
            out, lse = scored_attention_reference(q, k, v, layout, transform, scale)
            lse = lse.detach()
        else:
            out, lse = _ScoredAttention.apply(q, k, v, layout, transform, scale, return_lse)
    elif q.shape[0] == 0 or k.shape[0] == 0:
        out = torch.zeros(q.shape, dtype=q.dtype, device=q.device)
        lse = torch.full((q.shape[1], q.shape[0]), float("-inf"), dtype=torch.float32, device=q.device)
    else:
        with on_device(q):
            q, k, v = _operand(q), _operand(k), _operand(v)
            if _few(q.shape[0], k.shape[0], q.shape[1], k.shape[1]):
                out, lse = _forward_few_rows(q, k, v, layout, transform, scale)
            else:
                L = _plan(layout, k.shape[1])
                mod, _behind = _mod_args(transform, L)
                out, lse, _ = _forward(q, k, v, L, mod, scale)
                lse = lse[:, : q.shape[0]]
    return (out, lse) if return_lse else out
