"""Attention with transformed scores: layouts, refusals and the reference on the CPU, the sm_100a kernels against the
definition in 64 bits on the GPU, with element-wise bounds that follow from where the kernels round."""
import math

import pytest
import torch

from turbo_dllm_b200.ops.attention import MaskLayout, block_diffusion_layout
from turbo_dllm_b200.ops.scored_attention import (DEAD_KEY, ScoreTransform, document_layout, document_positions,
                                                  scored_attention, scored_attention_reference)

D = 128
HALF = torch.finfo(torch.bfloat16).eps / 2     # a rounding to bf16 is off by at most half a step, relative
# everything held in 32 bits: exponentials (two of them behind a cap, whose error grows with the cap's log2 e factor, 72
# for the largest cap here, at 2^-22 each), sums over at most a few thousand terms, the stored lse
FINE = 2.0 ** -14


def exact(q, k, v, layout, tr, scale, dout=None):
    """The definition in 64 bits, head by head, and the largest error a kernel may show in each output: P and dS are
    rounded to bf16 as operands of the next product, out enters the row sum dO.out as two bf16 terms, every result is rounded."""
    nq, Hq, _ = q.shape
    Hkv = k.shape[1]
    G = Hq // Hkv
    vis = layout.dense_mask()
    q, k, v = (t.detach().double() for t in (q, k, v))
    q = torch.where(vis.any(1)[:, None, None], q, torch.zeros_like(q))
    k, v = (torch.where(vis.any(0)[:, None, None], t, torch.zeros_like(t)) for t in (k, v))
    res = {n: torch.zeros_like(t) for n, t in (("out", q), ("dq", q), ("dk", k), ("dv", v))}
    res["lse"] = torch.full((Hq, nq), -math.inf, dtype=torch.float64, device=q.device)
    tol = {n: torch.zeros_like(t) for n, t in res.items()}
    for h in range(Hq):
        qh, kh, vh = q[:, h], k[:, h // G], v[:, h // G]
        s = scale * (qh @ kh.t())
        t = torch.zeros_like(s)
        z = s
        if tr is not None and tr.softcap:
            t = torch.tanh(s / tr.softcap)
            z = tr.softcap * t
        if tr is not None and tr.biased:
            z = z - tr.slopes[h].double() * (tr.q_pos.double()[:, None] - tr.k_pos.double()[None]).abs()
        z = z.masked_fill(~vis, -math.inf)
        top = z.amax(-1, keepdim=True).clamp_min(-1e300)
        e = torch.exp(z - top)
        total = e.sum(-1, keepdim=True)
        p = e / total.clamp_min(1e-300)
        o = p @ vh
        res["out"][:, h] = o
        live = total[:, 0] > 0
        res["lse"][h, live] = (top + torch.log(total))[live, 0]
        a = p @ vh.abs()
        eo = HALF * (o.abs() + a) + FINE * a
        tol["out"][:, h] = eo
        tol["lse"][h] = FINE * (1 + res["lse"][h].abs().nan_to_num(posinf=0))
        if dout is None:
            continue
        do = torch.where(vis.any(1)[:, None], dout[:, h].detach().double(), torch.zeros_like(qh))
        dp = do @ vh.t()
        delta = (do * o).sum(-1, keepdim=True)
        f = 1 - t * t
        ds = p * f * (dp - delta)
        res["dq"][:, h] = scale * (ds @ kh)
        res["dk"][:, h // G] += scale * (ds.t() @ qh)
        res["dv"][:, h // G] += p.t() @ do
        # out is P.V with rounded P; its own rounding is kept apart (to 2^-17 of it)
        edelta = (do.abs() * ((HALF + FINE) * a + FINE * o.abs())).sum(-1, keepdim=True)
        eds = HALF * ds.abs() + p * f * edelta + p * (f + FINE) * FINE * (dp.abs() + delta.abs())
        eds = eds + HALF * eds
        tol["dq"][:, h] += scale * (eds @ kh.abs())
        tol["dk"][:, h // G] += scale * (eds.t() @ qh.abs())
        tol["dv"][:, h // G] += (HALF + FINE) * (p.t() @ do.abs())
    for n in ("dq", "dk", "dv"):
        tol[n] += HALF * (res[n].abs() + tol[n])
    return res, tol


def near(got, want, tol, name):
    got = got.detach().double()
    fin = torch.isfinite(want)
    assert torch.equal(torch.isfinite(got), fin), name
    over = ((got - want).abs() - tol)[fin]
    # 1e-6: sums of products that cancel to zero
    assert over.numel() == 0 or float(over.max()) <= 1e-6, (name, float(over.max()), float((got - want).abs()[fin].max()))


def transform_for(kind, Hq, qpos, kpos, device):
    cap = {"cap": 50.0, "smallcap": 3.0, "both": 20.0}.get(kind, 0.0)
    if kind in ("bias", "both"):
        slopes = torch.exp2(-8.0 * (torch.arange(Hq, dtype=torch.float32) + 1) / Hq).to(device)
        return ScoreTransform(cap, slopes, qpos.to(device), kpos.to(device))
    return ScoreTransform(cap) if cap else None


# ------------------------------------------------------------------------------------------------ CPU
def test_document_layout_masks():
    L = document_layout([3, 0, 5], prefix=[2, 0, 3], rows=11)
    m = L.dense_mask()
    want = torch.zeros(11, 11, dtype=torch.bool)
    for s, n, pre in ((0, 3, 2), (3, 5, 3)):
        for i in range(n):
            want[s + i, s:s + max(i + 1, pre)] = True
    assert torch.equal(m, want)
    full = document_layout([3, 5], causal=False).dense_mask()
    assert torch.equal(full, torch.block_diag(torch.ones(3, 3), torch.ones(5, 5)).bool())
    assert document_positions([3, 0, 5], rows=11).tolist() == [0, 1, 2, 0, 1, 2, 3, 4, 0, 0, 0]
    assert document_layout([]).nq == 0


@pytest.mark.parametrize("kind", ["none", "cap", "smallcap", "bias", "both"])
def test_reference_gradients_against_differences(kind):
    torch.manual_seed(1)
    lens, rows = [4, 0, 3], 9
    L = document_layout(lens, prefix=[2, 0, 0], rows=rows)
    pos = document_positions(lens, rows=rows)
    tr = transform_for(kind, 4, pos, pos, "cpu")
    x = [torch.randn(rows, h, 8, dtype=torch.float64).requires_grad_() for h in (4, 2, 2)]
    assert torch.autograd.gradcheck(lambda *t: scored_attention(*t, L, tr), x)
    out, lse = scored_attention(*x, L, tr, return_lse=True)
    assert not lse.requires_grad and bool(torch.isinf(lse[:, 7:]).all()) and float(out[7:].abs().max()) == 0


def test_reference_matches_the_plain_operator_and_ignores_dead_rows():
    from turbo_dllm_b200.ops.attention import attention_reference

    torch.manual_seed(2)
    p = torch.arange(24)
    L = block_diffusion_layout(p, p // 8, p, 8)
    q, k, v = (torch.randn(48, h, 16) for h in (4, 2, 2))
    assert torch.allclose(scored_attention(q, k, v, L), attention_reference(q, k, v, L)[0], atol=1e-6)
    L = document_layout([20, 11], rows=40)
    clean = scored_attention(q[:40], k[:40], v[:40], L)
    for t in (q, k, v):
        t[31:40] = float("nan")
    got = scored_attention(q[:40], k[:40], v[:40], L)
    assert torch.equal(got, clean)


def test_refusals():
    L = document_layout([4, 4])
    pos = document_positions([4, 4])
    q, k = torch.zeros(8, 4, 16), torch.zeros(8, 2, 16)
    for bad in (-1.0, float("nan"), float("inf")):
        with pytest.raises(ValueError, match="softcap"):
            ScoreTransform(bad)
    s = torch.ones(4)
    with pytest.raises(ValueError, match="together"):
        ScoreTransform(0.0, s)
    with pytest.raises(ValueError, match="float32"):
        ScoreTransform(0.0, s.double(), pos, pos)
    with pytest.raises(ValueError, match="no gradient"):
        ScoreTransform(0.0, s.clone().requires_grad_(), pos, pos)
    with pytest.raises(ValueError, match="int32"):
        ScoreTransform(0.0, s, pos.float(), pos)
    with pytest.raises(ValueError, match="slopes"):
        scored_attention(q, k, k, L, ScoreTransform(0.0, torch.ones(3), pos, pos))
    with pytest.raises(ValueError, match="position"):
        scored_attention(q, k, k, L, ScoreTransform(0.0, s, pos[:5], pos))
    with pytest.raises(ValueError, match="divide"):
        scored_attention(q[:, :3], k, k, L)
    with pytest.raises(ValueError, match="divide"):
        scored_attention(q[:, :0], k, k, L)
    for bad in (0.0, -0.1, float("nan"), float("inf")):
        with pytest.raises(ValueError, match="scale"):
            scored_attention(q, k, k, L, scale=bad)
    with pytest.raises(ValueError, match="layout describes"):
        scored_attention(q[:5], k, k, L)
    with pytest.raises(ValueError, match="share"):
        scored_attention(q, k.double(), k.double(), L)
    with pytest.raises(ValueError, match="need q"):
        scored_attention(q, k, k[:, :1], L)
    with pytest.raises(ValueError, match="rows"):
        document_layout([4, 4], rows=7)
    with pytest.raises(ValueError, match="prefix"):
        document_layout([4, 4], prefix=[5, 0])
    with pytest.raises(ValueError, match="negative"):
        document_layout([4, -1])
    far = torch.full((8,), 1 << 24, dtype=torch.int32)
    with pytest.raises(ValueError, match="positions"):
        ScoreTransform(0.0, s, far, pos)._padded(128, 128)


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_positions_at_the_limit(dtype):
    lim = 1 << 24
    pos = torch.zeros(4, dtype=dtype)
    ends = [lim, -lim, torch.iinfo(dtype).min, torch.iinfo(dtype).max]
    for bad in ends:
        far = pos.clone()
        far[2] = bad
        with pytest.raises(ValueError, match="positions"):
            ScoreTransform(0.0, torch.ones(2), pos, far)._padded(128, 128)
    near_ = torch.tensor([lim - 1, 1 - lim, 0, 7], dtype=dtype)
    assert ScoreTransform(0.0, torch.ones(2), pos, near_)._padded(128, 128)[2][:4].tolist() == near_.tolist()
    # the reference holds any difference: 2^24 + 1 and 2^24 are one apart
    x = torch.randn(2, 2, 8)
    L = document_layout([2])
    tr = lambda at: ScoreTransform(0.0, torch.ones(2), torch.tensor([at, at + 1]), torch.tensor([at, at + 1]))   # noqa: E731
    assert torch.equal(scored_attention(x, x, x, L, tr(lim)), scored_attention(x, x, x, L, tr(0)))


def test_caps_and_scales_that_32_bits_do_not_hold_are_refused():
    L, x = document_layout([3]), torch.randn(3, 2, 8)
    for cap in (5e-324, 1e-46, 1e-19, 1e31, 1e39):
        with pytest.raises(ValueError, match="softcap"):
            ScoreTransform(cap)
    for scale in (1e-21, 1e19, 1e39):
        with pytest.raises(ValueError, match="scale"):
            scored_attention(x, x, x, L, scale=scale)
    for cap in (1e-18, 1e30):
        assert torch.isfinite(scored_attention(x, x, x, L, ScoreTransform(cap))).all()


def test_padded_positions_follow_the_tensors():
    pos = document_positions([5])
    tr = ScoreTransform(0.0, torch.ones(2), pos, pos)
    assert tr._padded(128, 128)[1][4] == 4
    pos[4] = 9
    assert tr._padded(128, 128)[1][4] == 9


def test_changed_copies_have_their_own_lists_and_positions():
    import dataclasses

    pos = torch.arange(5)
    tr = ScoreTransform(0.0, torch.ones(2), pos, pos)
    tr._padded(128, 128)
    new = dataclasses.replace(tr, k_pos=pos + 7, slopes=torch.full((2,), 3.0))
    slopes, q_pos, k_pos = new._padded(128, 128)
    assert k_pos[:5].tolist() == [7, 8, 9, 10, 11] and q_pos[:5].tolist() == [0, 1, 2, 3, 4]
    assert torch.allclose(slopes, torch.full((2,), 3.0 * math.log2(math.e)))
    assert tr._padded(128, 128)[2][:5].tolist() == [0, 1, 2, 3, 4]
    L = document_layout([3, 2])
    L._cache["mark"] = 1
    assert dataclasses.replace(L, q_hi=L.q_hi + 1)._cache == {}


def test_documents_under_another_default_device():
    with torch.device("meta"):
        got, at = document_layout([3, 5], prefix=[1, 0], rows=11), document_positions([3, 5], rows=11)
    want = document_layout([3, 5], prefix=[1, 0], rows=11)
    assert torch.equal(got.dense_mask(), want.dense_mask()) and torch.equal(at, document_positions([3, 5], rows=11))


@pytest.mark.parametrize("way", ["copy", "deepcopy", "pickle"])
def test_copies_keep_nothing_that_was_built(way):
    """What is kept holds addresses of one process's device memory, which a copy does not own."""
    import copy
    import pickle

    make = {"copy": copy.copy, "deepcopy": copy.deepcopy, "pickle": lambda t: pickle.loads(pickle.dumps(t))}[way]
    L, pos = document_layout([3, 2]), torch.arange(5)
    tr = ScoreTransform(2.0, torch.ones(2), pos, pos + 1)
    lists = L.tile_lists()
    tr._padded(128, 128)
    M, ts = make(L), make(tr)
    assert M._cache == {} and ts._cache == {} and L._cache["lists"] is lists and "padded" in tr._cache
    assert torch.equal(M.dense_mask(), L.dense_mask()) and ts.softcap == 2.0 and torch.equal(ts.k_pos, tr.k_pos)
    assert M.tile_lists()["f_idx"].tolist() == lists["f_idx"].tolist()


def test_writes_that_are_told():
    pos = torch.arange(5)
    tr = ScoreTransform(0.0, torch.ones(2), pos, pos)
    held = tr._padded(128, 128)
    assert tr._padded(128, 128)[2] is held[2]
    pos.data[4] = 9        # (not counted)
    tr.changed()
    assert tr._padded(128, 128)[2][:5].tolist() == [0, 1, 2, 3, 9]


@pytest.mark.parametrize("nq,nk", [(3, 0), (0, 3), (0, 0)])
@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_gradients_of_calls_without_rows_or_keys(nq, nk, device):
    """Zeros, whatever the operands hold, on the path of the caller's loss."""
    dtype = torch.float32 if device == "cpu" else torch.bfloat16
    z = torch.zeros(nq, dtype=torch.int32, device=device)
    L = MaskLayout(z, z + 9, z, torch.arange(nk, dtype=torch.int32, device=device))
    leaves = [torch.full((n, h, D), float("nan"), dtype=dtype, device=device).requires_grad_() for n, h in ((nq, 4), (nk, 2), (nk, 2))]
    out, lse = scored_attention(*leaves, L, ScoreTransform(3.0), return_lse=True)
    assert out.shape == (nq, 4, D) and out.dtype == dtype and lse.shape == (4, nq) and not lse.requires_grad
    assert lse.dtype == torch.float32 and bool((lse == -math.inf).all()) and bool((out == 0).all())
    for got, leaf in zip(torch.autograd.grad(out.sum(), leaves), leaves):
        assert got.shape == leaf.shape and got.dtype == dtype and bool((got == 0).all())


# ------------------------------------------------------------------------------------------------ GPU
def _operands(nq, nk, Hq, Hkv, seed, packed=False, gain=2.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    if packed:
        rows = torch.randn(nq, (Hq + 2 * Hkv) * D, generator=g, device="cuda").bfloat16() * gain
        return (rows[:, :Hq * D].view(nq, Hq, D), rows[:, Hq * D:(Hq + Hkv) * D].view(nk, Hkv, D),
                rows[:, (Hq + Hkv) * D:].view(nk, Hkv, D))
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")   # noqa: E731
    return (r(nq, Hq, D) * gain).bfloat16(), r(nk, Hkv, D).bfloat16(), r(nk, Hkv, D).bfloat16()


@pytest.fixture
def listed(monkeypatch):
    """Forward passes without gradients go by tile lists, whatever their size."""
    from turbo_dllm_b200.ops import scored_attention as sa

    monkeypatch.setattr(sa, "_few", lambda *a: False)


def run_case(q, k, v, layout, tr, backward=True, seed=3):
    """Forward (and backward) against 64 bits; the forward pass without gradients in both of its forms, too."""
    from turbo_dllm_b200.kernels import native
    from turbo_dllm_b200.ops import scored_attention as sa

    scale = 1.0 / math.sqrt(D)
    q, k, v = (t.detach().requires_grad_(backward) for t in (q, k, v))
    out, lse = scored_attention(q, k, v, layout, tr, return_lse=True)
    dout = torch.randn(out.shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").bfloat16()
    got = {"out": out.detach(), "lse": lse}
    if backward:
        got.update(zip(("dq", "dk", "dv"), torch.autograd.grad(out, [q, k, v], dout)))
    torch.cuda.synchronize()
    native.raise_on_device_error()
    want, tol = exact(q, k, v, layout, tr, scale, dout if backward else None)
    for n, t in got.items():
        near(t, want[n], tol[n], n)
    for few in (True, False):
        with pytest.MonkeyPatch.context() as mp, torch.no_grad():
            mp.setattr(sa, "_few", lambda *a: few)
            out, lse = scored_attention(q, k, v, layout, tr, return_lse=True)
        torch.cuda.synchronize()
        native.raise_on_device_error()
        near(out, want["out"], tol["out"], "out")
        near(lse, want["lse"], tol["lse"], "lse")
    return got


def blocks(tokens, block, device="cuda", window=None):
    p = torch.arange(tokens, device=device)
    L = block_diffusion_layout(p, p // block, p, block, window=window)
    return L, torch.cat([p, p]).to(torch.int32)


@pytest.mark.gpu
def test_document_lengths_that_lie_on_the_gpu():
    lens, pre = torch.tensor([3, 0, 5], device="cuda"), torch.tensor([2, 0, 3], device="cuda", dtype=torch.int32)
    for device in ("cpu", "cuda"):
        for causal in (True, False):
            got = document_layout(lens, prefix=pre, rows=11, causal=causal, device=device)
            want = document_layout([3, 0, 5], prefix=[2, 0, 3], rows=11, causal=causal)
            assert got.q_lo.device.type == device and torch.equal(got.dense_mask().cpu(), want.dense_mask())
        at = document_positions(lens, rows=11, device=device)
        assert at.device.type == device and torch.equal(at.cpu(), document_positions([3, 0, 5], rows=11))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["none", "cap", "smallcap", "bias", "both"])
@pytest.mark.parametrize("lens,prefix,rows", [([1], None, 1), ([5, 0, 2], None, 7), ([128], None, 128), ([129], [40], 129),
                                             ([100, 1, 200, 30], [0, 1, 150, 30], 345), ([700], [1], 719)])
def test_documents(kind, lens, prefix, rows):
    L = document_layout(lens, prefix=prefix, rows=rows, device="cuda")
    pos = document_positions(lens, rows=rows, device="cuda")
    run_case(*_operands(rows, rows, 4, 2, 0, packed=True), L, transform_for(kind, 4, pos, pos, "cuda"))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["cap", "both"])
@pytest.mark.parametrize("Hq,Hkv", [(1, 1), (3, 1), (8, 2), (6, 6)])
def test_blocks(kind, Hq, Hkv):
    L, pos = blocks(256, 32)
    run_case(*_operands(512, 512, Hq, Hkv, 1), L, transform_for(kind, Hq, pos, pos, "cuda"))


@pytest.mark.gpu
def test_windows_and_keys_of_another_length():
    L, pos = blocks(384, 16, window=100)
    run_case(*_operands(768, 768, 4, 2, 2), L, transform_for("both", 4, pos, pos, "cuda"))
    p = torch.arange(500, device="cuda")
    L = block_diffusion_layout(p[96:160], p[96:160] // 32, p[:77], 32, key_clean_pos=p[::3])
    qpos = torch.cat([p[96:160], p[:77]]).to(torch.int32)
    kpos = torch.cat([p[96:160], p[::3]]).to(torch.int32)
    run_case(*_operands(L.nq, L.nk, 4, 2, 3), L, transform_for("both", 4, qpos, kpos, "cuda"))


def step_layout(caches, new, device="cuda", capacity=None, window=None):
    """`new` rows per sequence against its own clean cache (rows behind a cache's length hold nothing) and each other."""
    s, span = len(caches), 1 << 20
    cap = capacity or max(max(caches), 1)
    seq = torch.arange(s, device=device)
    n = torch.tensor(caches, device=device)
    at = torch.arange(cap, device=device)
    kc = torch.where(at[None] < n[:, None], seq[:, None] * span + at[None], torch.full((), DEAD_KEY, device=device)).reshape(-1)
    sq, end = seq.repeat_interleave(new), n.repeat_interleave(new)
    lo = sq * span + (0 if window is None else (end - window).clamp_min(0))
    L = MaskLayout(*(t.to(torch.int32) for t in (lo, sq * span + end, -(sq + 1), torch.cat([kc, -(sq + 1)]))))
    qpos = (end + torch.arange(new, device=device).repeat(s)).to(torch.int32)
    return L, qpos, torch.cat([at.repeat(s).to(torch.int32), qpos])


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["none", "cap", "bias", "both"])
@pytest.mark.parametrize("caches,new,Hq,Hkv", [([1], 1, 1, 1), ([0], 1, 4, 2), ([5000], 1, 8, 2), ([700, 0, 1300], 1, 12, 4),
                                               ([300, 129], 32, 8, 2), ([4000], 32, 4, 1), ([260, 1, 513], 17, 6, 2),
                                               ([130], 128, 3, 1), ([2000], 5, 16, 2),
                                               ([1000], 100, 2, 2), ([300, 200], 64, 8, 1), ([5], 40, 16, 1),
                                               ([900], 300, 8, 2), ([500, 31], 137, 4, 4), ([600], 140, 6, 2)])
def test_few_rows(kind, caches, new, Hq, Hkv):
    L, qpos, kpos = step_layout(caches, new)
    for backward in (False, True):
        run_case(*_operands(L.nq, L.nk, Hq, Hkv, 8), L, transform_for(kind, Hq, qpos, kpos, "cuda"), backward=backward)


@pytest.mark.gpu
@pytest.mark.parametrize("new,Hq", [(1, 8), (9, 8), (30, 8), (9, 6)])
def test_few_rows_against_caches_with_junk_behind_their_lengths(new, Hq):
    L, qpos, kpos = step_layout([70, 900, 0], new, capacity=1000)
    q, k, v = _operands(L.nq, L.nk, Hq, 2, 9)
    dead = L.k_code == DEAD_KEY
    k[dead] = float("nan")
    v[dead] = float("inf")
    for backward in (False, True):
        run_case(q, k, v, L, transform_for("both", Hq, qpos, kpos, "cuda"), backward=backward)
    L, qpos, kpos = step_layout([3000], new, window=300)
    run_case(*_operands(L.nq, L.nk, Hq, 2, 9), L, transform_for("cap", Hq, qpos, kpos, "cuda"), backward=False)


@pytest.mark.gpu
@pytest.mark.parametrize("junk", [float("nan"), float("inf")])
@pytest.mark.parametrize("kind", ["none", "both"])
@pytest.mark.parametrize("caches,new,Hq,window", [([100] * 4, 9, 8, None), ([100, 250, 0, 180], 32, 8, None),
                                                  ([120, 256, 200], 20, 6, 60), ([30, 700], 3, 16, 20)])
def test_junk_in_unseen_cache_slots_between_seen_ones(caches, new, Hq, window, kind, junk):
    """Slots behind a sequence's length, or in front of its window, with running codes that no row sees: between the codes
    that the sequences before and behind it see. And unused noisy groups between used ones."""
    cap = max(caches) + 30
    L, qpos, kpos = step_layout(caches, new, capacity=cap, window=window)
    seqs, span = len(caches), 1 << 20
    at = torch.arange(cap, dtype=torch.int32, device="cuda")
    slots = (torch.arange(seqs, dtype=torch.int32, device="cuda")[:, None] * span + at[None]).reshape(-1)
    # (groups 1, 3, 5, ... used; a key of each even one in between)
    L = MaskLayout(L.q_lo, L.q_hi, 2 * L.q_grp, torch.cat([slots, 2 * L.k_code[seqs * cap:], -1 - 2 * torch.arange(
        1, seqs + 1, dtype=torch.int32, device="cuda")]))
    kpos = torch.cat([kpos, torch.zeros(seqs, dtype=torch.int32, device="cuda")])
    unseen = ~L.dense_mask().any(0)
    assert int(unseen[: seqs * cap].sum()) >= 30 * seqs and bool(unseen[-seqs:].all())
    q, k, v = _operands(L.nq, L.nk, Hq, 2, 15)
    k[unseen], v[unseen] = junk, -junk
    run_case(q, k, v, L, transform_for(kind, Hq, qpos, kpos, "cuda"), backward=False)


@pytest.mark.gpu
def test_few_rows_over_more_tiles_than_one_round():
    """148 KV heads leave one split of the keys, whose 1095 tiles exceed the 1024 of one visibility round."""
    L, qpos, kpos = step_layout([140000], 1)
    q, k, v = _operands(L.nq, L.nk, 1, 1, 10, gain=1.0)
    q, k, v = (t.expand(-1, 148, -1).contiguous() for t in (q, k, v))
    out, lse = scored_attention(q, k, v, L, ScoreTransform(30.0), return_lse=True)
    assert torch.equal(out, out[:, :1].expand_as(out)) and torch.equal(lse, lse[:1].expand_as(lse))
    want, tol = exact(q[:, :1], k[:, :1], v[:, :1], L, ScoreTransform(30.0), 1.0 / math.sqrt(D))
    near(out[:, :1], want["out"], tol["out"], "out")
    near(lse[:1], want["lse"], tol["lse"], "lse")


@pytest.mark.gpu
def test_few_rows_graph_follows_the_metadata():
    L, qpos, kpos = step_layout([500], 1, capacity=800)
    q, k, v = _operands(L.nq, L.nk, 8, 2, 12)
    tr = transform_for("both", 8, qpos, kpos, "cuda")
    scored_attention(q, k, v, L, tr)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = scored_attention(q, k, v, L, tr)
    M, mq, mk = step_layout([620], 1, capacity=800)
    for a, b in ((L.q_hi, M.q_hi), (L.k_code, M.k_code), (tr.q_pos, mq), (tr.k_pos, mk)):
        a.copy_(b)
    graph.replay()
    assert torch.equal(held, scored_attention(q, k, v, M, transform_for("both", 8, mq, mk, "cuda")))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("Hq,rows", [(2, 5), (6, 40), (8, 40)])
def test_positions_beyond_the_limit_are_refused_or_spoil_their_rows(Hq, rows, dtype):
    """One key position that floats do not hold: the call by tile lists refuses it, calls of few rows, whose positions stay on
    the device, and a captured graph give NaN to the rows that see the key, and to no other."""
    from turbo_dllm_b200.ops import scored_attention as sa

    n = 300
    whole, pos = document_layout([n], device="cuda"), torch.arange(n, device="cuda", dtype=dtype)
    at = torch.arange(n - rows, n, device="cuda")
    L = MaskLayout(whole.q_lo[at], whole.q_hi[at], whole.q_grp[at], whole.k_code)
    q, k, v = _operands(rows, n, Hq, 2, 21)
    bad = n - rows + 3        # rows 3 and later see it
    slopes = torch.full((Hq,), 0.25, device="cuda")
    want = scored_attention(q, k, v, L, ScoreTransform(0.0, slopes, pos[at], pos))
    for value in (1 << 24, -(1 << 24), torch.iinfo(dtype).min, torch.iinfo(dtype).max):
        far = pos.clone()
        far[bad] = value
        tr = ScoreTransform(0.0, slopes, pos[at], far)
        out, lse = scored_attention(q, k, v, L, tr, return_lse=True)
        assert torch.equal(out[:3], want[:3]) and bool(out[3:].isnan().all()) and bool(lse[:, 3:].isnan().all())
        leaf = q.detach().requires_grad_()
        with pytest.raises(ValueError, match="positions"):
            scored_attention(leaf, k, v, L, tr)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with pytest.MonkeyPatch.context() as mp, torch.no_grad():
        mp.setattr(sa, "_few", lambda *a: False)
        with torch.cuda.graph(graph):
            held = scored_attention(q, k, v, L, tr)
    graph.replay()
    assert not bool(held[:3].isnan().any()) and bool(held[3:].isnan().all())


@pytest.mark.gpu
@pytest.mark.parametrize("Hq", [4, 6, 32])
@pytest.mark.parametrize("kind", ["none", "cap", "bias"])
@pytest.mark.parametrize("rows", [100, 160])
def test_a_row_whose_scores_are_nan_says_so(rows, kind, Hq):
    """A query row of NaN that does see keys: NaN out, log-sum-exp and gradients, not those of a row without keys (which a
    merge of partial results would leave out). The other rows keep theirs."""
    from turbo_dllm_b200.ops import scored_attention as sa

    bad = 37
    L, pos = document_layout([rows], device="cuda"), document_positions([rows], device="cuda")
    tr = transform_for(kind, Hq, pos, pos, "cuda")
    q, k, v = _operands(rows, rows, Hq, 2, 18)
    spoilt = q.clone()
    spoilt[bad] = float("nan")
    rest = torch.arange(rows, device="cuda") != bad
    for few in (True, False):
        with pytest.MonkeyPatch.context() as mp:
            mp.setattr(sa, "_few", lambda *a: few)
            want, want_lse = scored_attention(q, k, v, L, tr, return_lse=True)
            out, lse = scored_attention(spoilt, k, v, L, tr, return_lse=True)
        assert bool(out[bad].isnan().all()) and bool(lse[:, bad].isnan().all())
        assert torch.equal(out[rest], want[rest]) and torch.equal(lse[:, rest], want_lse[:, rest])
    leaves = [t.requires_grad_() for t in (spoilt, k, v)]
    out, lse = scored_attention(*leaves, L, tr, return_lse=True)
    dq, dk, dv = torch.autograd.grad(out, leaves, torch.ones_like(out))
    assert bool(out[bad].isnan().all()) and bool(lse[:, bad].isnan().all()) and bool(dq[bad].isnan().all())
    assert not bool(dq[rest].isnan().any()) and bool(dv[:bad + 1].isnan().all()) and not bool(dv[bad + 1:].isnan().any())


@pytest.mark.gpu
@pytest.mark.parametrize("junk", [float("nan"), float("inf"), -3.0e38])
def test_contents_of_dead_rows_do_not_matter(junk):
    lens, rows = [90, 130], 300
    L = document_layout(lens, rows=rows, device="cuda")
    pos = document_positions(lens, rows=rows, device="cuda")
    tr = transform_for("both", 4, pos, pos, "cuda")
    q, k, v = (t.clone() for t in _operands(rows, rows, 4, 2, 4))
    for t in (q, k, v):
        t[220:] = junk
    got = run_case(q, k, v, L, tr)
    assert float(got["out"][220:].abs().max()) == 0 and all(float(got[n][220:].abs().max()) == 0 for n in ("dq", "dk", "dv"))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["none", "cap", "both"])
@pytest.mark.parametrize("masked", ["0" * 11, "1" * 11, "10000100010", "0001111011110", "01", "1000", "00000001", "0110" * 6])
def test_key_tiles_with_and_without_a_mask_in_turn(kind, masked):
    """Codes come into shared memory for the tiles that need them only; a tile after one without still reads its own. One dead
    key with junk in each masked tile, at another place each time."""
    n, nq = 128 * len(masked), 200
    code = torch.arange(n, dtype=torch.int32)
    for t, c in enumerate(masked):
        if c == "1":
            code[128 * t + (37 * t + 5) % 128] = DEAD_KEY
    z = torch.zeros(nq, dtype=torch.int32, device="cuda")
    L = MaskLayout(z, z + n, z, code.cuda())
    q, k, v = _operands(nq, n, 4, 2, 16)
    k[L.k_code == DEAD_KEY], v[L.k_code == DEAD_KEY] = float("nan"), float("nan")
    pos = torch.arange(n, dtype=torch.int32, device="cuda")
    run_case(q, k, v, L, transform_for(kind, 4, pos[:nq] if n >= nq else pos.new_zeros(nq), pos, "cuda"))


@pytest.mark.gpu
def test_masks_that_leave_every_row_empty():
    z = torch.zeros(70, dtype=torch.int32, device="cuda")
    L = MaskLayout(z, z, z, z + 5)
    got = run_case(*_operands(70, 70, 2, 1, 5), L, ScoreTransform(10.0))
    assert float(got["dk"].abs().max()) == 0


@pytest.mark.gpu
def test_strides_and_alignment():
    L = document_layout([150], device="cuda")
    q, k, v = _operands(150, 150, 4, 2, 6)
    base = scored_attention(q, k, v, L, ScoreTransform(20.0))
    odd = torch.empty(150 * 4 * D + 1, dtype=torch.bfloat16, device="cuda")[1:].view(150, 4, D)    # 2-byte aligned base
    odd.copy_(q)
    heads_first = k.permute(1, 0, 2).contiguous().permute(1, 0, 2)
    wide = torch.zeros(150, 2, 2 * D, dtype=torch.bfloat16, device="cuda")
    wide[..., :D] = v
    assert torch.equal(scored_attention(odd, heads_first, wide[..., :D], L, ScoreTransform(20.0)), base)
    qg = odd.detach().requires_grad_()
    out = scored_attention(qg, heads_first, wide[..., :D], L, ScoreTransform(20.0))
    (dq,) = torch.autograd.grad(out, [qg], torch.ones((), dtype=out.dtype, device="cuda").expand_as(out))
    assert torch.isfinite(dq).all()


def scattered_layout(seed, nq, nk):
    """Intervals, blocks and codes in no order; some rows see nothing, some keys are seen by none."""
    g = torch.Generator().manual_seed(seed)
    lo = torch.randint(0, 60, (nq,), generator=g)
    hi = lo + torch.randint(-5, 20, (nq,), generator=g)
    grp = -torch.randint(0, 6, (nq,), generator=g)
    code = torch.randint(-8, 90, (nk,), generator=g)
    code[5] = DEAD_KEY
    return MaskLayout(*(t.to(torch.int32).cuda() for t in (lo, hi, grp, code)))


@pytest.mark.gpu
@pytest.mark.parametrize("make", [lambda: document_layout([300, 0, 77], prefix=[40, 0, 0], rows=400, device="cuda"),
                                  lambda: blocks(640, 32, window=200)[0], lambda: step_layout([70, 900, 0], 60, capacity=1000)[0],
                                  lambda: document_layout([1], device="cuda"),
                                  *(lambda seed=seed, n=n: scattered_layout(seed, *n) for seed in (0, 1) for n in ((23, 57), (500, 700)))])
@pytest.mark.parametrize("Hkv", [1, 8, 64])
def test_plan_matches_the_dense_mask(make, Hkv):
    """Every visible pair lies in a listed tile, tiles without a mask are fully visible, lists are complete and in order."""
    import ctypes

    from turbo_dllm_b200.ops import scored_attention as sa

    L = make()
    P = sa._plan(L, Hkv)   # (few heads: chunks of one query tile; many: one chunk)
    off = (ctypes.c_longlong * 11)()
    from turbo_dllm_b200.kernels import native

    chunk = P["chunk"]
    native.lib().tdllm_attn_plan_size(L.nq, L.nk, chunk, off)
    buf = P["buf"].cpu().tolist()
    nqt, nkt = P["nqt"], P["nkt"]
    m = torch.zeros(nqt * 128, nkt * 128, dtype=torch.bool)
    m[: L.nq, : L.nk] = L.dense_mask().cpu()
    # keys that no row sees come in as dead
    codes = torch.where(m.any(0)[: L.nk], L.k_code.cpu(), torch.full((), DEAD_KEY, dtype=torch.int32)).tolist()
    assert buf[off[3]: off[3] + L.nk] == codes and set(buf[off[3] + L.nk: off[3] + nkt * 128]) <= {DEAD_KEY}
    any_ = m.view(nqt, 128, nkt, 128).any(3).any(1)
    real = torch.arange(nqt * 128) < L.nq
    all_ = (m | ~real[:, None]).view(nqt, 128, nkt, 128).all(3).all(1)
    part = lambda i, n: buf[off[i]: off[i] + n]   # noqa: E731
    f_ptr, f_order = part(4, nqt + 1), part(6, nqt)
    lists = [buf[off[5] + f_ptr[i]: off[5] + f_ptr[i + 1]] for i in range(nqt)]
    for i, l in enumerate(lists):
        tiles = [e >> 1 for e in l]
        assert tiles == sorted(set(tiles)) and set(any_[i].nonzero().flatten().tolist()) <= set(tiles)
        assert all(bool(all_[i, e >> 1]) for e in l if not e & 1)
    assert sorted(f_order) == list(range(nqt)) and all(len(lists[a]) >= len(lists[b]) for a, b in zip(f_order, f_order[1:]))
    nch = (nqt + chunk - 1) // chunk
    w_ptr, w_order = part(7, nch * nkt + 1), part(9, nch * nkt)
    back = {(e >> 1, it % nkt, e & 1) for it in range(nch * nkt) for e in buf[off[8] + w_ptr[it]: off[8] + w_ptr[it + 1]]}
    assert back == {(i, e >> 1, e & 1) for i, l in enumerate(lists) for e in l}
    assert all((e >> 1) // chunk == it // nkt for it in range(nch * nkt) for e in buf[off[8] + w_ptr[it]: off[8] + w_ptr[it + 1]])
    assert sorted(w_order) == list(range(nch * nkt))


@pytest.mark.gpu
def test_a_layout_that_is_written_to_and_a_plan_built_inside_a_capture(listed):
    q, k, v = _operands(300, 300, 4, 2, 13)
    L = document_layout([300], device="cuda")
    tr = ScoreTransform(20.0)
    scored_attention(q, k, v, L, tr)
    M = document_layout([100, 200], device="cuda")
    for a, b in ((L.q_lo, M.q_lo), (L.q_hi, M.q_hi)):
        a.copy_(b)
    want = scored_attention(q, k, v, M, tr)
    assert torch.equal(scored_attention(q, k, v, L, tr), want)
    torch.cuda.synchronize()
    fresh = document_layout([100, 200], device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = scored_attention(q, k, v, fresh, tr)
    # nothing of a capture is kept outside of it: its lists exist only once it has run
    assert not any(n.startswith("scored") for n in fresh._cache) and torch.equal(scored_attention(q, k, v, fresh, tr), want)
    graph.replay()
    assert torch.equal(held, want)
    # a graph that was captured with a layout's lists goes on using them when the layout moves on
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = scored_attention(q, k, v, fresh, tr)
    fresh.q_hi.copy_(document_layout([300], device="cuda").q_hi)
    scored_attention(q, k, v, fresh, tr)
    junk = [torch.full((4096,), 7, dtype=torch.int32, device="cuda") for _ in range(64)]
    graph.replay()
    assert torch.equal(held, want) and len(junk) == 64


@pytest.mark.gpu
def test_changed_copies_and_assigned_tensors_are_followed(listed):
    """A replaced layout or transform, and a layout with a new tensor in one of its fields, whose version counters are those of
    the tensors before them: the results of objects made from nothing."""
    import dataclasses

    q, k, v = _operands(300, 300, 4, 2, 14)
    pos = torch.arange(300, device="cuda", dtype=torch.int32)
    one, two = document_layout([300], device="cuda"), document_layout([100, 200], device="cuda")
    tr = transform_for("bias", 4, pos, pos, "cuda")
    other = transform_for("bias", 4, pos, pos * 3, "cuda")
    first = scored_attention(q, k, v, one, tr)
    want = scored_attention(q, k, v, two, ScoreTransform(0.0, other.slopes, other.q_pos, other.k_pos))
    L = dataclasses.replace(one, q_lo=two.q_lo, q_hi=two.q_hi)
    assert torch.equal(scored_attention(q, k, v, L, dataclasses.replace(tr, k_pos=other.k_pos)), want)
    out = scored_attention(q.detach().requires_grad_(), k, v, L, tr)
    assert torch.equal(out[100], v[100].repeat_interleave(2, 0))      # (the second document's first row sees itself alone)
    one.q_lo, one.q_hi = two.q_lo.clone(), two.q_hi.clone()
    assert not torch.equal(first, want) and torch.equal(scored_attention(q, k, v, one, other), want)


@pytest.mark.gpu
def test_a_replayed_graph_that_writes_the_layout_and_the_positions(listed):
    """Eager calls by tile lists after a replay that moved the metadata on, once they are told."""
    q, k, v = _operands(300, 300, 4, 2, 20)
    pos = torch.arange(300, dtype=torch.int32, device="cuda")
    L, tr = document_layout([300], device="cuda"), transform_for("bias", 4, pos.clone(), pos.clone(), "cuda")
    M = document_layout([100, 200], device="cuda")
    before = scored_attention(q, k, v, L, tr)
    want = scored_attention(q, k, v, M, transform_for("bias", 4, pos * 2, pos * 2, "cuda"))
    writes = [(L.q_lo, M.q_lo.clone()), (L.q_hi, M.q_hi.clone()), (tr.q_pos, pos * 2), (tr.k_pos, pos * 2)]
    back = [(a, a.clone()) for a, _ in writes]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for a, b in writes:
            a.copy_(b)
    for a, b in back:
        a.copy_(b)
    assert torch.equal(scored_attention(q, k, v, L, tr), before)
    graph.replay()
    L.changed()
    tr.changed()
    assert torch.equal(scored_attention(q, k, v, L, tr), want)


@pytest.mark.gpu
def test_layouts_of_inference_mode_are_followed(listed):
    q, k, v = _operands(300, 300, 4, 2, 19)
    want = scored_attention(q, k, v, document_layout([300], device="cuda"))
    with torch.inference_mode():
        L = document_layout([100, 200], device="cuda")
        scored_attention(q, k, v, L)
        M = document_layout([300], device="cuda")
        L.q_lo.copy_(M.q_lo)
        L.q_hi.copy_(M.q_hi)
        assert torch.equal(scored_attention(q, k, v, L), want)


@pytest.mark.gpu
def test_a_layout_that_dies_while_another_stream_uses_its_lists(listed):
    """The lists were allocated on the default stream; their memory must not go to a tensor there while the side stream
    still has the kernels that read them in front of it."""
    q, k, v = _operands(2000, 2000, 4, 2, 17)
    tr = ScoreTransform(20.0)
    want = scored_attention(q, k, v, document_layout([700, 1300], device="cuda"), tr)
    side = torch.cuda.Stream()
    for _ in range(3):
        L = document_layout([700, 1300], device="cuda")
        scored_attention(q, k, v, L, tr)
        side.wait_stream(torch.cuda.current_stream())
        busy = torch.randn(6000, 6000, device="cuda")
        with torch.cuda.stream(side):
            for _ in range(8):
                busy = busy @ busy * 1e-3
            got = scored_attention(q, k, v, L, tr)
        size = next(v for n, v in L._cache.items() if n.startswith("scored"))[1][0][0].numel()
        del L
        junk = [torch.zeros(size, dtype=torch.int32, device="cuda") for _ in range(8)]
        torch.cuda.synchronize()
        assert torch.equal(got, want) and len(junk) == 8


@pytest.mark.gpu
@pytest.mark.parametrize("cap", [1e-3, 0.7, 8.0, 300.0, 1e5])
@pytest.mark.parametrize("gain", [0.3, 6.0])
def test_caps_of_every_size(cap, gain):
    """Small and large scores against the cap take different forms of the tanh, and very small or large caps leave one whose
    coefficients 32 bits do not hold: whatever is taken, the row maximum's probability is right to the usual tolerance."""
    q, k, v = (t * gain for t in _operands(200, 200, 4, 2, 23))
    L, tr = document_layout([150, 50], device="cuda"), ScoreTransform(cap)
    want, lse = scored_attention_reference(q.double(), k.double(), v.double(), L, tr)
    for rows in (200, 40):
        M = MaskLayout(L.q_lo[:rows], L.q_hi[:rows], L.q_grp[:rows], L.k_code)
        out, got = scored_attention(q[:rows], k, v, M, tr, return_lse=True)
        # z is known to 2^-20 of the cap and 2^-22 of itself (a score of up to 600 here)
        tol = 2.0 ** -20 * min(cap, 600.0) + 2.0 ** -21 * min(cap, 600.0) + 2.0 ** -18
        assert float((got.double() - lse[:, :rows]).abs().max()) <= tol
        # probabilities are off by half a step (2^-8) and by tol, the output by half a step
        size = scored_attention_reference(q.double(), k.double(), v.double().abs(), L, tr)[0][:rows]
        assert bool(((out.double() - want[:rows]).abs() <= 2.0 ** -8 * want[:rows].abs() + (2.0 ** -8 + 4 * tol) * size).all())


@pytest.mark.gpu
@pytest.mark.parametrize("few", [True, False])
def test_caps_and_scales_at_their_limits(few, monkeypatch):
    """Caps of 1e-18 leave scores of nothing (the mean of v over the visible rows), caps of 1e30 leave them as they are."""
    from turbo_dllm_b200.ops import scored_attention as sa

    monkeypatch.setattr(sa, "_few", lambda *a: few)
    L = document_layout([200], causal=False, device="cuda")
    q, k, v = _operands(200, 200, 4, 2, 24)
    for cap, scale in ((1e-18, 1e18), (1e-18, 1e-20), (1e-18, 0.1), (1e30, 1e-20), (1e30, 0.1)):
        out, lse = scored_attention(q, k, v, L, ScoreTransform(cap), scale=scale, return_lse=True)
        want, want_lse = scored_attention_reference(q.double(), k.double(), v.double(), L, ScoreTransform(cap), scale)
        size = scored_attention_reference(q.double(), k.double(), v.double().abs(), L, ScoreTransform(cap), scale)[0]
        # scores up to 200 in 32 bits (2^-22 each), probabilities and the output off by half a step
        assert float((lse.double() - want_lse).abs().max()) <= 2.0 ** -14 * (1 + float(want_lse.abs().max()))
        assert bool(((out.double() - want).abs() <= HALF * want.abs() + (HALF + 2.0 ** -12) * size).all())


@pytest.mark.gpu
def test_empty_operands_and_other_types():
    e = torch.empty(0, 4, D, dtype=torch.bfloat16, device="cuda")
    L = document_layout([], device="cuda")
    out, lse = scored_attention(e, e[:, :2], e[:, :2], L, ScoreTransform(5.0), return_lse=True)
    assert out.shape == (0, 4, D) and lse.shape == (4, 0)
    z = torch.zeros(3, dtype=torch.int32, device="cuda")
    q = torch.randn(3, 4, D, device="cuda").bfloat16().requires_grad_()
    out, lse = scored_attention(q, e[:, :2], e[:, :2], MaskLayout(z, z + 9, z, z[:0]), return_lse=True)
    assert float(out.abs().max()) == 0 and bool(torch.isinf(lse).all())
    x = torch.randn(40, 2, 64, device="cuda")
    L = document_layout([40], device="cuda")
    ref = scored_attention_reference(x.double(), x.double(), x.double(), L, ScoreTransform(3.0))[0]
    assert torch.allclose(scored_attention(x, x, x, L, ScoreTransform(3.0)).double(), ref, atol=1e-5)
    from turbo_dllm_b200.kernels.native import NativeKernelError

    with pytest.raises(NativeKernelError, match="head_dim"):
        scored_attention(x.bfloat16(), x.bfloat16(), x.bfloat16(), L)


@pytest.mark.parametrize("heads,nq,nk,few", [((32, 8), 128, 1, True), ((32, 8), 129, 256, False), ((32, 8), 512, 512, True),
                                             ((32, 8), 577, 4096, False), ((8, 8), 2304, 2304, True), ((12, 4), 129, 4096, False)])
def test_which_form_a_forward_pass_takes(heads, nq, nk, few):
    from turbo_dllm_b200.ops import scored_attention as sa

    assert sa._few(nq, nk, *heads) is few


@pytest.mark.gpu
def test_another_stream_and_a_captured_graph():
    L = document_layout([200], device="cuda")
    q, k, v = _operands(200, 200, 4, 2, 7)
    tr = ScoreTransform(20.0)
    want = scored_attention(q, k, v, L, tr)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = scored_attention(q, k, v, L, tr)
    side.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = scored_attention(q, k, v, L, tr)
    q.copy_(q.flip(0))
    graph.replay()
    assert torch.equal(held, scored_attention(q, k, v, L, tr))


@pytest.mark.gpu
def test_threads_share_a_layout(listed):
    import threading

    L, tr = document_layout([400, 200], device="cuda"), ScoreTransform(20.0)
    q, k, v = _operands(600, 600, 8, 2, 29)
    want = scored_attention(q, k, v, document_layout([400, 200], device="cuda"), tr)
    torch.cuda.synchronize()
    wrong = []

    def work():
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            for _ in range(10):
                out = scored_attention(q, k, v, L, tr)
                side.synchronize()
                wrong.extend([] if torch.equal(out, want) else [1])

    threads = [threading.Thread(target=work) for _ in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


@pytest.mark.gpu
def test_two_captured_training_steps_replay_at_once():
    L, tr = document_layout([400, 200], device="cuda"), ScoreTransform(20.0)
    leaves = [t.requires_grad_() for t in _operands(600, 600, 8, 2, 31)]
    dout = torch.randn(600, 8, D, device="cuda").bfloat16()

    def step():
        out = scored_attention(*leaves, L, tr)
        return [out.detach(), *torch.autograd.grad(out, leaves, dout)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = [t.clone() for t in step()]
    torch.cuda.synchronize()
    graphs, held = [], []
    for _ in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            held.append(step())
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(5):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for got in held:
        assert torch.equal(got[0], want[0])
        for a, b in zip(got[1:], want[1:]):    # (sums in another order: a step of the type)
            assert float((a.double() - b.double()).norm()) <= HALF * float(b.double().norm())
