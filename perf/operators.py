"""Cases that time the operators between a decoder layer's matrix products: attention whose scores are capped or biased
by distance under a block, document or prefix mask (training, prompts, one token, one block of new tokens), rotary
positions (half and interleaved pairs, part of a head, scaled for long contexts), and the norms behind and in front of
a block with its gate and its residual.

`run` computes a case in plain torch operations, or, where `own` is true, through `turbo_dllm_b200.ops`. `exact` gives
the same outputs from the definitions in 64 bits."""
from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

DEV = "cuda"
DEAD = -(2 ** 31)        # code of a key that no row sees
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # attention, head width 128
        # one new token against one sequence's cache: the smallest call of a decoding loop
        dict(name="attn_token", op="attn", mask="step", seqs=1, new=1, cache=20001, heads=32, kv=8, cap=50.0, bias=False,
             back=False),
        # one denoising pass over a block of 32 tokens for each of four sequences, against their clean caches
        dict(name="attn_block_step", op="attn", mask="step", seqs=4, new=32, cache=8192, heads=32, kv=8, cap=50.0, bias=False,
             back=False),
        # a prompt whose first part is read in both directions; scores capped and biased by distance
        dict(name="attn_prefix_prompt", op="attn", mask="documents", rows=5000, docs=2, pad=0, prefix=0.3, heads=16, kv=8,
             cap=30.0, bias=True, back=False),
        # packed documents of odd lengths with padding behind the last one, distance bias, training
        dict(name="attn_train_documents", op="attn", mask="documents", rows=3001, docs=5, pad=37, prefix=0.0, heads=16, kv=8,
             cap=0.0, bias=True, back=True),
        # block-diffusion training rows (noisy and clean copy of 4096 tokens, blocks of 32), capped scores
        dict(name="attn_train_blocks", op="attn", mask="blocks", tokens=4096, block=32, heads=32, kv=8, cap=50.0, bias=False,
             back=True),
        # rotary positions
        # one decoding step of a batch of eight far into their contexts
        dict(name="rotary_step", op="rotary", rows=8, heads=40, dim=128, part=128, pairs="half", scaling="yarn", far=131072,
             dtype="bf16", back=False),
        # a long training row set, query and key heads inside the packed projection
        dict(name="rotary_train", op="rotary", rows=16384, heads=40, dim=128, part=128, pairs="half", scaling="yarn", far=16384,
             dtype="bf16", back=True),
        # part of each head, interleaved pairs, an odd row count, 32-bit values
        dict(name="rotary_part_interleaved", op="rotary", rows=3237, heads=12, dim=64, part=32, pairs="interleaved",
             scaling="linear", far=40000, dtype="fp32", back=True),
        # norms
        # the rows of one denoising block
        dict(name="norms_step", op="norms", rows=32, width=4096, gate="none", dtype="bf16", back=False),
        # training rows with a learned gate per channel
        dict(name="norms_train", op="norms", rows=16384, width=4096, gate="channel", dtype="bf16", back=True),
        # an odd width and row count, a gate for every value
        dict(name="norms_odd", op="norms", rows=2999, width=1411, gate="full", dtype="fp16", back=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attn", "attn", "attn", "rotary", "norms"])
    if op == "attn":
        kv = rng.choice([1, 2, 4, 8])
        heads = kv * rng.choice([1, 2, 3, 4])
        form = dict(heads=heads, kv=kv)
        form["cap"], form["bias"] = rng.choice([(50.0, False), (30.0, True), (0.0, True), (15.0, False)])
        kind = rng.choice(["step", "step", "documents", "documents", "blocks"])
        if kind == "step":
            seqs, new = rng.randint(1, 6), rng.choice([1, 1, 4, 16, 17, 32])
            return dict(op=op, mask=kind, seqs=seqs, new=new, cache=_log_int(rng, 1, 32000) // seqs + 1, back=False, **form)
        if kind == "documents":
            rows, back = _log_int(rng, 64, 5000), rng.random() < 0.6
            return dict(op=op, mask=kind, rows=rows, docs=rng.randint(1, 7), pad=rng.choice([0, 0, rng.randint(1, 60)]),
                        prefix=rng.choice([0.0, 0.0, round(rng.uniform(0.05, 0.9), 2)]), back=back, **form)
        block = rng.choice([8, 16, 32, 64])
        return dict(op=op, mask=kind, tokens=block * max(1, _log_int(rng, 64, 3000) // block), block=block, back=True, **form)
    if op == "rotary":
        dim = rng.choice([32, 64, 96, 128, 256])
        part = rng.choice([dim, dim, dim // 2, 3 * dim // 4])
        return dict(op=op, rows=_log_int(rng, 1, 8000), heads=rng.randint(1, 40), dim=dim, part=part,
                    pairs=rng.choice(["half", "interleaved"]), scaling=rng.choice(["none", "linear", "ntk", "llama3", "yarn"]),
                    far=_log_int(rng, 64, 1000000), dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]), back=rng.random() < 0.6)
    return dict(op=op, rows=_log_int(rng, 1, 9000), width=rng.choice([_log_int(rng, 64, 2900), 256 * rng.randint(1, 11), 4096, 5120]),
                gate=rng.choice(["none", "channel", "full"]), dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]),
                back=rng.random() < 0.6)


# ------------------------------------------------------------------------------------------------ masks
def _cuts(rows, parts, salt=0):
    """`parts` lengths that sum to `rows`, a length of zero now and then among them."""
    r = random.Random(1000003 * rows + 101 * parts + salt)
    at = sorted(r.randint(0, rows) for _ in range(parts - 1))
    return [b - a for a, b in zip([0] + at, at + [rows])]


def _mask(c):
    """Arrays of int64: q_lo, q_hi, q_grp of every query row, k_code of every key, and both sides' positions. A key of
    code >= 0 is seen where q_lo <= code < q_hi, a key of code < 0 where code == q_grp."""
    if c["mask"] == "step":
        # keys: per sequence its clean cache; then the new rows of all sequences, which see each other inside one sequence
        s, n, m, span = c["seqs"], c["new"], c["cache"], 1 << 24
        seq_k, pos_k = np.repeat(np.arange(s), m), np.tile(np.arange(m), s)
        seq_q, pos_q = np.repeat(np.arange(s), n), np.tile(np.arange(m, m + n), s)
        return (seq_q * span, seq_q * span + m, -(seq_q + 1), np.concatenate([seq_k * span + pos_k, -(seq_q + 1)]), pos_q,
                np.concatenate([pos_k, pos_q]))
    if c["mask"] == "documents":
        rows = c["rows"]
        pad = min(c["pad"], rows - 1)
        lens = _cuts(rows - pad, c["docs"])
        start = np.repeat(np.cumsum([0] + lens[:-1]), lens)
        first = np.repeat([int(math.ceil(c["prefix"] * n)) for n in lens], lens)
        at = np.arange(rows - pad)
        z = np.zeros(pad, dtype=np.int64)
        lo, hi = np.concatenate([start, z]), np.concatenate([np.maximum(at + 1, start + first), z])
        code = np.concatenate([at, z + DEAD])
        pos = np.concatenate([at - start, z])
        return lo, hi, np.zeros(rows, dtype=np.int64), code, pos, pos
    t, b = c["tokens"], c["block"]
    p = np.arange(t)
    blk = p // b
    lo = np.zeros(2 * t, dtype=np.int64)
    hi = np.concatenate([blk * b, (blk + 1) * b])
    grp = np.concatenate([-(blk + 1), np.zeros(t, dtype=np.int64)])
    return lo, hi, grp, np.concatenate([-(blk + 1), p]), np.concatenate([p, p]), np.concatenate([p, p])


def _pairs(c):
    lo, hi, grp, code, _, _ = _mask(c)
    clean = np.sort(code[code >= 0])
    noisy = np.sort(code[(code < 0) & (code != DEAD)])
    n = (np.searchsorted(clean, hi, "left") - np.searchsorted(clean, lo, "left")).clip(min=0)
    m = np.searchsorted(noisy, grp, "right") - np.searchsorted(noisy, grp, "left")
    return int(n.sum() + m.sum()), len(lo), len(code)


# ------------------------------------------------------------------------------------------------ states
def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed) * 7919 + 13)
    return g


def _randn(g, *shape, dtype=torch.float32, gain=1.0):
    return (torch.randn(*shape, generator=g, device=DEV) * gain).to(dtype)


def prepare(case, seed):
    c, g = case, _gen(seed)
    if c["op"] == "attn":
        H, K, D = c["heads"], c["kv"], 128
        mask = [torch.from_numpy(np.ascontiguousarray(a)).to(DEV).to(torch.int32) for a in _mask(c)]
        nq, nk = mask[0].numel(), mask[3].numel()
        s = dict(case=c, mask=mask, scale=1.0 / math.sqrt(D))
        if nq == nk:
            # self-attention reads the three parts of one packed projection
            rows = _randn(g, nq, (H + 2 * K) * D, dtype=torch.bfloat16, gain=1.4)
            s["q"] = rows[:, :H * D].view(nq, H, D)
            s["k"] = rows[:, H * D:(H + K) * D].view(nk, K, D)
            s["v"] = rows[:, (H + K) * D:].view(nk, K, D)
        else:
            s["q"] = _randn(g, nq, H, D, dtype=torch.bfloat16, gain=1.4)
            s["k"] = _randn(g, nk, K, D, dtype=torch.bfloat16, gain=1.4)
            s["v"] = _randn(g, nk, K, D, dtype=torch.bfloat16)
        s["slopes"] = torch.exp2(-8.0 * (torch.arange(H, device=DEV) + 1) / H).float() if c["bias"] else None
        if c["back"]:
            s["grad"] = _randn(g, nq, H, D, dtype=torch.bfloat16)
        if own:
            # the plan that a program keeps for a row layout
            from turbo_dllm_b200.ops.attention import MaskLayout
            from turbo_dllm_b200.ops.scored_attention import ScoreTransform

            s["layout"] = MaskLayout(*mask[:4])
            s["transform"] = ScoreTransform(softcap=c["cap"], slopes=s["slopes"], q_pos=mask[4] if c["bias"] else None,
                                            k_pos=mask[5] if c["bias"] else None)
        return s
    dt = DTYPES[c["dtype"]]
    if c["op"] == "rotary":
        R, H, D = c["rows"], c["heads"], c["dim"]
        # query and key heads lie in front of the value heads of a packed projection
        packed = _randn(g, R, (H + 2) * D, dtype=dt)
        freqs, scale = _frequencies(c)
        s = dict(case=c, x=packed[:, :H * D].view(R, H, D), scale=scale, freqs=torch.tensor(freqs, device=DEV).float(),
                 pos=torch.randint(0, c["far"], (R,), generator=g, device=DEV, dtype=torch.int32))
        if c["back"]:
            s["grad"] = _randn(g, R, H, D, dtype=dt)
        return s
    R, W = c["rows"], c["width"]
    s = dict(case=c, x=_randn(g, R, W, dtype=dt, gain=0.7), res=_randn(g, R, W, dtype=dt, gain=1.5),
             w_post=(1 + 0.2 * _randn(g, W)).to(dt), w_pre=(1 + 0.2 * _randn(g, W)).to(dt), gate=None, res_scale=0.9, eps=1e-6)
    if c["gate"] != "none":
        s["gate"] = _randn(g, *((W,) if c["gate"] == "channel" else (R, W)), dtype=dt, gain=0.8)
    if c["back"]:
        s["dy"], s["dh"] = _randn(g, R, W, dtype=dt), _randn(g, R, W, dtype=dt)
    return s


def _frequencies(c):
    """Inverse frequencies of the rotated pairs and the factor of cosine and sine, theta 1e6; a context of 8192
    stretched by 16 where the case scales."""
    n, theta, factor, old = c["part"], 1.0e6, 16.0, 8192
    base = [theta ** (-2.0 * i / n) for i in range(n // 2)]
    kind = c["scaling"]
    if kind == "linear":
        return [f / factor for f in base], 1.0
    if kind == "ntk":
        t = theta * factor ** (n / (n - 2))
        return [t ** (-2.0 * i / n) for i in range(n // 2)], 1.0
    if kind == "llama3":
        out = []
        for f in base:
            turns = old * f / (2 * math.pi)      # turns of the pair over the old context; kept above 4, divided below 1
            mix = min(1.0, max(0.0, (turns - 1.0) / (4.0 - 1.0)))
            out.append(f * (mix + (1 - mix) / factor))
        return out, 1.0
    if kind == "yarn":
        def at(turns):
            return n * math.log(old / (turns * 2 * math.pi)) / (2 * math.log(theta))

        lo, hi = max(math.floor(at(32.0)), 0), min(math.ceil(at(1.0)), n - 1)
        out = []
        for i, f in enumerate(base):
            ramp = min(1.0, max(0.0, (i - lo) / max(hi - lo, 1e-3)))
            out.append(f * ((1 - ramp) + ramp / factor))
        return out, 0.1 * math.log(factor) + 1.0
    return base, 1.0


# ------------------------------------------------------------------------------------------------ plain forms
def _seen(mask):
    lo, hi, grp, code = (m.long() for m in mask[:4])
    a = (code[None] >= 0) & (code[None] >= lo[:, None]) & (code[None] < hi[:, None])
    return a | ((code[None] < 0) & (code[None] == grp[:, None]))


def _plain_attn(s):
    c = s["case"]
    H, K = c["heads"], c["kv"]
    G = H // K
    q, k, v = (s[n].float() for n in "qkv")
    nq, D = q.shape[0], q.shape[2]
    q4 = q.view(nq, K, G, D).permute(1, 2, 0, 3)                          # [K, G, nq, D]
    k4, v4 = k.permute(1, 0, 2)[:, None], v.permute(1, 0, 2)[:, None]     # [K, 1, nk, D]
    z = (q4 @ k4.transpose(-1, -2)) * s["scale"]
    t = None
    if c["cap"]:
        t = torch.tanh(z / c["cap"])
        z = t * c["cap"]
    if c["bias"]:
        far = (s["mask"][4][:, None] - s["mask"][5][None]).abs().float()
        z = z - s["slopes"].view(K, G, 1, 1) * far
    seen = _seen(s["mask"])
    z = z.masked_fill(~seen, -math.inf)
    top = z.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    p = torch.exp(z - top)
    del z
    total = p.sum(-1, keepdim=True)
    lse = torch.where(total > 0, top + torch.log(total), torch.full_like(top, -math.inf))
    p = p / torch.where(total > 0, total, torch.ones_like(total))
    o = p @ v4
    rows = lambda x: x.permute(2, 0, 1, 3).reshape(nq, H, D)              # noqa: E731
    out = {"out": rows(o).to(s["q"].dtype), "lse": lse.reshape(H, nq)}
    if c["back"]:
        do = s["grad"].float().view(nq, K, G, D).permute(1, 2, 0, 3)
        dv = (p.transpose(-1, -2) @ do).sum(1)
        dz = do @ v4.transpose(-1, -2)
        dz = p * (dz - (do * o).sum(-1, keepdim=True))
        del p
        if t is not None:
            dz = dz * (1 - t * t)
        dz = dz * s["scale"]
        out["dq"] = rows(dz @ k4).to(s["q"].dtype)
        out["dk"] = (dz.transpose(-1, -2) @ q4).sum(1).permute(1, 0, 2).to(s["q"].dtype)
        out["dv"] = dv.permute(1, 0, 2).to(s["q"].dtype)
    return out


def _turn(x, cos, sin, n, pairs):
    """x [R, H, D] in 32 bits: its first n values of each head turned in pairs."""
    r, rest = x[..., :n], x[..., n:]
    if pairs == "half":
        a, b = r[..., :n // 2], r[..., n // 2:]
        r = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
    else:
        a, b = r[..., 0::2], r[..., 1::2]
        r = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).reshape(r.shape)
    return torch.cat([r, rest], dim=-1)


def _plain_rotary(s):
    c = s["case"]
    ang = s["pos"].double()[:, None, None] * s["freqs"].double()
    cos, sin = (torch.cos(ang) * s["scale"]).float(), (torch.sin(ang) * s["scale"]).float()
    out = {"out": _turn(s["x"].float(), cos, sin, c["part"], c["pairs"]).to(s["x"].dtype)}
    if c["back"]:
        out["dx"] = _turn(s["grad"].float(), cos, -sin, c["part"], c["pairs"]).to(s["x"].dtype)
    return out


def _plain_norms(s):
    c = s["case"]
    names = ["x", "res", "w_post", "w_pre"] + (["gate"] if s["gate"] is not None else [])
    f = {n: s[n].float().requires_grad_(c["back"]) for n in names}
    with torch.set_grad_enabled(c["back"]):
        x = f["x"]
        b = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + s["eps"]) * f["w_post"]
        if "gate" in f:
            b = b * f["gate"]
        h = s["res_scale"] * f["res"] + b
        y = h * torch.rsqrt((h * h).mean(-1, keepdim=True) + s["eps"]) * f["w_pre"]
    out = {"y": y.detach().to(s["x"].dtype), "h": h.detach().to(s["x"].dtype)}
    if c["back"]:
        got = torch.autograd.grad([y, h], [f[n] for n in names], [s["dy"].float(), s["dh"].float()])
        out.update({"d_" + n: d.to(s[n].dtype) for n, d in zip(names, got)})
    return out


# ------------------------------------------------------------------------------------------------ the framework's calls
def _own_attn(s):
    from turbo_dllm_b200.ops.scored_attention import scored_attention

    if not s["case"]["back"]:
        with torch.no_grad():
            out, lse = scored_attention(s["q"], s["k"], s["v"], s["layout"], s["transform"], scale=s["scale"], return_lse=True)
        return {"out": out, "lse": lse}
    q, k, v = (s[n].detach().requires_grad_() for n in "qkv")
    out, lse = scored_attention(q, k, v, s["layout"], s["transform"], scale=s["scale"], return_lse=True)
    dq, dk, dv = torch.autograd.grad(out, [q, k, v], s["grad"])
    return {"out": out.detach(), "lse": lse, "dq": dq, "dk": dk, "dv": dv}


def _own_rotary(s):
    from turbo_dllm_b200.ops.rotary import rotary

    c = s["case"]
    if not c["back"]:
        with torch.no_grad():
            return {"out": rotary(s["x"], s["pos"], s["freqs"], pairs=c["pairs"], scale=s["scale"])}
    x = s["x"].detach().requires_grad_()
    out = rotary(x, s["pos"], s["freqs"], pairs=c["pairs"], scale=s["scale"])
    (dx,) = torch.autograd.grad(out, [x], s["grad"])
    return {"out": out.detach(), "dx": dx}


def _own_norms(s):
    from turbo_dllm_b200.ops.norm import sandwich_norm

    more = dict(gate=s["gate"], res_scale=s["res_scale"], eps=s["eps"])
    if not s["case"]["back"]:
        with torch.no_grad():
            y, h = sandwich_norm(s["x"], s["res"], s["w_post"], s["w_pre"], **more)
        return {"y": y, "h": h}
    names = ["x", "res", "w_post", "w_pre"] + (["gate"] if s["gate"] is not None else [])
    f = {n: s[n].detach().requires_grad_() for n in names}
    more["gate"] = f.get("gate")
    y, h = sandwich_norm(f["x"], f["res"], f["w_post"], f["w_pre"], **more)
    got = torch.autograd.grad([y, h], [f[n] for n in names], [s["dy"], s["dh"]])
    return {"y": y.detach(), "h": h.detach(), **{"d_" + n: d for n, d in zip(names, got)}}


def run(state):
    op = state["case"]["op"]
    if own:
        return {"attn": _own_attn, "rotary": _own_rotary, "norms": _own_norms}[op](state)
    return {"attn": _plain_attn, "rotary": _plain_rotary, "norms": _plain_norms}[op](state)


# ------------------------------------------------------------------------------------------------ work
def work(case):
    c = case
    if c["op"] == "attn":
        pairs, nq, nk = _pairs(c)
        H, K, D = c["heads"], c["kv"], 128
        q, kv, lse = 2 * nq * H * D, 2 * 2 * nk * K * D, 4 * H * nq
        masks = 4 * (3 * nq + nk) + (4 * (nq + nk + H) if c["bias"] else 0)
        b, f = 2 * q + kv + lse + masks, 4 * pairs * D * H
        if c["back"]:
            b, f = b + 2 * q + kv, f + 10 * pairs * D * H        # reads the output's gradient, writes three gradients
        return {"bytes": b, "flops": f}
    size = torch.empty(0, dtype=DTYPES[c["dtype"]]).element_size()
    if c["op"] == "rotary":
        n = c["rows"] * c["heads"] * c["dim"]
        times = 2 if c["back"] else 1
        return {"bytes": times * 2 * n * size + 4 * c["rows"] + 2 * c["part"],
                "flops": times * 3 * c["rows"] * c["heads"] * c["part"]}
    n, w = c["rows"] * c["width"], c["width"]
    gate = {"none": 0, "channel": w, "full": n}[c["gate"]]
    b, f = size * (4 * n + 2 * w + gate), 10 * n
    if c["back"]:
        b, f = b + size * (4 * n + 2 * w + gate), f + 24 * n     # both gradients in, both inputs' and the weights' out
    return {"bytes": b, "flops": f}


# ------------------------------------------------------------------------------------------------ 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"attn": _exact_attn, "rotary": _exact_rotary, "norms": _exact_norms}[case["op"]](s)


def _exact_attn(s):
    """Head by head: softmax over the visible keys, gradients by automatic differentiation."""
    c = s["case"]
    H, G = c["heads"], c["heads"] // c["kv"]
    q, k, v = (s[n].detach().double() for n in "qkv")
    seen = _seen(s["mask"])
    none = ~seen.any(1)
    far = (s["mask"][4].double()[:, None] - s["mask"][5].double()[None]).abs() if c["bias"] else None
    out = {"out": torch.zeros_like(q), "lse": torch.zeros(H, q.shape[0], dtype=torch.float64, device=q.device)}
    if c["back"]:
        out.update(dq=torch.zeros_like(q), dk=torch.zeros_like(k), dv=torch.zeros_like(v))
    for h in range(H):
        leaves = [q[:, h].clone(), k[:, h // G].clone(), v[:, h // G].clone()]
        for x in leaves:
            x.requires_grad_(c["back"])
        with torch.set_grad_enabled(c["back"]):
            z = (leaves[0] @ leaves[1].t()) * s["scale"]
            if c["cap"]:
                z = c["cap"] * torch.tanh(z / c["cap"])
            if far is not None:
                z = z - s["slopes"][h].double() * far
            # rows that see no key keep finite scores here and are taken out behind the product
            z = torch.where(seen | none[:, None], z, torch.full_like(z, -math.inf))
            o = torch.where(none[:, None], torch.zeros_like(leaves[0]), torch.softmax(z, -1) @ leaves[2])
        out["out"][:, h] = o.detach()
        out["lse"][h] = torch.where(none, torch.full_like(z[:, 0], -math.inf), torch.logsumexp(z, -1)).detach()
        if c["back"]:
            d = torch.autograd.grad(o, leaves, s["grad"][:, h].double())
            out["dq"][:, h] = d[0]
            out["dk"][:, h // G] += d[1]
            out["dv"][:, h // G] += d[2]
        del z, o
    return out


def _exact_rotary(s):
    c = s["case"]
    n = c["part"]
    spin = torch.polar(torch.full((c["rows"], n // 2), float(s["scale"]), dtype=torch.float64, device=DEV),
                       torch.outer(s["pos"].double(), s["freqs"].double()))[:, None]

    def turned(x, by):
        x = x.double()
        r = x[..., :n].reshape(*x.shape[:2], *((2, n // 2) if c["pairs"] == "half" else (n // 2, 2)))
        r = r.transpose(-1, -2) if c["pairs"] == "half" else r
        r = torch.view_as_real(torch.view_as_complex(r.contiguous()) * by)
        r = r.transpose(-1, -2) if c["pairs"] == "half" else r
        return torch.cat([r.reshape(*x.shape[:2], n), x[..., n:]], dim=-1)

    out = {"out": turned(s["x"], spin)}
    if c["back"]:
        out["dx"] = turned(s["grad"], spin.conj())
    return out


def _exact_norms(s):
    """The gradients from the formulas: with u = x / rms(x), the pull-back of u is (d - u mean(d u)) / rms(x)."""
    x, res, wq, wp = (s[n].double() for n in ("x", "res", "w_post", "w_pre"))
    g = torch.ones((), dtype=torch.float64, device=DEV) if s["gate"] is None else s["gate"].double()
    rx = (x.square().mean(-1, keepdim=True) + s["eps"]).sqrt()
    u = x / rx
    h = s["res_scale"] * res + g * (u * wq)
    rh = (h.square().mean(-1, keepdim=True) + s["eps"]).sqrt()
    t = h / rh
    out = {"y": t * wp, "h": h}
    if s["case"]["back"]:
        dy, dh = s["dy"].double(), s["dh"].double()
        dt = dy * wp
        d = dh + (dt - t * (dt * t).mean(-1, keepdim=True)) / rh
        du = d * g * wq
        out["d_x"] = (du - u * (du * u).mean(-1, keepdim=True)) / rx
        out["d_res"] = s["res_scale"] * d
        out["d_w_post"] = (d * g * u).sum(0)
        out["d_w_pre"] = (dy * t).sum(0)
        if s["gate"] is not None:
            dg = d * u * wq
            out["d_gate"] = dg.sum(0) if s["gate"].dim() == 1 else dg
    return out
