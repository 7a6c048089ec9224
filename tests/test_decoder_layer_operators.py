"""Rotary, scored attention and the sandwich norm together, as a decoder layer has them: packed documents in training, a
prompt and then single tokens against a cache in serving."""
import pytest
import torch

from turbo_dllm_b200.kernels.native import NativeKernelError
from turbo_dllm_b200.ops.norm import sandwich_norm, sandwich_norm_reference
from turbo_dllm_b200.ops.rotary import RotaryScaling, rotary, rotary_frequencies, rotary_reference
from turbo_dllm_b200.ops.scored_attention import (ScoreTransform, document_layout, document_positions, scored_attention,
                                                  scored_attention_reference)

HQ, HKV, D, WIDTH, INNER, CAP, RES = 4, 2, 128, 320, 448, 20.0, 0.8


def weights(dtype, device, seed=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)   # noqa: E731
    w = dict(qkv=r((HQ + 2 * HKV) * D, WIDTH) / WIDTH ** 0.5, out=r(WIDTH, HQ * D) / (HQ * D) ** 0.5,
             up=r(INNER, WIDTH) / WIDTH ** 0.5, down=r(WIDTH, INNER) / INNER ** 0.5, gate=0.5 + 0.1 * r(WIDTH),
             **{n: 1 + 0.1 * r(WIDTH) for n in ("first", "post1", "pre1", "post2", "pre2")})
    return {n: t.to(dtype).to(device) for n, t in w.items()}


OWN = (rotary, scored_attention, sandwich_norm)
PLAIN = (rotary_reference, lambda q, k, v, layout, t: scored_attention_reference(q, k, v, layout, t)[0],
         lambda x, res, a, b, gate, res_scale: sandwich_norm_reference(x, res, a, b, gate, res_scale))


def layer(w, h, pos, layout, transform, freqs, ops, cache=None):
    """One layer on residual rows h: (the next layer's input, the residual stream). `cache` = (k, v, rows held so far)."""
    turn, attend, norms = ops
    y = torch.nn.functional.rms_norm(h, (WIDTH,), w["first"], 1e-6)
    qkv = (y @ w["qkv"].T).view(-1, HQ + 2 * HKV, D)
    q, k, v = qkv[:, :HQ], qkv[:, HQ: HQ + HKV], qkv[:, HQ + HKV:]
    q, k = turn(q, pos, freqs), turn(k, pos, freqs)
    if cache is not None:
        kc, vc, at = cache
        kc[at: at + k.shape[0]] = k
        vc[at: at + k.shape[0]] = v
        k, v = kc, vc
    a = attend(q, k, v, layout, transform).flatten(1) @ w["out"].T
    y, h = norms(a, h, w["post1"], w["pre1"], gate=w["gate"], res_scale=RES)
    f = torch.nn.functional.silu(y @ w["up"].T) @ w["down"].T
    return norms(f, h, w["post2"], w["pre2"], gate=w["gate"], res_scale=RES)


def frequencies(device):
    return rotary_frequencies(D, 10000.0, RotaryScaling("yarn", 4.0, 64))[0].to(device)


def served(w, h, device, prompt, room, ops=OWN):
    """The rows of h through a prompt and then single tokens, against a cache of `room` rows."""
    freqs = frequencies(device)
    slopes = torch.tensor([2.0 ** -i for i in range(1, HQ + 1)], device=device)
    n = h.shape[0]
    kc, vc = (torch.zeros(room, HKV, D, dtype=h.dtype, device=device) for _ in range(2))
    whole = document_layout([n], rows=room, device=device)
    places = torch.arange(room, dtype=torch.int32, device=device)
    out = []
    for at, m in [(0, prompt)] + [(i, 1) for i in range(prompt, n)]:
        rows = slice(at, at + m)
        layout = type(whole)(whole.q_lo[rows], whole.q_hi[rows], whole.q_grp[rows], whole.k_code)
        t = ScoreTransform(CAP, slopes, places[rows], places)
        with torch.no_grad():
            out.append(torch.cat(layer(w, h[rows], places[rows].long(), layout, t, freqs, ops, (kc, vc, at)), 1))
    return torch.cat(out)


def whole(w, h, device, lens, ops=OWN):
    """All rows at once, documents packed."""
    slopes = torch.tensor([2.0 ** -i for i in range(1, HQ + 1)], device=device)
    n = h.shape[0]
    pos = document_positions(lens, rows=n, device=device)
    t = ScoreTransform(CAP, slopes, pos, pos)
    return torch.cat(layer(w, h, pos.long(), document_layout(lens, rows=n, device=device), t, frequencies(device), ops), 1)


def far(got, want):
    return float((got.detach().double() - want).norm() / want.norm())


def test_serving_matches_the_whole_sequence():
    w = weights(torch.float64, "cpu")
    h = torch.randn(9, WIDTH, dtype=torch.float64, generator=torch.Generator().manual_seed(1))
    # 64 bits; positions are at most 8, so angles and distances are exact to 2^-45 and better
    assert far(served(w, h, "cpu", 5, 16), whole(w, h, "cpu", [9])) < 2.0 ** -40


def test_gradients_match_differences():
    w = weights(torch.float64, "cpu")
    h = torch.randn(7, WIDTH, dtype=torch.float64, generator=torch.Generator().manual_seed(2)).requires_grad_()
    to = torch.randn(7, 2 * WIDTH, dtype=torch.float64, generator=torch.Generator().manual_seed(3))
    loss = lambda t: (whole(w, t, "cpu", [4, 3]) * to).sum()   # noqa: E731
    grad, = torch.autograd.grad(loss(h), h)
    step = torch.randn(h.shape, dtype=torch.float64, generator=torch.Generator().manual_seed(4))
    e = 2.0 ** -17     # (the difference's own error: e^2 of the value by the third derivative, 2^-52 / e by rounding)
    with torch.no_grad():
        diff = float(loss(h + e * step) - loss(h - e * step)) / (2 * e)
    assert abs(diff - float((grad * step).sum())) <= 2.0 ** -20 * float((grad * step).abs().sum())


def grads(ops, dtype, w, h, to, lens):
    w = {n: t.to(dtype).requires_grad_() for n, t in w.items()}
    h = h.to(dtype).requires_grad_()
    out = whole(w, h, "cuda", lens, ops)
    got = torch.autograd.grad((out * to.to(dtype)).sum(), [h, *w.values()])
    return [out, *got]


@pytest.mark.gpu
@pytest.mark.parametrize("lens,rows", [([300, 1, 77, 0, 200], 600), ([129], 129), ([1], 1)])
def test_training_is_as_exact_as_the_plain_layer(lens, rows):
    """Both chains round to bf16 at the same places (the operators' own form at fewer), so against 64 bits the kernels'
    error is at most the plain chain's up to scatter; that of a norm over WIDTH or more values is a few per cent, and 1.25
    leaves room for it. A single row has attention weights of exactly 1, whose true gradient by the scores is 0: q's and
    k's rows of the projection's gradient are rounding alone there, so that its norm is v's."""
    w = weights(torch.bfloat16, "cuda")
    g = torch.Generator(device="cuda").manual_seed(5)
    h = torch.randn(rows, WIDTH, generator=g, device="cuda").bfloat16()
    to = torch.randn(rows, 2 * WIDTH, generator=g, device="cuda").bfloat16()
    exact = grads(PLAIN, torch.float64, w, h, to, lens)
    plain = grads(PLAIN, torch.bfloat16, w, h, to, lens)
    own = grads(OWN, torch.bfloat16, w, h, to, lens)
    for name, e, p, o in zip(["out", "h", *w], exact, plain, own):
        assert o.dtype == torch.bfloat16
        assert far(o, e.detach()) <= 1.25 * far(p, e.detach()) + 2.0 ** -10, (name, far(o, e.detach()), far(p, e.detach()))


@pytest.mark.gpu
def test_serving_on_the_gpu():
    """Prompt and single tokens (the few-row form) are as exact as the plain layer over the whole sequence."""
    w = weights(torch.bfloat16, "cuda")
    h = torch.randn(300, WIDTH, generator=torch.Generator(device="cuda").manual_seed(6), device="cuda").bfloat16()
    exact = whole({n: t.double() for n, t in w.items()}, h.double(), "cuda", [300], PLAIN)
    plain = whole(w, h, "cuda", [300], PLAIN)
    for prompt in (296, 100):
        got = served(w, h, "cuda", prompt, 333)
        for rows in (slice(0, prompt), slice(prompt, 300)):
            assert far(got[rows], exact[rows]) <= 1.25 * far(plain[rows], exact[rows])


@pytest.mark.gpu
def test_a_training_step_in_a_graph():
    """Forward and backward captured, replayed on other rows: the eager step's results. dQ's sums run in another order, so
    what depends on them agrees to a step of the type; the rest has the same bits."""
    lens, rows = [200, 130], 333
    w = {n: t.requires_grad_() for n, t in weights(torch.bfloat16, "cuda").items()}
    g = torch.Generator(device="cuda").manual_seed(7)
    data = [torch.randn(rows, WIDTH, generator=g, device="cuda").bfloat16() for _ in range(2)]
    to = torch.randn(rows, 2 * WIDTH, generator=g, device="cuda").bfloat16()
    h = data[0].clone().requires_grad_()
    slopes = torch.tensor([0.5, 0.25, 0.125, 0.0625], device="cuda")
    pos = document_positions(lens, rows=rows, device="cuda")
    t, layout, freqs, far_pos = ScoreTransform(CAP, slopes, pos, pos), document_layout(lens, rows=rows, device="cuda"), \
        frequencies("cuda"), pos.long()

    def step():
        out = torch.cat(layer(w, h, far_pos, layout, t, freqs, OWN), 1)
        return [out.detach(), *torch.autograd.grad(out, [h, *w.values()], to)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for rows_in in reversed(data):
        with torch.no_grad():
            h.copy_(rows_in)
        graph.replay()
        replayed = [x.clone() for x in held]
        eager = step()
        assert torch.equal(replayed[0], eager[0])
        for name, a, b in zip(["h", *w], replayed[1:], eager[1:]):
            if name in ("h", "qkv", "first"):
                assert far(a, b.double()) <= 2.0 ** -8, name
            else:
                assert torch.equal(a, b), name


@pytest.mark.gpu
@pytest.mark.parametrize("which", ["rotary", "attention", "norm"])
def test_a_second_differentiation_is_refused(which):
    x = torch.randn(4, 1, 128, device="cuda").bfloat16().requires_grad_()
    if which == "rotary":
        out = rotary(x, torch.arange(4, device="cuda"), frequencies("cuda"))
    elif which == "attention":
        out = scored_attention(x, x, x, document_layout([4], device="cuda"), ScoreTransform(5.0))
    else:
        out = sandwich_norm(x, x, *torch.ones(2, 128, device="cuda").bfloat16())[0]
    with pytest.raises(RuntimeError, match="twice"):
        torch.autograd.grad(out.float().square().sum(), x, create_graph=True)


@pytest.mark.gpu
def test_the_split_backward_is_refused(monkeypatch):
    monkeypatch.setenv("TDLLM_ATTN_BWD", "split")
    x = torch.randn(4, 1, 128, device="cuda").bfloat16().requires_grad_()
    layout = document_layout([4], device="cuda")
    with pytest.raises(NativeKernelError, match="TDLLM_ATTN_BWD"):
        scored_attention(x, x, x, layout)
    with torch.no_grad():
        assert scored_attention(x, x, x, layout).shape == x.shape


def test_tangents_are_refused_where_kernels_run_and_nowhere_else():
    from torch.autograd import forward_ad

    from turbo_dllm_b200.ops._util import refuse_tangents

    x, t = torch.randn(4, 1, 128), torch.randn(4, 1, 128)
    freqs = frequencies("cpu")
    refuse_tangents("this", x)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, t)
        refuse_tangents("this", x, None)
        with pytest.raises(NotImplementedError, match="this has no forward-mode"):
            refuse_tangents("this", x, None, dual)
        # (the reference, which the CPU takes, has the derivative: the rotation is linear)
        turned = forward_ad.unpack_dual(rotary(dual, torch.arange(4), freqs)).tangent
    assert torch.equal(turned, rotary(t, torch.arange(4), freqs))


@pytest.mark.gpu
@pytest.mark.parametrize("which", ["rotary", "attention", "norm"])
def test_tangents_are_refused_on_the_gpu(which):
    from torch.autograd import forward_ad

    x = torch.randn(4, 1, 128, device="cuda").bfloat16()
    w, freqs, pos = torch.ones(128, device="cuda").bfloat16(), frequencies("cuda"), torch.arange(4, device="cuda")
    L = document_layout([4], device="cuda")
    call, places = {"rotary": (lambda t: rotary(t[0], pos, freqs), 1),
                    "attention": (lambda t: scored_attention(*t, L, ScoreTransform(5.0)), 3),
                    "norm": (lambda t: sandwich_norm(t[0], t[1], w, w, gate=t[2]), 3)}[which]
    with forward_ad.dual_level():
        call([x] * 3)
        for at in range(places):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call([forward_ad.make_dual(x, x) if i == at else x for i in range(3)])
