"""Rotary positions: frequencies, refusals and the reference on the CPU, the kernel against 64 bits on the GPU."""
import math

import pytest
import torch

from turbo_dllm_b200.ops.rotary import RotaryScaling, rotary, rotary_frequencies, rotary_reference


def exact(x, pos, freqs, pairs, scale, back=False):
    """Complex product in 64 bits."""
    n = 2 * freqs.shape[0]
    spin = torch.polar(torch.full((len(pos), n // 2), float(scale), dtype=torch.float64, device=x.device),
                       torch.outer(pos.double(), freqs.double()))[:, None]
    r = x[..., :n].double().unflatten(-1, (2, n // 2) if pairs == "half" else (n // 2, 2))
    r = r.transpose(-1, -2) if pairs == "half" else r
    r = torch.view_as_real(torch.view_as_complex(r.contiguous()) * (spin.conj() if back else spin))
    r = r.transpose(-1, -2) if pairs == "half" else r
    return torch.cat([r.flatten(-2), x[..., n:].double()], dim=-1)


def check(got, x, want, n):
    """Half a step of the type for the stored result, and 2^-22 of the pair's length for 32-bit cosines and products:
    the angle's rest is rounded to 2^-25 half turns, cosine, sine, two products and a sum add a few 2^-24 each."""
    half = torch.finfo(x.dtype).eps / 2
    pairmag = x[..., :n].double().abs().amax() * 2 + 1e-30
    err = (got.double() - want).abs()
    assert bool((err[..., :n] <= half * want[..., :n].abs() + 2.0 ** -21 * pairmag + torch.finfo(x.dtype).tiny).all()), float(err.max())
    assert torch.equal(got[..., n:], x[..., n:])


# ------------------------------------------------------------------------------------------------ CPU
def test_frequencies():
    f, s = rotary_frequencies(64, 1e4)
    assert s == 1.0 and torch.allclose(f.double(), 1e4 ** (-torch.arange(0, 64, 2).double() / 64))
    lin, _ = rotary_frequencies(64, 1e4, RotaryScaling("linear", 4.0))
    assert torch.allclose(lin * 4, f)
    ntk, _ = rotary_frequencies(64, 1e4, RotaryScaling("ntk", 4.0))
    assert ntk[0] == f[0] and abs(float(f[-1] / ntk[-1]) - 4.0) < 1e-5
    l3, _ = rotary_frequencies(128, 5e5, RotaryScaling("llama3", 8.0, 8192, 1.0, 4.0))
    base, _ = rotary_frequencies(128, 5e5)
    turns = 8192 * base.double() / (2 * math.pi)
    assert torch.equal(l3[turns >= 4], base[turns >= 4]) and torch.allclose(l3[turns <= 1] * 8, base[turns <= 1])
    assert bool((l3 <= base).all()) and bool((l3 * 8 >= base * (1 - 1e-6)).all())
    y, s = rotary_frequencies(128, 1e6, RotaryScaling("yarn", 16.0, 8192))
    base, _ = rotary_frequencies(128, 1e6)
    assert abs(s - (0.1 * math.log(16) + 1)) < 1e-12 and y[0] == base[0] and abs(float(base[-1] / y[-1]) - 16) < 1e-4
    assert rotary_frequencies(128, 1e6, RotaryScaling("yarn", 16.0, attention_factor=1.0))[1] == 1.0
    assert rotary_frequencies(2, 1e4, RotaryScaling("ntk", 4.0))[0].tolist() == [1.0]


@pytest.mark.parametrize("pairs", ["half", "interleaved"])
def test_reference(pairs):
    torch.manual_seed(0)
    f, _ = rotary_frequencies(6, 1e4)
    x = torch.randn(4, 3, 10, dtype=torch.float64, requires_grad=True)
    pos = torch.tensor([0, 5, 1 << 20, -3])
    check(rotary(x, pos, f, pairs=pairs, scale=1.3).detach(), x.detach(), exact(x.detach(), pos, f, pairs, 1.3), 6)
    assert torch.autograd.gradcheck(lambda t: rotary(t, pos, f, pairs=pairs, scale=1.3), [x])


def test_half_pairs_match_the_fused_operator():
    from turbo_dllm_b200.ops.rope import qk_norm_rope_reference, rope_inv_freq

    torch.manual_seed(0)
    x, pos, inv = torch.randn(5, 4 * 16), torch.arange(5), rope_inv_freq(16, 1e4)
    want = qk_norm_rope_reference(x, pos, inv, None, None, 2, 1, 16, 1e-6)[:, :48]
    got = rotary(x.view(5, 4, 16)[:, :3], pos, inv).reshape(5, 48)
    assert torch.allclose(got, want, atol=1e-6)


def test_refusals():
    f, _ = rotary_frequencies(8, 1e4)
    x, pos = torch.zeros(3, 2, 8), torch.arange(3)
    for kw, match in ((dict(kind="other", factor=2.0), "linear"), (dict(kind="ntk", factor=0.5), "factor"),
                      (dict(kind="linear", factor=float("nan")), "factor"), (dict(kind="ntk", factor=2.0, original_length=0), "length"),
                      (dict(kind="llama3", factor=2.0, low_freq_factor=4.0), "low"), (dict(kind="yarn", factor=2.0, beta_slow=40.0), "beta")):
        with pytest.raises(ValueError, match=match):
            RotaryScaling(**kw)
    for part in (0, 7):
        with pytest.raises(ValueError, match="even"):
            rotary_frequencies(part, 1e4)
    with pytest.raises(ValueError, match="position per row"):
        rotary(x, pos[:2], f)
    with pytest.raises(ValueError, match="int32"):
        rotary(x, pos.float(), f)
    with pytest.raises(ValueError, match="float32 vector"):
        rotary(x[..., :6], pos, f)
    with pytest.raises(ValueError, match="float32 vector"):
        rotary(x, pos, f.double())
    with pytest.raises(ValueError, match="pairs"):
        rotary(x, pos, f, pairs="quarter")


@pytest.mark.parametrize("device", ["meta", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_more_rows_than_32_bits_count_are_refused(device):
    x, pos = torch.zeros(1, 1, 2, device=device).expand(2 ** 31 + 5, 1, 2), torch.zeros(1, dtype=torch.int32, device=device)
    with pytest.raises(ValueError, match="rows"):
        rotary(x, pos.expand(2 ** 31 + 5), torch.ones(1, device=device))


def test_frequencies_that_want_a_gradient_are_refused():
    f = rotary_frequencies(8, 1e4)[0].requires_grad_()
    x, pos = torch.randn(3, 2, 8), torch.arange(3)
    with pytest.raises(ValueError, match="no gradient"):
        rotary(x, pos, f)
    with torch.no_grad():
        assert torch.equal(rotary(x, pos, f), rotary(x, pos, f.detach()))


# ------------------------------------------------------------------------------------------------ GPU
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("pairs", ["half", "interleaved"])
@pytest.mark.parametrize("rows,H,D,part", [(1, 1, 2, 2), (7, 3, 33, 32), (65, 5, 128, 128), (130, 2, 96, 72), (9, 40, 64, 32),
                                           (17, 1, 256, 256), (3, 2, 31, 10)])
def test_kernel(dtype, pairs, rows, H, D, part):
    g = torch.Generator(device="cuda").manual_seed(rows * D)
    x = torch.randn(rows, H, D, generator=g, device="cuda").to(dtype).requires_grad_()
    pos = torch.randint(-1000, 1 << 20, (rows,), generator=g, device="cuda", dtype=torch.int32)
    pos[-1] = 2 ** 31 - 1
    f, s = rotary_frequencies(part, 1e6, RotaryScaling("yarn", 8.0), device="cuda")
    out = rotary(x, pos, f, pairs=pairs, scale=s)
    check(out.detach(), x.detach(), exact(x.detach(), pos, f, pairs, s), part)
    do = torch.randn(out.shape, generator=g, device="cuda").to(dtype)
    (dx,) = torch.autograd.grad(out, [x], do)
    check(dx, do, exact(do, pos, f, pairs, s, back=True), part)


@pytest.mark.gpu
@pytest.mark.parametrize("pairs", ["half", "interleaved"])
def test_strides_and_positions_of_64_bits(pairs):
    g = torch.Generator(device="cuda").manual_seed(0)
    packed = torch.randn(50, 6 * 64 + 1, generator=g, device="cuda").bfloat16()
    f, _ = rotary_frequencies(64, 1e4, device="cuda")
    pos = torch.arange(50, device="cuda")
    views = [packed[:, :5 * 64].view(50, 5, 64), packed[:, 1:5 * 64 + 1].unflatten(1, (5, 64)), packed[::2, 64:5 * 64].unflatten(1, (4, 64)),
             packed[:, :384].reshape(50, 64, 6).transpose(1, 2)]
    for x in views:
        p = pos[: x.shape[0]]
        got = rotary(x, p, f, pairs=pairs)
        check(got, x, exact(x, p, f, pairs, 1.0), 64)
        assert torch.equal(got, rotary(x.contiguous(), p.int(), f, pairs=pairs))
    x = views[0].detach().requires_grad_()
    (dx,) = torch.autograd.grad(rotary(x, pos, f, pairs=pairs), [x], torch.ones((), device="cuda", dtype=x.dtype).expand(x.shape))
    one = torch.ones_like(x)
    check(dx, one, exact(one, pos, f, pairs, 1.0, back=True), 64)
    assert rotary(x[:0], pos[:0], f).shape == (0, 5, 64)
    assert rotary_reference(x.detach().double(), pos, f).dtype == torch.float64


@pytest.mark.gpu
def test_graph_replay_with_new_positions():
    f, _ = rotary_frequencies(64, 1e4, device="cuda")
    x, pos = torch.randn(8, 4, 64, device="cuda").bfloat16(), torch.arange(8, device="cuda", dtype=torch.int32)
    rotary(x, pos, f)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = rotary(x, pos, f)
    pos += 100000
    graph.replay()
    assert torch.equal(held, rotary(x, pos, f))
