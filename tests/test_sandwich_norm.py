"""The norms around a block: refusals and the reference on the CPU, the kernels against 64 bits on the GPU."""
import pytest
import torch

from turbo_dllm_b200.ops.norm import rmsnorm_reference, sandwich_norm

EPS = 1e-6
FINE = 2.0 ** -18    # 32-bit arithmetic: a row sum adds up to 16 values per thread and ten tree levels at 2^-24 each
SUMS = 2.0 ** -15    # sums over rows: up to 400 sequential 32-bit additions


def exact(x, res, wq, wp, gate, a, dy=None, dh=None):
    """Outputs and gradients in 64 bits with the error each may have: half a step of the type on what is stored, FINE
    (SUMS) of the summed magnitudes."""
    half = torch.finfo(x.dtype).eps / 2
    x, res, wq, wp = (t.detach().double() for t in (x, res, wq, wp))
    gate = torch.ones((), dtype=torch.float64, device=x.device) if gate is None else gate.detach().double()
    mean = lambda t: t.mean(-1, keepdim=True)   # noqa: E731
    rx = (mean(x * x) + EPS).sqrt()
    u = x / rx
    b = gate * u * wq
    h = a * res + b
    size = (a * res).abs() + b.abs()
    rh = (mean(h * h) + EPS).sqrt()
    t = h / rh
    tsize = size / rh * (1 + mean(size * size) / (rh * rh))
    want = {"y": t * wp, "h": h}
    tol = {"y": half * want["y"].abs() + FINE * tsize * wp.abs(), "h": half * h.abs() + FINE * size}
    if dy is not None or dh is not None:
        dy = torch.zeros_like(x) if dy is None else dy.detach().double()
        dh = torch.zeros_like(x) if dh is None else dh.detach().double()
        dt = dy * wp
        d = dh + (dt - t * mean(dt * t)) / rh
        dsize = dh.abs() + (dt.abs() + tsize * mean(dt.abs() * tsize)) / rh
        gw = gate * wq
        du = d * gw
        want["x"] = (du - u * mean(du * u)) / rx
        tol["x"] = half * want["x"].abs() + FINE * (dsize * gw.abs() + u.abs() * mean(dsize * gw.abs() * u.abs())) / rx
        want["res"] = a * d
        tol["res"] = half * want["res"].abs() + FINE * abs(a) * dsize
        for n, term, mag in (("w_post", d * gate * u, dsize * gate.abs() * u.abs()), ("w_pre", dy * t, dy.abs() * tsize),
                             ("gate", d * u * wq, dsize * u.abs() * wq.abs())):
            if n == "gate" and gate.dim() == 2:
                want[n], tol[n] = term, half * term.abs() + FINE * mag
            else:
                want[n] = term.sum(0)
                tol[n] = half * want[n].abs() + SUMS * mag.sum(0)
    return want, tol


def near(got, want, tol, name):
    tiny = torch.finfo(got.dtype).tiny
    over = (got.detach().double() - want).abs() - tol - tiny
    assert over.numel() == 0 or float(over.max()) <= 0, (name, float(over.max()))


def operands(rows, H, gate, dtype, device, seed=0):
    g = torch.Generator(device=device).manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device=device)   # noqa: E731
    out = dict(x=(0.7 * r(rows, H)).to(dtype), res=(1.5 * r(rows, H)).to(dtype), w_post=(1 + 0.2 * r(H)).to(dtype),
               w_pre=(1 + 0.2 * r(H)).to(dtype))
    if gate:
        out["gate"] = r(*((H,) if gate == "channel" else (rows, H))).to(dtype)
    return out, r(rows, H).to(dtype), r(rows, H).to(dtype)


def run(t, dy, dh, a=0.9):
    leaves = {n: v.detach().requires_grad_() for n, v in t.items()}
    y, h = sandwich_norm(leaves["x"], leaves["res"], leaves["w_post"], leaves["w_pre"], gate=leaves.get("gate"), res_scale=a, eps=EPS)
    outs, grads = zip(*[(o, g) for o, g in ((y, dy), (h, dh)) if g is not None])
    got = dict(zip(leaves, torch.autograd.grad(outs, list(leaves.values()), grads, allow_unused=True)))
    got = {n: torch.zeros_like(leaves[n]) if g is None else g for n, g in got.items()}
    return {"y": y, "h": h, **got}


# ------------------------------------------------------------------------------------------------ CPU
@pytest.mark.parametrize("gate", [None, "channel", "full"])
def test_reference(gate):
    t, dy, dh = operands(5, 7, gate, torch.float64, "cpu")
    want, _ = exact(t["x"], t["res"], t["w_post"], t["w_pre"], t.get("gate"), 0.9, dy, dh)
    got = run(t, dy, dh)
    for n in got:
        assert torch.allclose(got[n], want[n], rtol=1e-10, atol=1e-12), n
    leaves = [v.requires_grad_() for v in t.values()]
    assert torch.autograd.gradcheck(lambda *v: sandwich_norm(*v[:4], gate=v[4] if gate else None, res_scale=0.9), leaves)


def test_it_is_two_norms():
    t, _, _ = operands(3, 8, None, torch.float32, "cpu")
    y, h = sandwich_norm(t["x"].view(3, 1, 8), t["res"].view(3, 1, 8), t["w_post"], t["w_pre"])
    want = t["res"] + rmsnorm_reference(t["x"], t["w_post"], EPS)[0]
    assert y.shape == (3, 1, 8) and torch.allclose(h.view(3, 8), want)
    assert torch.allclose(y.view(3, 8), rmsnorm_reference(want, t["w_pre"], EPS)[0], atol=1e-6)


def test_refusals():
    t, _, _ = operands(3, 8, None, torch.float32, "cpu")
    x, res, wq, wp = t.values()
    with pytest.raises(ValueError, match="one shape"):
        sandwich_norm(x, res[:2], wq, wp)
    with pytest.raises(ValueError, match="vectors"):
        sandwich_norm(x, res, wq[:7], wp)
    with pytest.raises(ValueError, match="gate"):
        sandwich_norm(x, res, wq, wp, gate=x[:1])
    with pytest.raises(ValueError, match="share"):
        sandwich_norm(x, res, wq.double(), wp)
    with pytest.raises(ValueError, match="one shape"):
        sandwich_norm(x[:, :0], res[:, :0], wq[:0], wp[:0])


@pytest.mark.parametrize("device", ["meta", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_more_rows_than_32_bits_count_are_refused(device):
    x, w = torch.zeros(1, 2, device=device).expand(2 ** 31 + 5, 2), torch.zeros(2, device=device)
    with pytest.raises(ValueError, match="rows"):
        sandwich_norm(x, x, w, w)


# ------------------------------------------------------------------------------------------------ GPU
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("gate", [None, "channel", "full"])
@pytest.mark.parametrize("rows,H", [(1, 1), (3, 7), (5, 256), (33, 1000), (700, 1411), (2, 4096), (601, 4104), (3, 16384), (1300, 96),
                                    (2, 16383)])
def test_kernels(dtype, gate, rows, H):
    t, dy, dh = operands(rows, H, gate, dtype, "cuda", rows + H)
    want, tol = exact(t["x"], t["res"], t["w_post"], t["w_pre"], t.get("gate"), 0.9, dy, dh)
    got = run(t, dy, dh)
    for n in got:
        near(got[n], want[n], tol[n], n)
    again = run(t, dy, dh)
    assert all(torch.equal(got[n], again[n]) for n in got)      # sums in a fixed order
    y, h = sandwich_norm(t["x"], t["res"], t["w_post"], t["w_pre"], gate=t.get("gate"), res_scale=0.9, eps=EPS)
    assert torch.equal(y, got["y"]) and torch.equal(h, got["h"])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("gate", [None, "full"])
@pytest.mark.parametrize("H", [1, 2, 3, 5, 9])
@pytest.mark.parametrize("rows", [20001, 20004, 20008])
def test_many_rows_of_a_few_values(dtype, gate, H, rows):
    """Several rows to a line of 16 bytes, more rows than blocks, ends of the tensors at every place in a line."""
    t, dy, dh = operands(rows, H, gate, dtype, "cuda", rows + H)
    got = run(t, dy, dh)
    part = slice(rows - 300, rows)
    less = {n: v[part] if v.dim() == 2 else v for n, v in t.items()}
    want, tol = exact(less["x"], less["res"], less["w_post"], less["w_pre"], less.get("gate"), 0.9, dy[part], dh[part])
    for n in ("y", "h", "x", "res") + (("gate",) if gate else ()):
        near(got[n][part], want[n], tol[n], n)


@pytest.mark.gpu
def test_rows_that_overlap_or_repeat():
    g = torch.Generator(device="cuda").manual_seed(3)
    for H, ld in ((16, 0), (16, 8), (12, 4), (9, 1), (7, 0)):
        rows = 4000
        flat = torch.randn(rows * max(ld, 1) + H, generator=g, device="cuda").bfloat16()
        x = flat.as_strided((rows, H), (ld, 1))
        w = torch.ones(H, dtype=torch.bfloat16, device="cuda")
        for a, b in zip(sandwich_norm(x, x, w, w), sandwich_norm(x.contiguous(), x.contiguous(), w, w)):
            assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("which", ["dy", "dh"])
@pytest.mark.parametrize("gate", [None, "full"])
def test_one_incoming_gradient(which, gate):
    t, dy, dh = operands(40, 512, gate, torch.bfloat16, "cuda")
    dy, dh = (dy, None) if which == "dy" else (None, dh)
    want, tol = exact(t["x"], t["res"], t["w_post"], t["w_pre"], t.get("gate"), 0.9, dy, dh)
    got = run(t, dy, dh)
    for n in got:
        near(got[n], want[n], tol[n], n)


@pytest.mark.gpu
def test_strides_and_empty_rows():
    t, dy, dh = operands(30, 256, "full", torch.bfloat16, "cuda")
    base = run(t, dy, dh)
    wide = torch.zeros(30, 3 * 256 + 1, dtype=torch.bfloat16, device="cuda")
    views = {n: wide[:, i * 256 + 1:(i + 1) * 256 + 1] for i, n in enumerate(("x", "res", "gate"))}
    for n, v in views.items():
        v.copy_(t[n])
    # (a base that is not 16-byte aligned goes value by value: other sums, the same bounds)
    want, tol = exact(t["x"], t["res"], t["w_post"], t["w_pre"], t["gate"], 0.9, dy, dh)
    for n, got in run({**t, **views}, dy, dh).items():
        near(got, want[n], tol[n], n)
    turned = {**t, "x": t["x"].t().contiguous().t()}
    assert torch.equal(run(turned, dy, dh)["y"], base["y"])
    none = {n: v[:0] if v.dim() == 2 else v for n, v in t.items()}
    got = run(none, dy[:0], dh[:0])
    assert got["y"].shape == (0, 256) and float(got["w_post"].abs().max()) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,H", [(torch.bfloat16, 4096), (torch.float16, 264), (torch.float32, 516), (torch.bfloat16, 12288)])
@pytest.mark.parametrize("gate", [None, "channel", "full"])
@pytest.mark.parametrize("off", [1, 3])
@pytest.mark.parametrize("rows", [40, 4000])
def test_weights_that_start_anywhere(dtype, H, gate, off, rows):
    """Vectors that are slices of a flat buffer, `off` values behind a 16-byte boundary, with and without more rows than blocks."""
    rows = min(rows, (1 << 24) // H)
    t, dy, dh = operands(rows, H, gate, dtype, "cuda", rows + H)
    want, tol = exact(t["x"], t["res"], t["w_post"], t["w_pre"], t.get("gate"), 0.9, dy, dh)
    for n in ("w_post", "w_pre", "gate"):
        if n in t and t[n].dim() == 1:
            flat = torch.full((H + 16,), float("nan"), dtype=dtype, device="cuda")
            flat[off: off + H] = t[n]
            t[n] = flat[off: off + H]
            assert t[n].is_contiguous() and t[n].data_ptr() % 16
    got = run(t, dy, dh)
    for n in got:
        near(got[n], want[n], tol[n], n)
    y, h = sandwich_norm(t["x"], t["res"], t["w_post"], t["w_pre"], gate=t.get("gate"), res_scale=0.9, eps=EPS)
    assert torch.equal(y, got["y"]) and torch.equal(h, got["h"])


@pytest.mark.gpu
def test_gradients_go_to_the_flat_buffers():
    t, dy, dh = operands(60, 512, "channel", torch.bfloat16, "cuda")
    plain = run(t, dy, dh)
    for sink_type in (torch.float32, torch.bfloat16):
        leaves = {n: v.detach().requires_grad_() for n, v in t.items()}
        for n in ("w_post", "w_pre", "gate"):
            leaves[n].main_grad = torch.full((512,), 7.0, dtype=sink_type, device="cuda")
            leaves[n].grad_acc = False
        for step in (1, 2):
            y, h = sandwich_norm(leaves["x"], leaves["res"], leaves["w_post"], leaves["w_pre"], gate=leaves["gate"], res_scale=0.9, eps=EPS)
            torch.autograd.backward([y, h], [dy, dh])
            for n in ("w_post", "w_pre", "gate"):
                assert leaves[n].grad is None and leaves[n].grad_acc
                # (two roundings to bf16 apart: the plain result's and, for the second step, the buffer's)
                assert torch.allclose(leaves[n].main_grad.float(), step * plain[n].float(), rtol=2.0 ** -6, atol=2.0 ** -8), (n, step)
    # one parameter in all three places
    w = t["w_post"].detach().requires_grad_()
    w.main_grad, w.grad_acc = torch.full((512,), 7.0, device="cuda"), False
    same = run({**t, "w_post": w.detach(), "w_pre": w.detach(), "gate": w.detach()}, dy, dh)
    y, h = sandwich_norm(t["x"], t["res"], w, w, gate=w, res_scale=0.9, eps=EPS)
    torch.autograd.backward([y, h], [dy, dh])
    total = sum(same[n].double() for n in ("w_post", "w_pre", "gate"))
    size = sum(same[n].double().abs() for n in ("w_post", "w_pre", "gate"))
    # (the separate gradients come rounded to bf16, the buffer holds 32 bits)
    assert bool(((w.main_grad.double() - total).abs() <= 2.0 ** -8 * size + 2.0 ** -20).all())
    from turbo_dllm_b200.kernels.native import NativeKernelError

    leaves["w_post"].main_grad = torch.zeros(512, dtype=torch.float16, device="cuda")
    y, h = sandwich_norm(leaves["x"], leaves["res"], leaves["w_post"], leaves["w_pre"])
    with pytest.raises(NativeKernelError, match="gradient buffer"):
        y.sum().backward()
    x = torch.zeros(1, 16385, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(NativeKernelError, match="widths"):
        sandwich_norm(x, x, x[0], x[0])


@pytest.mark.gpu
def test_threads_with_rows_of_different_widths():
    """Widths of one kernel that need different amounts of shared memory, launched from several threads at once."""
    import threading

    cases = [operands(600, H, "full", torch.bfloat16, "cuda", H) for H in (4096, 4608, 5120, 6144)]
    want = [run(*c) for c in cases]
    torch.cuda.synchronize()
    wrong = []

    def work(mine, expected):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(60):
                    y, h = sandwich_norm(mine["x"], mine["res"], mine["w_post"], mine["w_pre"], gate=mine["gate"], res_scale=0.9, eps=EPS)
                torch.cuda.current_stream().synchronize()
                wrong.extend([] if torch.equal(y, expected["y"]) and torch.equal(h, expected["h"]) else ["result"])
        except Exception as e:   # noqa: BLE001 (a thread's exception is not pytest's)
            wrong.append(repr(e))

    threads = [threading.Thread(target=work, args=(c[0], w)) for c, w in zip(cases, want)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


@pytest.mark.gpu
@pytest.mark.parametrize("gate", [None, "full"])
@pytest.mark.parametrize("rows,H", [(4000, 4096), (3000, 136), (3000, 1411)])
def test_a_recorded_error_of_another_kernel(rows, H, gate):
    """While it stands, waits give up at once; the rows' own copies still land, and the results are right."""
    from turbo_dllm_b200.kernels import native

    t, dy, dh = operands(rows, H, gate, torch.bfloat16, "cuda", 6)
    want = run(t, dy, dh)
    lib = native.lib()
    native.check(lib.tdllm_set_wait_timeout_ns(2_000_000), "set timeout")
    try:
        native.check(lib.tdllm_test_wait_timeout(None), "launch")      # (a wait that nobody ends records an error)
        during = [run(t, dy, dh) for _ in range(3)]
        torch.cuda.synchronize()
        err = native.device_error()
        assert err["code"] == 1 and err["kernel"] == 99
    finally:
        lib.tdllm_clear_error()
        lib.tdllm_set_wait_timeout_ns(2_000_000_000)
    for got in (*during, run(t, dy, dh)):
        assert all(torch.equal(got[n], want[n]) for n in want)
    native.raise_on_device_error()


@pytest.mark.gpu
def test_two_captured_graphs_side_by_side():
    t, dy, dh = operands(300, 512, None, torch.bfloat16, "cuda")
    u, ey, eh = operands(300, 512, None, torch.bfloat16, "cuda", seed=5)
    want = [run(t, dy, dh), run(u, ey, eh)]
    torch.cuda.synchronize()
    graphs, held = [], []
    for args in ((t, dy, dh), (u, ey, eh)):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            held.append(run(*args))
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for h, w in zip(held, want):
        assert all(torch.equal(h[n], w[n]) for n in w)
