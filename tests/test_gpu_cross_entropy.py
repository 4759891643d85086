"""Cross entropy over a vocabulary matrix (stored, or noise) on the GPU against a plain 64-bit implementation.

Tolerances.  bf16: the inputs' products are exact in float32, so a logit is off by float32 accumulation only: at most
2^-23 (R / 16 + 16) sum |x_i w_i| (the tensor core adds 16 products at a time, each addition may cut instead of round); the same
goes for the sum of exponentials.  A loss (or log-sum-exp) moves by at most the largest logit's error plus 2^-20 for the exponential and
the row's sum.  Gradients in bf16 carry two roundings, of the probability (2^-9 relative after averaging, 2^-8 at most) and of the
result (2^-8): 2^-7 of sum |p w| bounds the worst element; elements are compared with 2^-7 of that sum.
"""
import math

import pytest
import torch
import torch.nn.functional as F

from oracle import oracle as O

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def rb():
    import randumb_b200
    assert torch.cuda.is_available()
    return randumb_b200


def noise_matrix(V, R, seed, row0, dtype):
    return torch.from_numpy(O.noise_f32(V, R, seed, row0)).to(dtype)


def plain(x, w, target, ignore, reduction, gout):
    """Loss, dx, dw, logit and gradient error scales, in 64 bits on the GPU, from the definition; ignored rows are left out before anything is computed."""
    keep = torch.ones_like(target, dtype=torch.bool) if ignore is None else target != ignore
    rows = torch.nonzero(keep)[:, 0]
    xd, wd, t = x.double()[rows], w.double(), target[rows]
    logits = xd @ wd.t()
    lse = torch.logsumexp(logits, 1)
    l = lse - logits.gather(1, t[:, None])[:, 0]
    losses = torch.zeros(x.shape[0], dtype=torch.float64, device=x.device)
    losses[rows] = l
    n = rows.numel()
    if reduction == "none":
        loss, g = losses, gout.double()[rows]
    else:
        loss = losses.sum() / (1 if reduction == "sum" else n) if n else torch.tensor(0.0 if reduction == "sum" else float("nan"), dtype=torch.float64)
        g = torch.full((n,), float(gout) / (1 if reduction == "sum" else max(n, 1)), dtype=torch.float64, device=x.device)
    p = torch.softmax(logits, 1)
    # p - 1 at the target as the sum of the others: 1 - p itself is lost in 64 bits where p is nearly 1
    at = torch.arange(n, device=x.device)
    p[at, t] = 0
    p[at, t] = -p.sum(1)
    pa = p.abs()
    dx = torch.zeros(x.shape, dtype=torch.float64, device=x.device)
    dx[rows] = (p * g[:, None]) @ wd
    dxa = torch.zeros_like(dx)
    dxa[rows] = (pa * g.abs()[:, None]) @ wd.abs()
    dw = (p * g[:, None]).t() @ xd
    dwa = (pa * g.abs()[:, None]).t() @ xd.abs()
    terms = (xd.abs() @ wd.abs().t()).amax().item() if n else 0.0
    return loss, losses, dx, dxa, dw, dwa, terms


def tolerances(dtype, R, V, terms):
    """(absolute error of a logit and a loss, relative factor of a gradient on the sum of its terms' magnitudes)."""
    steps = (R / 16 + 16) * (1 if dtype == torch.bfloat16 else 6)
    logit = 2.0 ** -23 * steps * terms + 2.0 ** -19
    # exponent offset and argument in powers of two: 2 u of up to `terms` * log2(e), twice
    logit += 4 * 2.0 ** -24 * 1.5 * terms
    acc = 2.0 ** -23 * (V / 16 + 64) * (1 if dtype == torch.bfloat16 else 6)
    return logit, (2.0 ** -7 if dtype == torch.bfloat16 else 2.0 ** -22) + 3 * logit + acc


def inputs(kind, T, R, V, dtype, seed, std=2.0):
    g = torch.Generator().manual_seed(seed)
    if kind == "noise":
        w = noise_matrix(V, R, 1000 + seed, 5, dtype).cuda()
        x = (torch.randn(T, R, generator=g) * std * (3.0 / R) ** 0.5).to(dtype).cuda()
    else:
        w = (torch.randn(V, R, generator=g) * std / R ** 0.5).to(dtype).cuda()
        x = torch.randn(T, R, generator=g).to(dtype).cuda()
    target = torch.randint(0, V, (T,), generator=g).cuda()
    return x, w, target


def call(rb, kind, x, w, target, seed, ignore=-100, reduction="mean"):
    if kind == "noise":
        return rb.ops.noise_cross_entropy(x, 1000 + seed, w.shape[0], target, row0=5, ignore_index=ignore, reduction=reduction)
    return rb.ops.linear_cross_entropy(x, w, target, ignore_index=ignore, reduction=reduction)


def check(rb, kind, x, w, target, seed, ignore, reduction, gout=None):
    T, R = x.shape
    V = w.shape[0]
    if gout is None:
        gout = torch.rand(T, device="cuda") - 0.3 if reduction == "none" else torch.tensor(1.7, device="cuda")
    loss_w, losses, dx_w, dxa, dw_w, dwa, terms = plain(x, w, target, ignore, reduction, gout)
    xl = x.detach().clone().requires_grad_()
    wl = w.detach().clone().requires_grad_()
    loss = call(rb, kind, xl, wl, target, seed, ignore, reduction)
    assert loss.dtype == torch.float32 and loss.shape == ((T,) if reduction == "none" else ())
    grads = torch.autograd.grad(loss, [xl] if kind == "noise" else [xl, wl], gout)
    rb.kernels.check_status()
    logit, fac = tolerances(x.dtype, R, V, terms)
    scale = 1 if reduction != "sum" else max(1, int((target != ignore).sum()))
    assert torch.allclose(loss.double(), loss_w.to(loss.device), rtol=2.0 ** -21, atol=logit * scale, equal_nan=True), (loss, loss_w)
    assert ((grads[0].double() - dx_w).abs() <= fac * dxa + 1e-30).all(), ((grads[0].double() - dx_w).abs() / (dxa + 1e-30)).max()
    if kind == "linear":
        accT = 2.0 ** -23 * (T / 16 + 64) * 6
        assert ((grads[1].double() - dw_w).abs() <= (fac + accT) * dwa + 1e-30).all(), ((grads[1].double() - dw_w).abs() / (dwa + 1e-30)).max()
    # the loss alone, without autograd, is the same number
    with torch.no_grad():
        alone = call(rb, kind, x, w, target, seed, ignore, reduction)
    assert torch.allclose(alone, loss.detach(), rtol=2.0 ** -20, atol=2 * logit * scale, equal_nan=True)
    return loss, grads


SHAPES = [(1, 8, 1), (1, 128, 50257), (2, 1, 3), (3, 5, 300), (31, 64, 256), (128, 72, 257), (129, 256, 1000), (255, 250, 511), (257, 264, 513),
          (600, 40, 2049), (1000, 513, 777), (2048, 128, 4096), (2500, 136, 700)]


@pytest.mark.parametrize("kind", ["noise", "linear"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape", SHAPES)
def test_loss_and_gradients(rb, kind, dtype, shape):
    T, R, V = shape
    x, w, target = inputs(kind, T, R, V, dtype, T + R)
    check(rb, kind, x, w, target, T + R, -100, "mean")


@pytest.mark.parametrize("kind", ["noise", "linear"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("reduction", ["none", "mean", "sum"])
def test_ignored_rows_may_hold_anything(rb, kind, dtype, reduction):
    T, R, V, seed = 700, 96, 1111, 3
    x, w, target = inputs(kind, T, R, V, dtype, seed)
    skip = torch.rand(T, generator=torch.Generator().manual_seed(1)).cuda() < 0.45
    target[skip] = -7
    want, _ = check(rb, kind, x, w, target, seed, -7, reduction, torch.linspace(-1, 2, T, device="cuda") if reduction == "none" else None)
    dirty = x.clone()
    dirty[skip] = torch.tensor([float("nan"), float("inf"), -float("inf"), torch.finfo(dtype).max], device="cuda").to(dtype).repeat(R // 4)
    g = torch.linspace(-1, 2, T, device="cuda") if reduction == "none" else torch.tensor(1.7, device="cuda")
    both = []
    for xx in (x, dirty):
        leaves = [xx.clone().requires_grad_()] + ([w.clone().requires_grad_()] if kind == "linear" else [])
        loss = call(rb, kind, leaves[0], leaves[-1] if kind == "linear" else w, target, seed, -7, reduction)
        both.append([loss.detach()] + list(torch.autograd.grad(loss, leaves, g)))
    for a, b in zip(*both):
        assert torch.equal(a, b) and torch.isfinite(a).all()
    assert (both[1][1][skip] == 0).all()


@pytest.mark.parametrize("kind", ["noise", "linear"])
def test_no_row_counts(rb, kind):
    x, w, target = inputs(kind, 300, 64, 500, torch.bfloat16, 2)
    target[:] = -100
    for reduction in ("mean", "sum", "none"):
        leaves = [x.clone().requires_grad_(), w.clone().requires_grad_()]
        loss = call(rb, kind, *leaves, target, 2, -100, reduction)
        assert torch.isnan(loss) if reduction == "mean" else (loss == 0).all()
        for g in torch.autograd.grad(loss.sum(), leaves[:1 if kind == "noise" else 2]):
            assert (g == 0).all()
    # no rows at all
    for reduction in ("mean", "sum", "none"):
        leaves = [x[:0].clone().requires_grad_(), w.clone().requires_grad_()]
        loss = call(rb, kind, *leaves, target[:0], 2, -100, reduction)
        assert torch.isnan(loss) if reduction == "mean" else loss.sum() == 0
        grads = torch.autograd.grad(loss.sum(), leaves[:1 if kind == "noise" else 2])
        assert grads[0].shape == (0, 64) and all((g == 0).all() for g in grads)


@pytest.mark.parametrize("kind", ["noise", "linear"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape", [(300, 128, 900), (2500, 520, 600)])
def test_logits_far_above_the_target(rb, kind, dtype, shape):
    """Rows whose sum relative to the target's logit leaves float32 (other logits hundreds above it), beside ordinary rows and rows
    that the model knows almost for sure."""
    T, R, V = shape
    seed = 8
    x, w, target = inputs(kind, T, R, V, dtype, seed)
    far = torch.arange(0, T, 7, device="cuda")
    sure = torch.arange(3, T, 7, device="cuda")
    norm = (w.float() ** 2).sum(1, keepdim=True)
    x[far] = (w[(target[far] + 1) % V].float() / norm[(target[far] + 1) % V] * torch.linspace(60, 900, far.numel(), device="cuda")[:, None]).to(dtype)
    x[sure] = (w[target[sure]].float() / norm[target[sure]] * torch.linspace(15, 300, sure.numel(), device="cuda")[:, None]).to(dtype)
    loss, grads = check(rb, kind, x, w, target, seed, -100, "none", torch.ones(T, device="cuda"))
    assert loss[far].max() > 300 and loss[sure].min() < 1e-6


@pytest.mark.parametrize("kind", ["noise", "linear"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("std", [15.0, 40.0, 300.0])
def test_logits_of_large_scale(rb, kind, dtype, std):
    """Logits spread far wider than a trained model's: the largest lies 60, 150 or 1000 above the target's in an ordinary row."""
    T, R, V, seed = 400, 200, 3000, 12
    x, w, target = inputs(kind, T, R, V, dtype, seed, std)
    x[::50] *= 0.01
    loss, _ = check(rb, kind, x, w, target, seed, -100, "none", torch.ones(T, device="cuda"))
    assert loss.median() > 2 * std


def test_target_outside_the_vocabulary(rb):
    for kind in ("noise", "linear"):
        x, w, target = inputs(kind, 40, 32, 100, torch.bfloat16, 4)
        for bad in (100, -1, 2 ** 40, -2 ** 40):
            t = target.clone()
            t[17] = bad
            leaves = [x.clone().requires_grad_(), w.clone().requires_grad_()]
            loss = call(rb, kind, *leaves, t, 4, -100, "none")
            ok = torch.arange(40, device="cuda") != 17
            assert torch.isnan(loss[17]) and torch.isfinite(loss[ok]).all()
            dx = torch.autograd.grad(loss, leaves[0], torch.ones_like(loss))[0]
            assert torch.isnan(dx[17]).all() and torch.isfinite(dx[ok]).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_strided_and_misaligned_operands(rb, dtype):
    T, R, V, seed = 200, 100, 333, 6
    x, w, target = inputs("linear", T, R, V, dtype, seed)
    want = [t.clone() for t in _value(rb, x, w, target)]
    bx = torch.zeros(T, R + 13, device="cuda", dtype=dtype)
    bw = torch.zeros(V, R + 24, device="cuda", dtype=dtype)
    bx[:, 3:3 + R], bw[:, 8:8 + R] = x, w
    odd = torch.zeros(V * R + 1, device="cuda", dtype=dtype)[1:].view(V, R).copy_(w)
    for xx, ww in ((bx[:, 3:3 + R], w), (x, bw[:, 8:8 + R]), (x, odd), (x.t().contiguous().t(), w.t().contiguous().t())):
        for a, b in zip(_value(rb, xx, ww, target), want):
            assert torch.equal(a, b)
    # a target that is a slice of a wider matrix; leading dimensions
    wide = torch.zeros(T, 3, dtype=torch.int64, device="cuda")
    wide[:, 1] = target
    assert torch.equal(rb.linear_cross_entropy(x, w, wide[:, 1]), want[0])
    l3 = rb.linear_cross_entropy(x.view(4, 50, R), w, target.view(4, 50), reduction="none")
    assert l3.shape == (4, 50) and torch.equal(l3.reshape(-1), rb.linear_cross_entropy(x, w, target, reduction="none"))


def _value(rb, x, w, target):
    x, w = x.detach().requires_grad_(), w.detach().requires_grad_()
    loss = rb.linear_cross_entropy(x, w, target)
    return [loss.detach()] + list(torch.autograd.grad(loss, [x, w]))


def test_only_what_is_asked_for(rb):
    x, w, target = inputs("linear", 150, 64, 400, torch.bfloat16, 5)
    both = _value(rb, x, w, target)
    xl = x.clone().requires_grad_()
    assert torch.equal(torch.autograd.grad(rb.linear_cross_entropy(xl, w, target), xl)[0], both[1])
    wl = w.clone().requires_grad_()
    assert torch.equal(torch.autograd.grad(rb.linear_cross_entropy(x, wl, target), wl)[0], both[2])
    # twice through the same graph: the second gradient is the first
    xl = x.clone().requires_grad_()
    loss = call(rb, "noise", xl, w, target, 5)
    a = torch.autograd.grad(loss, xl, torch.tensor(3.0, device="cuda"), retain_graph=True)[0]
    b = torch.autograd.grad(loss, xl, torch.tensor(3.0, device="cuda"))[0]
    assert torch.equal(a, b)


@pytest.mark.parametrize("kind", ["noise", "linear"])
@pytest.mark.parametrize("T,R,V,dtype", [(40000, 64, 20000, torch.bfloat16), (30000, 250, 20000, torch.bfloat16), (20000, 36, 8100, torch.float32)])
def test_several_pieces_and_repeatability(rb, kind, T, R, V, dtype):
    """Enough rows that the vocabulary is taken in several pieces; the same call gives the same bits."""
    seed = 11
    g = torch.Generator(device="cuda").manual_seed(1)
    x = (torch.randn(T, R, device="cuda", generator=g) * (3.0 / R) ** 0.5 * 2).to(dtype)
    w = (noise_matrix(V, R, 1000 + seed, 5, dtype).cuda() if kind == "noise" else (torch.randn(V, R, device="cuda", generator=g) * 2 / R ** 0.5).to(dtype))
    target = torch.randint(0, V, (T,), device="cuda", generator=g)
    target[torch.rand(T, device="cuda", generator=g) < 0.2] = -100
    out = []
    for _ in range(2):
        leaves = [x.clone().requires_grad_(), w.clone().requires_grad_()]
        loss = call(rb, kind, *leaves, target, seed)
        out.append([loss.detach()] + list(torch.autograd.grad(loss, leaves[:1 if kind == "noise" else 2])))
    for a, b in zip(*out):
        assert torch.equal(a, b)
    xs, ws = x.float().requires_grad_(), w.float().requires_grad_()
    want = F.cross_entropy(xs @ ws.t(), target)
    gx, gw = torch.autograd.grad(want, [xs, ws])
    # norms: rounding errors of single elements average out; 2^-8 covers the two bf16 roundings; float32 either side's sums of up to 20000 terms
    tol = 2.0 ** -8 if dtype == torch.bfloat16 else 1e-5
    assert abs(out[0][0].item() / want.item() - 1) < 1e-5
    assert O.rel_fro(out[0][1].float().cpu(), gx.cpu()) < tol
    if kind == "linear":
        assert O.rel_fro(out[0][2].float().cpu(), gw.cpu()) < tol


def test_noise_in_several_pieces_without_a_gradient(rb):
    """The noise matrix is staged 256 MB at a time."""
    T, R, V = 70, 512, 300001
    x = (torch.randn(T, R, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3)) * (3.0 / R) ** 0.5 * 2).bfloat16()
    target = torch.randint(0, V, (T,), device="cuda")
    target[0], target[1] = V - 1, 262144                             # the last row; the first of the second piece
    S = rb.kernels.noise(V, R, 77, 9, 0, torch.bfloat16).float()
    want = F.cross_entropy(x.float() @ S.t(), target, reduction="none")
    got = rb.noise_cross_entropy(x, 77, V, target, row0=9, reduction="none")
    # float32 sums of 512 products either side, logits up to 10: 2^-23 * 48 * 30 at most
    assert (got - want).abs().max() < 2.0 ** -23 * 48 * 30

def test_gradient_is_the_slope(rb):
    """float32: the loss along a direction, by differences, against the gradient."""
    for kind in ("noise", "linear"):
        x, w, target = inputs(kind, 64, 40, 200, torch.float32, 9)
        xl, wl = x.clone().requires_grad_(), w.clone().requires_grad_()
        leaves = [xl] if kind == "noise" else [xl, wl]
        grads = torch.autograd.grad(call(rb, kind, xl, wl, target, 9, reduction="sum"), leaves)
        for i, (leaf, gr) in enumerate(zip(leaves, grads)):
            d = gr / gr.norm()
            h = 0.05
            with torch.no_grad():
                f = [call(rb, kind, x + s * h * d if i == 0 else x, w + s * h * d if i == 1 else w, target, 9, reduction="sum").double().item() for s in (-1, 1)]
            # third derivatives of the sum along a unit direction stay below its second's scale: h^2 / 6 of them is under 1 %; losses of 64 rows
            # are off by 64 * 2e-6 each: 64 * 4e-6 / (2 h) / |g|
            assert abs((f[1] - f[0]) / (2 * h) / gr.norm().item() - 1) < 0.01 + 64 * 4e-6 / (2 * h) / gr.norm().item()


def test_captured_and_on_a_side_stream(rb):
    for kind in ("noise", "linear"):
        x, w, target = inputs(kind, 500, 128, 3001, torch.bfloat16, 7)
        xl, wl = x.clone().requires_grad_(), w.clone().requires_grad_()
        leaves = [xl] if kind == "noise" else [xl, wl]
        st = torch.cuda.Stream()
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            loss = call(rb, kind, xl, wl, target, 7)
            eager = [loss.detach()] + list(torch.autograd.grad(loss, leaves))
        torch.cuda.synchronize()
        del loss
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            loss = call(rb, kind, xl, wl, target, 7)
            out = [loss.detach()] + list(torch.autograd.grad(loss, leaves))
        del loss
        x2, _, target2 = inputs(kind, 500, 128, 3001, torch.bfloat16, 70)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, eager))
        with torch.no_grad():
            xl.copy_(x2)
        target2[100:300] = -100
        target.copy_(target2)
        graph.replay()
        torch.cuda.synchronize()
        xn = x2.clone().requires_grad_()
        wn = w.clone().requires_grad_()
        fresh = call(rb, kind, xn, wn, target2, 7)
        want = [fresh.detach()] + list(torch.autograd.grad(fresh, [xn] if kind == "noise" else [xn, wn]))
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_capture_as_the_first_call_of_a_process():
    """Forward and backward captured before the library has been used: nothing in a first call may disturb a capture."""
    import os
    import subprocess
    import sys
    code = """
import torch, randumb_b200 as rb
x = torch.randn(70, 64, device="cuda").bfloat16().requires_grad_()
w = torch.randn(300, 64, device="cuda").bfloat16().requires_grad_()
t = torch.randint(0, 300, (70,), device="cuda")
rb.kernels.status_buffer(x.device)
st = torch.cuda.Stream()
st.wait_stream(torch.cuda.current_stream())
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g, stream=st):
    out = [rb.linear_cross_entropy(x, w, t), *torch.autograd.grad(rb.linear_cross_entropy(x, w, t), [x, w]),
           *torch.autograd.grad(rb.noise_cross_entropy(x, 5, 300, t), x)]
g.replay()
torch.cuda.synchronize()
want = [rb.linear_cross_entropy(x, w, t), *torch.autograd.grad(rb.linear_cross_entropy(x, w, t), [x, w]),
        *torch.autograd.grad(rb.noise_cross_entropy(x, 5, 300, t), x)]
assert all(torch.equal(a, b) for a, b in zip(out, want))
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", code], cwd=root, env=dict(os.environ, PYTHONPATH=root), capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]


def test_one_row_of_a_strided_matrix(rb):
    x, w, target = inputs("linear", 1, 128, 50, torch.bfloat16, 1)
    wide = torch.zeros(1, 256, device="cuda", dtype=torch.bfloat16)
    wide[:, ::2] = x
    assert torch.equal(rb.linear_cross_entropy(wide[:, ::2], w, target), rb.linear_cross_entropy(x, w, target))
    one = w[:1].clone()
    widew = torch.zeros(1, 256, device="cuda", dtype=torch.bfloat16)
    widew[:, ::2] = one
    z = torch.zeros(1, dtype=torch.int64, device="cuda")
    assert rb.linear_cross_entropy(x, widew[:, ::2], z).item() == 0.0


def test_two_streams_at_once(rb):
    """Two calls whose kernels may run side by side give what they give alone."""
    sets = [inputs("linear", 900, 128, 5003, torch.bfloat16, s) for s in (1, 2)]
    alone = [_value(rb, *s) for s in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(5):
        for st, s, out in zip(streams, sets, outs):
            with torch.cuda.stream(st):
                out.append(_value(rb, *s))
    torch.cuda.synchronize()
    for a, out in zip(alone, outs):
        for o in out:
            assert all(torch.equal(x, y) for x, y in zip(a, o))


# up to four rows without a gradient have a kernel of their own; 3004 (four rows) and 12028 (one) are the widest that take it
@pytest.mark.parametrize("kind", ["noise", "linear"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,R,V", [(1, 1, 1), (1, 3, 2), (2, 31, 5), (3, 33, 1000), (4, 250, 511), (4, 513, 40003), (5, 64, 300), (4, 3004, 70), (4, 3005, 70),
                                   (1, 12028, 90), (1, 12029, 90)])
@pytest.mark.parametrize("std", [2.0, 40.0, 300.0])
def test_a_few_rows(rb, kind, dtype, T, R, V, std):
    x, w, target = inputs(kind, T, R, V, dtype, T + R, std)
    _, losses, _, _, _, _, terms = plain(x, w, target, None, "none", torch.ones(T, device="cuda"))
    logit, _ = tolerances(dtype, R, V, terms)
    for reduction, want in (("none", losses), ("mean", losses.mean()), ("sum", losses.sum())):
        with torch.no_grad():
            got = call(rb, kind, x, w, target, T + R, None, reduction)
            again = call(rb, kind, x, w, target, T + R, None, reduction)
        assert torch.equal(got, again)
        assert torch.allclose(got.double(), want, rtol=2.0 ** -21, atol=logit * (T if reduction == "sum" else 1)), (got, want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_few_rows_ignored_strided_and_infinite(rb, dtype):
    g = torch.Generator().manual_seed(5)
    wide = torch.randn(700, 131, generator=g).to(dtype).cuda()
    x = torch.randn(4, 140, generator=g).to(dtype).cuda()[:, 3:132]
    for w in (wide[:, 1:130], wide[:, :129]):
        target = torch.tensor([5, -100, 699, -100]).cuda()
        with torch.no_grad():
            want = torch.nn.functional.cross_entropy(x.double() @ w.double().t(), target, reduction="none")
            terms = (x.double().abs() @ w.double().abs().t()).max().item()
            bad = x.clone()
            bad[1], bad[3, 0] = float("nan"), float("inf")
            for xx in (x, bad):
                got = rb.ops.linear_cross_entropy(xx, w, target, reduction="none")
                assert torch.allclose(got.double(), want, rtol=2.0 ** -21, atol=tolerances(dtype, 129, 700, terms)[0])
                mean = rb.ops.linear_cross_entropy(xx, w, target)
                assert torch.allclose(mean.double(), want.sum() / 2, rtol=2.0 ** -20, atol=tolerances(dtype, 129, 700, terms)[0])
            none = torch.full((4,), -100).cuda()
            assert torch.isnan(rb.ops.linear_cross_entropy(bad, w, none))
            assert rb.ops.linear_cross_entropy(bad, w, none, reduction="sum") == 0
            out = rb.ops.linear_cross_entropy(x, w, torch.tensor([5, 700, 699, -1]).cuda(), reduction="none", ignore_index=None)
            assert torch.equal(torch.isnan(out).cpu(), torch.tensor([False, True, False, True]))
    # a logit of minus infinity leaves the sum alone; one of plus infinity beside a finite target makes the loss infinite
    w = torch.ones(40, 8, dtype=dtype).cuda()
    one = torch.ones(1, 8, dtype=dtype).cuda()
    t = torch.tensor([0]).cuda()
    with torch.no_grad():
        w[7, 0] = float("-inf")
        assert abs(rb.ops.linear_cross_entropy(one, w, t).item() - math.log(39)) < 1e-5
        w[9, 0] = w[33, 0] = float("inf")
        assert rb.ops.linear_cross_entropy(one, w, t).item() == float("inf")


@pytest.mark.parametrize("T", [3, 1060])
def test_offsets_past_32_bits(rb, T):
    """Rows 2^22 elements apart: the last ones lie more than 2^32 elements behind the first."""
    R, V, pitch = 72, 1060, 2 ** 22
    x, w, target = inputs("linear", T, R, V, torch.bfloat16, 6)
    target[:2] = torch.tensor([V - 1, 0])
    far = torch.empty((V - 1) * pitch + R, dtype=torch.bfloat16, device="cuda").as_strided((V, R), (pitch, 1))
    far.copy_(w)
    check(rb, "linear", x, w, target, 6, -100, "mean")
    with torch.no_grad():
        assert torch.equal(rb.ops.linear_cross_entropy(x, far, target, reduction="none"), rb.ops.linear_cross_entropy(x, w, target, reduction="none"))
    one, other = ([t.requires_grad_() for t in (x.clone(), m)] for m in (w, far.detach()))
    want, got = (torch.autograd.grad(rb.ops.linear_cross_entropy(a, m, target), [a, m]) for a, m in (one, other))
    assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])
    far = far.detach()
    rows = far[V - T:]
    rows.copy_(x.detach())
    for call_it in (lambda a: rb.ops.linear_cross_entropy(a, w.detach(), target), lambda a: rb.ops.noise_cross_entropy(a, 9, V, target)):
        (a, b) = (t.detach().requires_grad_() for t in (x, rows))
        la, lb = call_it(a), call_it(b)
        assert torch.equal(la, lb) and torch.equal(torch.autograd.grad(la, a)[0], torch.autograd.grad(lb, b)[0])


@pytest.mark.parametrize("kind", ["noise", "linear"])
def test_operators_through_the_dispatcher(rb, kind):
    """rten::*_ce_*: schema, fake kernels and autograd registration; the same numbers as the eager functions."""
    x, w, target = inputs(kind, 60, 40, 90, torch.float32, 3)
    xl, wl = x.clone().requires_grad_(), w.clone().requires_grad_()
    checks = ("test_schema", "test_faketensor", "test_autograd_registration")
    if kind == "noise":
        args = (xl, target, 1003, 90, 5, -100, "mean", True)
        torch.library.opcheck(torch.ops.rten.noise_ce_fwd.default, args, test_utils=checks)
        loss = torch.ops.rten.noise_ce_fwd(*args)[0]
        leaves = [xl]
    else:
        args = (xl, wl, target, -100, "mean")
        torch.library.opcheck(torch.ops.rten.linear_ce_fwd.default, args, test_utils=checks)
        loss = torch.ops.rten.linear_ce_fwd(*args)[0]
        leaves = [xl, wl]
    grads = torch.autograd.grad(loss, leaves)
    x2, w2 = x.clone().requires_grad_(), w.clone().requires_grad_()
    loss2 = call(rb, kind, x2, w2, target, 3)
    grads2 = torch.autograd.grad(loss2, [x2] if kind == "noise" else [x2, w2])
    assert torch.equal(loss, loss2) and all(torch.equal(a, b) for a, b in zip(grads, grads2))


@pytest.mark.parametrize("dtype,tol", [(torch.bfloat16, 2e-2), (torch.float32, 2e-5)])
def test_layer_loss(rb, dtype, tol):
    """RandumbLinear.cross_entropy against the layer's weight in 64 bits.  bf16: z and dz are rounded to bf16 on the way, as the
    layer's forward and backward round them (the tolerance of the layer's own tests); float32: the CUDA-core products' 1e-5 and the loss's."""
    torch.manual_seed(0)
    head = rb.RandumbLinear(96, 1234, 64, seed=21, device="cuda", dtype=dtype)
    x = torch.randn(3, 100, 96, device="cuda", dtype=dtype)
    target = torch.randint(0, 1234, (3, 100), device="cuda")
    target[1, 20:70] = -100
    xl = x.clone()
    xl[1, 20:70] = float("nan")
    xl.requires_grad_()
    loss = head.cross_entropy(xl, target)
    dx, dc = torch.autograd.grad(loss, [xl, head.weight_coef])
    S = noise_matrix(1234, 64, 21, 0, dtype).double().cuda()
    C = head.weight_coef.detach().double().requires_grad_()
    xd = x.double().requires_grad_()
    want = F.cross_entropy(((xd @ C.t()) @ S.t()).reshape(-1, 1234), target.reshape(-1))
    wx, wc = torch.autograd.grad(want, [xd, C])
    assert abs(loss.item() - want.item()) < tol * want.item()
    assert (dx[1, 20:70] == 0).all()
    assert O.rel_fro(dx.double().cpu(), wx.cpu()) < tol and O.rel_fro(dc.double().cpu(), wc.cpu()) < tol
    with pytest.raises(RuntimeError, match="bias"):
        rb.RandumbLinear(96, 12, 8, seed=1, bias=True, device="cuda", dtype=dtype).cross_entropy(x, target)


def test_training_steps_with_all_operators(rb):
    """A pseudorandom layer and head, the fused loss, clipping and AdamW together: gradients of a step against autograd on dense weights,
    the update against torch's AdamW on the same gradients."""
    torch.manual_seed(1)
    dev = "cuda"
    body = rb.RandumbLinear(64, 96, 32, seed=3, device=dev)
    head = rb.RandumbLinear(96, 517, 48, seed=10, device=dev)
    params = [body.weight_coef, head.weight_coef]
    opt = rb.optim.AdamW(params, lr=1e-2, weight_decay=0.05, max_grad_norm=0.5)
    ref = [p.detach().clone().requires_grad_() for p in params]
    topt = torch.optim.AdamW(ref, lr=1e-2, weight_decay=0.05)
    S1, S2 = (torch.from_numpy(O.noise_f32(n, r, s)).cuda() for n, r, s in ((96, 32, 3), (517, 48, 10)))
    for k in range(3):
        x = torch.randn(200, 64, device=dev)
        target = torch.randint(0, 517, (200,), device=dev)
        target[::9] = -100
        loss = head.cross_entropy(torch.tanh(body(x)), target)
        opt.zero_grad()
        loss.backward()
        topt.zero_grad()
        want = F.cross_entropy(torch.tanh(x @ (S1 @ ref[0]).t()) @ (S2 @ ref[1]).t(), target)
        want.backward()
        assert abs(loss.item() / want.item() - 1) < 1e-4
        for p, r in zip(params, ref):
            assert O.rel_fro(p.grad.cpu(), r.grad.cpu()) < 1e-4
        norm = torch.nn.utils.clip_grad_norm_(ref, 0.5)
        opt.step()
        topt.step()
        assert abs(opt.last_grad_norm.item() / norm.item() - 1) < 1e-4
        with torch.no_grad():
            for p, r in zip(params, ref):
                # m / sqrt(v) of the first steps is near the gradient's sign: elements whose gradient is all rounding may go either way
                assert (p - r).abs().mean() < 1e-5
                r.copy_(p)


def test_refusals(rb):
    x, w, target = inputs("linear", 8, 16, 20, torch.bfloat16, 1)
    ce, nce = rb.linear_cross_entropy, rb.noise_cross_entropy
    with pytest.raises(RuntimeError, match="does not match"):
        ce(x, w, target[:7])
    with pytest.raises(RuntimeError, match="does not match"):
        ce(x, w[:, :8], target)
    with pytest.raises(RuntimeError, match="does not match"):
        ce(x, w.float(), target)
    with pytest.raises(RuntimeError, match="int64"):
        ce(x, w, target.int())
    with pytest.raises(RuntimeError, match="reduction"):
        ce(x, w, target, reduction="average")
    with pytest.raises(RuntimeError, match="float32 and bfloat16"):
        nce(x.half(), 1, 20, target)
    with pytest.raises(RuntimeError, match="at least one"):
        nce(x, 1, 0, target)
    with pytest.raises(RuntimeError, match="does not match"):
        rb.rlinear_cross_entropy(x, torch.zeros(4, 15, device="cuda", dtype=torch.bfloat16), 1, 20, target)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        ce(x, w, target.cpu())


def planned(kind, dtype, logits, ups, seed, R=400):
    """Rows of x, a matrix of few rows and targets with chosen logits: logits [T, V] with V < R fixes x up to the matrix's null space, from which each
    row gets as much as makes |x| |w_t| / sqrt(R) * (mean of the largest of V standard normal values) lie ups[i] above its target's logit (the largest
    one): long rows that are not well aligned with their targets."""
    T, V = logits.shape
    g = torch.Generator().manual_seed(seed)
    w = (noise_matrix(V, R, 1000 + seed, 5, dtype) if kind == "noise" else (torch.randn(V, R, generator=g) * 0.5).to(dtype)).double()
    target = logits.argmax(1)
    x = logits.double() @ torch.linalg.pinv(w).t()
    n = torch.randn(T, R, generator=g, dtype=torch.float64)
    n -= n @ torch.linalg.pinv(w) @ w
    a = math.sqrt(2 * math.log(V))
    spread = a + (0.5772 - 0.5 * (math.log(math.log(V)) + math.log(4 * 3.14159265))) / a
    want = (logits.amax(1).double() + ups) * math.sqrt(R) / spread / w[target].norm(dim=1)
    more = want ** 2 - (x ** 2).sum(1)
    assert (more > 0).all()
    x += n * (more.sqrt() / n.norm(dim=1))[:, None]
    return x.to(dtype).cuda(), w.to(dtype).cuda(), target.cuda()


def small_losses(x, w, target):
    """(losses, largest sum of a logit's terms) in 64 bits, without the difference of log-sum-exp and logit: 2^-52 of a logit is more than
    2^-20 of the smallest of these losses."""
    xd, wd = x.double(), w.double()
    logits = xd @ wd.t()
    e = torch.exp(logits - logits.gather(1, target[:, None]))
    e[torch.arange(x.shape[0]), target] = 0
    return torch.log1p(e.sum(1)), (xd.abs() @ wd.abs().t()).amax().item()


@pytest.mark.parametrize("kind", ["noise", "linear"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("top", [0.0, 30.0])
@pytest.mark.parametrize("ups", [(41.0, 48.0, 55.0, 62.0, 69.0), (76.0, 85.0, 110.0, 150.0, 400.0)])
def test_a_likely_target_of_a_long_row(rb, kind, dtype, top, ups):
    """The target is the most likely token by 10 to 35, in rows whose length says that some other logit should lie `ups` above it."""
    gaps = (10.0, 15.0, 18.8, 22.0, 25.0, 35.0)
    T, V, seed = len(gaps) * len(ups), 50, 4
    g = torch.Generator().manual_seed(3)
    logits = top - torch.tensor(gaps).repeat_interleave(len(ups))[:, None] + torch.randn(T, V, generator=g)
    logits[torch.arange(T), torch.randint(0, V, (T,), generator=g)] = top
    x, w, target = planned(kind, dtype, logits, torch.tensor(ups, dtype=torch.float64).repeat(len(gaps)), seed)
    loss, _ = check(rb, kind, x, w, target, seed, -100, "none", torch.ones(T, device="cuda"))
    # such a loss is the sum of e^(l_v - l_t): it is off, relative to itself, by the error of a difference of logits
    losses, terms = small_losses(x, w, target)
    logit, _ = tolerances(dtype, x.shape[1], V, terms)
    assert losses.max() < 0.1 and ((loss.double() - losses).abs() <= 2 * logit * losses).all(), ((loss.double() - losses) / losses)


@pytest.mark.parametrize("kind", ["noise", "linear"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_the_likeliest_of_widely_spread_logits(rb, kind, dtype):
    """Logits of deviation 200, rows whose target is the largest by 5 to 30 and lies far below where the largest usually does."""
    R, V, seed = 64, 1000, 6
    x, w, _ = inputs(kind, 30000, R, V, dtype, seed, 200.0)
    logits = x.double() @ w.double().t()
    two = logits.topk(2)
    gap = two.values[:, 0] - two.values[:, 1]
    rows = torch.nonzero((gap > 5) & (gap < 30))[:, 0]
    rows = rows[two.values[rows, 0].argsort()[:80]]
    target = two.indices[rows, 0]
    assert rows.numel() == 80 and two.values[rows, 0].max() < 560
    x = x[rows].contiguous()
    loss, _ = check(rb, kind, x, w, target, seed, -100, "none", torch.ones(80, device="cuda"))
    losses, terms = small_losses(x, w, target)
    logit, _ = tolerances(dtype, R, V, terms)
    assert ((loss.double() - losses).abs() <= 2 * logit * losses).all(), ((loss.double() - losses) / losses)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("common", [-100.0, 60.0])
def test_logits_with_a_common_part(rb, dtype, common):
    """Rows of a stored matrix that share a component, as trained ones do: all logits about `common`, of deviation 3."""
    T, R, V, seed = 700, 96, 2000, 9
    g = torch.Generator().manual_seed(seed)
    u = torch.randn(R, generator=g)
    u /= u.norm()
    x = torch.randn(T, R, generator=g)
    x += (10 - x @ u)[:, None] * u
    w = torch.randn(V, R, generator=g) * 0.3
    w += (common / 10 - w @ u)[:, None] * u
    target = torch.randint(0, V, (T,), generator=g).cuda()
    check(rb, "linear", x.to(dtype).cuda(), w.to(dtype).cuda(), target, seed, -100, "none", torch.ones(T, device="cuda"))


def test_logits_with_a_common_part_take_the_ordinary_way(rb):
    """Rows about -100 with deviation 3 are no harder than rows about 0: no row needs the slow way (which takes a hundred times as long)."""
    T, R, V = 2048, 256, 20000
    g = torch.Generator(device="cuda").manual_seed(1)
    u = torch.randn(R, device="cuda", generator=g)
    u /= u.norm()
    x = torch.randn(T, R, device="cuda", generator=g)
    x += (10 - x @ u)[:, None] * u
    w = torch.randn(V, R, device="cuda", generator=g) * (3 / R ** 0.5)
    target = torch.randint(0, V, (T,), device="cuda", generator=g)
    took = []
    for common in (0.0, -100.0):
        ww, xx = (w + (common / 10 - w @ u)[:, None] * u).bfloat16(), x.bfloat16()
        times = []
        with torch.no_grad():
            for _ in range(8):
                a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
                a.record()
                rb.linear_cross_entropy(xx, ww, target)
                b.record()
                b.synchronize()
                times.append(a.elapsed_time(b))
        took.append(sorted(times)[2])
    assert took[1] < 8 * took[0], took


@pytest.mark.parametrize("T", [5, 70, 700])
def test_vocabulary_rows_masked_by_minus_infinity(rb, T):
    """Vocabulary rows that hold minus infinity in a column where every x is positive have probability 0: they reach neither the loss nor another
    row's weight gradient, and their own is 0, whatever number of rows the last tile holds."""
    R, V, seed, dtype = 40, 300, 2, torch.bfloat16
    x, w, target = inputs("linear", T, R, V, dtype, seed)
    x[:, 0] = x[:, 0].abs() + 0.5
    off = torch.tensor([7, 100, 299], device="cuda")
    target[torch.isin(target, off)] = 3
    w[off, 0] = -math.inf
    keep = torch.ones(V, dtype=torch.bool, device="cuda")
    keep[off] = False
    place = keep.cumsum(0) - 1
    wl, kl = w.clone().requires_grad_(), w[keep].clone().requires_grad_()
    loss, want = rb.linear_cross_entropy(x, wl, target), rb.linear_cross_entropy(x, kl, place[target])
    dw, dk = torch.autograd.grad(loss, wl)[0], torch.autograd.grad(want, kl)[0]
    assert (dw[off] == 0).all()
    # the same numbers added in another order
    assert abs(loss.item() / want.item() - 1) < 2.0 ** -19
    assert (dw[keep].double() - dk.double()).abs().max() <= 2.0 ** -8 * dk.double().abs().max()


def test_no_second_derivatives(rb):
    """A gradient of a gradient is refused by every form of the loss; none of its parts drops out silently."""
    x, w, target = inputs("linear", 20, 16, 30, torch.float32, 1)
    c = torch.randn(8, 16, device="cuda")
    for make in (lambda a: rb.linear_cross_entropy(a, w, target), lambda a: rb.noise_cross_entropy(a, 3, 30, target),
                 lambda a: rb.rlinear_cross_entropy(a, c, 3, 30, target), lambda a: rb.rlinear_cross_entropy(a, c.requires_grad_(), 3, 30, target),
                 lambda a: rb.linear_cross_entropy(a, w.requires_grad_(), target, reduction="none").square().sum(),
                 lambda a: torch.ops.rten.noise_ce_fwd(a, target, 3, 30, 0, -100, "mean", True)[0],
                 lambda a: torch.ops.rten.linear_ce_fwd(a, w.detach(), target, -100, "mean")[0]):
        a = x.clone().requires_grad_()
        grad = torch.autograd.grad(make(a), a, create_graph=True)[0]
        b = x.clone().requires_grad_()
        assert torch.equal(grad, torch.autograd.grad(make(b), b)[0])
        with pytest.raises(RuntimeError):
            (make(a) + grad.pow(2).sum()).backward()


def test_layer_loss_through_the_dispatcher(rb):
    """The product in front of the noise head as an operator: schema, fake kernel, autograd, the same numbers as the eager function."""
    x, _, target = inputs("linear", 60, 40, 90, torch.bfloat16, 3)
    c = (torch.randn(24, 40, device="cuda") * 0.2).bfloat16()
    xl, cl = x.clone().requires_grad_(), c.clone().requires_grad_()
    torch.library.opcheck(torch.ops.rten.matmul_nt_fwd.default, (xl, cl), test_utils=("test_schema", "test_faketensor", "test_autograd_registration"))
    loss = torch.ops.rten.noise_ce_fwd(torch.ops.rten.matmul_nt_fwd(xl, cl), target, 1003, 90, 5, -100, "mean", True)[0]
    grads = torch.autograd.grad(loss, [xl, cl])
    x2, c2 = x.clone().requires_grad_(), c.clone().requires_grad_()
    loss2 = rb.rlinear_cross_entropy(x2, c2, 1003, 90, target, row0=5)
    grads2 = torch.autograd.grad(loss2, [x2, c2])
    assert torch.equal(loss, loss2) and all(torch.equal(a, b) for a, b in zip(grads, grads2))


def test_vmap_takes_the_calls_one_by_one(rb):
    x, w, target = inputs("linear", 40, 16, 30, torch.float32, 1)
    c = torch.randn(8, 16, device="cuda")
    xs, ts = x.view(4, 10, 16), target.view(4, 10)
    for f in (lambda a, t: rb.linear_cross_entropy(a, w, t), lambda a, t: rb.noise_cross_entropy(a, 3, 30, t), lambda a, t: rb.rlinear_cross_entropy(a, c, 3, 30, t)):
        with torch.no_grad():
            got = torch.func.vmap(f)(xs, ts)
            assert torch.equal(got, torch.stack([f(a, t) for a, t in zip(xs, ts)]))


@pytest.mark.parametrize("kind", ["noise", "linear"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V", [1, 2, 5, 31, 32, 33, 40, 70])
def test_wide_logits_of_small_vocabularies(rb, kind, dtype, V):
    """Rows whose length asks for a look at other logits, over vocabularies that are all looked at, and just not."""
    T, R, seed = 90, 72, V
    x, w, target = inputs(kind, T, R, V, dtype, seed, 60.0)
    check(rb, kind, x, w, target, seed, -100, "none", torch.ones(T, device="cuda"))


def test_traced_by_torch_compile(rb):
    """One graph without breaks, forward and backward, and the eager numbers."""
    x, w, target = inputs("linear", 40, 16, 30, torch.float32, 1)
    c = torch.randn(8, 16, device="cuda", requires_grad=True)
    x, w = x.requires_grad_(), w.requires_grad_()
    for f, leaves in ((lambda: rb.linear_cross_entropy(x, w, target), [x, w]), (lambda: rb.noise_cross_entropy(x, 3, 30, target), [x]),
                      (lambda: rb.rlinear_cross_entropy(x, c, 3, 30, target), [x, c])):
        want = f()
        got = torch.compile(f, backend="aot_eager", fullgraph=True)()
        assert torch.equal(got, want)
        assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(got, leaves), torch.autograd.grad(want, leaves)))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T", [3, 70, 700])
def test_vocabulary_rows_masked_by_the_lowest_value(rb, dtype, T):
    """The same with the type's lowest finite value: the masked rows' logits are -1e38 or below, and all gradients are finite."""
    R, V, seed = 40, 300, 2
    x, w, target = inputs("linear", T, R, V, dtype, seed)
    x[:, 0] = x[:, 0].abs() + 0.5
    off = torch.tensor([7, 100, 299], device="cuda")
    target[torch.isin(target, off)] = 3
    w[off, 0] = torch.finfo(dtype).min
    keep = torch.ones(V, dtype=torch.bool, device="cuda")
    keep[off] = False
    place = keep.cumsum(0) - 1
    xl, wl, xk, kl = (t.clone().requires_grad_() for t in (x, w, x, w[keep]))
    loss, want = rb.linear_cross_entropy(xl, wl, target), rb.linear_cross_entropy(xk, kl, place[target])
    with torch.no_grad():
        alone = rb.linear_cross_entropy(x, w, target)
    (dx, dw), (dk_x, dk) = torch.autograd.grad(loss, [xl, wl]), torch.autograd.grad(want, [xk, kl])
    # the same numbers added in another order
    assert abs(loss.item() / want.item() - 1) < 2.0 ** -19 and abs(alone.item() / want.item() - 1) < 2.0 ** -19
    step = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -18
    assert (dw[off] == 0).all() and (dw[keep].double() - dk.double()).abs().max() <= step * dk.double().abs().max()
    assert (dx.double() - dk_x.double()).abs().max() <= step * dk_x.double().abs().max()


@pytest.mark.parametrize("mean,dev,idle", [(60.0, 15.0, 0.0), (400.0, 10.0, 0.0), (0.0, 10.0, 30.0), (-300.0, 10.0, 100.0), (0.0, 20.0, 0.0)])
def test_logits_of_any_mean_take_the_ordinary_way(rb, mean, dev, idle):
    """Logits of the given mean and deviation; `idle`: a common component of the matrix's rows that the rows of x do not have, which lengthens the
    first and moves no logit.  No row needs the slow way, and losses are those of 64 bits."""
    T, R, V = 2048, 256, 20000
    g = torch.Generator(device="cuda").manual_seed(2)
    q, _ = torch.linalg.qr(torch.randn(R, 2, device="cuda", generator=g))
    u, away = q[:, 0], q[:, 1]
    x = torch.randn(T, R, device="cuda", generator=g)
    x += (10 - x @ u)[:, None] * u
    x -= (x @ away)[:, None] * away
    target = torch.randint(0, V, (T,), device="cuda", generator=g)
    noise = torch.randn(V, R, device="cuda", generator=g) / R ** 0.5
    took = []
    for m, s, i in ((0.0, 1.0, 0.0), (mean, dev, idle)):
        w = noise * s
        w = (w + (m / 10 - w @ u)[:, None] * u + (i - w @ away)[:, None] * away).bfloat16()
        xx = x.bfloat16()
        times = []
        with torch.no_grad():
            for _ in range(8):
                a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
                a.record()
                loss = rb.linear_cross_entropy(xx, w, target, reduction="none")
                b.record()
                b.synchronize()
                times.append(a.elapsed_time(b))
        took.append(sorted(times)[2])
        _, losses, *_, terms = plain(xx, w, target, None, "none", torch.ones(T, device="cuda"))
        assert ((loss.double() - losses).abs() <= 2.0 ** -21 * losses + tolerances(torch.bfloat16, R, V, terms)[0]).all()
    assert took[1] < 8 * took[0], took
