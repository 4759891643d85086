"""AdamW and the gradient norm on the GPU against plain 64-bit implementations.

Tolerances.  One float32 operation is off by at most half a step, u = 2^-24 of its value.  A moment is a sum of two rounded products:
|dm| <= 2 u (|b1 m| + |(1 - b1) g|) and one u more where the gradient is scaled first.  The update m / (sqrt(v) / root + eps) adds
the roundings of v (3 u, halved by the root), sqrt, product, sum, quotient, size: below 10 u relative to the update's own terms.
"""
import copy
import math

import numpy as np
import pytest
import torch

from oracle import oracle as O

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
SIZES = [1, 3, 255, 256, 257, 1000, 8192, 8193, 20001]


@pytest.fixture(scope="module")
def rb():
    import randumb_b200
    assert torch.cuda.is_available()
    return randumb_b200


def make(sizes, pdtype, gdtype, seed, shift=0):
    """Tensors carved out of one buffer, `shift` elements off its start: most of them begin on no vector boundary."""
    g = torch.Generator().manual_seed(seed)
    n = sum(sizes)

    def carve(flat):
        buf = torch.zeros(n + shift, dtype=flat.dtype, device="cuda")
        buf[shift:] = flat.cuda()
        out, at = [], shift
        for k in sizes:
            out.append(buf[at:at + k])
            at += k
        return out

    p = torch.randn(n, generator=g) * 0.05
    gr = torch.randn(n, generator=g) * torch.exp(2 * torch.randn(n, generator=g)) * 1e-3
    m = torch.randn(n, generator=g) * 1e-3
    v = torch.rand(n, generator=g) * 1e-6
    return carve(p.to(pdtype)), carve(gr.to(gdtype)), carve(m), carve(v), carve


def plain(p, g, m, v, t, lr, b1, b2, eps, wd, gs=1.0):
    """The definition in 64 bits."""
    g = g.double() * gs
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    upd = (m / (1 - b1 ** t)) / (torch.sqrt(v / (1 - b2 ** t)) + eps)
    return p * (1 - lr * wd) - lr * upd, m, v, upd


@pytest.mark.parametrize("pdtype,gdtype,master", [(torch.float32, torch.float32, False), (torch.float32, torch.bfloat16, False),
                                                  (torch.bfloat16, torch.bfloat16, False), (torch.bfloat16, torch.float32, True),
                                                  (torch.bfloat16, torch.bfloat16, True)])
@pytest.mark.parametrize("shift", [0, 1])
def test_adamw_32_bit_moments(rb, pdtype, gdtype, master, shift):
    lr, b1, b2, eps, wd, gs = 3e-3, 0.9, 0.95, 1e-8, 0.1, 0.25
    ps, grads, ms, vs, carve = make(SIZES, pdtype, gdtype, 3, shift)
    masters = carve(torch.cat([p.float().cpu() * 1.001 for p in ps])) if master else None
    steps = torch.tensor([float(7 * i) for i in range(len(SIZES))], device="cuda")
    want = []
    for i, (p, g, m, v) in enumerate(zip(masters or ps, grads, ms, vs)):
        want.append(plain(p.double(), g, m.double(), v.double(), 7 * i + 1, lr, b1, b2, eps, wd, gs) + (m.double().abs(), g.double().abs() * gs, p.double().abs()))
    before = [g.clone() for g in grads]
    rb.optim.adamw_step(ps, grads, ms, vs, steps, lr=lr, betas=(b1, b2), eps=eps, weight_decay=wd, masters=masters,
                        grad_scale=torch.full((1,), gs, device="cuda"))
    assert steps.tolist() == [7 * i + 1 for i in range(len(SIZES))]
    for i in range(len(SIZES)):
        wp, wm, wv, upd, am, ag, ap = want[i]
        assert torch.equal(before[i], grads[i])
        # |m| can be far below its terms: the bound is on the terms.  eps of v: three roundings of its larger term
        assert ((ms[i].double() - wm).abs() <= 4 * U * (am + ag)).all()
        assert ((vs[i].double() - wv).abs() <= 5 * U * wv).all()
        dm = 4 * U * (am + ag) / (1 - b1 ** (7 * i + 1)) / (torch.sqrt(wv / (1 - b2 ** (7 * i + 1))) + eps)
        bound = lr * (dm + 16 * U * upd.abs()) + 4 * U * ap
        got = (masters or ps)[i]
        if pdtype == torch.float32 or master:
            assert ((got.double() - wp).abs() <= bound).all()
        if master:
            assert torch.equal(ps[i], masters[i].to(torch.bfloat16))
        elif pdtype == torch.bfloat16:
            # rounded to bf16 at the end: half a step, 2^-8 of the value, on top
            assert ((got.double() - wp).abs() <= bound + 2.0 ** -8 * (wp.abs() + bound)).all()


def _v_values(codes):
    return (codes.to(torch.int32) << 19).view(torch.float32).double() * 2.0 ** 112


def _e4m3_neighbours_ok(code, q):
    """Rounded to nearest: off by at most half a step -- 2^-4 of the value, or half the smallest step 2^-9 -- and 4 u of q."""
    return (code.double() - q).abs() <= torch.clamp(q.abs() * 2.0 ** -4, min=2.0 ** -10) * (1 + 8 * U)


@pytest.mark.parametrize("pdtype,gdtype", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16)])
@pytest.mark.parametrize("shift", [0, 3])
def test_adamw_8_bit_moments(rb, pdtype, gdtype, shift):
    lr, b1, b2, eps, wd, seed = 1e-3, 0.9, 0.999, 1e-8, 0.01, 77
    ps, grads, _, _, carve = make(SIZES, pdtype, gdtype, 5, shift)
    n = sum(SIZES)
    ms = carve(torch.zeros(n, dtype=torch.uint8))
    ms = [t.view(torch.float8_e4m3fn) for t in ms]
    vs = carve(torch.zeros(n, dtype=torch.uint8))
    blocks = [-(-k // 256) for k in SIZES]
    msc = [torch.zeros(b, device="cuda") for b in blocks]
    vsc = [torch.zeros(b, device="cuda") for b in blocks]
    steps = torch.zeros(len(SIZES), device="cuda")
    for it in range(3):
        for k, g in enumerate(grads):
            g.copy_(torch.randn(g.shape, generator=torch.Generator().manual_seed(100 * it + k)).to(g.dtype) * 1e-3)
        old = [(p.double().cpu(), rb.optim.first_moment_values(m, a).double().cpu(), rb.optim.second_moment_values(v, b).double().cpu())
               for p, m, v, a, b in zip(ps, ms, vs, msc, vsc)]
        rb.optim.adamw_step(ps, grads, ms, vs, steps, lr=lr, betas=(b1, b2), eps=eps, weight_decay=wd, exp_avg_scales=msc, exp_avg_sq_scales=vsc, seed=seed)
        for i, k in enumerate(SIZES):
            p0, m0, v0 = old[i]
            wp, wm, wv, upd = plain(p0, grads[i].cpu(), m0, v0, it + 1, lr, b1, b2, eps, wd)
            pad = blocks[i] * 256 - k
            top = lambda x: torch.nn.functional.pad(x, (0, pad)).reshape(-1, 256).amax(1)
            a, b = msc[i].double().cpu(), vsc[i].double().cpu()
            at = (m0.abs() + grads[i].double().cpu().abs())
            # the largest magnitude's own rounding error and the division's
            assert ((a * 448 - top(wm.abs())).abs() <= 6 * U * top(at)).all() and ((b * 1.9375 - top(wv)).abs() <= 8 * U * top(wv)).all()
            sa, sb = a.repeat_interleave(256)[:k], b.repeat_interleave(256)[:k]
            q = torch.where(sa > 0, wm / sa, 0.0)
            slack = 16 * U * torch.where(sa > 0, at / sa, 0.0)
            assert (((ms[i].cpu().double() - q).abs() - slack) <= torch.clamp(q.abs() * 2.0 ** -4, min=2.0 ** -10)).all()
            # second moment: one of the two neighbours, the one that the noise word picks (a value within 2^-20 of a border may fall either way)
            qv = torch.where(sb > 0, wv / sb, 0.0)
            word = O.noise_bits_1d(k, (seed + (it + 1) * 0x9E3779B1 + i * 0x85EBCA6B) & 0xFFFFFFFF) >> np.uint32(13)
            frac = torch.from_numpy(word.astype(np.float64)) * 2.0 ** -19
            lo = torch.where(qv >= 2.0 ** -14, torch.floor(torch.log2(qv.clamp(min=1e-300))), torch.full_like(qv, -14.0))
            step = torch.exp2(lo - 4)
            cell = torch.floor(qv / step + frac + 1e-9) * step
            got = _v_values(vs[i].cpu())
            border = ((qv / step + frac) - torch.round(qv / step + frac)).abs() < 2.0 ** -16
            want = torch.where((wv > 0) & (cell == 0), torch.full_like(cell, 2.0 ** -18), cell).clamp(max=1.9375)
            assert ((got == want) | border).all()
            assert ((got > 0) == (wv > 0)).all()
            bound = lr * 32 * U * (upd.abs() + 1) + 4 * U * p0.abs()
            rnd = 0 if pdtype == torch.float32 else 2.0 ** -8 * (wp.abs() + bound)
            slack_m = lr * 8 * U * at / (1 - b1 ** (it + 1)) / (torch.sqrt(wv / (1 - b2 ** (it + 1))) + eps)
            assert ((ps[i].double().cpu() - wp).abs() <= bound + slack_m + rnd).all()


def test_adamw_8_bit_second_moment_keeps_its_expectation(rb):
    """With no gradient v decays by b2 each step, far below a step of the format: the random rounding follows it on average.
    64 blocks of 256 equal values start at 1; after 400 steps of b2 = 0.998 the expectation is 0.998^400 = 0.449.  The first
    element of each block is fed so that the scale stays; one rounding has variance below (step/2)^2, step <= 2^-4 of the value,
    so 400 of them on 16320 values leave the mean within 400^0.5 * 2^-5 / 16320^0.5 * 5 sigma = 2.5 %."""
    n, b2 = 64 * 256, 0.998
    p, g = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda")
    head = torch.zeros(n, dtype=torch.bool, device="cuda")
    head[::256] = True
    g[head] = 1.0
    m = torch.zeros(n, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    v = torch.full((n,), 247, dtype=torch.uint8, device="cuda")
    v[head] = 247
    ms, vs = torch.zeros(64, device="cuda"), torch.full((64,), 1 / 1.4375, device="cuda")
    steps = torch.zeros(1, device="cuda")
    for _ in range(400):
        rb.optim.adamw_step([p], [g], [m], [v], steps, lr=0.0, betas=(0.9, b2), exp_avg_scales=[ms], exp_avg_sq_scales=[vs], seed=5)
    mean = rb.optim.second_moment_values(v, vs)[~head].double().mean().item()
    assert abs(mean / b2 ** 400 - 1) < 0.025


@pytest.mark.parametrize("dtypes", [(torch.float32,), (torch.bfloat16,), (torch.float32, torch.bfloat16)])
def test_grad_norm(rb, dtypes):
    g = torch.Generator().manual_seed(1)
    grads = [(torch.randn(k, generator=g) * 10 ** (i % 5 - 2)).to(dtypes[i % len(dtypes)]).cuda() for i, k in enumerate(SIZES * 60)]   # 540 tensors: two launches
    grads.append(torch.zeros(0, device="cuda", dtype=dtypes[0]))
    want = math.sqrt(sum(float((t.double() ** 2).sum()) for t in grads))
    norm, none = rb.optim.grad_norm(grads)
    # the eight squares a lane adds in float32: 8 roundings of u each at most, halved by the root, and the result's own
    assert none is None and abs(norm.item() / want - 1) <= 8 * U
    n2, f = rb.optim.grad_norm(grads, max_norm=0.5)
    assert torch.equal(n2, norm) and abs(f.item() * want / 0.5 - 1) <= 12 * U + 1e-6 / want
    assert rb.optim.grad_norm(grads, max_norm=1e9)[1].item() == 1.0
    bad = grads[:3] + [torch.full((5,), float("nan"), device="cuda", dtype=dtypes[0])]
    nn, ff = rb.optim.grad_norm(bad, max_norm=1.0)
    assert math.isnan(nn.item()) and math.isnan(ff.item())


def test_step_on_a_side_stream_and_in_a_graph(rb):
    sizes = [5000, 300, 77]
    ps, grads, ms, vs, _ = make(sizes, torch.float32, torch.float32, 9)
    ref = [[t.clone() for t in x] for x in (ps, ms, vs)]
    steps, rsteps = torch.zeros(3, device="cuda"), torch.zeros(3, device="cuda")
    lr = torch.full((1,), 1e-2, device="cuda")
    for k in range(3):
        _, f = rb.optim.grad_norm(grads, 1.0)
        rb.optim.adamw_step(ref[0], grads, ref[1], ref[2], rsteps, lr=1e-2 * (k + 1), grad_scale=f)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        _, f = rb.optim.grad_norm(grads, 1.0)
        rb.optim.adamw_step(ps, grads, ms, vs, steps, lr=lr, grad_scale=f)
    assert steps.tolist() == [0, 0, 0]
    for k in range(3):
        lr.fill_(1e-2 * (k + 1))
        graph.replay()
    torch.cuda.synchronize()
    assert steps.tolist() == [3, 3, 3]
    for a, b in zip(ps + ms + vs, ref[0] + ref[1] + ref[2]):
        # the learning rate is 1e-2 in float32 here and in float64 there: u of the update
        assert (a - b).abs().max() <= 1e-6


def test_optimizer_class(rb):
    """Two groups, bf16 with masters beside float32, a channels-last weight, a parameter whose gradient comes later, a checkpoint."""
    torch.manual_seed(0)

    def build():
        g = torch.Generator().manual_seed(4)
        a = torch.nn.Parameter(torch.randn(33, 65, generator=g).cuda().bfloat16())
        b = torch.nn.Parameter(torch.randn(8, 3, 5, 5, generator=g).cuda().to(memory_format=torch.channels_last))
        c = torch.nn.Parameter(torch.randn(70, generator=g).cuda())
        return a, b, c

    def grads(ps, k, skip_c):
        g = torch.Generator().manual_seed(50 + k)
        for i, p in enumerate(ps):
            p.grad = None if (i == 2 and skip_c) else torch.randn(p.shape, generator=g).cuda().to(p.dtype)

    for bits in (32, 8):
        ps = build()
        opt = rb.optim.AdamW([{"params": ps[:2], "lr": 1e-2}, {"params": ps[2:], "weight_decay": 0.0}], lr=1e-3, state_bits=bits, max_grad_norm=0.7, seed=3)
        ref = [p.detach().float().clone().requires_grad_() for p in ps]
        topt = torch.optim.AdamW([{"params": ref[:2], "lr": 1e-2}, {"params": ref[2:], "weight_decay": 0.0}], lr=1e-3)
        for k in range(4):
            grads(ps, k, k == 0)
            for p, r in zip(ps, ref):
                r.grad = None if p.grad is None else p.grad.float().clone()  # clip_grad_norm_ writes to it
            want = torch.nn.utils.clip_grad_norm_([r for r in ref if r.grad is not None], 0.7)
            opt.step()
            topt.step()
            assert abs(opt.last_grad_norm.item() / want.item() - 1) < 1e-5
            if k == 1:                                             # save, rebuild, load
                sd = opt.state_dict()
                saved = [p.detach().clone() for p in ps]
                ps2 = build()
                for p, s in zip(ps2, saved):
                    p.data.copy_(s)
                opt = rb.optim.AdamW([{"params": ps2[:2], "lr": 1e-2}, {"params": ps2[2:], "weight_decay": 0.0}], lr=1e-3, state_bits=bits,
                                     max_grad_norm=0.7, seed=3)
                opt.load_state_dict(sd)
                ps = ps2
        assert opt.state[ps[0]]["step"].item() == 4 and opt.state[ps[2]]["step"].item() == 3
        assert opt.state[ps[1]]["exp_avg"].stride() == ps[1].stride()
        if bits == 8:                                              # the channels-last moment decodes in its own layout, near the float32 one
            st, want = opt.state[ps[1]], topt.state[ref[1]]["exp_avg"]
            got = rb.optim.first_moment_values(st["exp_avg"], st["exp_avg_scale"])
            assert got.stride() == ps[1].stride() and (got - want).norm() < 0.1 * want.norm()
        for i, (p, r) in enumerate(zip(ps, ref)):
            got = opt.state[p]["master"] if "master" in opt.state[p] else p
            # each of the four updates is at most lr * (1 + a few) in size; 8-bit moments are within 2^-4 (first), and the second's random rounding
            # within 2^-4 a step, of the float32 ones: at most a quarter of the distance walked.  32 bits: roundings only
            walked = 4 * (1e-2 if i < 2 else 1e-3) * 1.2
            assert (got.float() - r).abs().max().item() <= (walked * 0.25 if bits == 8 else 1e-5)
        other = rb.optim.AdamW([{"params": build()[:2]}, {"params": build()[2:]}], state_bits=40 - bits)
        other.load_state_dict(opt.state_dict())                    # the checkpoint's format comes with it
        assert [g["state_bits"] for g in other.param_groups] == [bits, bits]
    ckpt = topt.state_dict()
    c = [torch.nn.Parameter(r.detach().clone()) for r in ref]
    mine = rb.optim.AdamW([{"params": c[:2]}, {"params": c[2:]}])
    mine.load_state_dict(ckpt)                                     # torch's own AdamW
    assert torch.equal(mine.state[c[0]]["exp_avg"], topt.state[ref[0]]["exp_avg"]) and mine.state[c[0]]["step"].item() == 4
    low = build()
    with pytest.raises(RuntimeError, match="other state_bits or masters"):
        rb.optim.AdamW([{"params": low[:2]}, {"params": low[2:]}]).load_state_dict(ckpt)   # no masters for the bfloat16 parameter in it


def test_refusals(rb):
    p, g, m, v = (torch.zeros(4, device="cuda") for _ in range(4))
    s = torch.zeros(1, device="cuda")
    step = rb.optim.adamw_step
    with pytest.raises(RuntimeError, match="twice"):
        step([p, p], [g, g], [m, m], [v, v], torch.zeros(2, device="cuda"))
    two = lambda: [torch.zeros(4, device="cuda") for _ in range(2)]                   # noqa: E731
    with pytest.raises(RuntimeError, match="twice"):
        step(two(), [g, g], two(), two(), [s, s])
    with pytest.raises(RuntimeError, match="twice"):
        step(two(), [g, g], [m, m], two(), torch.zeros(2, device="cuda"))
    with pytest.raises(RuntimeError, match="twice"):
        step([p], [g], [m], [m], s)
    with pytest.raises(RuntimeError, match="differ in size"):
        step([p], [torch.zeros(5, device="cuda")], [m], [v], s)
    with pytest.raises(RuntimeError, match="one type"):
        step([p], [g.half()], [m], [v], s)
    with pytest.raises(RuntimeError, match="one type"):
        step([p], [g], [m.bfloat16()], [v], s)
    with pytest.raises(RuntimeError, match="contiguous"):
        step([torch.zeros(4, 2, device="cuda")[:, 0]], [g], [m], [v], s)
    with pytest.raises(RuntimeError, match="live on"):
        step([p], [g.cpu()], [m], [v], s)
    with pytest.raises(RuntimeError, match="steps"):
        step([p], [g], [m], [v], torch.zeros(2, device="cuda"))
    with pytest.raises(RuntimeError, match="masters"):
        step([p], [g], [m], [v], s, masters=[p.clone()])
    with pytest.raises(RuntimeError, match="one-element"):
        step([p], [g], [m], [v], s, grad_scale=torch.zeros(2, device="cuda"))
    with pytest.raises(RuntimeError, match="not supported"):
        step([p], [g], [m], [v], s, betas=(1.0, 0.9))
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        step([p.cpu()], [g], [m], [v], s)
    with pytest.raises(RuntimeError, match="scales"):
        step([p], [g], [m.to(torch.float8_e4m3fn)], [v.to(torch.uint8)], s, exp_avg_scales=[m[:2]], exp_avg_sq_scales=[m[:1]])
    step([], [], [], [], s)
    assert p.abs().sum() == 0


def test_more_tensors_than_one_launch_holds(rb):
    """500 tensors, some empty, in 8 bits and 32: each as if it were alone (tensor i of the list rounds with its own seed)."""
    sizes = [(7 * i) % 600 for i in range(500)]
    g = torch.Generator().manual_seed(2)
    p0 = [torch.randn(k, generator=g).cuda() for k in sizes]
    gr = [torch.randn(k, generator=g).cuda() for k in sizes]
    for bits in (32, 8):
        def state():
            if bits == 32:
                return [torch.zeros(k, device="cuda") for k in sizes], [torch.zeros(k, device="cuda") for k in sizes], {}
            m = [torch.zeros(k, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn) for k in sizes]
            v = [torch.zeros(k, dtype=torch.uint8, device="cuda") for k in sizes]
            return m, v, dict(exp_avg_scales=[torch.zeros(-(-k // 256), device="cuda") for k in sizes],
                              exp_avg_sq_scales=[torch.zeros(-(-k // 256), device="cuda") for k in sizes])
        p = [t.clone() for t in p0]
        m, v, sc = state()
        steps = torch.zeros(500, device="cuda")
        rb.optim.adamw_step(p, gr, m, v, steps, lr=1e-2, seed=11, **sc)
        assert (steps == 1).all()
        q = [t.clone() for t in p0]
        m2, v2, sc2 = state()
        s2 = [torch.zeros((), device="cuda") for _ in sizes]
        for i in (1, 44, 383, 384, 385, 499):
            one = {k: [x[i]] for k, x in sc2.items()}
            # tensor i of a list of its own rounds with seed + i * 0x85EBCA6B
            rb.optim.adamw_step([q[i]], [gr[i]], [m2[i]], [v2[i]], [s2[i]], lr=1e-2, seed=11 + i * 0x85EBCA6B, **one)
            assert torch.equal(p[i], q[i]) and torch.equal(m[i].view(torch.uint8), m2[i].view(torch.uint8)) and torch.equal(v[i], v2[i])


def test_optimizer_follows_its_parameters(rb):
    """Between steps a parameter's storage is exchanged, another gets its first gradient, one group is added."""
    a, b, c = (torch.nn.Parameter(torch.ones(k, device="cuda")) for k in (300, 40, 5))
    opt = rb.optim.AdamW([a, b], lr=0.1, weight_decay=0.0)
    ref = [torch.nn.Parameter(torch.ones(k, device="cuda")) for k in (300, 40, 5)]
    topt = torch.optim.AdamW(ref[:2], lr=0.1, weight_decay=0.0)
    for k in range(5):
        for p, r in zip((a, b, c), ref):
            if p is not b or k >= 2:
                p.grad = torch.full_like(p, 0.5 + k)
                r.grad = p.grad.clone()
        if k == 3:
            a.data = a.data.clone()
            opt.add_param_group({"params": [c], "lr": 0.01, "weight_decay": 0.0})
            topt.add_param_group({"params": [ref[2]], "lr": 0.01, "weight_decay": 0.0})
        opt.step()
        topt.step()
        for p, r in zip((a, b, c), ref):
            # a few roundings of values of size 1 in either program
            assert (p - r).abs().max() < 8 * 2.0 ** -23


@pytest.mark.parametrize("bits", [32, 8])
def test_state_that_moves(rb, bits):
    """The state's memory is exchanged between steps (moved to the host and back): the next step works on the new one."""
    g = torch.Generator().manual_seed(4)
    start = torch.randn(700, generator=g).cuda()
    a, b = torch.nn.Parameter(start.clone()), torch.nn.Parameter(start.clone())
    opt, ref = (rb.optim.AdamW([p], lr=0.01, state_bits=bits) for p in (a, b))
    old = []
    for _ in range(4):
        a.grad = torch.randn(700, generator=g).cuda()
        b.grad = a.grad.clone()
        opt.step()
        ref.step()
        assert torch.equal(a, b)
        for t in opt.state[a].values():
            old.append((t.data, t.data.clone()))
            t.data = t.data.cpu().cuda()
    for t, before in old:
        assert torch.equal(t.float(), before.float())         # what was left behind is not written any more


def test_a_graph_that_kept_a_parameter_notices_the_step(rb):
    p = torch.nn.Parameter(torch.ones(8, device="cuda"))
    q = torch.nn.Parameter(torch.ones(4, 2, device="cuda").t())
    opt = rb.optim.AdamW([p, q])
    loss = (p * p).sum() + (q * q).sum()
    loss.backward(retain_graph=True)
    opt.step()
    assert p._version > 0 and q._version > 0
    with pytest.raises(RuntimeError, match="inplace operation"):
        loss.backward()


def test_a_copied_optimizer_steps_by_itself(rb):
    p = torch.nn.Parameter(torch.ones(300, device="cuda"))
    opt = rb.optim.AdamW([p], lr=0.1, max_grad_norm=1.0, state_bits=8)
    for k in range(2):
        p.grad = torch.full_like(p, 1.0 + k)
        opt.step()
    q, twin = copy.deepcopy((p, opt))
    q.grad = p.grad = torch.full_like(p, 3.0)
    opt.step()
    assert not torch.equal(p, q)
    twin.step()
    assert torch.equal(p, q) and torch.equal(opt.last_grad_norm, twin.last_grad_norm)


@pytest.mark.parametrize("bits", [32, 8])
def test_a_tensor_past_32_bit_offsets(rb, bits):
    """2^31 + 300 elements: what lies behind 2^31 is updated as in a small tensor."""
    n, head = 2 ** 31 + 300, 2 ** 31 - 256
    kw = dict(device="cuda")
    p, g = torch.zeros(n, dtype=torch.bfloat16, **kw), torch.zeros(n, dtype=torch.bfloat16, **kw)
    tail = torch.randn(n - head, generator=torch.Generator().manual_seed(9)).bfloat16().cuda()
    p[head:], g[head:] = tail, tail.flip(0)

    def state(k):
        if bits == 32:
            return [torch.zeros(k, **kw)], [torch.zeros(k, **kw)], {}
        return [torch.zeros(k, dtype=torch.uint8, **kw).view(torch.float8_e4m3fn)], [torch.zeros(k, dtype=torch.uint8, **kw)], \
            dict(exp_avg_scales=[torch.zeros(-(-k // 256), **kw)], exp_avg_sq_scales=[torch.zeros(-(-k // 256), **kw)])

    m, v, sc = state(n)
    assert torch.equal(rb.optim.grad_norm([g])[0], rb.optim.grad_norm([g[head:].clone()])[0])
    rb.optim.adamw_step([p], [g], m, v, torch.zeros(1, **kw), lr=0.1, weight_decay=0.0, **sc)
    q, m2, v2 = [tail.clone()], *state(n - head)[:2]
    sc2 = state(n - head)[2]
    rb.optim.adamw_step(q, [tail.flip(0)], m2, v2, torch.zeros(1, **kw), lr=0.1, weight_decay=0.0, **sc2)
    assert torch.equal(m[0].view(torch.uint8)[(head if bits == 8 else 4 * head):], m2[0].view(torch.uint8))
    # the random rounding of an 8-bit second moment goes by the element's place, the update of a first step does not hang on it
    assert torch.equal(p[head:], q[0]) and (p[:head:1 << 20] == 0).all()


@pytest.mark.parametrize("pdtype,bits", [(torch.float32, 32), (torch.float32, 8), (torch.bfloat16, 32)])
@pytest.mark.parametrize("eps", [0.0, 1e-30, 1e-25, 1e-20, 1e-18, 1e-16, 1e-15, 1e-13, 1e-11, 1e-8])
def test_a_small_eps_and_small_gradients(rb, pdtype, bits, eps):
    """First step from zero with lr 1, gradients of 1e-19 to 1e-15: v is below float32's normal range for most of them, its root is not, and eps
    may be far below that.  The moments are taken as float32 rounds them (v by steps of 2^-149 here); what is left is the update:
    quotient and root within 2^-21 as the kernel states, and eight roundings of 2^-24 each, 2^-21 together."""
    b1, b2, n = 0.9, 0.999, 600
    g = torch.logspace(-19, -15, n, dtype=torch.float64).float() * (1 - 2 * (torch.arange(n) % 2))
    p = torch.zeros(n, dtype=pdtype, device="cuda")
    kw = {}
    if bits == 32:
        m, v = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda")
    else:
        m, v = torch.zeros(n, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn), torch.zeros(n, dtype=torch.uint8, device="cuda")
        kw = dict(exp_avg_scales=[torch.zeros(3, device="cuda")], exp_avg_sq_scales=[torch.zeros(3, device="cuda")])
    if pdtype == torch.bfloat16:
        kw["masters"] = [torch.zeros(n, device="cuda")]
    rb.optim.adamw_step([p], [g.cuda()], [m], [v], torch.zeros(1, device="cuda"), lr=1.0, betas=(b1, b2), eps=eps, weight_decay=0.0, **kw)
    m64 = (g * np.float32(1 - b1)).double()
    v64 = torch.from_numpy((g.numpy() * g.numpy()) * np.float32(1 - b2)).double()
    assert (v64 > 0).all() and (v64 < 2.0 ** -126).sum() > 100
    want = -(m64 / (1 - b1)) / (torch.sqrt(v64 / (1 - b2)) + float(np.float32(eps)))
    got = (kw["masters"][0] if pdtype == torch.bfloat16 else p).double().cpu()
    assert ((got - want).abs() <= 2.0 ** -20 * want.abs()).all(), ((got - want).abs() / want.abs()).max()


def _eight(k):
    return [torch.zeros(k, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)], [torch.zeros(k, dtype=torch.uint8, device="cuda")], \
        dict(exp_avg_scales=[torch.zeros(-(-k // 256), device="cuda")], exp_avg_sq_scales=[torch.zeros(-(-k // 256), device="cuda")])


@pytest.mark.parametrize("shift", [0, 1])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan, 1e25])
def test_8_bit_moments_lose_one_element_to_a_gradient_out_of_range(rb, bad, shift):
    """One infinity, NaN or value whose square is infinite in one step: that element's parameter and first moment are NaN from then on, and
    every other element has the bytes of a run in which the gradient was 0 there."""
    n, at = 700, 261
    runs = []
    for first in (bad, 0.0):
        p = torch.zeros(n + shift, device="cuda")[shift:]
        m, v, kw = _eight(n + shift)
        m, v = [m[0][shift:]], [v[0][shift:]]
        kw = {k: [t[0][:3].clone()] for k, t in kw.items()}
        steps = torch.zeros(1, device="cuda")
        for k in range(4):
            g = torch.randn(n, generator=torch.Generator().manual_seed(k)).cuda()
            g[at] = first if k == 0 else 0.0
            rb.optim.adamw_step([p], [g], m, v, steps, lr=0.1, **kw)
        runs.append((p, m[0].view(torch.uint8), v[0], rb.optim.first_moment_values(m[0], kw["exp_avg_scales"][0]), *[t[0] for t in kw.values()]))
    rest = torch.arange(n, device="cuda") != at
    assert torch.isnan(runs[0][0][at]) and torch.isnan(runs[0][3][at])
    for a, b in zip(*runs):
        keep = rest if a.numel() == n else slice(None)
        assert torch.equal(a[keep], b[keep])


def test_8_bit_moments_of_a_gradient_just_in_range(rb):
    """g = 1e19: the second moment, 1e35, is the largest of its block and stays finite; the parameters stay numbers."""
    n = 300
    p = torch.zeros(n, device="cuda")
    m, v, kw = _eight(n)
    steps = torch.zeros(1, device="cuda")
    for k in range(4):
        g = torch.randn(n, generator=torch.Generator().manual_seed(k)).cuda()
        if k == 0:
            g[7] = 1e19
        rb.optim.adamw_step([p], [g], m, v, steps, lr=0.1, **kw)
        assert torch.isfinite(p).all() and p.abs().max() < 0.1 * 40 * (k + 1)
        values = rb.optim.second_moment_values(v[0], kw["exp_avg_sq_scales"][0])
        assert torch.isfinite(rb.optim.first_moment_values(m[0], kw["exp_avg_scales"][0])).all()
        assert torch.isfinite(values).all() and values[7] == values.max() and values[7] > 9e34


def test_8_bit_moments_that_are_nothing_but_nan(rb):
    """A tensor of one element, and a clipping factor that is NaN: no element of the block is a number, and the state says so."""
    for n, gs in ((1, None), (300, torch.full((), math.nan, device="cuda"))):
        p = torch.ones(n, device="cuda")
        m, v, kw = _eight(n)
        steps = torch.zeros(1, device="cuda")
        rb.optim.adamw_step([p], [torch.full((n,), math.nan if gs is None else 1.0, device="cuda")], m, v, steps, grad_scale=gs, **kw)
        assert torch.isnan(p).all() and torch.isnan(rb.optim.first_moment_values(m[0], kw["exp_avg_scales"][0])).all()
        rb.optim.adamw_step([p.fill_(1.0)], [torch.ones(n, device="cuda")], m, v, steps, **kw)
        assert torch.isnan(p).all()


def test_the_first_step_is_not_captured(rb):
    p = torch.nn.Parameter(torch.ones(8, device="cuda"))
    p.grad = torch.ones_like(p)
    opt = rb.optim.AdamW([p], lr=0.1)
    torch.cuda.synchronize()
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        with pytest.raises(RuntimeError, match="cannot be captured"):
            opt.step()
    opt.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    graph.replay()
    torch.cuda.synchronize()
    assert opt.state[p]["step"].item() == 2


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("sizes", [(1e25,), (1e-25,), (1e20, 1e-3), (1e-25, 1e-22, 0.0)])
def test_grad_norm_of_values_whose_squares_leave_the_range(rb, dtype, sizes):
    """g^2 is infinite or 0 in float32, the norm is neither."""
    g = torch.Generator().manual_seed(1)
    grads = [(torch.randn(k, generator=g).double() * s).to(dtype).cuda() for k in (3, 8192, 20001) for s in sizes]
    want = math.sqrt(sum(float((t.double() ** 2).sum()) for t in grads))
    norm, f = rb.optim.grad_norm(grads, max_norm=0.5)
    # the eight squares a lane adds, as in test_grad_norm
    assert abs(norm.item() / want - 1) <= 8 * U
    assert abs(f.item() / min(1.0, 0.5 / (want + 1e-6)) - 1) <= 12 * U


@pytest.mark.parametrize("gdtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("shift", [0, 1])
def test_masters_step_as_float32_parameters_do(rb, gdtype, bits, shift):
    """bf16 parameters with masters, either moments, either gradient type: masters and state are bit for bit those of float32 parameters, the
    parameters their rounding."""
    n = sum(SIZES)
    runs = []
    for pdtype in (torch.float32, torch.bfloat16):
        ps, grads, ms, vs, carve = make(SIZES, pdtype, gdtype, 11, shift)
        start = carve(torch.randn(n, generator=torch.Generator().manual_seed(12)))
        kw = {}
        if bits == 8:
            ms, vs = [t.view(torch.float8_e4m3fn) for t in carve(torch.zeros(n, dtype=torch.uint8))], carve(torch.zeros(n, dtype=torch.uint8))
            kw = {k: [torch.zeros(-(-t.numel() // 256), device="cuda") for t in ps] for k in ("exp_avg_scales", "exp_avg_sq_scales")}
        if pdtype == torch.bfloat16:
            kw["masters"] = start
        else:
            ps = start
        steps = torch.zeros(len(SIZES), device="cuda")
        for _ in range(3):
            rb.optim.adamw_step(ps, grads, ms, vs, steps, lr=1e-2, seed=5, **kw)
        runs.append((start, [t.view(torch.uint8) for t in ms], [t.view(torch.uint8) for t in vs]))
    for a, b in zip(*runs):
        assert all(torch.equal(x, y) for x, y in zip(a, b))
    assert all(torch.equal(p, w.to(torch.bfloat16)) for p, w in zip(ps, runs[1][0]))
