"""The training-step operators of a model with a large output vocabulary, as they are measured.

Three operators that one training step uses one after the other:

* ``noise_cross_entropy``   softmax cross entropy over a pseudorandom vocabulary matrix: logits = z S^T with S the layer's
                            Squirrel5 noise, regenerated from a seed; gives the loss and the gradient of z;
* ``linear_cross_entropy``  the same over a stored vocabulary matrix W: loss, gradient of x, gradient of W;
* ``adamw_step``            AdamW over a list of tensors, moments in 32 or in 8 bits, with ``grad_norm`` for clipping.

``run`` computes each in its plain form (elementary torch operations in 32 bits) or, where ``own`` is true, with the calls of
this package that a training program makes.  ``exact`` computes the same from the definitions in 64 bits.
"""
import math

import numpy as np
import torch

own = False

DEV = "cuda"
IGNORE = -100
N1, N2, N3, N4, N5, PRIME = 0xD2A80A3F, 0xA884F197, 0x6C736F4B, 0xB79F3ABB, 0x1B56C4F5, 198491317
MASK = 0xFFFFFFFF
BLOCK = 256                     # elements that share one scale of an 8-bit moment
TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # scoring one token with a pseudorandom head: all latency
        dict(name="noise head, 1 token, loss", op="noise_ce", T=1, R=128, V=50257, dtype="bf16", grad=False, ignored=0.0, reduction="mean"),
        # a training step of a pseudorandom head: 8 sequences of 1024 tokens, coefficient dimension of the headline layer
        dict(name="noise head, 8192 tokens, training", op="noise_ce", T=8192, R=1024, V=50257, dtype="bf16", grad=True, ignored=0.0, reduction="mean"),
        # fine-tuning on answers only: a padded batch whose prompts carry no loss, sizes that divide by nothing, weighted outside
        dict(name="noise head, 1531 tokens, 40 % ignored", op="noise_ce", T=1531, R=200, V=32003, dtype="bf16", grad=True, ignored=0.4, reduction="none"),
        # the same layer trained in float32
        dict(name="noise head, 1024 tokens, float32", op="noise_ce", T=1024, R=256, V=10007, dtype="fp32", grad=True, ignored=0.1, reduction="sum"),
        # the stored head of the benchmark's whole training step: d 768, vocabulary 50257, 8 x 1024 tokens
        dict(name="stored head, 8192 tokens, training", op="linear_ce", T=8192, R=768, V=50257, dtype="bf16", grad=True, ignored=0.0, reduction="mean"),
        # validation of a wider model: the loss of every token
        dict(name="stored head, 4096 tokens, loss", op="linear_ce", T=4096, R=2048, V=32000, dtype="bf16", grad=False, ignored=0.05, reduction="none"),
        # a short batch in float32, odd sizes
        dict(name="stored head, 777 tokens, float32", op="linear_ce", T=777, R=250, V=8191, dtype="fp32", grad=True, ignored=0.2, reduction="mean"),
        # the coefficient matrices of 24 layers: many small tensors
        dict(name="AdamW, 24 coefficient matrices", op="adamw", sizes="24x98304", dtype="fp32", bits=32, master=False, clip=False),
        # every weight of the benchmark's training step in bf16, kept beside in float32, gradients clipped
        dict(name="AdamW, whole model, bf16 with float32 masters, clipped", op="adamw",
             sizes="1x38597376,1x786432,48x768,48x589824,24x98304", dtype="bf16", bits=32, master=True, clip=True),
        # the same model's float32 weights with 8-bit moments
        dict(name="AdamW, whole model, 8-bit moments", op="adamw", sizes="1x38597376,1x786432,48x768,48x589824,24x98304", dtype="fp32", bits=8,
             master=False, clip=False),
        # odd tensors (biases, a convolution, scales) with 8-bit moments, clipped
        dict(name="AdamW, odd tensors, 8-bit moments, clipped", op="adamw", sizes="40x1,30x777,20x50001,3x1000003", dtype="fp32", bits=8, master=False,
             clip=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["noise_ce", "linear_ce", "adamw"])
    if kind == "adamw":
        left, parts = 66_000_000, []
        for _ in range(rng.randint(1, 5)):
            n = _log(rng, 1, 20_000_000)
            c = max(1, min(_log(rng, 1, 60), left // n))
            if c * n <= left:
                left -= c * n
                parts.append("%dx%d" % (c, n))
        dtype = rng.choice(["bf16", "fp32"])
        return dict(op="adamw", sizes=",".join(parts or ["1x1000"]), dtype=dtype, bits=rng.choice([8, 32]), master=dtype == "bf16" and rng.random() < 0.5,
                    clip=rng.random() < 0.5)
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    most = 4.2e11 if dtype == "bf16" else 6e9                  # T V R of the largest listed case of the type
    while True:
        T, R, V = _log(rng, 1, 16384), _log(rng, 16, 2048), _log(rng, 300, 65536)
        if rng.random() < 0.5:
            R = max(8, R // 8 * 8)
        if T * V * R <= most:
            break
    return dict(op=kind, T=T, R=R, V=V, dtype=dtype, grad=rng.random() < 0.7, ignored=rng.choice([0.0, 0.1, 0.5]),
                reduction=rng.choice(["mean", "sum", "none"]))


def _tensors(case):
    return [int(n) for part in case["sizes"].split(",") for n in [part.split("x")[1]] * int(part.split("x")[0])]


def work(case):
    if case["op"] == "adamw":
        n = sum(_tensors(case))
        ps = 2 if case["dtype"] == "bf16" else 4
        moments = 2 * (4 if case["bits"] == 32 else 1 + 4 / BLOCK)
        # parameter (and float32 master) read and written, gradient read, both moments read and written
        return {"bytes": n * (2 * ps + (8 if case["master"] else 0) + ps + 2 * moments), "flops": 0}
    T, R, V = case["T"] * (1 - case["ignored"]), case["R"], case["V"]
    es = 2 if case["dtype"] == "bf16" else 4
    stored = case["op"] == "linear_ce"
    products = (3 if stored else 2) if case["grad"] else 1     # logits; gradient of the rows; gradient of the matrix
    nbytes = case["T"] * R * es + case["T"] * 8 + (V * R * es if stored else 0)
    if case["grad"]:
        nbytes += case["T"] * R * es + (V * R * es if stored else 0)
    return {"bytes": nbytes, "flops": 2.0 * T * V * R * products}


# ------------------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    dt = TYPES[case["dtype"]]
    if case["op"] == "adamw":
        sizes = _tensors(case)
        n = sum(sizes)
        offs = np.concatenate([[0], np.cumsum(sizes)]).tolist()

        def split(flat):
            return [flat[a:b] for a, b in zip(offs, offs[1:])]

        s = {"case": case, "sizes": sizes}
        # parameters of a trained model; gradients whose scale changes from one stretch of rows to the next, some exactly zero
        base = torch.randn(n, device=DEV, generator=g) * 0.02
        stretch = torch.exp(torch.randn((n + 767) // 768, device=DEV, generator=g)).repeat_interleave(768)[:n]
        grad = torch.randn(n, device=DEV, generator=g) * 1e-3 * stretch
        grad *= torch.rand(n, device=DEV, generator=g) > 0.02
        m = (0.7 * torch.randn(n, device=DEV, generator=g) * 1e-3 * stretch)
        v = (torch.rand(n, device=DEV, generator=g) + 0.3) * 1e-6 * stretch * stretch
        s["param"], s["grad"] = base.to(dt), grad.to(dt)
        s["params"], s["grads"] = split(s["param"]), split(s["grad"])
        s["masters"] = None
        if case["master"]:
            s["master"] = base.clone()
            s["masters"] = split(s["master"])
        s["steps"] = torch.full((len(sizes),), 100.0, device=DEV)
        s["seed"] = int(seed) & 0x7FFF
        if case["bits"] == 32:
            s["m"], s["v"] = m, v
            s["ms"], s["vs"] = split(m), split(v)
        else:
            s["lay"] = lay = _layout(sizes)
            (s["m"], s["m_scale"]), (s["v"], s["v_scale"]) = _quant_m(m, lay), _quant_v(v, lay, None)
            s["ms"], s["vs"] = split(s["m"]), split(s["v"])
            boffs = lay["block_offsets"]
            s["m_scales"] = [s["m_scale"][a:b] for a, b in zip(boffs, boffs[1:])]
            s["v_scales"] = [s["v_scale"][a:b] for a, b in zip(boffs, boffs[1:])]
        s["hyper"] = dict(lr=3e-4, betas=(0.9, 0.95), eps=1e-8, weight_decay=0.1)
        return s
    T, R, V = case["T"], case["R"], case["V"]
    target = torch.randint(0, V, (T,), device=DEV, generator=g)
    known = torch.rand(T, 1, device=DEV, generator=g) * 8.0    # how far the model has learned each token, in logits
    s = {"case": case, "noise_seed": int(seed) * 7919 + 17, "row0": 0}
    if case["op"] == "noise_ce":
        # logits of standard deviation 2 around the rows of the targets: noise has variance 1/3
        rows = _noise(target, R, s["noise_seed"])
        x = torch.randn(T, R, device=DEV, generator=g) * (2.0 * (3.0 / R) ** 0.5) + rows * (known * 3.0 / R)
        s["x"] = x.to(dt)
    else:
        w = torch.randn(V, R, device=DEV, generator=g) * (2.0 / R ** 0.5)
        s["w"] = w.to(dt)
        s["x"] = (torch.randn(T, R, device=DEV, generator=g) + w[target] * (known / 4.0)).to(dt)
    if case["ignored"]:
        skip = torch.rand(T, device=DEV, generator=g) < case["ignored"]
        target = target.masked_fill(skip, IGNORE)
    if case["reduction"] == "none":
        s["weights"] = torch.rand(T, device=DEV, generator=g)  # what the program weighs each token's loss with
    s["target"] = target
    return s


# ------------------------------------------------------------------------------------------------ one pass
def run(s):
    if s["case"]["op"] == "adamw":
        return _adamw_own(s) if own else _adamw_plain(s)
    return _ce_own(s) if own else _ce_plain(s)


def _ce_own(s):
    import randumb_b200 as rb
    c = s["case"]
    x = s["x"].detach()
    leaves = [x] if c["op"] == "noise_ce" else [x, s["w"].detach()]
    if c["grad"]:
        leaves = [t.requires_grad_() for t in leaves]
    if c["op"] == "noise_ce":
        loss = rb.ops.noise_cross_entropy(leaves[0], s["noise_seed"], c["V"], s["target"], row0=s["row0"], ignore_index=IGNORE, reduction=c["reduction"])
    else:
        loss = rb.ops.linear_cross_entropy(leaves[0], leaves[1], s["target"], ignore_index=IGNORE, reduction=c["reduction"])
    if not c["grad"]:
        return {"loss": loss}
    grads = torch.autograd.grad(loss, leaves, s["weights"] if c["reduction"] == "none" else None)
    return {"loss": loss.detach(), "dx": grads[0], "dw": grads[1] if len(grads) > 1 else []}


def _ce_plain(s):
    c = s["case"]
    w = _noise(torch.arange(c["V"], device=DEV), c["R"], s["noise_seed"]).to(s["x"].dtype) if c["op"] == "noise_ce" else s["w"]
    x, w = s["x"].float(), w.float()
    keep = s["target"] != IGNORE
    t = s["target"].clamp(min=0)
    logits = x @ w.t()
    top = logits.amax(1, keepdim=True)
    e = torch.exp(logits - top)
    total = e.sum(1, keepdim=True)
    rows = (top + torch.log(total) - logits.gather(1, t[:, None]))[:, 0]
    rows = torch.where(keep, rows, torch.zeros_like(rows))
    count = keep.sum().float()
    loss = rows if c["reduction"] == "none" else rows.sum() if c["reduction"] == "sum" else rows.sum() / count
    if not c["grad"]:
        return {"loss": loss}
    share = s["weights"] if c["reduction"] == "none" else torch.ones_like(rows) if c["reduction"] == "sum" else torch.ones_like(rows) / count
    share = torch.where(keep, share, torch.zeros_like(share))
    p = e / total
    p[torch.arange(c["T"], device=DEV), t] -= 1.0
    p *= share[:, None]
    dt = s["x"].dtype
    return {"loss": loss, "dx": (p @ w).to(dt), "dw": (p.t() @ x).to(dt) if c["op"] == "linear_ce" else []}


def _adamw_own(s):
    import randumb_b200 as rb
    c, scale = s["case"], None
    out = {"param": s["param"]}
    if c["clip"]:
        out["norm"], scale = rb.optim.grad_norm(s["grads"], max_norm=1.0)
    eight = {} if c["bits"] == 32 else dict(exp_avg_scales=s["m_scales"], exp_avg_sq_scales=s["v_scales"], seed=s["seed"])
    rb.optim.adamw_step(s["params"], s["grads"], s["ms"], s["vs"], s["steps"], masters=s["masters"], grad_scale=scale, **s["hyper"], **eight)
    return _adamw_out(s, out)


def _adamw_out(s, out):
    if s["case"]["master"]:
        out["master"] = s["master"]
    # 8-bit moments: the first as what it is, float8 values and their scales; the second, whose bytes are no float type of torch, as numbers
    out["m"] = s["m"]
    out["v"] = s["v"] if s["case"]["bits"] == 32 else _ue4m4(s["v"])
    if s["case"]["bits"] == 8:
        out["m_scale"], out["v_scale"] = s["m_scale"], s["v_scale"]
    out["steps"] = s["steps"]
    return out


def _adamw_plain(s):
    c, h = s["case"], s["hyper"]
    b1, b2 = h["betas"]
    g = s["grad"].float()
    out = {"param": s["param"]}
    if c["clip"]:
        out["norm"] = torch.sqrt((g * g).sum())
        g = g * torch.clamp(1.0 / (out["norm"] + 1e-6), max=1.0)
    s["steps"] += 1.0
    t = s["steps"].double()
    sizes = torch.tensor(s["sizes"], device=DEV)

    def spread(per_tensor):
        return torch.repeat_interleave(per_tensor.float(), sizes, output_size=g.numel())

    size = spread(h["lr"] / (1.0 - b1 ** t))
    root = spread(torch.sqrt(1.0 - b2 ** t))
    m = s["m"] if c["bits"] == 32 else s["m"].float() * _per_element(s["m_scale"], s["lay"])
    v = s["v"] if c["bits"] == 32 else _ue4m4(s["v"]) * _per_element(s["v_scale"], s["lay"])
    m = m * b1 + g * (1.0 - b1)
    v = v * b2 + g * g * (1.0 - b2)
    p = s["master"] if c["master"] else s["param"].float()
    p = p * (1.0 - h["lr"] * h["weight_decay"]) - size * (m / (torch.sqrt(v) / root + h["eps"]))
    if c["master"]:
        s["master"].copy_(p)
    s["param"].copy_(p)
    if c["bits"] == 32:
        s["m"].copy_(m)
        s["v"].copy_(v)
    else:
        for name, (codes, scale) in (("m", _quant_m(m, s["lay"])), ("v", _quant_v(v, s["lay"], _round_bits(s)))):
            s[name].copy_(codes)
            s[name + "_scale"].copy_(scale)
    return _adamw_out(s, out)


# ------------------------------------------------------------------------------------------------ pieces of the plain forms
def _mix(b):
    """Squirrel5's mixing of 32-bit words held in int64."""
    b = b ^ (b >> 9)
    b = (b + N2) & MASK
    b = b ^ (b >> 11)
    b = (b * N3) & MASK
    b = b ^ (b >> 13)
    b = (b + N4) & MASK
    b = b ^ (b >> 15)
    b = (b * N5) & MASK
    return b ^ (b >> 17)


def _noise(rows, cols, seed):
    """float32 noise rows: word of position PRIME * row + col, as a signed number times 2^-31."""
    pos = (rows[:, None] * PRIME + torch.arange(cols, device=rows.device)[None, :]) & MASK
    bits = _mix((pos * N1 + (seed & MASK)) & MASK)
    return bits.to(torch.int32).float() * 2.0 ** -31


def _layout(sizes):
    """Blocks of BLOCK consecutive elements of each tensor share a scale: block of every element, and each tensor's first block."""
    per = [-(-n // BLOCK) for n in sizes]
    block_offsets = np.concatenate([[0], np.cumsum(per)]).tolist()
    n = torch.tensor(sizes, device=DEV)
    which = torch.repeat_interleave(torch.arange(len(sizes), device=DEV), n)
    first = torch.cumsum(n, 0) - n
    index = torch.arange(int(sum(sizes)), device=DEV) - first[which]
    block = torch.tensor(block_offsets[:-1], device=DEV)[which] + index // BLOCK
    return {"block": block, "which": which.int(), "index": index.int(), "blocks": block_offsets[-1], "block_offsets": block_offsets}


def _per_element(scale, lay):
    return scale[lay["block"]]


def _block_max(x, lay):
    return torch.zeros(lay["blocks"], device=x.device, dtype=x.dtype).scatter_reduce_(0, lay["block"], x, "amax")


def _quant_m(m, lay):
    """First moment: float8 e4m3, the block's largest magnitude at 448, rounded to nearest."""
    scale = _block_max(m.abs(), lay) / 448.0
    at = _per_element(scale, lay)
    q = torch.where(at > 0, m / at, torch.zeros_like(m)).clamp(-448.0, 448.0)
    return q.float().to(torch.float8_e4m3fn), scale.float()


def _ue4m4(codes):
    """Values of the second moment's bytes: 4 exponent bits (bias 15) and 4 mantissa bits, no sign; byte 255 stands for 1.9375."""
    return (codes.to(torch.int32) << 19).view(torch.float32) * 2.0 ** 112


def _quant_v(v, lay, bits):
    """Second moment: the byte at or below v / scale, or the next one, by 19 random bits (none: the one below); never 0 for a positive value."""
    scale = _block_max(v, lay) / 1.9375
    at = _per_element(scale, lay)
    q = torch.where(at > 0, v / at, torch.zeros_like(v)).float() * 2.0 ** -112
    word = q.view(torch.int32)
    codes = ((word + (0 if bits is None else bits)) >> 19).clamp(max=255)
    codes = torch.where((codes == 0) & (v > 0), torch.ones_like(codes), codes)
    return codes.to(torch.uint8), scale.float()


def _round_bits(s):
    """19 bits for each element: the noise word of position (index in the tensor) under a seed of its own for each tensor and step."""
    lay = s["lay"]
    step = s["steps"].long()[lay["which"].long()]
    seed = (s["seed"] + step * 0x9E3779B1 + lay["which"].long() * 0x85EBCA6B) & MASK
    return (_mix(((lay["index"].long() & MASK) * N1 + seed) & MASK) >> 13).int()


# ------------------------------------------------------------------------------------------------ definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return _adamw_exact(s) if case["op"] == "adamw" else _ce_exact(s)


def _noise_words(rows, cols, seed):
    """The noise words again, in numpy's wrapping 32-bit arithmetic."""
    with np.errstate(over="ignore"):
        r = np.asarray(rows).astype(np.uint32)[:, None]
        h = (np.uint32(PRIME) * r + np.arange(cols, dtype=np.uint32)[None, :]) * np.uint32(N1) + np.uint32(seed & MASK)
        for shift, add, mul in ((9, N2, None), (11, None, N3), (13, N4, None), (15, None, N5)):
            h ^= h >> np.uint32(shift)
            h = h + np.uint32(add) if add is not None else h * np.uint32(mul)
        h ^= h >> np.uint32(17)
    return h


def _ce_exact(s):
    c, dt = s["case"], torch.float64
    T, V, R = c["T"], c["V"], c["R"]
    if c["op"] == "noise_ce":
        words = _noise_words(np.arange(V), R, s["noise_seed"])
        w = (torch.from_numpy(words.view(np.int32)).to(DEV).to(torch.float32) * 2.0 ** -31).to(s["x"].dtype).to(dt)
    else:
        w = s["w"].to(dt)
    x = s["x"].to(dt)
    valid = torch.nonzero(s["target"] != IGNORE)[:, 0]
    n = max(int(valid.numel()), 0)
    loss_rows = torch.zeros(T, device=DEV, dtype=dt)
    dx = torch.zeros(T, R, device=DEV, dtype=dt)
    dw = torch.zeros(V, R, device=DEV, dtype=dt)
    for part in torch.split(valid, 1024):
        xt, tt = x[part], s["target"][part]
        lp = torch.log_softmax(xt @ w.t(), dim=1)
        loss_rows[part] = -lp.gather(1, tt[:, None])[:, 0]
        if c["grad"]:
            k = s["weights"][part].to(dt) if c["reduction"] == "none" else torch.full((part.numel(),), 1.0 if c["reduction"] == "sum" else 1.0 / n, device=DEV, dtype=dt)
            p = torch.exp(lp)
            p.scatter_add_(1, tt[:, None], torch.full_like(tt[:, None], -1, dtype=dt))
            p = p * k[:, None]
            dx[part] = p @ w
            if c["op"] == "linear_ce":
                dw += p.t() @ xt
    loss = loss_rows if c["reduction"] == "none" else loss_rows.sum() if c["reduction"] == "sum" else loss_rows.sum() / (n if n else float("nan"))
    if not c["grad"]:
        return {"loss": loss}
    return {"loss": loss, "dx": dx, "dw": dw if c["op"] == "linear_ce" else []}


def _adamw_exact(s):
    c, h, dt = s["case"], s["hyper"], torch.float64
    out = {}
    g = s["grad"].to(dt)
    if c["clip"]:
        out["norm"] = torch.linalg.vector_norm(g)
        g = g * min(1.0, 1.0 / (float(out["norm"]) + 1e-6))
    t = float(s["steps"][0]) + 1.0
    s["steps"].fill_(t)
    eight = c["bits"] == 8
    m = s["m"].to(dt) if not eight else s["m"].to(dt) * s["m_scale"].to(dt)[s["lay"]["block"]]
    v = s["v"].to(dt) if not eight else _ue4m4(s["v"]).to(dt) * s["v_scale"].to(dt)[s["lay"]["block"]]
    b1, b2 = h["betas"]
    m += (g - m) * (1.0 - b1)
    v += (g * g - v) * (1.0 - b2)
    p = (s["master"] if c["master"] else s["param"]).to(dt)
    p -= h["lr"] * (h["weight_decay"] * p + (m / (1.0 - b1 ** t)) / ((v / (1.0 - b2 ** t)).sqrt() + h["eps"]))
    out["param"] = p
    if c["master"]:
        out["master"] = p
    if eight:
        # a moment next to a border between two 8-bit values may round to either: their scales have a value in 64 bits, the bytes have none
        out["m"] = out["v"] = None
        out["m_scale"] = _block_max(m.abs(), s["lay"]) / 448.0
        out["v_scale"] = _block_max(v, s["lay"]) / 1.9375
    else:
        out["m"], out["v"] = m, v
    out["steps"] = s["steps"]
    return out
