"""Host side of the training operators (cross entropy, AdamW, gradient norm): refusals before any launch, CPU tensors, tracing,
planning.  CPU only -- no kernel runs here."""
import copy
import ctypes
import pickle

import pytest
import torch

import randumb_b200 as rb
from randumb_b200 import _lib

OK, WS, BIG = 0x7F0000001000, 0x7F0000100000, 1 << 40          # addresses that are checked, never dereferenced
LOSS, LOSS_GRAD, GRADS = _lib.CE_LOSS, _lib.CE_LOSS_GRAD, _lib.CE_GRADS
NONE, MEAN, SUM = (_lib.CE_REDUCTIONS[k] for k in ("none", "mean", "sum"))


def fwd(L, loss=OK, aux=OK, unit=None, x=OK, ldx=64, w=None, ldw=0, target=OK, ws=WS, nbytes=BIG, T=10, R=64, V=100, dtype=_lib.BF16, reduction=MEAN):
    return L.rdb_ce_fwd(loss, aux, unit, x, ldx, w, ldw, target, ws, nbytes, T, R, V, 0, 0, -100, 1, dtype, reduction, None, None)


def bwd(L, dx=OK, dw=OK, dloss=OK, x=OK, ldx=64, w=OK, ldw=64, target=OK, aux=OK, ws=WS, nbytes=BIG, T=10, R=64, V=100, dtype=_lib.BF16, reduction=MEAN):
    return L.rdb_ce_bwd(dx, dw, dloss, x, ldx, w, ldw, target, aux, ws, nbytes, T, R, V, -100, 1, dtype, reduction, None, None)


def test_cross_entropy_refusals(built_lib):
    L = _lib.lib()
    assert fwd(L, T=-1) == -2 and fwd(L, V=0) == -2 and fwd(L, R=0) == -2 and fwd(L, ldx=63) == -2 and fwd(L, w=OK, ldw=63) == -2
    assert fwd(L, dtype=5) == -3 and fwd(L, reduction=7) == -6
    assert fwd(L, aux=None) == -1 and fwd(L, loss=None) == -1 and fwd(L, x=None) == -1 and fwd(L, target=None) == -1
    assert fwd(L, x=OK + 1) == -4 and fwd(L, target=OK + 4) == -4 and fwd(L, x=OK + 2, dtype=_lib.F32) == -4
    assert fwd(L, w=OK, ldw=64, unit=OK) == -6                      # a stored matrix has its gradients in the backward call
    assert fwd(L, T=1 << 40) == -8 and fwd(L, V=1 << 40) == -8 and fwd(L, R=1 << 30, ldx=1 << 30) == -8
    need = L.rdb_ce_workspace_bytes(LOSS, 10, 64, 100, _lib.BF16, None, 0)
    assert fwd(L, nbytes=need - 1) == -5 and fwd(L, ws=WS + 8) == -5 and fwd(L, ws=None) == -5
    assert bwd(L, dx=None, dw=None) == 0                            # nothing asked for
    assert bwd(L, w=None) == -1 and bwd(L, dloss=None) == -1 and bwd(L, aux=None) == -1 and bwd(L, dw=OK + 1) == -4
    assert bwd(L, nbytes=1024) == -5 and bwd(L, T=-1) == -2
    assert L.rdb_ce_scale(OK, OK, OK, None, 4, 8, _lib.BF16, MEAN, None) == -1
    assert L.rdb_ce_scale(None, None, None, None, 0, 8, _lib.BF16, MEAN, None) == 0
    assert L.rdb_ce_scale(OK, OK, OK, OK, 4, 8, _lib.BF16, 9, None) == -6


def test_cross_entropy_workspace(built_lib):
    """The logits never fit the workspace of a large problem: pieces of at most 512 MB; a stored bf16 matrix with aligned rows is read in
    place, any other goes through the workspace piece by piece."""
    L = _lib.lib()
    T, R, V = 65536, 1024, 50257
    logits = T * V * 2
    for op, w in ((LOSS_GRAD, None), (GRADS, OK)):
        need = L.rdb_ce_workspace_bytes(op, T, R, V, _lib.BF16, w, R)
        assert need < 0.5 * logits
    assert L.rdb_ce_workspace_bytes(LOSS, 8192, R, V, _lib.BF16, OK, R) < 64 << 20
    in_place = L.rdb_ce_workspace_bytes(LOSS, 512, R, V, _lib.BF16, OK, R)
    assert L.rdb_ce_workspace_bytes(LOSS, 512, R, V, _lib.BF16, OK, R + 1) >= in_place + V * R * 2      # rows off the 16-byte boundary
    assert L.rdb_ce_workspace_bytes(LOSS, 512, R, V, _lib.BF16, OK + 2, R) >= in_place + V * R * 2
    assert L.rdb_ce_workspace_bytes(LOSS, 512, R, V, _lib.F32, OK, R) >= in_place                        # three bf16 parts of a piece
    assert L.rdb_ce_workspace_bytes(LOSS, 0, R, V, _lib.BF16, OK, R) > 0


def lists(n=1, **over):
    words = dict(param=OK, grad=OK, exp_avg=OK, exp_avg_sq=OK, step=OK)
    words.update(over)
    keep = {k: (ctypes.c_uint64 * n)(*([v] * n if not isinstance(v, list) else v)) for k, v in words.items() if k != "numel" and v is not None}
    keep["numel"] = (ctypes.c_int64 * n)(*([over.get("numel", 8)] * n))
    return _lib.AdamwLists(n=n, **{k: ctypes.addressof(v) for k, v in keep.items()}), keep


def test_adamw_and_norm_refusals(built_lib):
    L = _lib.lib()
    h = _lib.AdamwHyper(1e-3, 0.9, 0.99, 1e-8, 0.0, None, 0)

    def step(pd=_lib.F32, gd=_lib.F32, bits=32, hyper=h, **over):
        arg, keep = lists(**over)
        return L.rdb_adamw_step(ctypes.byref(arg), pd, gd, bits, ctypes.byref(hyper), None, None)

    assert L.rdb_adamw_step(None, 0, 0, 32, ctypes.byref(h), None, None) == -1
    assert step(param=None) == -1 and step(numel=-1) == -2 and step(step=0) == -1 and step(grad=0) == -1
    assert step(pd=7) == -3 and step(bits=16) == -3 and step(bits=8) == -1
    assert step(param=OK + 2) == -4 and step(pd=_lib.BF16, param=OK + 1) == -4 and step(exp_avg=OK + 1) == -4 and step(step=OK + 2) == -4
    assert step(bits=8, exp_avg_scale=OK + 2, exp_avg_sq_scale=OK) == -4 and step(bits=8, exp_avg_scale=OK, exp_avg_sq_scale=OK + 1) == -4
    assert step(hyper=_lib.AdamwHyper(1e-3, 0.9, 0.99, 1e-8, 0.0, OK + 2, 0)) == -4
    assert step(master=OK) == -6                                    # masters are the float32 copies of bf16 parameters
    for bad in (_lib.AdamwHyper(1e-3, 1.0, 0.99, 1e-8, 0.0, None, 0), _lib.AdamwHyper(1e-3, 0.9, float("nan"), 1e-8, 0.0, None, 0),
                _lib.AdamwHyper(1e-3, 0.9, 0.99, -1.0, 0.0, None, 0)):
        assert step(hyper=bad) == -6
    empty = _lib.AdamwLists(n=0)
    assert L.rdb_adamw_step(ctypes.byref(empty), 0, 0, 32, ctypes.byref(h), None, None) == 0
    ptr, num, typ = (ctypes.c_uint64 * 1)(OK), (ctypes.c_int64 * 1)(8), (ctypes.c_int32 * 1)(0)
    need = L.rdb_grad_norm_workspace_bytes(1)
    norm = lambda *a: L.rdb_grad_norm(*a, None)                     # noqa: E731
    assert norm(None, None, ptr, num, typ, 1, 1.0, WS, need) == -1 and norm(OK, None, None, num, typ, 1, 1.0, WS, need) == -1
    assert norm(OK, OK, ptr, num, typ, 1, -1.0, WS, need) == -6 and norm(OK, OK, ptr, num, typ, 1, float("nan"), WS, need) == -6
    assert norm(OK, None, ptr, num, typ, 1, 0.0, WS, need - 1) == -5 and norm(OK, None, ptr, num, typ, -1, 0.0, WS, need) == -2
    assert norm(OK, None, ptr, num, (ctypes.c_int32 * 1)(3), 1, 0.0, WS, need) == -3
    assert norm(OK, None, (ctypes.c_uint64 * 1)(OK + 2), num, typ, 1, 0.0, WS, need) == -4


def test_cpu_tensors_are_refused():
    x, w, t = torch.ones(2, 3), torch.ones(5, 3), torch.zeros(2, dtype=torch.int64)
    with pytest.raises(NotImplementedError, match="Unsupported CPU implementation"):
        rb.noise_cross_entropy(x, 1, 5, t)
    with pytest.raises(NotImplementedError, match="Unsupported CPU implementation"):
        rb.linear_cross_entropy(x, w, t)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        rb.kernels.ce_fwd(x, w, t)
    for far in (2 ** 63, -2 ** 63 - 1, 2 ** 64):                     # would be another value in 64 bits
        with pytest.raises(RuntimeError, match="ignore_index"):
            rb.kernels.ce_fwd(x, w, t, far)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        rb.optim.adamw_step([x], [x], [x], [x], torch.zeros(1))
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        rb.optim.grad_norm([x])
    with pytest.raises(RuntimeError, match="no gradients"):
        rb.optim.grad_norm([])
    with pytest.raises(RuntimeError, match="does not match"):
        rb.noise_cross_entropy(x, 1, 5, t[:1])
    rb.optim.adamw_step([], [], [], [], torch.zeros(0))


def test_fake_tensors_give_shapes():
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        z = torch.empty(4, 6, 16, device="cuda", dtype=torch.bfloat16, requires_grad=True)
        w = torch.empty(30, 16, device="cuda", dtype=torch.bfloat16, requires_grad=True)
        t = torch.empty(4, 6, device="cuda", dtype=torch.int64)
        loss = rb.noise_cross_entropy(z, 1, 30, t)
        assert loss.shape == () and loss.dtype == torch.float32
        _, aux, unit = rb.ops.noise_ce_fwd(z.reshape(24, 16), t.reshape(24), 1, 30, 0, -100, "mean", True)
        dz = rb.ops.noise_ce_bwd(loss, unit, aux, "mean", z.dtype)          # (the engine itself needs a device)
        assert dz.shape == (24, 16) and dz.dtype == z.dtype
        rows = rb.linear_cross_entropy(z, w, t, reduction="none")
        assert rows.shape == (4, 6)
        dz, dw = rb.ops.linear_ce_bwd(rows.reshape(24), z.reshape(24, 16), w, t.reshape(24), aux, None, "none", False, True)
        assert dz.shape == (0,) and dw.shape == w.shape and dw.dtype == w.dtype


def test_optimizer_arguments():
    p = torch.nn.Parameter(torch.zeros(3))
    for bad in (dict(lr=-1.0), dict(lr=float("nan")), dict(betas=(1.0, 0.9)), dict(betas=(0.9, -0.1)), dict(eps=-1.0), dict(weight_decay=-1.0),
                dict(state_bits=16), dict(max_grad_norm=-1.0)):
        with pytest.raises(ValueError):
            rb.optim.AdamW([p], **bad)
    opt = rb.optim.AdamW([p])
    opt.step()                                                      # no gradients: nothing to do
    two = rb.optim.AdamW([p], max_grad_norm=0.5, seed=7, state_bits=8)
    for c in (copy.deepcopy(two), pickle.loads(pickle.dumps(two))):
        assert (c.max_grad_norm, c.seed, c.last_grad_norm, c.param_groups[0]["state_bits"]) == (0.5, 7, None, 8)
        c.step()
    p.grad = torch.ones(3)
    with pytest.raises(RuntimeError, match="CUDA parameters"):
        opt.step()
    with pytest.raises(RuntimeError, match="one block of memory"):
        rb.optim._flat(torch.zeros(4, 4)[:, :2])
    assert rb.optim._flat(torch.arange(12).view(3, 4).t()).tolist() == list(range(12))


def test_optimizer_refuses_options_that_it_does_not_have():
    """maximize, amsgrad, differentiable and coupled weight decay (torch.optim.Adam's) are refused where a group or a checkpoint asks for them, and
    a refused checkpoint leaves the optimiser as it was."""
    p = torch.nn.Parameter(torch.zeros(3))
    for bad in (dict(maximize=True), dict(amsgrad=True), dict(differentiable=True), dict(decoupled_weight_decay=False, weight_decay=0.1), dict(state_bits=16)):
        with pytest.raises(ValueError):
            rb.optim.AdamW([{"params": [p], **bad}])
    rb.optim.AdamW([{"params": [p], "maximize": False, "decoupled_weight_decay": False, "weight_decay": 0.0}])
    q = torch.nn.Parameter(torch.zeros(3))
    for other in (torch.optim.AdamW([q], maximize=True), torch.optim.AdamW([q], amsgrad=True), torch.optim.Adam([q], weight_decay=0.1)):
        opt = rb.optim.AdamW([p], lr=0.5, state_bits=8)
        with pytest.raises(ValueError):
            opt.load_state_dict(other.state_dict())
        assert opt.param_groups[0]["lr"] == 0.5 and opt.param_groups[0]["state_bits"] == 8 and "maximize" not in opt.param_groups[0]
    for other in (torch.optim.AdamW([q], lr=0.25), torch.optim.Adam([q], lr=0.25)):      # without weight decay the two are the same
        opt = rb.optim.AdamW([p], lr=0.5)
        opt.load_state_dict(other.state_dict())
        assert opt.param_groups[0]["lr"] == 0.25


def test_a_checkpoint_that_does_not_fit_changes_nothing():
    p = torch.nn.Parameter(torch.zeros(3, dtype=torch.bfloat16))
    opt = rb.optim.AdamW([p], lr=0.5)
    opt.state[p]["step"] = torch.zeros(())
    groups, state = opt.param_groups, opt.state
    other = rb.optim.AdamW([torch.nn.Parameter(torch.zeros(3))], lr=0.25).state_dict()
    other["state"] = {0: {"step": torch.tensor(3.0)}}
    with pytest.raises(RuntimeError):
        opt.load_state_dict(other)
    assert opt.param_groups is groups and opt.state is state and groups[0]["lr"] == 0.5


def test_fake_tensors_through_the_layer_loss():
    """rlinear_cross_entropy and RandumbLinear.cross_entropy can be traced like their parts; on CPU tensors they say what the parts say."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    layer = rb.RandumbLinear(16, 30, 8, seed=1, device="cpu", dtype=torch.bfloat16)
    with FakeTensorMode():
        x = torch.empty(4, 6, 16, device="cuda", dtype=torch.bfloat16, requires_grad=True)
        c = torch.empty(8, 16, device="cuda", dtype=torch.bfloat16, requires_grad=True)
        t = torch.empty(4, 6, device="cuda", dtype=torch.int64)
        loss = rb.rlinear_cross_entropy(x, c, 1, 30, t)
        assert loss.shape == () and loss.dtype == torch.float32 and loss.requires_grad
        assert rb.rlinear_cross_entropy(x, c, 1, 30, t, reduction="none", ignore_index=None).shape == (4, 6)
        layer.weight_coef = torch.nn.Parameter(torch.empty(8, 16, device="cuda", dtype=torch.bfloat16))
        assert layer.cross_entropy(x, t).shape == ()
        z = rb.ops.matmul_nt_fwd(x.reshape(24, 16), c)
        assert z.shape == (24, 8) and z.dtype == torch.bfloat16
        da, db = rb.ops.matmul_nt_bwd(z, x.reshape(24, 16), c, False, True)
        assert da.shape == (0,) and db.shape == c.shape and db.dtype == c.dtype
    with pytest.raises(NotImplementedError, match="Unsupported CPU implementation"):
        rb.rlinear_cross_entropy(torch.ones(2, 3), torch.ones(4, 3), 1, 5, torch.zeros(2, dtype=torch.int64))


def test_tangents_are_refused():
    """Forward-mode differentiation is not implemented, and says so where a tangent would be dropped."""
    import torch.autograd.forward_ad as fw
    x, w, c, t = torch.ones(2, 3), torch.ones(5, 3), torch.ones(4, 3), torch.zeros(2, dtype=torch.int64)
    calls = (lambda a: rb.noise_cross_entropy(a, 1, 5, t), lambda a: rb.linear_cross_entropy(a, w, t), lambda a: rb.rlinear_cross_entropy(a, c, 1, 5, t))
    for call in calls + (lambda a: rb.linear_cross_entropy(x, a.repeat(3, 1)[:5], t), lambda a: rb.rlinear_cross_entropy(x, a.repeat(2, 1), 1, 5, t)):
        with fw.dual_level():
            with pytest.raises(RuntimeError, match="forward-mode"):
                call(fw.make_dual(x, torch.ones_like(x)))
        with pytest.raises(RuntimeError, match="forward-mode"):
            torch.func.jvp(call, (x,), (torch.ones_like(x),))
    with fw.dual_level():                                           # no tangent among the inputs: as ever
        for call in calls:
            with pytest.raises((NotImplementedError, RuntimeError), match="CPU"):
                call(x)
