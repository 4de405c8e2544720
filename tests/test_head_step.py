"""The head's loss, its gradients and the optimizer step run together, as a trainer runs them."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

from anni_b200 import capi, head, lm_adam
from anni_b200.capi import DT_BF16, DT_F32, DT_Q8
from anni_b200.engine import LM_SHAPES, OptStep, lm_segments
from anni_b200.head import head_loss, head_loss_grad
from anni_b200.mtstep import MultiStep
from test_head import Exact, check_grads, check_loss

gpu = pytest.mark.gpu
D, V = LM_SHAPES["tiny"]["d_model"], LM_SHAPES["tiny"]["vocab"]
KIND = {DT_F32: torch.float32, DT_BF16: torch.bfloat16}


def batch(t, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(t, D, generator=g).bfloat16().cuda()
    target = torch.randint(-1, V, (t,), generator=g).int().cuda()
    return x, target


def engine(grad_dtype, seed=1):
    segs = lm_segments(**LM_SHAPES["tiny"], wd="matrices")
    eng = OptStep(segs, grad_dtype=grad_dtype).allocate()
    eng.master.copy_(torch.randn(segs.n, generator=torch.Generator().manual_seed(seed)) * 0.1)
    eng.twin_bf16.copy_(eng.master)
    return segs, eng


@gpu
@pytest.mark.parametrize("grad_dtype", [DT_F32, DT_BF16])
def test_engine_adds_the_heads_gradients_and_steps(grad_dtype):
    """Two micro-batches into the flat, a step, and the loss on the stepped twin."""
    segs, eng = engine(grad_dtype)
    w, b = segs.slice_of("w_head"), segs.slice_of("b_head")
    for step in (1, 2):
        want = [torch.zeros(D, V, dtype=torch.float64, device="cuda"), torch.zeros(V, dtype=torch.float64, device="cuda")]
        for micro in (0, 1):
            x, target = batch(130, 10 * step + micro)
            dx = torch.empty(130, D, dtype=KIND[grad_dtype], device="cuda")
            before = dict(dw=eng.grad[w].view(D, V).clone(), db=eng.grad[b].clone())
            nll = eng.head_loss(x, target, grad_scale=0.5, dx=dx)
            ex = Exact(x, eng.twin_bf16[w].view(D, V), target, eng.master[b], scale=0.5)
            assert ((nll.double() - ex.nll).abs() <= torch.where(ex.counted, ex.e_nll, 0.0)).all()
            check_grads(ex, KIND[grad_dtype], before, dx=dx, dw=eng.grad[w].view(D, V), db=eng.grad[b])
            want[0] += ex.grads(KIND[grad_dtype])["dw"][0]
            want[1] += ex.grads(KIND[grad_dtype])["db"][0]
        g = eng.grad.double()
        old = eng.master.clone()
        eng.step(OptStep.hyper(lr=1e-3, t=step, clip=1.0))
        st = eng.status()
        assert st.skipped == 0 and abs(st.norm - float(g.norm())) <= 1e-9 * st.norm
        assert not eng.grad.any() and not torch.equal(old[w], eng.master[w])
        assert torch.equal(eng.twin_bf16, eng.master.bfloat16())


@gpu
def test_engine_refusals():
    segs, eng = engine(DT_BF16)
    x, target = batch(4, 1)
    with pytest.raises(ValueError):
        eng.head_loss(x[:, :63], target)
    with pytest.raises(ValueError):
        eng.head_loss(x, target, w="nothing")
    with pytest.raises(TypeError):
        eng.head_loss(x, target, dx=torch.empty(4, D, device="cuda"))
    with pytest.raises(TypeError):
        eng.head_loss(x, target, b="blk0.b1")
    assert not eng.grad.any()


@gpu
@pytest.mark.parametrize("grad_dtype", [DT_F32, DT_BF16])
def test_optimizer_object(grad_dtype):
    """The C optimizer object: its head call, the gradients in its flat, its step against an engine given the same."""
    segs, eng = engine(grad_dtype)
    host = eng.master.cpu().numpy().copy()
    opt = lm_adam.create(segs, host.ctypes.data, 0, grad_dtype=grad_dtype)
    L, H = lm_adam.lib(), head.lib()
    o = opt.contents
    c = head.Call()
    c.d_model, c.vocab, c.tokens = D, V, 130
    iw, ib = segs.index("w_head"), segs.index("b_head")
    assert H.anni_lm_adam_head_call(opt, iw, ib, C.byref(c)) == capi.E_ARG         # no flats yet
    assert L.anni_lm_adam_prepare(opt) == capi.OK
    assert H.anni_lm_adam_head_call(opt, ib, iw, C.byref(c)) == capi.E_ARG
    assert H.anni_lm_adam_head_call(opt, iw, iw, C.byref(c)) == capi.E_ARG
    assert H.anni_lm_adam_head_call(opt, iw, len(segs), C.byref(c)) == capi.E_ARG
    assert H.anni_lm_adam_head_call(opt, iw, ib, C.byref(c)) == capi.OK
    assert (c.ldw, c.lddw, c.grad_dtype, c.flags, c.grad_scale) == (V, V, grad_dtype, head.HEAD_ACCUMULATE, 1.0)
    o.loss_scale = 8.0
    assert H.anni_lm_adam_head_call(opt, iw, ib, C.byref(c)) == capi.OK and c.grad_scale == 8.0
    x, target = batch(130, 5)
    nll, lse = torch.empty(2, 130, device="cuda").unbind(0)
    c.x, c.ldx, c.target, c.nll, c.lse = x.data_ptr(), D, target.data_ptr(), nll.data_ptr(), lse.data_ptr()
    need = C.c_size_t()
    size = 0
    for grad in (0, 1):
        assert H.anni_head_workspace(C.byref(c), grad, C.byref(need)) == capi.OK
        size = max(size, need.value)
    ws = torch.empty(size, dtype=torch.uint8, device="cuda")
    c.workspace, c.workspace_bytes = ws.data_ptr(), size
    torch.cuda.synchronize()
    assert H.anni_head_loss(C.byref(c), None) == capi.OK and H.anni_head_loss_grad(C.byref(c), None) == capi.OK
    torch.cuda.synchronize()
    mine = eng.head_loss(x, target, grad_scale=8.0)
    assert torch.equal(nll, mine)
    flat = torch.empty_like(eng.grad)
    assert capi.lib().anni_peer_copy(flat.data_ptr(), o.d_grad, flat.numel() * flat.element_size(), None) == capi.OK
    torch.cuda.synchronize()
    assert torch.equal(flat, eng.grad)
    o.grad_clip = 1.0
    assert L.anni_lm_adam_step_scaled(opt, 1e-3, 0.5) == capi.OK and o.last_skipped == 0
    eng.step(OptStep.hyper(lr=1e-3, t=1, clip=1.0, grad_scale=0.5 / 8.0, exact=True))
    assert L.anni_lm_adam_sync_host(opt) == capi.OK
    assert np.array_equal(host, eng.master.cpu().numpy())
    L.anni_lm_adam_free(C.byref(C.pointer(opt.contents)))


def test_head_call_refuses_without_a_device():
    c = head.Call()
    assert head.lib().anni_lm_adam_head_call(None, 0, 1, C.byref(c)) == capi.E_ARG


@gpu
@pytest.mark.parametrize("state_dtype", [DT_F32, DT_Q8])
def test_a_list_of_tensors_trained_through_the_head(state_dtype):
    """W and b as tensors of their own: loss, gradients and list step over four steps, each against the formula."""
    g = torch.Generator().manual_seed(2)
    wm, bm = (torch.randn(D, V, generator=g) * 0.1).cuda(), torch.zeros(V, device="cuda")
    twin = wm.bfloat16()
    dw, db = torch.zeros(D, V, dtype=torch.bfloat16, device="cuda"), torch.zeros(V, dtype=torch.bfloat16, device="cuda")
    opt = MultiStep([wm, bm], grads=[dw, db], state_dtype=state_dtype, decay=[True, False], twins=[twin, None])
    x, target = batch(200, 3)
    for t in range(1, 5):
        nll, lse = head_loss(x, twin, target, bias=bm)
        head_loss_grad(x, twin, target, lse, bias=bm, grad_scale=1 / 200, dw=dw, dbias=db, accumulate=True)
        ex = Exact(x, twin, target, bm, scale=1 / 200)
        check_loss(ex, nll, lse)
        check_grads(ex, torch.bfloat16, dw=dw, db=db)
        norm = math.sqrt(float((dw.double() ** 2).sum() + (db.double() ** 2).sum()))
        hp = OptStep.hyper(lr=1e-3, t=t, clip=0.5, wd=0.1)
        if state_dtype == DT_Q8:
            hp.flags |= capi.STEP_STOCHASTIC
        opt.step(hp, seed=t)
        st = opt.status()
        assert st.skipped == 0 and st.steps_done == t and abs(st.norm - norm) <= 1e-12 * norm
        assert torch.equal(twin, wm.bfloat16()) and not dw.any() and not db.any()
        for k in opt.moments()[1]:
            assert torch.isfinite(k).all() and (k >= 0).all()
