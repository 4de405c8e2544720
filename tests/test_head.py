"""The head's loss and gradients against the definition in 64 bits.

Error bounds, element by element, all from quantities of the definition.
* A logit is a sum of exact products in fp32: each of the at most D / 16 + 8 additions may lose one unit in the
  last place (2^-23) of at most A = sum_d |x w| + |b|:  e_l = (D / 16 + 8) 2^-23 A.
* lse: the largest e_l of the row; exponentials good to 2^-21 and a sum whose longest chain is under 300 + V / 64
  additions of 2^-24; the value itself a few roundings of |lse| and of the largest logit.
* nll: the errors of lse and of the target's logit, and one rounding.
* delta: the factor times p (e_l + e_lse + 2^-20), and its own rounding -- bf16: half a step, 2^-8 of it; fp32:
  three bf16 terms, 2^-24 of it (and one rounding of the difference with the one-hot, 2^-23 of the factor).
* dx, dw: those errors times |W|, |x|; each of K / 16 + 8 additions per term 2^-23 of the sum of |delta W|; the result's
  rounding (2^-8 or 2^-24 of it).  dbias: a sum of fp32 values, (T + 8) 2^-24 of the sum of |delta|.
"""
import ctypes as C
import math

import pytest
import torch

from anni_b200 import capi, head
from anni_b200.head import head_loss, head_loss_grad

gpu = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


def inputs(t, d, v, seed=0, ignored=0.2, bias=True, sharp=2.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(t, d, generator=g).to(BF)
    w = (torch.randn(d, v, generator=g) * (sharp / math.sqrt(d))).to(BF)
    target = torch.randint(0, v, (t,), generator=g).int()
    target[torch.rand(t, generator=g) < ignored] = -1
    b = torch.randn(v, generator=g) * 0.5 if bias else None
    return [None if a is None else a.cuda() for a in (x, w, target, b)]


class Exact:
    """The definition in 64 bits with the bounds above."""

    def __init__(self, x, w, target, bias, weight=None, scale=1.0):
        xd, wd = x.double(), w.double()
        self.t, self.d = x.shape
        self.v = w.shape[1]
        b = torch.zeros(self.v, dtype=torch.float64, device=x.device) if bias is None else bias.double()
        z = xd @ wd + b
        self.counted = (target >= 0) & (target < self.v)
        size = xd.abs() @ wd.abs() + torch.where(b.isfinite(), b.abs(), 0)
        el = (self.d / 16 + 8) * 2.0 ** -23 * size
        self.lse = torch.logsumexp(z, 1)
        top = z.masked_fill(~z.isfinite(), 0).abs().amax(1)
        self.e_lse = el.amax(1) + 2.0 ** -21 + (300 + self.v / 64) * 2.0 ** -24 + 8 * 2.0 ** -24 * (self.lse.abs() + top)
        at = target.clamp(0, self.v - 1).long().view(-1, 1)
        hit = z.gather(1, at).view(-1)
        self.nll = torch.where(self.counted, self.lse - hit, 0.0)
        self.e_nll = self.e_lse + el.gather(1, at).view(-1) + 2.0 ** -24 * (self.nll.abs() + 2 * hit.abs())
        f = self.counted.double() * scale * (1.0 if weight is None else weight.double())
        f = torch.where(self.counted & (self.lse != -math.inf), f, 0.0)
        p = (z - self.lse[:, None]).exp()
        onehot = torch.zeros_like(p).scatter_(1, at, 1.0)
        self.delta = torch.where(f[:, None] != 0, f[:, None] * (p - onehot), 0.0)
        self.f, self.p, self.el = f, torch.where(f[:, None] != 0, p, 0.0), el
        self.xd = torch.where(f[:, None] != 0, xd, 0.0)
        self.wd = wd

    def grads(self, kind):
        """{name: (value, bound)}; the bound without the rounding of an accumulated result."""
        own = 2.0 ** -8 if kind == BF else 2.0 ** -24
        terms = 1 if kind == BF else 3
        e = self.f.abs()[:, None] * (self.p * (self.el + self.e_lse[:, None] + 2.0 ** -20) + 2.0 ** -23 * (self.p > 0))
        e = e + own * self.delta.abs()
        ad, wa, xa = self.delta.abs(), self.wd.abs(), self.xd.abs()
        e_unrounded = e - own * self.delta.abs()
        dx, dw, db = self.delta @ self.wd.t(), self.xd.t() @ self.delta, self.delta.sum(0)
        add = lambda k: (k / 16 + 8) * terms * 2.0 ** -23  # noqa: E731
        return {"dx": (dx, e @ wa.t() + add(self.v) * (ad @ wa.t())), "dw": (dw, xa.t() @ e + add(self.t) * (xa.t() @ ad)),
                "db": (db, e_unrounded.sum(0) + (self.t + 8) * 2.0 ** -24 * ad.sum(0))}


def check_loss(ex, nll, lse):
    assert ((lse.double() - ex.lse).abs() <= ex.e_lse).all()
    assert ((nll.double() - ex.nll).abs() <= torch.where(ex.counted, ex.e_nll, 0.0)).all()


def check_grads(ex, kind, before=None, **got):
    own = 2.0 ** -8 if kind == BF else 2.0 ** -24
    for name, (want, bound) in ex.grads(kind).items():
        if name not in got:
            continue
        if before is not None and name in before:
            want = want + before[name].double()
        g = got[name].double()
        off = (g - want).abs() - (bound * (1 + own) + own * want.abs() + 1e-38)
        assert (off <= 0).all(), (name, float(off.max()), int((off > 0).sum()))


def buffers(t, d, v, kind, fill=float("nan")):
    return tuple(torch.full(s, fill, dtype=kind, device="cuda") for s in ((t, d), (d, v), (v,)))


def both(x, w, target, b, kind, weight=None, scale=1.0):
    nll, lse = head_loss(x, w, target, bias=b)
    dx, dw, db = buffers(*x.shape, w.shape[1], kind)
    head_loss_grad(x, w, target, lse, bias=b, weight=weight, grad_scale=scale, dx=dx, dw=dw, dbias=db)
    return nll, lse, dx, dw, db


SHAPES = [(1, 1, 1), (1, 64, 300), (2, 8, 8), (5, 3, 7), (127, 64, 300), (128, 64, 256), (129, 65, 257), (300, 200, 1000),
          (257, 136, 5003), (64, 1536, 4096), (1000, 72, 264), (3, 520, 20001), (8, 1536, 1000), (4, 64, 512), (7, 100, 777),
          (8, 2056, 264), (9, 64, 300)]


@gpu
@pytest.mark.parametrize("kind", [BF, F32])
@pytest.mark.parametrize("t,d,v", SHAPES)
def test_sizes(t, d, v, kind):
    x, w, target, b = inputs(t, d, v, seed=t + d + v, bias=d % 2 == 0)
    nll, lse, dx, dw, db = both(x, w, target, b, kind)
    ex = Exact(x, w, target, b)
    check_loss(ex, nll, lse)
    check_grads(ex, kind, dx=dx, dw=dw, db=db)


@gpu
@pytest.mark.parametrize("kind", [BF, F32])
def test_several_pieces_of_the_vocabulary(kind):
    """More rows times entries than the workspace holds of delta: the gradients of x are summed over pieces."""
    t, d, v = 8200, 40, 26000
    x, w, target, b = inputs(t, d, v, seed=3)
    nll, lse, dx, dw, db = both(x, w, target, b, kind)
    ex = Exact(x, w, target, b)
    check_loss(ex, nll, lse)
    check_grads(ex, kind, dx=dx, dw=dw, db=db)


@gpu
@pytest.mark.parametrize("kind", [BF, F32])
def test_weights_scale_and_accumulation(kind):
    t, d, v = 200, 96, 777
    x, w, target, b = inputs(t, d, v, seed=4)
    weight = torch.rand(t, generator=torch.Generator().manual_seed(1)).cuda() * 2
    weight[::7] = 0
    weight[3] = -1.5
    nll, lse = head_loss(x, w, target, bias=b)
    dx, dw, db = buffers(t, d, v, kind)
    dw.normal_()
    db.normal_()
    before = dict(dw=dw.clone(), db=db.clone())
    head_loss_grad(x, w, target, lse, bias=b, weight=weight, grad_scale=-0.25, dx=dx, dw=dw, dbias=db, accumulate=True)
    ex = Exact(x, w, target, b, weight, -0.25)
    check_grads(ex, kind, before, dx=dx, dw=dw, db=db)
    assert not dx[::7].any()


@gpu
@pytest.mark.parametrize("kind", [BF, F32])
@pytest.mark.parametrize("wanted", ["dx", "dw", "db"])
def test_one_output_alone(kind, wanted):
    t, d, v = 150, 64, 520
    x, w, target, b = inputs(t, d, v, seed=5)
    _, lse, *full = both(x, w, target, b, kind)
    out = dict(zip(("dx", "dw", "db"), buffers(t, d, v, kind)))
    names = dict(dx="dx", dw="dw", db="dbias")
    head_loss_grad(x, w, target, lse, bias=b, **{names[wanted]: out[wanted]})
    assert torch.equal(out[wanted], dict(zip(("dx", "dw", "db"), full))[wanted])


@gpu
@pytest.mark.parametrize("kind", [BF, F32])
def test_ignored_rows_may_hold_anything(kind):
    """Rows without a target or with factor 0: nll 0 (or their own), no gradient, and no effect on any other."""
    t, d, v = 140, 72, 500
    x, w, target, b = inputs(t, d, v, seed=6, ignored=0.0)
    target[10:20] = -1
    target[139] = -100
    weight = torch.ones(t, device="cuda")
    weight[30:40] = 0
    clean = both(x, w, target, b, kind, weight)
    y = x.clone()
    y[10] = math.nan
    y[11:20] = math.inf
    y[30:40] = -math.inf
    y[139, 0] = math.nan
    nll, lse, dx, dw, db = both(y, w, target, b, kind, weight)
    assert (nll[target < 0] == 0).all()
    on = torch.ones(t, dtype=torch.bool, device="cuda")
    on[30:40] = False
    assert torch.equal(nll[on], clean[0][on])
    for a, c in zip((dx, dw, db), clean[2:]):
        assert torch.equal(a, c)
    assert not dx[10:20].any() and not dx[30:40].any() and not dx[139].any()


@gpu
@pytest.mark.parametrize("kind", [BF, F32])
def test_every_row_ignored(kind):
    x, w, target, b = inputs(70, 64, 300, seed=7)
    target.fill_(-1)
    x.fill_(math.nan)
    nll, lse, dx, dw, db = both(x, w, target, b, kind)
    assert not nll.any() and not dx.any() and not dw.any() and not db.any()


@gpu
def test_targets_beyond_the_vocabulary():
    x, w, target, b = inputs(130, 64, 300, seed=8, ignored=0.0)
    target[5], target[129] = 300, 2 ** 31 - 1
    nll, lse, dx, dw, db = both(x, w, target, b, F32)
    bad = torch.zeros(130, dtype=torch.bool, device="cuda")
    bad[5] = bad[129] = True
    assert torch.isnan(nll[bad]).all() and torch.isfinite(nll[~bad]).all() and not dx[bad].any()
    check_grads(Exact(x, w, target, b), F32, dx=dx, dw=dw, db=db)


@gpu
@pytest.mark.parametrize("kind", [BF, F32])
def test_masked_vocabulary(kind):
    """-inf bias: entries leave the softmax, also whole tiles of them and the first ones; one that is a target; all."""
    t, d, v = 66, 64, 1500
    x, w, target, b = inputs(t, d, v, seed=9, ignored=0.1)
    b[:700] = -math.inf
    b[1490:] = -math.inf
    target = torch.where(target >= 0, 700 + target % 790, target).int()
    nll, lse, dx, dw, db = both(x, w, target, b, kind)
    ex = Exact(x, w, target, b)
    check_loss(ex, nll, lse)
    check_grads(ex, kind, dx=dx, dw=dw, db=db)
    few = Exact(x[:5], w, target[:5], b)
    check_loss(few, *head_loss(x[:5], w, target[:5], bias=b))
    assert not dw[:, :700].any() and not db[1490:].any()
    target[0] = 3
    nll, lse, dx, dw, db = both(x, w, target, b, kind)
    assert nll[0] == math.inf and torch.isfinite(nll[1:]).all()
    assert abs(float(db[3]) + 1.0) <= 2.0 ** -8
    b.fill_(-math.inf)
    nll, lse, dx, dw, db = both(x, w, target, b, kind)
    assert (lse == -math.inf).all() and torch.isnan(nll[target >= 0]).all() and (nll[target < 0] == 0).all()
    assert not dx.any() and not dw.any() and not db.any()


@gpu
def test_large_logits_and_lowest_bias():
    """Logits of some thousands and biases of the type's lowest value: no overflow, the largest wins."""
    t, d, v = 40, 64, 600
    x, w, target, b = inputs(t, d, v, seed=10, ignored=0.0, sharp=1500.0)
    b[100:300] = torch.finfo(torch.float32).min
    target = torch.where((target >= 100) & (target < 300), 5, target).int()
    nll, lse, dx, dw, db = both(x, w, target, b, F32)
    ex = Exact(x, w, target, b)
    ex.e_lse, ex.e_nll = (Exact(x, w, target, torch.where(b < -1e30, -math.inf, b)).__dict__[k] for k in ("e_lse", "e_nll"))
    check_loss(ex, nll, lse)
    for a in (dx, dw, db):
        assert torch.isfinite(a).all()
    assert not dw[:, 100:300].any()
    b.fill_(torch.finfo(torch.float32).min)         # nothing but the lowest value: an even softmax, for one row and for many
    for rows in (1, 40):
        nll, lse = head_loss(x[:rows], w, target[:rows], bias=b)
        assert torch.isfinite(lse).all() and (lse < -3e38).all()
        dbias = torch.empty(v, device="cuda")
        head_loss_grad(x[:rows], w, target[:rows], lse, bias=b, dbias=dbias)
        assert torch.isfinite(dbias).all()


@gpu
def test_nan_row_with_a_target():
    """A NaN in a counted row shows in its loss and leaves the other rows' losses alone."""
    x, w, target, b = inputs(130, 64, 300, seed=11, ignored=0.0)
    clean, _ = head_loss(x, w, target, bias=b)
    x[7, 3] = math.nan
    nll, _ = head_loss(x, w, target, bias=b)
    assert torch.isnan(nll[7])
    nll[7] = clean[7]
    assert torch.equal(nll, clean)
    few, _ = head_loss(x[4:8], w, target[4:8], bias=b)
    assert torch.isnan(few[3]) and torch.isfinite(few[:3]).all()


@gpu
@pytest.mark.parametrize("kind", [BF, F32])
@pytest.mark.parametrize("off", [0, 1, 8])
def test_strides_and_addresses(kind, off):
    """Slices of wider matrices, on and off the 16-byte grid; what lies around the outputs stays."""
    t, d, v = 140, 72, 520
    x, w, target, b = inputs(t, d, v, seed=12)
    pad = lambda a, n: torch.full((a.shape[0], a.shape[1] + n), math.nan, dtype=a.dtype, device="cuda")  # noqa: E731
    X, W = pad(x, off + 8), pad(w, off + 16)
    X[:, off:off + d], W[:, off:off + v] = x, w
    xs, ws = X[:, off:off + d], W[:, off:off + v]
    DX, DW = pad(x.to(kind), off + 3), pad(w.to(kind), off + 5)
    DX.fill_(7)
    DW.fill_(7)
    dbw = torch.full((v + off + 1,), 7, dtype=kind, device="cuda")
    nll, lse = head_loss(xs, ws, target, bias=b)
    head_loss_grad(xs, ws, target, lse, bias=b, dx=DX[:, off:off + d], dw=DW[:, off:off + v], dbias=dbw[off:off + v])
    ex = Exact(x, w, target, b)
    check_loss(ex, nll, lse)
    check_grads(ex, kind, dx=DX[:, off:off + d], dw=DW[:, off:off + v], db=dbw[off:off + v])
    assert (DX[:, :off] == 7).all() and (DX[:, off + d:] == 7).all() and (DW[:, :off] == 7).all() and (DW[:, off + v:] == 7).all()
    assert (dbw[:off] == 7).all() and dbw[-1] == 7


@gpu
def test_gradients_against_differences():
    """d sum(nll) / d bias and / d x by central differences of the loss itself.

    Step h: the loss's error is under 1e-5 a row (40 rows: 4e-4 / 2h), the third derivative of a row's loss in one
    logit is under 0.1 (40 * 0.1 h^2 / 6; in x times the cube of |w| <= 1)."""
    t, d, v = 40, 32, 50
    x, w, target, b = inputs(t, d, v, seed=13, ignored=0.0)
    _, _, dx, dw, db = both(x, w, target, b, F32)
    total = lambda xx, bb: float(head_loss(xx, w, target, bias=bb)[0].double().sum())  # noqa: E731
    h = 0.125
    for k in (0, 7, 49):
        hi, lo = b.clone(), b.clone()
        hi[k] += h
        lo[k] -= h
        assert abs((total(x, hi) - total(x, lo)) / (2 * h) - float(db[k])) <= 4e-4 / (2 * h) + 40 * 0.1 * h * h / 6
    for i, k in ((0, 0), (39, 31), (17, 5)):
        hi, lo = x.clone(), x.clone()
        hi[i, k], lo[i, k] = float(x[i, k]) + h, float(x[i, k]) - h
        step = float(hi[i, k]) - float(lo[i, k])
        mid = (float(hi[i, k]) + float(lo[i, k])) / 2 - float(x[i, k])       # bf16 may not hold x + h: the middle moves
        curve = float((w[k].double() ** 2).max())
        assert abs((total(hi, b) - total(lo, b)) / step - float(dx[i, k])) <= 2e-5 / step + 0.1 * h * h / 6 + curve * abs(mid)


# ---- how it is called ------------------------------------------------------------------------------------

@gpu
def test_same_bits_every_time_and_on_another_stream():
    x, w, target, b = inputs(300, 200, 1000, seed=14)
    first = both(x, w, target, b, BF)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    nll, lse = head_loss(x, w, target, bias=b, stream=st)
    dx, dw, db = buffers(300, 200, 1000, BF)
    st.wait_stream(torch.cuda.current_stream())
    head_loss_grad(x, w, target, lse, bias=b, dx=dx, dw=dw, dbias=db, stream=st)
    torch.cuda.synchronize()
    for a, c in zip(first, (nll, lse, dx, dw, db)):
        assert torch.equal(a, c)


@gpu
def test_two_captured_graphs():
    """Two graphs of two calls replayed on two streams at once: each has its own workspace."""
    runs = []
    for seed in (15, 16):
        x, w, target, b = inputs(300, 136, 1000, seed=seed)
        want = both(x, w, target, b, BF)
        out = buffers(300, 136, 1000, BF)
        gr, st = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.graph(gr, stream=st):
            nll, lse = head_loss(x, w, target, bias=b)
            head_loss_grad(x, w, target, lse, bias=b, dx=out[0], dw=out[1], dbias=out[2])
        runs.append((gr, st, (nll, lse) + out, want, (x, w, target, b)))
    torch.cuda.synchronize()
    for _ in range(3):
        for gr, st, *_ in runs:
            with torch.cuda.stream(st):
                gr.replay()
    torch.cuda.synchronize()
    for _, _, got, want, _ in runs:
        assert all(torch.equal(a, c) for a, c in zip(got, want))


@gpu
def test_no_rows():
    w = torch.zeros(64, 300, dtype=BF, device="cuda")
    x, target = torch.zeros(0, 64, dtype=BF, device="cuda"), torch.zeros(0, dtype=torch.int32, device="cuda")
    nll, lse = head_loss(x, w, target)
    assert nll.shape == lse.shape == (0,)
    for add, want in ((True, 3.0), (False, 0.0)):
        dw, db = torch.full((64, 300), 3.0, device="cuda"), torch.full((300,), 3.0, device="cuda")
        head_loss_grad(x, w, target, lse, dx=torch.empty(0, 64, device="cuda"), dw=dw, dbias=db, accumulate=add)
        assert (dw == want).all() and (db == want).all()


@gpu
def test_python_refusals():
    x, w, target, b = inputs(4, 8, 16)
    nll, lse = head_loss(x, w, target, bias=b)
    for bad in (dict(x=x.float()), dict(x=x.t()), dict(x=x[:, :4]), dict(w=w.t()), dict(w=w.float()), dict(target=target.long()),
                dict(target=target[:2]), dict(bias=b[:5]), dict(bias=b.double()), dict(x=x[:1].expand(4, 8))):
        with pytest.raises((TypeError, ValueError)):
            head_loss(**{**dict(x=x, w=w, target=target, bias=b), **bad})
    for bad in (dict(dx=x.float(), dw=w), dict(dx=x.half()), dict(dx=torch.empty(4, 9, device="cuda")), dict(lse=lse[:2]),
                dict(weight=lse.double()), dict(dbias=b[:3])):
        with pytest.raises((TypeError, ValueError)):
            head_loss_grad(x, w, target, **{**dict(lse=lse), **bad})


# ---- refusals of the C entry points: no device needed --------------------------------------------------

def _c(**kw):
    c = head.Call()
    base = dict(x=0x10000000, ldx=64, w=0x20000000, ldw=300, bias=0x30000000, target=0x31000000, tokens=10, d_model=64,
                vocab=300, nll=0x32000000, lse=0x33000000, weight=0x34000000, grad_scale=1.0, grad_dtype=capi.DT_BF16,
                flags=0, dx=0x40000000, lddx=64, dw=0x50000000, lddw=300, dbias=0x60000000, workspace=0x70000000,
                workspace_bytes=1 << 40)
    for k, x in {**base, **kw}.items():
        setattr(c, k, x)
    return c


COMMON = [dict(tokens=-1), dict(d_model=0), dict(vocab=0), dict(ldx=63), dict(ldw=299), dict(x=0x10000001), dict(w=0x20000001),
          dict(x=None), dict(w=None), dict(target=None), dict(lse=None), dict(workspace=None), dict(workspace=0x70000080),
          dict(workspace_bytes=256), dict(bias=0x30000002), dict(target=0x31000002), dict(lse=0x33000001)]
GRAD = [dict(grad_dtype=2), dict(flags=2), dict(lddx=63), dict(lddw=299), dict(dx=0x40000001), dict(dbias=0x60000001),
        dict(dw=0x50000002, grad_dtype=capi.DT_F32), dict(weight=0x34000001)]


@pytest.mark.parametrize("kw", COMMON + [dict(nll=None)])
def test_loss_refuses(kw):
    assert head.lib().anni_head_loss(C.byref(_c(**kw)), None) == capi.E_ARG


@pytest.mark.parametrize("kw", COMMON + GRAD)
def test_grad_refuses(kw):
    assert head.lib().anni_head_loss_grad(C.byref(_c(**kw)), None) == capi.E_ARG


@pytest.mark.parametrize("kw", [dict(tokens=(1 << 24) + 1), dict(d_model=(1 << 16) + 1, ldx=1 << 20), dict(vocab=(1 << 24) + 1, ldw=1 << 26)])
def test_limits(kw):
    L = head.lib()
    n = C.c_size_t()
    for grad in (0, 1):
        assert L.anni_head_workspace(C.byref(_c(**kw)), grad, C.byref(n)) == capi.E_LIMIT
    assert L.anni_head_loss(C.byref(_c(**kw)), None) == capi.E_LIMIT


def test_null_and_empty_calls():
    L = head.lib()
    n = C.c_size_t()
    assert L.anni_head_loss(None, None) == L.anni_head_loss_grad(None, None) == capi.E_ARG
    assert L.anni_head_workspace(None, 0, C.byref(n)) == capi.E_ARG and L.anni_head_workspace(C.byref(_c()), 0, None) == capi.E_ARG
    assert L.anni_head_loss(C.byref(_c(tokens=0, x=None, workspace=None)), None) == capi.OK
    assert L.anni_head_loss_grad(C.byref(_c(dx=None, dw=None, dbias=None, workspace=None)), None) == capi.OK


def test_workspace_is_bounded():
    """Delta of a piece, not of the vocabulary: 16384 rows of 100,000 entries fit a few hundred megabytes."""
    n = C.c_size_t()
    for kind in (capi.DT_BF16, capi.DT_F32):
        c = _c(tokens=16384, d_model=1536, ldx=1536, lddx=1536, vocab=100000, ldw=100000, lddw=100000, grad_dtype=kind)
        assert head.lib().anni_head_workspace(C.byref(c), 1, C.byref(n)) == capi.OK
        assert n.value < 700 << 20


def test_every_declared_symbol_is_exported():
    from test_abi_cpu import _declared_symbols
    names = _declared_symbols("anni_head.h")
    assert len(names) == 4 and not [k for k in names if not hasattr(head.lib(), k)]


@gpu
@pytest.mark.parametrize("t", [1, 2, 3])
@pytest.mark.parametrize("d,v,ld,at", [(1536, 4097, 4097, 0), (2567, 1001, 1001, 0), (700, 20001, 20001, 0), (1, 9, 9, 0),
                                       (9, 7, 7, 0), (513, 496, 500, 3), (130, 260, 264, 1), (200, 1000, 1008, 8),
                                       (8192, 300, 302, 0), (64, 248, 249, 1), (1200, 33000, 33000, 0)])
def test_few_rows_of_any_layout(t, d, v, ld, at):
    """A few rows read W in whole 16-byte granules wherever its rows begin; what lies between them is NaN."""
    x, w, target, b = inputs(t, d, v, seed=t + d + v)
    target[0] = v - 1
    wide = torch.full((d * ld + at,), float("nan"), dtype=BF, device="cuda")
    view = wide[at:at + (d - 1) * ld + v].as_strided((d, v), (ld, 1))
    view.copy_(w)
    ex = Exact(x, w, target, b)
    first = head_loss(x, view, target, bias=b)
    check_loss(ex, *first)
    for again in zip(first, head_loss(x, view, target, bias=b)):
        assert torch.equal(*again)
