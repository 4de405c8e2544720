"""The step over a list of tensors against its formula in 64 bits, and against the packed-arena step.

Error bounds.  u = 2^-24 is half a step of float, relative to the value.
* 32-bit moments are computed in double and rounded once: within u of the formula, and 1e-12 for the clip
  factor, whose norm is summed in another order.  Parameter: the bar of the arena step, two steps of the larger
  of the old and the new value and 1e-6 of the change (SFU square root and reciprocal, two products).
* 8-bit moments are computed in float: the stored value code * scale, beta, 1 - beta, the clip factor and the
  gradient's product with it are each rounded once (u), the product of the second term (for v: two) once, and
  their sum once: at most 8 u of |b1 m| + |(1 - b1) g|, resp. of b2 v + (1 - b2) g^2.  The scale inherits the
  error of the largest element and adds a constant's and a product's: 10 u of the largest such sum in the block.  A
  value over its scale, y, carries those 8 u of its terms, 8 u of the largest element's, and the roundings of a
  reciprocal and two products: at most DELTA below.  The stored number must be as near to the exact y as the nearest one, but for 2 DELTA.
"""
import ctypes as C
import math

import numpy as np
import pytest
import torch

from anni_b200 import capi, mtstep
from anni_b200.capi import DT_BF16, DT_F32, DT_Q8
from anni_b200.engine import LM_SHAPES, OptStep, Segments, lm_segments
from anni_b200.mtstep import MultiStep

gpu = pytest.mark.gpu
U = 2.0 ** -24
SIZES = [1, 5, 255, 256, 257, 2047, 2048, 2049, 4097, 70001, 0, 33]
HYP = dict(lr=3e-4, beta1=0.9, beta2=0.95, eps=1e-8, wd=0.1)


# ---- the formula in 64 bits --------------------------------------------------------------------

def _table(kind):
    """The non-negative finite numbers of an 8-bit type."""
    codes = torch.arange(127 if kind == torch.float8_e4m3fn else 124, dtype=torch.uint8)
    return codes.view(kind).double()


def _mix(h):
    h = ((h ^ (h >> 16)) * 0x85EBCA6B) & 0xFFFFFFFF
    h = ((h ^ (h >> 13)) * 0xC2B2AE35) & 0xFFFFFFFF
    return h ^ (h >> 16)


def _bits(seed, block0, n):
    """The 32 random bits of the n elements of a tensor whose first block has the number block0 in the list."""
    i = torch.arange(n, dtype=torch.int64)
    block = block0 + i // 256
    key = _mix((seed & 0xFFFFFFFF) ^ _mix((block + (seed >> 32) * 0x9E3779B9) & 0xFFFFFFFF))
    return _mix((key + (i % 256) * 0x9E3779B9) & 0xFFFFFFFF)


def _per_block(x):
    """Largest |x| of each block of 256, one value per element."""
    pad = torch.nn.functional.pad(x.abs(), (0, -len(x) % 256)).view(-1, 256).amax(1)
    return pad, pad.repeat_interleave(256)[:len(x)]


def _formula(p, g, m, v, coef, wd, *, lr, beta1, beta2, eps, t):
    g = g * coef
    tm, tv = beta1 * m.abs() + (1 - beta1) * g.abs(), beta2 * v + (1 - beta2) * g * g
    m = beta1 * m + (1 - beta1) * g
    v = tv
    den = (v / (1 - beta2 ** t)).sqrt() + eps
    q = p - lr / (1 - beta1 ** t) * m / den
    return q - lr * wd * q, m, v, tm, lr / (1 - beta1 ** t) * tm / den


def _check_codes(y, got, delta, kind, draws=None, floor=None):
    """got (8-bit numbers) are the roundings of the exact y >= 0 that an error of delta allows."""
    tab = _table(kind)
    y = y.clamp_max(float(tab[-1]))
    lo = (torch.searchsorted(tab, y, right=True) - 1).clamp(0, len(tab) - 2)
    a, b = tab[lo], tab[lo + 1]
    gotv = got.float().double().abs()
    if draws is None:
        near = torch.minimum(y - a, b - y)
        ok = (gotv - y).abs() <= near + 2 * delta + 1e-300
    else:
        frac = (y - a) / (b - a) + draws.double() / 65536.0 - 1.0
        edge = frac.abs() * (b - a) <= 2 * delta + (b - a) * 2.0 ** -18        # 2^-20: what the float's own cut drops
        ok = torch.where(frac >= 0, gotv == b, gotv == a) | (edge & ((gotv == a) | (gotv == b)))
        # an error may also carry y over a number itself
        ok |= (torch.minimum(y - a, b - y) <= 2 * delta) & ((gotv - y).abs() <= (b - a) + 2 * delta)
    if floor is not None:
        ok |= floor & (gotv == tab[1])
    bad = (~ok).nonzero().view(-1)
    assert not len(bad), (len(bad), [(float(y[i]), float(gotv[i]), float(delta[i])) for i in bad[:5]])


# ---- inputs --------------------------------------------------------------------------------------

class Case:
    """A list of tensors on the GPU, each `shift` elements into its own allocation, and its copy in 64 bits."""

    def __init__(self, sizes, grad_dtype, state_dtype, seed=0, shift=0, twin=True, gscale=1e-3):
        r = torch.Generator().manual_seed(seed)
        cut = lambda x: torch.cat([torch.zeros(shift, dtype=x.dtype), x]).cuda()[shift:] if x.element_size() > 1 else \
            torch.cat([torch.zeros(shift, dtype=torch.uint8), x.view(torch.uint8)]).cuda()[shift:].view(x.dtype)  # noqa: E731
        rn = lambda n, s: torch.randn(n, generator=r) * s  # noqa: E731
        self.sizes, self.eight = sizes, state_dtype == DT_Q8
        self.p = [cut(rn(n, 0.02)) for n in sizes]
        self.g = [cut(rn(n, gscale).to(torch.bfloat16 if grad_dtype == DT_BF16 else torch.float32)) for n in sizes]
        m, v = [rn(n, 3e-4) for n in sizes], [rn(n, 1e-3) ** 2 + 1e-10 for n in sizes]
        self.ms = self.vs = None
        if self.eight:
            em, ev = [mtstep.encode(x, torch.float8_e4m3fn) for x in m], [mtstep.encode(x, torch.float8_e5m2) for x in v]
            m, v = [x for x, _ in em], [x for x, _ in ev]
            self.ms, self.vs = [s.cuda() for _, s in em], [s.cuda() for _, s in ev]
        self.m, self.v = [cut(x) for x in m], [cut(x) for x in v]
        self.twin = [cut(torch.zeros(n, dtype=torch.bfloat16)) for n in sizes] if twin else None
        self.decay = [k % 2 == 0 for k in range(len(sizes))]
        self.step = MultiStep(self.p, grads=self.g, state_dtype=state_dtype, grad_dtype=grad_dtype, decay=self.decay,
                              twins=self.twin, moments=(self.m, self.v), scales=(self.ms, self.vs) if self.eight else None)
        self.before = self.snapshot()

    def snapshot(self):
        out = dict(p=self.p, g=self.g, m=self.m, v=self.v, ms=self.ms, vs=self.vs, twin=self.twin)
        return {k: [y.clone().cpu() for y in x] if x is not None else None for k, x in out.items()}

    def check(self, hyp, *, clip=0.0, grad_scale=1.0, t=1000, seed=0, stochastic=False, out=None):
        """The state after one step from `before` against the formula."""
        b, a = self.before, self.snapshot()
        taken = [g is not None for g in self.step.grads]
        norm = math.sqrt(sum(float((g.double() ** 2).sum()) for g, on in zip(b["g"], taken) if on)) * abs(grad_scale)
        coef = grad_scale * (clip / (norm + 1e-12) if clip > 0 and norm > clip else 1.0)
        block0 = 0
        for k, n in enumerate(self.sizes):
            first, block0 = block0, block0 + -(-n // 256)
            if not taken[k] or n == 0:
                for key in ("p", "m", "v", "twin"):
                    if a[key] is not None:
                        assert torch.equal(a[key][k].view(torch.uint8 if a[key][k].element_size() == 1 else a[key][k].dtype),
                                           b[key][k].view(torch.uint8 if b[key][k].element_size() == 1 else b[key][k].dtype))
                continue
            p0, g = b["p"][k].double(), b["g"][k].double()
            if self.eight:
                m0 = b["m"][k].float().double() * b["ms"][k].double().repeat_interleave(256)[:n]
                v0 = b["v"][k].float().double() * b["vs"][k].double().repeat_interleave(256)[:n]
            else:
                m0, v0 = b["m"][k].double(), b["v"][k].double()
            q, m, v, tm, tu = _formula(p0, g, m0, v0, coef, hyp["wd"] if self.decay[k] else 0.0, t=t,
                                       **{x: hyp[x] for x in ("lr", "beta1", "beta2", "eps")})
            big = torch.maximum(p0.abs(), q.abs())
            bar = 2 * 2 * U * big + 1e-6 * (q - p0).abs()
            if self.eight:
                bar += 2 * 8 * U * tu
            assert ((a["p"][k].double() - q).abs() <= bar + 1e-45).all(), (k, n)
            if self.twin is not None:
                assert torch.equal(a["twin"][k], a["p"][k].bfloat16())
            if not self.eight:
                assert ((a["m"][k].double() - m).abs() <= U * m.abs() + 1e-12 * tm + 1e-45).all(), (k, n)
                assert ((a["v"][k].double() - v).abs() <= (U + 2e-12) * v + 1e-45).all(), (k, n)
                continue
            r = _bits(seed, first, n) if stochastic else None
            for x, terms, key, top, kind in ((m, tm, "m", 448.0, torch.float8_e4m3fn), (v, v, "v", 57344.0, torch.float8_e5m2)):
                amax, each = _per_block(x)
                worst = _per_block(terms)[0]
                scale = a[key + "s"][k].double()
                assert ((scale - amax / top).abs() <= 10 * U * worst / top + 1e-45).all(), (k, n, key)
                y = x.abs() * top / each
                delta = 8 * U * terms * top / each + (10 * worst / amax).repeat_interleave(256)[:n] * U * y + 3 * U * y
                got = a[key][k]
                assert (torch.sign(got.float().double()) * x >= 0).all()
                _check_codes(y, got, delta, kind, None if r is None else ((r & 0xFFFF) if key == "m" else (r >> 16)),
                             (x > 0) if key == "v" else None)
        return norm


def hyper(clip=0.0, grad_scale=1.0, t=1000, check=True, zero=False, stochastic=False, **kw):
    h = OptStep.hyper(**{**HYP, **kw}, t=t, clip=clip, grad_scale=grad_scale, check_finite=check, zero_grad=zero)
    if stochastic:
        h.flags |= capi.STEP_STOCHASTIC
    return h


# ---- against the formula ---------------------------------------------------------------------------

@gpu
@pytest.mark.parametrize("shift", [0, 1])
@pytest.mark.parametrize("grad_dtype", [DT_F32, DT_BF16])
@pytest.mark.parametrize("clip,grad_scale", [(0.0, 1.0), (0.05, 0.5)])
def test_32_bit_step(grad_dtype, clip, grad_scale, shift):
    c = Case(SIZES, grad_dtype, DT_F32, seed=1, shift=shift)
    c.step.step(hyper(clip, grad_scale))
    norm = c.check(HYP, clip=clip, grad_scale=grad_scale)
    st = c.step.status()
    assert st.error == 0 and st.skipped == 0 and st.steps_done == 1
    assert abs(st.norm - norm) <= 1e-12 * norm


@gpu
@pytest.mark.parametrize("shift", [0, 1])
@pytest.mark.parametrize("grad_dtype", [DT_F32, DT_BF16])
@pytest.mark.parametrize("clip,check", [(0.0, False), (0.05, True)])
@pytest.mark.parametrize("stochastic", [False, True])
def test_8_bit_step(grad_dtype, clip, check, stochastic, shift):
    c = Case(SIZES, grad_dtype, DT_Q8, seed=2, shift=shift)
    seed = (5 << 40) + 12345
    c.step.step(hyper(clip, check=check, stochastic=stochastic), seed=seed)
    c.check(HYP, clip=clip, seed=seed, stochastic=stochastic)


@gpu
@pytest.mark.parametrize("state_dtype", [DT_F32, DT_Q8])
def test_many_small_tensors(state_dtype):
    """More tensors than one launch of the address upload carries, single elements among them."""
    sizes = [1 + (k * 37) % 700 for k in range(1000)]
    c = Case(sizes, DT_BF16, state_dtype, seed=3, twin=False)
    c.step.set_grads(c.g)
    c.step.step(hyper(1.0))
    c.check(HYP, clip=1.0)


@gpu
@pytest.mark.parametrize("grad_dtype", [DT_F32, DT_BF16])
@pytest.mark.parametrize("clip", [0.0, 0.3])
def test_32_bit_step_has_the_arena_steps_bits(grad_dtype, clip):
    """The unit-test LM's tensors, once packed in an arena and once apart: the same parameters and moments."""
    segs = lm_segments(**LM_SHAPES["tiny"], wd="matrices")
    c = Case(list(segs.sizes), grad_dtype, DT_F32, seed=4)
    eng = OptStep(segs, grad_dtype=grad_dtype, state_dtype=DT_F32).allocate()
    for name, xs in (("master", c.p), ("m", c.m), ("v", c.v), ("grad", c.g)):
        getattr(eng, name).copy_(torch.cat([x.view(-1) for x in xs]))
    c.decay = [bool(f & capi.SEG_WD) for f in segs.flags]
    c.step = MultiStep(c.p, grads=c.g, decay=c.decay, twins=c.twin, moments=(c.m, c.v))
    for t in (1, 2, 3):
        eng.step(OptStep.hyper(**HYP, t=t, clip=clip, zero_grad=False))
        c.step.step(hyper(clip, t=t))
    assert eng.status().skipped == 0
    if clip == 0.0:             # the clip factor's norm is summed in another order: bits only without it
        for name, xs in (("master", c.p), ("m", c.m), ("v", c.v), ("twin_bf16", c.twin)):
            assert torch.equal(getattr(eng, name), torch.cat(xs)), name
    else:
        assert abs(eng.status().norm - c.step.status().norm) <= 1e-12 * eng.status().norm
        assert (eng.master - torch.cat(c.p)).abs().max() <= 1e-7


@gpu
@pytest.mark.parametrize("state_dtype", [DT_F32, DT_Q8])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_non_finite_norm_skips(state_dtype, bad):
    c = Case([300, 5000, 7], DT_F32, state_dtype, seed=5)
    c.g[1][4321] = bad
    c.step.step(hyper(1.0, zero=True))
    st = c.step.status()
    assert st.skipped == 1 and not math.isfinite(st.norm)
    after = c.snapshot()
    for k in ("p", "m", "v", "ms", "vs", "twin"):
        if after[k] is not None:
            assert all(torch.equal(x.contiguous().view(torch.uint8), y.contiguous().view(torch.uint8)) for x, y in zip(after[k], c.before[k]))
    assert not any(g.any() for g in c.g)


@gpu
@pytest.mark.parametrize("state_dtype", [DT_F32, DT_Q8])
def test_sitting_out_and_zeroing(state_dtype):
    """A tensor without a gradient has no share in the norm and stays; the others' gradients are left zeroed."""
    c = Case([300, 5000, 7, 2048], DT_BF16, state_dtype, seed=6)
    kept = c.g[1]
    c.step.step(hyper(0.01, zero=True), grads=[c.g[0], None, c.g[2], c.g[3]])
    norm = c.check(HYP, clip=0.01)
    assert abs(c.step.status().norm - norm) <= 1e-12 * norm
    assert kept.any() and not any(g.any() for g in (c.g[0], c.g[2], c.g[3]))
    c.step.step(hyper(0.0), grads=[None] * 4)
    assert c.step.status().norm == 0.0 and c.step.status().steps_done == 2


@gpu
def test_8_bit_edges():
    """A zero block, a block below 2^-100, one element that dwarfs the others, a NaN without the finite check."""
    n = 256 * 5 + 3
    p = torch.ones(n, device="cuda")
    g = torch.zeros(n, device="cuda")
    g[256:512] = 1e-25                  # m about 1e-26, v about 1e-51: v vanishes
    g[512:768] = 1e-6
    g[512] = 1e3                        # v of the others is 1e-18 of the largest: kept at the smallest number
    g[768 + 9] = math.nan
    g[1024:] = 1.0
    s = MultiStep([p], grads=[g], state_dtype=DT_Q8, decay=[False])
    s.step(hyper(check=False, t=1))
    m, v = s.moments()[0][0], s.moments()[1][0]
    assert not m[:256].any() and not v[:256].any() and (p[:256] == 1).all()
    assert (v[256:512] == 0).all() and s.v_scale[0][1] == 0 and (m[256:512] > 0).all()
    assert (s.v[0].view(torch.uint8)[513:768] == 1).all() and s.v[0].float()[512] == 57344
    assert torch.isfinite(p[512:768]).all()
    assert torch.isnan(p[777]) and torch.isfinite(p[768:777]).all() and torch.isnan(m[768:1024]).any()
    assert torch.isfinite(m[1024:]).all() and (v[1024:] > 0).all() and torch.isfinite(p[1024:]).all()
    g.zero_()
    q = p.clone()
    s.step(hyper(check=False, t=2))
    moved = (p - q)[512:768].abs()      # m of the small ones was rounded away or divides by a v that is not too small
    assert torch.isfinite(moved).all() and (moved <= HYP["lr"] / (1 - 0.9 ** 2) * 1.5).all()


@gpu
@pytest.mark.parametrize("stochastic", [False, True])
def test_8_bit_codes_are_those_of_the_float_formula(stochastic):
    """Every product and sum is rounded on its own: the formula in torch's fp32 gives the same codes and scales."""
    n = 256 * 400
    c = Case([n], DT_F32, DT_Q8, seed=21, twin=False)
    m0, v0, ms0, vs0, g = (x[0].clone() for x in (c.m, c.v, c.ms, c.vs, c.g))
    c.step.step(hyper(check=False, stochastic=stochastic), seed=77)
    at = lambda codes, scale: codes.float().view(-1, 256) * scale.view(-1, 1)  # noqa: E731
    b1, b2 = HYP["beta1"], HYP["beta2"]
    g = g.view(-1, 256)
    m = b1 * at(m0, ms0) + (1 - b1) * g
    v = b2 * at(v0, vs0) + (1 - b2) * g * g
    for x, codes, scale, top in ((m, c.m[0], c.ms[0], 448.0), (v, c.v[0], c.vs[0], 57344.0)):
        amax = x.abs().amax(1, keepdim=True)
        assert torch.equal(scale, (amax / top).view(-1))
        if not stochastic:
            want = (x * (top / amax)).clamp(-top, top).to(codes.dtype)
            if top > 448:
                want = torch.maximum(want.view(torch.uint8), (x > 0).to(torch.uint8)).view(codes.dtype)
            assert torch.equal(codes.view(torch.uint8), want.view(-1).view(torch.uint8))


@gpu
def test_stochastic_rounding_is_unbiased():
    """v decays by 0.1 % a step; to nearest it stays where it is, stochastically it follows on average.

    One element of each block holds the scale (its gradient keeps its v).  A step moves one of the others by D, at
    most a quarter of its value v, with probability 0.001 v / D: variance 0.001 v D <= 2.5e-4 v^2.  After 400 steps
    at most 0.1 v^2, for the mean of 4096 elements a deviation of at most sqrt(0.1 / 4096) = 0.005: six of them."""
    n = 4096 + 16
    start = 0.3 + 0.2 * torch.rand(n, generator=torch.Generator().manual_seed(8))
    start[::256] = 50.0
    g = torch.zeros(n, device="cuda")
    g[::256] = math.sqrt(50.0)
    inner = torch.ones(n, dtype=torch.bool, device="cuda")
    inner[::256] = False
    ends = {}
    for stochastic in (False, True):
        p = torch.zeros(n, device="cuda")
        v, vs = mtstep.encode(start, torch.float8_e5m2)
        m = torch.zeros(n, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
        s = MultiStep([p], grads=[g], state_dtype=DT_Q8, moments=([m], [v.cuda()]),
                      scales=([torch.zeros_like(vs).cuda()], [vs.cuda()]))
        first = s.moments()[1][0].double()
        for t in range(400):
            s.step(hyper(check=False, t=t + 1, beta2=0.999, stochastic=stochastic), seed=1000 + t)
        ends[stochastic] = float((s.moments()[1][0].double() / first)[inner].mean())
    assert abs(ends[True] - 0.999 ** 400) <= 0.03
    assert abs(ends[False] - 1.0) <= 1e-4


# ---- how it is called --------------------------------------------------------------------------------

@gpu
@pytest.mark.parametrize("state_dtype", [DT_F32, DT_Q8])
def test_captured_and_replayed(state_dtype):
    """Three replays of a captured set_grads + step = three eager steps; two graphs of two handles side by side."""
    a, b, c = (Case([300, 5000, 70001], DT_BF16, state_dtype, seed=9) for _ in range(3))
    for _ in range(3):
        a.step.step(hyper(1.0), seed=3)
    graphs = []
    for x in (b, c):
        st = torch.cuda.Stream()
        st.wait_stream(torch.cuda.current_stream())
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=st):
            x.step.step(hyper(1.0), seed=3, grads=x.g)
        graphs.append((gr, st))
    torch.cuda.synchronize()
    for _ in range(3):
        for gr, st in graphs:
            with torch.cuda.stream(st):
                gr.replay()
    torch.cuda.synchronize()
    want = a.snapshot()
    for x in (b, c):
        got = x.snapshot()
        for k in ("p", "m", "v", "twin"):
            assert all(torch.equal(y.contiguous().view(torch.uint8), z.contiguous().view(torch.uint8)) for y, z in zip(got[k], want[k])), k


@gpu
@pytest.mark.parametrize("state_dtype", [DT_F32, DT_Q8])
def test_gradients_move_between_replays(state_dtype):
    """A captured step takes the addresses that the handle has when it is replayed, on the 16-byte grid or off it."""
    c = Case([300, 5000, 70001, 2048], DT_BF16, state_dtype, seed=13)
    gr, st = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(gr, stream=st):
        c.step.step(hyper(0.5, zero=True))
    room = [torch.zeros(g.numel() + 3, dtype=g.dtype, device="cuda") for g in c.g]
    moved = [r[1 + k % 3:][:g.numel()] for k, (r, g) in enumerate(zip(room, c.g))]
    for a, b in zip(moved, c.g):
        a.copy_(b)
    c.step.set_grads(moved)
    torch.cuda.synchronize()
    gr.replay()
    torch.cuda.synchronize()
    kept = c.snapshot()["g"]
    assert all(torch.equal(a, b) for a, b in zip(kept, c.before["g"])) and not any(r.any() for r in room)
    c.check(HYP, clip=0.5)


@gpu
def test_two_lists_on_two_streams():
    """Steps of different handles overlap and do not disturb each other."""
    cs = [Case([70001, 300], DT_F32, DT_Q8, seed=10 + k) for k in range(2)]
    streams = [torch.cuda.Stream() for _ in cs]
    torch.cuda.synchronize()
    for c, st in zip(cs, streams):
        c.step.step(hyper(0.1), stream=st)
    torch.cuda.synchronize()
    for c in cs:
        c.check(HYP, clip=0.1)


@gpu
def test_the_same_inputs_give_the_same_bits():
    outs = []
    for _ in range(2):
        c = Case([70001, 4097, 300], DT_BF16, DT_Q8, seed=12)
        for t in range(3):
            c.step.step(hyper(0.1, t=t + 1, stochastic=True), seed=t)
        outs.append(c.snapshot())
    for k in ("p", "m", "v", "ms", "vs"):
        assert all(torch.equal(x.contiguous().view(torch.uint8), y.contiguous().view(torch.uint8)) for x, y in zip(outs[0][k], outs[1][k]))


@gpu
@pytest.mark.parametrize("state_dtype", [DT_F32, DT_Q8])
def test_nothing_to_step(state_dtype):
    """Empty tensors alone, and tensors that all sit out: the step closes, the norm is 0."""
    for n in (0, 5000):
        p = torch.ones(n, device="cuda")
        s = MultiStep([p, torch.zeros(0, device="cuda")], grads=[torch.zeros(0, device="cuda") if n == 0 else None, None],
                      state_dtype=state_dtype)
        s.step(hyper(1.0))
        st = s.status()
        assert st.error == 0 and st.skipped == 0 and st.norm == 0.0 and st.steps_done == 1 and (p == 1).all()


@gpu
def test_python_refusals():
    p, g = torch.zeros(8, device="cuda"), torch.zeros(8, device="cuda")
    for bad in (dict(grads=[g[:4]]), dict(grads=[g, g]), dict(decay=[True, False]), dict(twins=[g]),
                dict(moments=([g], [g]), state_dtype=DT_Q8), dict(grads=[g.half()]), dict(state_dtype=DT_BF16)):
        with pytest.raises((ValueError, TypeError)):
            MultiStep([p], **bad)
    with pytest.raises(TypeError):
        MultiStep([torch.zeros(4, 4, device="cuda").t()[1:]])
    with pytest.raises(capi.AnniError):         # the same tensor twice
        MultiStep([p, p], grads=[g, g.clone()])
    with pytest.raises(capi.AnniError):         # a gradient inside a parameter
        MultiStep([p], grads=[p])
    s = MultiStep([p], grads=[g])
    for h in (hyper(stochastic=True), OptStep.hyper(lr=1e-3, t=1, exact=True), OptStep.hyper(lr=1e-3, t=1, dev_loss_scale=True)):
        with pytest.raises(capi.AnniError):
            s.step(h)
    with pytest.raises(ValueError):
        s.set_grads([g, g])


# ---- refusals of the C entry points: no device needed ------------------------------------------------

def _create(edit=lambda t: None, n=1, grad_dtype=DT_F32, state_dtype=DT_F32):
    """Create over n entries of made-up addresses, `edit`ed; the code it answers (E_CUDA: the arguments passed)."""
    L = mtstep.lib()
    arr = (mtstep.Tensor * max(n, 1))()
    for k, t in enumerate(arr):
        base = 0x10000000 * (k + 1)
        t.param, t.grad, t.m, t.v = base, base + 0x100000, base + 0x200000, base + 0x300000
        t.m_scale, t.v_scale, t.twin_bf16 = base + 0x400000, base + 0x500000, base + 0x600000
        t.n, t.flags = 1000, capi.SEG_WD | capi.SEG_TWIN_BF16
    edit(arr[0])
    h = C.c_void_p()
    rc = L.anni_mtstep_create(arr, n, grad_dtype, state_dtype, C.byref(h))
    if rc == capi.OK:
        L.anni_mtstep_destroy(h)
    return rc


def _set(**kw):
    def edit(t):
        for k, x in kw.items():
            setattr(t, k, x)
    return edit


@pytest.mark.parametrize("kw", [
    dict(n=0), dict(n=-1), dict(grad_dtype=2), dict(grad_dtype=-1), dict(state_dtype=DT_BF16), dict(state_dtype=3),
    dict(edit=_set(n=-1)), dict(edit=_set(flags=capi.SEG_TWIN_FP8)), dict(edit=_set(param=None)),
    dict(edit=_set(m=None)), dict(edit=_set(v=None)), dict(edit=_set(twin_bf16=None)),
    dict(edit=_set(m_scale=None), state_dtype=DT_Q8), dict(edit=_set(v_scale=None), state_dtype=DT_Q8),
    dict(edit=_set(param=0x10000002)), dict(edit=_set(m=0x10200001)), dict(edit=_set(twin_bf16=0x10600001)),
    dict(edit=_set(m_scale=0x10400002), state_dtype=DT_Q8), dict(edit=_set(grad=0x10100002)),
    dict(edit=_set(grad=0x10100001), grad_dtype=DT_BF16),
    dict(edit=_set(m=0x10000000)), dict(edit=_set(v=0x10200000 + 3996)), dict(edit=_set(grad=0x10000000)),
    dict(edit=_set(param=0x20000000), n=2), dict(edit=_set(grad=0x20100000), n=2)])
def test_create_refuses(kw):
    assert _create(**kw) == capi.E_ARG


def test_create_accepts_what_the_header_allows():
    """Odd addresses of 8-bit moments, empty tensors without addresses, missing gradients: only the device is missing."""
    if torch.cuda.is_available():
        pytest.skip("made-up addresses: for a machine without a device")
    empty = _set(n=0, param=None, m=None, v=None, m_scale=None, v_scale=None, twin_bf16=None, grad=None)
    for kw in (dict(), dict(state_dtype=DT_Q8), dict(edit=empty), dict(edit=_set(grad=None)),
               dict(edit=_set(m=0x10200001, v=0x10300003), state_dtype=DT_Q8),
               dict(edit=_set(m_scale=None, v_scale=None)), dict(n=300)):
        assert _create(**kw) == capi.E_CUDA


def test_null_handles_are_refused():
    L = mtstep.lib()
    hp, st = capi.Hyper(), capi.Status()
    arr = (C.c_void_p * 1)()
    assert L.anni_mtstep_create(None, 1, 0, 0, C.byref(C.c_void_p())) == capi.E_ARG
    assert L.anni_mtstep_create((mtstep.Tensor * 1)(), 1, 0, 0, None) == capi.E_ARG
    assert L.anni_mtstep_set_grads(None, arr, None) == capi.E_ARG
    assert L.anni_mtstep_step(None, C.byref(hp), 0, None) == capi.E_ARG
    assert L.anni_mtstep_status_read(None, C.byref(st), None) == capi.E_ARG
    L.anni_mtstep_destroy(None)


def test_every_declared_symbol_is_exported():
    from test_abi_cpu import _declared_symbols
    names = _declared_symbols("anni_mtstep.h")
    assert len(names) == 5 and not [n for n in names if not hasattr(mtstep.lib(), n)]


def test_encode_decode_on_the_host():
    """The host helpers: every number within half a step of its type, blocks of zeros, short last block."""
    x = torch.randn(1000, generator=torch.Generator().manual_seed(1), dtype=torch.float32)
    x[256:512] = 0
    for kind, half, y in ((torch.float8_e4m3fn, 2.0 ** -4, x), (torch.float8_e5m2, 2.0 ** -3, x * x)):
        codes, scale = mtstep.encode(y, kind)
        assert codes.dtype == kind and len(codes) == 1000 and len(scale) == 4 and scale[1] == 0
        back = mtstep.decode(codes, scale)
        small = scale.repeat_interleave(256)[:1000] * (2.0 ** -9 if kind == torch.float8_e4m3fn else 2.0 ** -16)
        assert ((back - y).abs() <= half * y.abs() * (1 + 1e-6) + small).all()
