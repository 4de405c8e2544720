"""What the operators of a training step cost: AdamW over a list of tensors, and the loss of the head.

Two operators.  ``list``: one AdamW step over tensors that lie wherever the program put them, moments in 32
bits or in 8 (e4m3 / e5m2 numbers with one fp32 scale per 256 elements), with the global norm, the clip and
the skip of a non-finite norm, decay by tensor, bf16 twins.  ``head``: softmax cross entropy of x W + b over a
vocabulary, rows of loss and log-sum-exp, and with ``grad`` the gradients of x, W and b.

``own`` says which side ``run`` computes: False the plain form in elementary torch operations, True the
calls of ``anni_b200``.
"""
import math
import random

import torch

own = False

BLOCK = 256         # elements that share a scale
STEP = dict(lr=3e-4, beta1=0.9, beta2=0.95, eps=1e-8, wd=0.1, clip=1.0, t=1000)


# ---------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------

def listed():
    lists = [
        # the unit-test language model: 28 tensors, 138,156 elements; what a call costs at least
        dict(name="list32_tiny", op="list", layout="lm", d=64, ff=256, blocks=2, vocab=300, tied=False, bits=32,
             grad="f32", twin=True, clip=True, stochastic=False),
        # low-rank adapters beside a frozen model: many small matrices, 8-bit moments rounded at random
        dict(name="list8_adapters", op="list", layout="ragged", tensors=448, least=1000, most=60000, pick=11,
             bits=8, grad="bf16", twin=True, clip=True, stochastic=True),
        # 184.7 M parameters whose gradients arrive in bf16, 32-bit moments
        dict(name="list32_184m", op="list", layout="lm", d=1024, ff=4096, blocks=12, vocab=16384, tied=False,
             bits=32, grad="bf16", twin=True, clip=True, stochastic=False),
        # the same with moments in 8 bits: a quarter of the optimizer's memory
        dict(name="list8_184m", op="list", layout="lm", d=1024, ff=4096, blocks=12, vocab=16384, tied=False,
             bits=8, grad="bf16", twin=True, clip=True, stochastic=False),
        # wide blocks, fp32 gradients already clipped elsewhere, 8 bits rounded at random, no twins
        dict(name="list8_98m_f32", op="list", layout="lm", d=1536, ff=6272, blocks=3, vocab=8000, tied=True,
             bits=8, grad="f32", twin=False, clip=False, stochastic=True),
    ]
    heads = [
        # the unit-test language model's head, its vocabulary no multiple of a vector
        dict(name="head_tiny", op="head", tokens=127, d=64, vocab=300, grad="bf16", bias=True, ignored=0.1,
             weights=False, masked=0, add=False),
        # one token scored against the large vocabulary: W is read once
        dict(name="head_one_row", op="head", tokens=1, d=1536, vocab=100000, grad="", bias=True, ignored=0.0,
             weights=False, masked=0, add=False),
        # validation: losses only
        dict(name="head_eval", op="head", tokens=4096, d=1024, vocab=16384, grad="", bias=True, ignored=0.0,
             weights=False, masked=0, add=False),
        # a micro-batch of the 184.7 M model, gradients added to those of the micro-batches before
        dict(name="head_train_16k", op="head", tokens=8192, d=1024, vocab=16384, grad="bf16", bias=True,
             ignored=0.1, weights=False, masked=0, add=True),
        # the largest head: 100,000 entries, the last 64 of them padding that a -inf bias masks
        dict(name="head_train_100k", op="head", tokens=4096, d=1536, vocab=100000, grad="bf16", bias=True,
             ignored=0.0, weights=False, masked=64, add=False),
        # fp32 gradients, rows weighted one by one, every size odd
        dict(name="head_train_odd_f32", op="head", tokens=1001, d=1001, vocab=5003, grad="f32", bias=False,
             ignored=0.2, weights=True, masked=0, add=False),
    ]
    return lists + heads


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    if rng.random() < 0.5:
        most = _log_int(rng, 300, 30_000_000)
        tensors = _log_int(rng, 1, max(1, min(2000, 150_000_000 // most)))
        return dict(op="list", layout="ragged", tensors=tensors, least=1, most=most, pick=rng.randrange(1 << 30),
                    bits=rng.choice((8, 8, 32)), grad=rng.choice(("f32", "bf16")), twin=rng.random() < 0.5,
                    clip=rng.random() < 0.7, stochastic=rng.random() < 0.5)
    tokens = _log_int(rng, 1, 8192)
    d = _log_int(rng, 64, 2560)
    vocab = _log_int(rng, 300, 100000)
    if rng.random() < 0.6:          # sizes of models are mostly round
        d, vocab = -(-d // 64) * 64, -(-vocab // 8) * 8
    while tokens * d * vocab > 4096 * 1536 * 100000:
        tokens = max(1, tokens // 2)
    return dict(op="head", tokens=tokens, d=d, vocab=vocab, grad=rng.choice(("", "bf16", "bf16", "f32")),
                bias=rng.random() < 0.7, ignored=rng.choice((0.0, 0.1, 0.5)), weights=rng.random() < 0.3,
                masked=rng.choice((0, 0, 17)), add=rng.random() < 0.3)


def _sizes(case):
    """Element counts of the list's tensors and which of them decay."""
    if case["layout"] == "lm":
        d, ff, v = case["d"], case["ff"], case["vocab"]
        block = [(d * d, 1)] * 4 + [(d * ff, 1), (ff, 0), (ff * d, 1)] + [(d, 0)] * 5
        return [(d * v, 1), (v, 0)] + ([] if case["tied"] else [(v * d, 1)]) + block * case["blocks"]
    r = random.Random(case["pick"])
    return [(_log_int(r, case["least"], case["most"]), r.randrange(2)) for _ in range(case["tensors"])]


def work(case):
    if case["op"] == "list":
        n = sum(k for k, _ in _sizes(case))
        moments = 16.0 if case["bits"] == 32 else 4.0 + 16.0 / BLOCK
        per = (2 if case["grad"] == "bf16" else 4) + 8 + moments + (2 if case["twin"] else 0)
        return {"bytes": per * n, "flops": 20.0 * n}
    t, d, v = case["tokens"], case["d"], case["vocab"]
    size = {"": 0, "bf16": 2, "f32": 4}[case["grad"]]
    read = 2 * t * d + 2 * d * v + 4 * t + (4 * v if case["bias"] else 0)
    written = 8 * t + size * (t * d + (2 if case["add"] else 1) * (d * v + v))
    return {"bytes": float(read + written), "flops": 2.0 * t * d * v * (3 if case["grad"] else 1)}


# ---------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------

def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return (_prepare_list if case["op"] == "list" else _prepare_head)(case, seed, gen)


def _normal(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda")


def _prepare_list(case, seed, gen):
    # The tensors lie in buffers that give each of them whole blocks of 256 elements, as an allocator does; what
    # lies between them is zero and stays so.
    sizes = torch.tensor([k for k, _ in _sizes(case)])
    blocks = (sizes + BLOCK - 1) // BLOCK
    start = (torch.cumsum(blocks, 0) - blocks) * BLOCK
    total = int(blocks.sum())
    owner = torch.repeat_interleave(torch.arange(len(sizes)), blocks).cuda()
    decays = torch.tensor([float(k) for _, k in _sizes(case)]).cuda()[owner]
    last = (start + sizes).cuda()[owner].view(-1, 1)
    inside = torch.arange(total * BLOCK, device="cuda").view(-1, BLOCK) < last
    spread = torch.exp(0.5 * _normal(gen, total, 1))       # gradients of one block are alike, of two less so
    s = {"case": case, "seed": seed, "decays": decays.view(-1, 1), "block": torch.arange(total, device="cuda").view(-1, 1)}
    grad = torch.where(inside, _normal(gen, total, BLOCK) * spread * 1e-3, 0)
    s["grad"] = grad.to(torch.bfloat16 if case["grad"] == "bf16" else torch.float32).view(-1)
    del grad
    s["param"] = torch.where(inside, _normal(gen, total, BLOCK) * 0.02, 0).view(-1)
    m = torch.where(inside, _normal(gen, total, BLOCK) * spread * 3e-4, 0)
    v = torch.where(inside, (_normal(gen, total, BLOCK) * spread * 1e-3).square() + 1e-9, 0)
    if case["bits"] == 32:
        s["m"], s["v"] = m.view(-1), v.view(-1)
    else:
        s["m_scale"], s["v_scale"] = m.abs().amax(1) / 448.0, v.amax(1) / 57344.0
        s["m"] = (m / s["m_scale"].view(-1, 1)).to(torch.float8_e4m3fn).view(-1)
        s["v"] = (v / s["v_scale"].view(-1, 1)).to(torch.float8_e5m2).view(-1)
    if case["twin"]:
        s["twin"] = s["param"].bfloat16()
    if own:
        from anni_b200 import capi
        from anni_b200.engine import OptStep
        from anni_b200.mtstep import MultiStep
        at = list(zip(start.tolist(), sizes.tolist()))
        piece = lambda x, per=1: [x[a // per:a // per + -(-k // per)] for a, k in at]  # noqa: E731
        eight = case["bits"] == 8
        s["engine"] = MultiStep(
            piece(s["param"]), state_dtype=capi.DT_Q8 if eight else capi.DT_F32, grads=piece(s["grad"]),
            decay=[bool(k) for _, k in _sizes(case)], twins=piece(s["twin"]) if case["twin"] else None,
            moments=(piece(s["m"]), piece(s["v"])),
            scales=(piece(s["m_scale"], BLOCK), piece(s["v_scale"], BLOCK)) if eight else None)
        s["hyper"] = OptStep.hyper(**{**STEP, "clip": STEP["clip"] if case["clip"] else 0.0},
                                   check_finite=case["clip"], zero_grad=False)
        if case["stochastic"] and eight:
            s["hyper"].flags |= capi.STEP_STOCHASTIC
    return s


def _prepare_head(case, seed, gen):
    t, d, v = case["tokens"], case["d"], case["vocab"]
    s = {"case": case}
    s["x"] = _normal(gen, t, d).bfloat16()
    s["w"] = (_normal(gen, d, v) * (1.5 / math.sqrt(d))).bfloat16()
    target = torch.randint(0, v - case["masked"], (t,), generator=gen, device="cuda")
    skip = torch.rand(t, generator=gen, device="cuda") < case["ignored"]
    s["target"] = torch.where(skip, -1, target).int()
    # some of the rows are predicted well: the row of x has the target's column in it
    known = torch.rand(t, 1, generator=gen, device="cuda") < 0.5
    s["x"] = torch.where(known, (s["x"] + 4.0 * s["w"][:, target].t()).bfloat16(), s["x"]).contiguous()
    s["bias"] = s["weight"] = None
    if case["bias"] or case["masked"]:
        s["bias"] = 0.1 * _normal(gen, v)
        s["bias"][v - case["masked"]:] = -math.inf
    if case["weights"]:
        s["weight"] = torch.rand(t, generator=gen, device="cuda") * 2.0
    if case["grad"]:
        kind = torch.bfloat16 if case["grad"] == "bf16" else torch.float32
        s["dx"] = torch.empty(t, d, dtype=kind, device="cuda")
        s["dw"] = torch.randn(d, v, generator=gen, device="cuda", dtype=kind) if case["add"] else torch.empty(d, v, dtype=kind, device="cuda")
        s["db"] = torch.randn(v, generator=gen, device="cuda", dtype=kind) if case["add"] else torch.empty(v, dtype=kind, device="cuda")
    return s


# ---------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------

def run(s):
    if s["case"]["op"] == "list":
        if own:
            s["engine"].step(s["hyper"], seed=s["seed"])
        else:
            _plain_list(s)
        return {k: s[k] for k in ("param", "m", "v", "m_scale", "v_scale", "twin") if k in s}
    return _own_head(s) if own else _plain_head(s)


def _own_head(s):
    from anni_b200.head import head_loss, head_loss_grad
    nll, lse = head_loss(s["x"], s["w"], s["target"], bias=s["bias"])
    out = {"nll": nll, "lse": lse}
    if s["case"]["grad"]:
        head_loss_grad(s["x"], s["w"], s["target"], lse, bias=s["bias"], weight=s["weight"], dx=s["dx"], dw=s["dw"],
                       dbias=s["db"], accumulate=s["case"]["add"])
        out.update(dx=s["dx"], dw=s["dw"], db=s["db"])
    return out


def _plain_head(s):
    keep = s["target"] >= 0
    at = s["target"].clamp_min(0).long().view(-1, 1)
    logits = s["x"].float() @ s["w"].float()
    if s["bias"] is not None:
        logits += s["bias"]
    top = logits.amax(1, keepdim=True)
    lse = (logits - top).exp().sum(1).log() + top.view(-1)
    nll = torch.where(keep, lse - logits.gather(1, at).view(-1), 0)
    out = {"nll": nll, "lse": lse}
    if not s["case"]["grad"]:
        return out
    delta = (logits - lse.view(-1, 1)).exp_()
    del logits
    delta.scatter_add_(1, at, torch.full_like(at, -1, dtype=torch.float32))
    delta *= (keep.float() * (1.0 if s["weight"] is None else s["weight"])).view(-1, 1)
    dx, dw, db = delta @ s["w"].float().t(), s["x"].float().t() @ delta, delta.double().sum(0)
    if s["case"]["add"]:
        dw, db = dw + s["dw"].float(), db + s["db"].double()
    s["dx"].copy_(dx)
    s["dw"].copy_(dw)
    s["db"].copy_(db)
    out.update(dx=s["dx"], dw=s["dw"], db=s["db"])
    return out


def _bits32(x):
    return x & 0xFFFFFFFF


def _mix(h):
    """The 32-bit finaliser of MurmurHash3 (Appleby, public domain)."""
    h = _bits32((h ^ (h >> 16)) * 0x85EBCA6B)
    h = _bits32((h ^ (h >> 13)) * 0xC2B2AE35)
    return h ^ (h >> 16)


def _draws(seed, block):
    """Random 32 bits of each element: of the seed, its block's number in the list and its place in the block."""
    key = _mix(_bits32(seed ^ _mix(_bits32(block + (seed >> 32) * 0x9E3779B9))))
    return _mix(_bits32(key + torch.arange(BLOCK, device=block.device) * 0x9E3779B9))


def _stochastic(x, draws, kept, least):
    """x rounded to ``kept`` bits of mantissa: up with the chance of the part cut off, in 16 random bits; below
    ``least``, the smallest normal number, to multiples of its last place."""
    cut = 23 - kept
    y = x.abs()
    y = y + torch.where(y < least, least, 0.0)
    bits = y.view(torch.int32) + (draws << (cut - 16)).int()
    r = ((bits >> cut) << cut).view(torch.float32)
    return torch.copysign(r - torch.where(x.abs() < least, least, 0.0), x)


def _eight(x, top, kind, draws, kept, least):
    """Blocks of x as 8-bit numbers and their scales."""
    amax = x.abs().amax(1, keepdim=True)
    some = amax >= 2.0 ** -100
    scale = torch.where(some, amax / top, 0)
    y = x * torch.where(some, top / amax, 0)
    if draws is not None:
        y = _stochastic(y, draws, kept, least)
    return y.clamp(-top, top).to(kind), scale


def _plain_list(s):
    case = s["case"]
    lr, b1, b2, eps, wd, t = (STEP[k] for k in ("lr", "beta1", "beta2", "eps", "wd", "t"))
    g = s["grad"].view(-1, BLOCK).float()
    fine = None
    if case["clip"]:
        norm = g.double().square().sum().sqrt()
        fine = norm.isfinite()
        g = g * torch.where(norm > STEP["clip"], STEP["clip"] / (norm + 1e-12), 1.0).float()
    p = s["param"].view(-1, BLOCK)
    m, v = s["m"].float().view(-1, BLOCK), s["v"].float().view(-1, BLOCK)
    if case["bits"] == 8:
        m, v = m * s["m_scale"].view(-1, 1), v * s["v_scale"].view(-1, 1)
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    q = p - (lr / (1 - b1 ** t)) * m / ((v / (1 - b2 ** t)).sqrt() + eps)
    q = q - lr * wd * s["decays"] * q
    new = {"param": q}
    if case["bits"] == 8:
        draws = _draws(s["seed"], s["block"]) if case["stochastic"] else None
        new["m"], new["m_scale"] = _eight(m, 448.0, torch.float8_e4m3fn, None if draws is None else draws & 0xFFFF, 3, 2.0 ** -6)
        e, new["v_scale"] = _eight(v, 57344.0, torch.float8_e5m2, None if draws is None else draws >> 16, 2, 2.0 ** -14)
        new["v"] = torch.maximum(e.view(torch.uint8), (v > 0).to(torch.uint8) * (new["v_scale"] > 0)).view(torch.float8_e5m2)
    else:
        new["m"], new["v"] = m, v
    if case["twin"]:
        new["twin"] = q.bfloat16()
    for k, x in new.items():
        x = x.reshape(-1)
        if fine is not None:
            raw = {1: torch.uint8, 2: torch.int16, 4: torch.int32}[x.element_size()]
            x = torch.where(fine, x.view(raw), s[k].view(raw)).view(x.dtype)
        s[k].copy_(x)


# ---------------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------------

def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    return _exact_list(s, seed) if case["op"] == "list" else _exact_head(s)


def _exact_head(s):
    x, w, target = s["x"].double(), s["w"].double(), s["target"].long()
    b = 0.0 if s["bias"] is None else s["bias"].double()
    grad = bool(s["case"]["grad"])
    t, v = len(x), w.shape[1]
    nll, lse = torch.zeros(t, dtype=torch.float64, device="cuda"), torch.zeros(t, dtype=torch.float64, device="cuda")
    dx, dw, db = (torch.zeros_like(x), torch.zeros_like(w), torch.zeros(v, dtype=torch.float64, device="cuda")) if grad else (None,) * 3
    for a in range(0, t, 1024):
        rows = torch.arange(a, min(t, a + 1024), device="cuda")
        z = torch.addmm(torch.zeros(1, dtype=torch.float64, device="cuda"), x[rows], w) + b
        lse[rows] = torch.logsumexp(z, 1)
        counted = rows[target[rows] >= 0]
        nll[counted] = lse[counted] - z[counted - a, target[counted]]
        if grad:
            factor = torch.zeros(len(rows), dtype=torch.float64, device="cuda")
            factor[counted - a] = 1.0 if s["weight"] is None else s["weight"][counted].double()
            z = torch.softmax(z, 1)
            z[counted - a, target[counted]] -= 1.0
            z *= factor[:, None]
            dx[rows] = torch.mm(z, w.t())
            dw += torch.mm(x[rows].t(), z)
            db += z.sum(0)
    out = {"nll": nll, "lse": lse}
    if grad:
        if s["case"]["add"]:
            dw, db = dw + s["dw"].double(), db + s["db"].double()
        out.update(dx=dx, dw=dw, db=db)
    return out


def _values(exponent_bits, mantissa_bits, count):
    """The non-negative finite numbers of an 8-bit type, ascending."""
    bias = 2 ** (exponent_bits - 1) - 1
    of = lambda e, f: math.ldexp(f / 2 ** mantissa_bits + (e > 0), max(e, 1) - bias)  # noqa: E731
    return torch.tensor([of(c >> mantissa_bits, c & (2 ** mantissa_bits - 1)) for c in range(count)], dtype=torch.float64, device="cuda")


def _rounded(y, table, draws):
    """|y| taken to a number of the table, the nearest (of two equally near the even one), or by chance."""
    y = y.clamp_max(table[-1])
    lo = (torch.searchsorted(table, y, right=True) - 1).clamp(0, len(table) - 2)
    part = (y - table[lo]) / (table[lo + 1] - table[lo])
    if draws is None:
        up = (part > 0.5) | ((part == 0.5) & (lo % 2 == 1))
    else:
        up = part + draws.double() / 65536.0 >= 1.0
    return lo + up.long()


def _exact_list(s, seed):
    case, h = s["case"], STEP
    grad = s["grad"].double()
    coef = 1.0
    if case["clip"]:
        norm = float(torch.linalg.vector_norm(grad))
        coef = h["clip"] / (norm + 1e-12) if norm > h["clip"] else 1.0
    tables = (_values(4, 3, 127), _values(5, 2, 124)) if case["bits"] == 8 else None
    out = {k: torch.empty(s[k].shape, dtype=torch.float64, device="cuda") for k in ("param", "m", "v", "m_scale", "v_scale", "twin") if k in s}
    piece = 1 << 14         # blocks at a time
    for a in range(0, len(s["decays"]), piece):
        here = slice(a, a + piece)
        flat = slice(a * BLOCK, (a + piece) * BLOCK)
        g = grad[flat] * coef
        p, m, v = s["param"][flat].double(), s["m"][flat].double(), s["v"][flat].double()
        if tables:
            m = m * s["m_scale"][here].double().repeat_interleave(BLOCK)
            v = v * s["v_scale"][here].double().repeat_interleave(BLOCK)
        m = m * h["beta1"] + g * (1 - h["beta1"])
        v = v * h["beta2"] + g ** 2 * (1 - h["beta2"])
        p = p - h["lr"] * (m / (1 - h["beta1"] ** h["t"])) / (torch.sqrt(v / (1 - h["beta2"] ** h["t"])) + h["eps"])
        p = p * (1 - h["lr"] * h["wd"] * s["decays"][here].double().view(-1).repeat_interleave(BLOCK))
        out["param"][flat] = p
        if case["twin"]:
            out["twin"][flat] = p
        if not tables:
            out["m"][flat], out["v"][flat] = m, v
            continue
        draws = _draws(seed, s["block"][here]).view(-1) if case["stochastic"] else None
        for name, x, table, shift, floor in (("m", m, tables[0], 0, 0), ("v", v, tables[1], 16, 1)):
            amax = x.abs().view(-1, BLOCK).amax(1)
            scale = amax / table[-1]
            y = torch.nan_to_num(x.abs() / scale.repeat_interleave(BLOCK), nan=0.0)
            code = _rounded(y, table, None if draws is None else (draws >> shift) & 0xFFFF)
            if floor:
                code = torch.maximum(code, (x > 0).long())
            out[name + "_scale"][here] = scale
            out[name][flat] = table[code] * torch.sign(x)
    return out
