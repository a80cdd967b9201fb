"""The sequence-block operators (gated residual norm, block-scaled fp8 product, gated linear recurrence) against their definitions in
64 bits.  Tolerances: half a step of the output's type, plus the number of fp32 roundings on a value's way times 2^-24 times the size
of what is added up there (the formula over absolute values)."""
import math

import pytest
import torch

import seqblock_ref as R
from tecogan_amd import kernels as K
from tecogan_amd._lib import TecoHipError

pytestmark = pytest.mark.gpu
DEV = "cuda"
KINDS = dict(none=K.NORM_NONE, rms=K.NORM_RMS, layer=K.NORM_LAYER)
ACTS = dict(none=K.ACT_NONE, sigmoid=K.ACT_SIGMOID, tanh=K.ACT_TANH, silu=K.ACT_SILU)
BF, F32 = torch.bfloat16, torch.float32


def rnd(*shape, seed=0, dtype=F32, scale=1.0, mean=0.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale + mean).to(dtype)


def within(got, want, bound, what):
    got, want, bound = got.detach().double().cpu(), want.detach().double().cpu(), bound.detach().double().cpu()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    bad = ~((got - want).abs() <= bound)
    bad &= ~(torch.isnan(got) & torch.isnan(want))
    assert not bad.any(), "%s: %d of %d outside; worst %g times its bound (got %g, want %g)" % (
        what, int(bad.sum()), bad.numel(), float(((got - want).abs() / bound.clamp_min(1e-300))[bad].max()), float(got[bad][0]), float(want[bad][0]))


# ---- gated norm ----------------------------------------------------------------------------------------------------------------
# rows, C, dtype, res, post, pre, gate (None / rows per gate), act, scale, row stride factor
NORM_CASES = [
    (1, 1, F32, F32, "none", "rms", 1, "none", False, 1),
    (1, 2048, BF, BF, "rms", "rms", 1, "none", True, 1),
    (3, 7, BF, BF, "rms", "layer", 2, "silu", True, 1),              # scalar path, a short last gate row
    (37, 24, F32, F32, "layer", "layer", 5, "tanh", True, 1),        # several rows a wave, whole gate rows in an item
    (130, 64, BF, F32, "none", "layer", None, "none", True, 1),
    (257, 136, BF, BF, "layer", "rms", 257, "sigmoid", False, 1),    # one gate row for all: pieces
    (64, 520, F32, F32, "rms", "rms", 1, "sigmoid", True, 3),        # strided rows; a row over several waves, lanes past its end
    (19, 1000, BF, F32, "rms", "none", 1, "silu", True, 1),          # no pre norm: the residual stream alone
    (9, 4104, BF, BF, "rms", "layer", 4, "tanh", True, 2),           # two vectors a lane
    (5, 8193, BF, F32, "layer", "rms", 1, "none", True, 1),          # four vectors a lane, scalar path
    (4, 16384, F32, F32, "rms", "layer", 2, "sigmoid", True, 1),     # the widest row
    (2100, 96, BF, BF, "rms", "rms", 700, "none", True, 1),          # pieces of several gate rows
    (11, 5000, BF, F32, "layer", "layer", 3, "sigmoid", True, 1),    # more parameter sums than one pass over wide rows holds
    (40, 1003, BF, BF, "layer", "rms", 1, "tanh", True, 1),          # rows that begin at every alignment
    (40, 1003, F32, F32, "rms", "layer", 8, "silu", True, 1),
    (29, 7740, BF, F32, "layer", "rms", 6, "tanh", True, 1),         # wide rows value by value, gate rows in pieces of one row
    (6, 12001, BF, BF, "rms", "layer", 1, "silu", True, 1),
    (30000, 88, BF, BF, "rms", "rms", 13, "sigmoid", False, 1),      # whole gate rows longer than an even share of the rows
    (9000, 89, BF, F32, "none", "layer", None, "none", True, 1),
]


def norm_inputs(case, seed=0):
    rows, C, dt, res, post, pre, k, act, scale, f = case
    i = dict(x=rnd(rows, C, seed=seed, dtype=res, scale=2.0, mean=0.5), o=rnd(rows, C, seed=seed + 1, dtype=dt, scale=1.5),
             gate=None if k is None else rnd(-(-rows // k), C, seed=seed + 2, dtype=dt))
    p = dict(w_post=rnd(C, seed=3, scale=0.1, mean=1.0) if post != "none" else None,
             b_post=rnd(C, seed=4, scale=0.1) if post == "layer" else None, scale=rnd(C, seed=5, scale=0.3) if scale else None,
             w_pre=rnd(C, seed=6, scale=0.1, mean=1.0) if pre != "none" else None, b_pre=rnd(C, seed=7, scale=0.1) if pre == "layer" else None)
    return i, p


def dev(t, f=1):
    """On the GPU; f > 1: every f-th slice of a wider tensor, as a part of a projection is."""
    if t is None:
        return None
    if f == 1:
        return t.to(DEV)
    wide = torch.full((t.shape[0], t.shape[1] * f), float("nan"), device=DEV, dtype=t.dtype)
    wide[:, t.shape[1]:2 * t.shape[1]] = t.to(DEV)
    return wide[:, t.shape[1]:2 * t.shape[1]]


def norm_how(case, p, alpha=0.7, eps=1e-5):
    rows, C, dt, res, post, pre, k, act, scale, f = case
    return dict(post=KINDS[post], pre=KINDS[pre], alpha=alpha, gate_act=ACTS[act], rows_per_gate=k or 1, eps=eps,
                **{n: dev(v) for n, v in p.items()})


def d64(i):
    return {n: None if v is None else v.double() for n, v in i.items()}


def size_of_norm(kind, z, eps):
    """|z^| + 1 + |mean| r: what a normalised value's error is relative to."""
    if kind == "none":
        return z.abs()
    mu, r = R.moments(kind, z, eps)
    return ((z - mu) * r).abs() + 1 + mu.abs() * r


# fp32 roundings on a value's way: sums over a row (at most 32 additions in a lane, 6 exchanges, 8 waves), twice, and about 40
# operations, exponentials (argument below 16: 16 units) among them
N_VALUE = 160


@pytest.mark.parametrize("case", NORM_CASES)
def test_gated_norm_forward(case):
    rows, C, dt, res, post, pre, k, act, scale, f = case
    i, p = norm_inputs(case)
    alpha, eps = 0.7, 1e-5
    y = dev(torch.zeros(rows, C, dtype=res), f)
    h = dev(torch.zeros(rows, C, dtype=dt), f) if pre != "none" else None
    K.gated_norm_forward(dev(i["x"], f), dev(i["o"], f), dev(i["gate"]), y, h, **norm_how(case, p))
    a, q = d64(i), d64(p)
    wy, wh = R.norm_forward(a["x"], a["o"], a["gate"], q, post, pre, act, k or 1, alpha, eps)
    s = size_of_norm(post, a["o"], eps) * (1 if q["w_post"] is None else q["w_post"].abs()) + (0 if q["b_post"] is None else q["b_post"].abs())
    s = s * alpha * (1 if q["scale"] is None else q["scale"].abs())
    if k is not None:
        s = s * (R.act(act, R.gate_rows(a["gate"], k, rows)).abs() + R.U32)
    err = N_VALUE * R.U32 * (s + a["x"].abs())
    within(y, wy, err + R.HALF[res] * wy.abs() * 1.01, "y %s" % (case,))
    if h is not None:
        _, r = R.moments(pre, wy, eps)
        w = 1 if q["w_pre"] is None else q["w_pre"].abs()
        eh = (r * (err + err.mean(-1, keepdim=True)) + N_VALUE * R.U32 * size_of_norm(pre, wy, eps)) * w + 4 * R.U32
        eh = eh + size_of_norm(pre, wy, eps) * w * (r * err).square().mean(-1, keepdim=True).sqrt()       # through 1 / deviation
        within(h, wh, eh + R.HALF[dt] * wh.abs() * 1.01, "h %s" % (case,))


def norm_gradients(case, i, p, d_y, d_h, alpha, eps):
    """fp64 gradients by autograd (of y's rounded value as the backward pass gets it) and their bounds by the absolute formula."""
    rows, C, dt, res, post, pre, k, act, scale, f = case
    a = {n: None if v is None else v.double() for n, v in {**i, **p}.items()}
    y, o, gate = a["x"], a["o"], a["gate"]                         # i["x"] holds y here
    g = act_rows = slope = None
    if gate is not None:
        g = R.gate_rows(gate, k, rows)
        act_rows, slope = R.act(act, g), R.act_slope(act, g)
    one = torch.ones(C, dtype=torch.float64)
    wpost, wpre = one if a["w_post"] is None else a["w_post"], one if a["w_pre"] is None else a["w_pre"]
    sc = one if a["scale"] is None else a["scale"]
    bp = 0 * one if a["b_post"] is None else a["b_post"]
    A = torch.ones_like(o) if gate is None else act_rows
    # gradients by autograd through the two halves
    yl = y.clone().requires_grad_()
    wl, bl = wpre.clone().requires_grad_(), torch.zeros(C, dtype=torch.float64, requires_grad=True)
    G = d_y.double()
    want, mag = {}, {}
    if pre != "none":
        hh = R.normed(pre, yl, wl, bl, eps)
        gy, gw, gb = torch.autograd.grad(hh, (yl, wl, bl), d_h.double())
        G = G + gy
        want["d_w_pre"], want["d_b_pre"] = gw, gb
        mu, r = R.moments(pre, y, eps)
        n = ((y - mu) * r).abs() + (mu.abs() * r)
        t = (d_h.double() * wpre).abs()
        Gm = d_y.double().abs() + r * (t + (n + 1) * (t * (n + 1)).mean(-1, keepdim=True) + t.mean(-1, keepdim=True))
        mag["d_w_pre"], mag["d_b_pre"] = (d_h.double().abs() * (n + 1)).sum(0), d_h.double().abs().sum(0)
    else:
        Gm = d_y.double().abs()
    want["d_x"], mag["d_x"] = G, Gm
    leaves = {"o": o, "w_post": wpost, "b_post": bp, "scale": sc}
    if gate is not None:
        leaves["gate"] = gate
    leaves = {n: v.clone().requires_grad_() for n, v in leaves.items()}
    q = dict(w_post=leaves["w_post"], b_post=leaves["b_post"], scale=leaves["scale"], w_pre=None, b_pre=None)
    v, _ = R.norm_forward(torch.zeros_like(y), leaves["o"], leaves.get("gate"), q, post, "none", act, k or 1, alpha, eps)
    for n, gr in zip(leaves, torch.autograd.grad(v, list(leaves.values()), G, allow_unused=True)):
        want["d_" + n] = torch.zeros_like(leaves[n]) if gr is None else gr
    no = size_of_norm(post, o, eps)
    um = no * wpost.abs() + bp.abs()
    D = alpha * Gm
    mag["d_scale"] = (D * A.abs() * um).sum(0)
    dum = D * sc.abs() * A.abs()
    mag["d_w_post"], mag["d_b_post"] = (dum * no).sum(0), dum.sum(0)
    if post != "none":
        _, r = R.moments(post, o, eps)
        t = dum * wpost.abs()
        mag["d_o"] = r * (t + no * (t * no).mean(-1, keepdim=True) + t.mean(-1, keepdim=True))
    else:
        mag["d_o"] = dum
    if gate is not None:
        terms = D * sc.abs() * um * (slope.abs() + (1 + g.abs()) * 2.0 ** -3)       # derivative: a difference of values of this size
        mag["d_gate"] = torch.zeros_like(gate).index_add_(0, torch.arange(rows) // k, terms)
    return want, mag


# Backward: three row sums deep (each at most 46 additions) and about 60 operations; parameter sums add an item's rows (at most 64 in
# these cases), up to 32 sub-rows and 16 + 4 partial sums, a gate row's pieces (at most 256)
N_GRAD, N_SUM = 320, 640


@pytest.mark.parametrize("case", NORM_CASES)
def test_gated_norm_backward(case):
    rows, C, dt, res, post, pre, k, act, scale, f = case
    i, p = norm_inputs(case)
    alpha, eps = 0.7, 1e-5
    d_y, d_h = rnd(rows, C, seed=11, dtype=res), (rnd(rows, C, seed=12, dtype=dt) if pre != "none" else None)
    want, mag = norm_gradients(case, i, p, d_y, d_h, alpha, eps)
    got = dict(d_x=dev(torch.zeros(rows, C, dtype=res), f), d_o=dev(torch.zeros(rows, C, dtype=dt), f))
    d_gate = None if k is None else torch.zeros(-(-rows // k), C, dtype=dt, device=DEV)
    params = {n: torch.full((C,), float("nan"), device=DEV) for n in ("d_w_post", "d_b_post", "d_scale", "d_w_pre", "d_b_pre")
              if not (post == "none" and "post" in n) and not (pre == "none" and "pre" in n)}
    ws = torch.full((K.gated_norm_ws(rows, C, k or 1),), float("nan"), device=DEV)
    args = (dev(d_y, f), dev(d_h, f), dev(i["x"], f), dev(i["o"], f), dev(i["gate"]), got["d_x"], got["d_o"], d_gate, ws)
    K.gated_norm_backward(*args, **norm_how(case, p), **params)
    got.update(params)
    if d_gate is not None:
        got["d_gate"] = d_gate
    for n, v in got.items():
        count = N_GRAD if n in ("d_x", "d_o") or (n == "d_gate" and k == 1) else N_SUM
        within(v, want[n], count * R.U32 * mag[n] + R.HALF[v.dtype] * want[n].abs() * 1.01 + 1e-30, "%s %s" % (n, case))
    first = {n: v.clone() for n, v in got.items()}
    K.gated_norm_backward(*args, **norm_how(case, p), **params)
    assert all(torch.equal(v, first[n]) for n, v in got.items()), "the same inputs give other bits"


def test_gated_norm_without_a_block_output():
    x = rnd(33, 72, seed=1)
    h = torch.empty(33, 72, device=DEV)
    K.gated_norm_forward(dev(x), None, None, None, h, pre=K.NORM_LAYER, eps=1e-5)
    w = R.normed("layer", x.double(), None, None, 1e-5)
    within(h, w, N_VALUE * R.U32 * size_of_norm("layer", x.double(), 1e-5) + R.U32 * w.abs(), "h")
    d_x, d_w, ws = torch.empty(33, 72, device=DEV), torch.empty(72, device=DEV), torch.empty(K.gated_norm_ws(33, 72), device=DEV)
    dh = rnd(33, 72, seed=2)
    K.gated_norm_backward(None, dev(dh), dev(x), None, None, d_x, None, None, ws, pre=K.NORM_LAYER, eps=1e-5, d_w_pre=d_w)
    xl = x.double().requires_grad_()
    g, = torch.autograd.grad(R.normed("layer", xl, None, None, 1e-5), xl, dh.double())
    _, r = R.moments("layer", x.double(), 1e-5)
    n = size_of_norm("layer", x.double(), 1e-5)
    t = dh.double().abs()
    within(d_x, g, N_GRAD * R.U32 * r * (t + n * (t * n).mean(-1, keepdim=True) + t.mean(-1, keepdim=True)), "d_x")


def test_gated_norm_in_place_and_empty():
    case = (50, 128, BF, BF, "rms", "rms", 1, "sigmoid", True, 1)
    i, p = norm_inputs(case)
    y, h, h2 = (torch.empty(50, 128, device=DEV, dtype=BF) for _ in range(3))
    x = dev(i["x"])
    K.gated_norm_forward(x, dev(i["o"]), dev(i["gate"]), y, h, **norm_how(case, p))
    K.gated_norm_forward(x, dev(i["o"]), dev(i["gate"]), x, h2, **norm_how(case, p))
    assert torch.equal(x, y) and torch.equal(h, h2)
    d_w = torch.full((128,), 7.0, device=DEV)
    e = torch.empty(0, 128, device=DEV, dtype=BF)
    K.gated_norm_forward(e, e, None, e, e, post=K.NORM_RMS)
    K.gated_norm_backward(e, e, e, e, None, e, e, None, torch.empty(K.gated_norm_ws(0, 128), device=DEV), post=K.NORM_RMS, d_w_pre=d_w)
    assert (d_w == 0).all()


@pytest.mark.parametrize("C", [128, 5000])
def test_gated_norm_gradients_over_their_inputs(C):
    """d_x over d_y, d_o over d_h's place would be another row's; d_x = d_y and d_o = o are element for element: same bits as apart."""
    case = (21, C, BF, BF, "layer", "layer", 1, "silu", True, 1)
    i, p = norm_inputs(case)
    d_y, d_h = rnd(21, C, seed=11, dtype=BF), rnd(21, C, seed=12, dtype=BF)
    ws = torch.empty(K.gated_norm_ws(21, C), device=DEV)

    def run(over):
        a = dict(d_y=dev(d_y), d_h=dev(d_h), y=dev(i["x"]), o=dev(i["o"]), gate=dev(i["gate"]))
        d_x, d_o, d_g = (a["d_y"], a["o"], a["gate"]) if over else (torch.empty_like(a[n]) for n in ("d_y", "o", "gate"))
        params = {n: torch.empty(C, device=DEV) for n in ("d_w_post", "d_b_post", "d_scale", "d_w_pre", "d_b_pre")}
        K.gated_norm_backward(a["d_y"], a["d_h"], a["y"], a["o"], a["gate"], d_x, d_o, d_g, ws, **norm_how(case, p), **params)
        return [d_x, d_o, d_g] + list(params.values())
    assert all(torch.equal(a, b) for a, b in zip(run(False), run(True)))


def test_gated_norm_rows_of_zeros_and_of_nan_do_not_touch_their_neighbours():
    x, o = rnd(9, 40, seed=1), rnd(9, 40, seed=2)
    x[3], o[3] = 0, 0
    x[5, 7] = float("nan")
    y, h = torch.empty(9, 40, device=DEV), torch.empty(9, 40, device=DEV)
    K.gated_norm_forward(dev(x), dev(o), None, y, h, post=K.NORM_RMS, pre=K.NORM_LAYER, eps=1e-6)
    wy, wh = R.norm_forward(x.double(), o.double(), None, dict.fromkeys(("w_post", "b_post", "scale", "w_pre", "b_pre")), "rms", "layer",
                            "none", 1, 1.0, 1e-6)
    assert torch.isnan(h[5]).all() and not h[3].any()
    ok = [r for r in range(9) if r != 5]
    within(h[ok], wh[ok], torch.full((8, 40), 1e-4, dtype=torch.float64), "h")        # far above rounding: neighbours are whole


def test_gated_norm_directional_difference():
    """<gradient, direction> against a central difference of the 64-bit forward pass: the kernel's gradients are those of this function."""
    case = (12, 48, F32, F32, "layer", "rms", 4, "silu", True, 1)
    i, p = norm_inputs(case)
    alpha, eps, step = 0.7, 1e-5, 1e-5
    d_y, d_h = rnd(12, 48, seed=11), rnd(12, 48, seed=12)
    a, q = d64(i), d64(p)
    y, _ = R.norm_forward(a["x"], a["o"], a["gate"], q, "layer", "rms", "silu", 4, alpha, eps)
    out = dict(d_x=torch.empty(12, 48, device=DEV), d_o=torch.empty(12, 48, device=DEV), d_gate=torch.empty(3, 48, device=DEV))
    K.gated_norm_backward(dev(d_y), dev(d_h), dev(y.float()), dev(i["o"]), dev(i["gate"]), out["d_x"], out["d_o"], out["d_gate"],
                          torch.empty(K.gated_norm_ws(12, 48, 4), device=DEV), **norm_how(case, p))
    for n, key in (("d_x", "x"), ("d_o", "o"), ("d_gate", "gate")):
        direction = rnd(*a[key].shape, seed=21).double()

        def loss(t):
            yy, hh = R.norm_forward(*[a[m] + t * direction if m == key else a[m] for m in ("x", "o", "gate")], q, "layer", "rms", "silu", 4,
                                    alpha, eps)
            return ((yy * d_y.double()).sum() + (hh * d_h.double()).sum()).item()
        want = (loss(step) - loss(-step)) / (2 * step)
        got = (out[n].double().cpu() * direction).sum().item()
        size = (out[n].double().cpu() * direction).abs().sum().item()
        # y is rounded to fp32 before the backward pass (2^-24 of values up to 10, times gradients): 1e-5 of the terms; the difference's
        # own error is step^2 times the third derivative, about 1e-9 of them
        assert abs(got - want) <= 1e-5 * size, (n, got, want)


# ---- fp8 -----------------------------------------------------------------------------------------------------------------------
def values8(q):
    return q.cpu().float().double()


@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
@pytest.mark.parametrize("tile", [False, True])
@pytest.mark.parametrize("shape,dtype", [((1, 1), F32), ((3, 130), BF), ((128, 128), BF), ((129, 700), F32), ((260, 513), BF), ((7, 1037), BF)])
def test_fp8_quantize_is_exact_in_both_orders(fmt, tile, shape, dtype):
    x = rnd(*shape, seed=3, dtype=F32) * torch.exp(3 * rnd(1, shape[1], seed=4))
    x[0, 0] = 0
    x = x.to(dtype)
    if shape[0] > 2:
        x[2, :] = 0                                                    # a block of nothing
    q, s, qt, st = K.fp8_alloc(*shape, DEV, fmt, tile=tile, transposed=True)
    for t in (q, qt):
        t.view(torch.uint8).fill_(0x55)
    K.fp8_quantize(dev(x), q, s, qt, st, tile=tile)
    for got, code, m in ((q, s, x), (qt, st, x.t())):
        want, e = R.quantized(m, fmt, tile)
        assert torch.equal(code.cpu()[:, :e.shape[1]].long() - 127, e)
        assert torch.equal(values8(got), want)
    only, so = K.fp8_alloc(*shape, DEV, fmt, tile=tile)
    K.fp8_quantize(dev(x), only, so, tile=tile)
    assert torch.equal(only.view(torch.uint8), q.view(torch.uint8)) and torch.equal(so, s)


@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
def test_fp8_quantize_every_bf16_value(fmt):
    """All 65536 bit patterns: subnormals, infinities, NaN; each row of 128 has its own scale."""
    x = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(BF).reshape(512, 128)
    x = x[:, torch.randperm(128, generator=torch.Generator().manual_seed(1))]
    q, s = K.fp8_alloc(512, 128, DEV, fmt)
    K.fp8_quantize(dev(x), q, s)
    want, e = R.quantized(x, fmt, False)
    assert torch.equal(s.cpu()[:, :1].long() - 127, e)
    got = values8(q)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    ok = ~torch.isnan(want)
    assert torch.equal(got[ok], want[ok])


def test_fp8_quantize_reads_strided_rows_and_leaves_the_rest():
    x = rnd(70, 96, seed=1, dtype=BF)
    a, b = K.fp8_alloc(70, 96, DEV), K.fp8_alloc(70, 96, DEV)
    K.fp8_quantize(dev(x), *a)
    K.fp8_quantize(dev(x, 3), *b)
    assert torch.equal(a[0].view(torch.uint8), b[0].view(torch.uint8)) and torch.equal(a[1], b[1])


def operand(rows, cols, fmt, tile, seed):
    m = rnd(rows, cols, seed=seed) * torch.exp(rnd(1, cols, seed=seed + 50))
    q, s = K.fp8_alloc(rows, cols, DEV, fmt, tile=tile)
    K.fp8_quantize(dev(m), q, s, tile=tile)
    v, e = R.quantized(m, fmt, tile)
    e = e.repeat_interleave(128, 0)[:rows] if tile else e
    return (q, s), v * R.power(e.repeat_interleave(128, 1))


def product_bound(a, b, dtype, want):
    """One addition for each k, rounded relative to what has been added up, then the output's own rounding.  bf16 outputs: the 8-bit
    matrix instruction cuts 7 of 8 neighbouring products to 2^-13 of a power of two that is at most the largest of the 8."""
    kk = a.shape[1]
    bound = (kk + 8) * R.U32 * (a.abs() @ b.abs().t()) + 1.01 * R.HALF[dtype] * want.abs() + 1e-30
    if dtype == BF:
        a, b, cut = a.abs().float().to(DEV), b.abs().float().to(DEV), torch.zeros(a.shape[0], b.shape[0], device=DEV)
        for k in range(0, kk, 8):
            most = torch.zeros_like(cut)
            for j in range(k, k + 8):
                most = torch.maximum(most, a[:, j, None] * b[None, :, j])
            cut += most
        bound = bound + 7 * 2.0 ** -13 * 1.001 * cut.double().cpu()
    return bound


MATMUL = [
    # M, N, K, format and tile of a, of b, output, bias
    (1, 1, 1, "e4m3", False, "e4m3", True, F32, True),
    (1, 200, 256, "e4m3", False, "e4m3", True, BF, True),
    (16, 4096, 512, "e4m3", False, "e4m3", True, BF, False),
    (17, 130, 1300, "e5m2", False, "e4m3", True, F32, False),
    (64, 64, 640, "e4m3", False, "e5m2", True, BF, True),
    (129, 257, 129, "e5m2", False, "e5m2", False, F32, True),
    (300, 511, 700, "e5m2", False, "e4m3", False, F32, False),
    (256, 256, 1024, "e4m3", True, "e4m3", True, BF, False),
    (513, 770, 2049, "e4m3", False, "e4m3", True, BF, True),
    (1024, 512, 4096, "e4m3", False, "e4m3", False, F32, False),
    (33, 2048, 8192, "e4m3", False, "e4m3", True, BF, True),
    (40, 70, 128, "e4m3", False, "e4m3", True, BF, False),        # one to five blocks of K for the groups of a tile to share
    (40, 70, 256, "e4m3", False, "e5m2", True, F32, False),
    (65, 130, 384, "e4m3", True, "e4m3", False, BF, True),
    (70, 100, 640, "e5m2", False, "e4m3", True, F32, True),
    (64, 64, 8320, "e4m3", False, "e4m3", True, F32, False),
    (1030, 1700, 300, "e4m3", False, "e4m3", True, F32, True),    # two of the smallest tiles a compute unit
    (2048, 2040, 1100, "e4m3", False, "e4m3", True, BF, False),   # one of the middle ones
]


@pytest.mark.parametrize("case", MATMUL)
def test_fp8_matmul(case):
    M, N, Kc, fa, ta, fb, tb, odt, has_bias = case
    (qa, sa), a = operand(M, Kc, fa, ta, 1)
    (qb, sb), b = operand(N, Kc, fb, tb, 2)
    bias = rnd(N, seed=9) if has_bias else None
    out = torch.full((M, N), float("nan"), device=DEV, dtype=odt)
    K.fp8_matmul(qa, sa, qb, sb, out, bias=dev(bias))
    want = a @ b.t() + (0 if bias is None else bias.double())
    bound = product_bound(a, b, odt, want)
    within(out, want, bound, "product %s" % (case,))
    if odt == F32:
        prior = rnd(M, N, seed=10)
        acc = dev(prior)
        K.fp8_matmul(qa, sa, qb, sb, acc, bias=dev(bias), accumulate=True)
        within(acc, want + prior.double(), bound + R.U32 * (want + prior.double()).abs() + R.U32 * prior.double().abs(), "accumulated %s" % (case,))
    wide = torch.full((M, 2 * N + 3), 5.0, device=DEV, dtype=odt)
    K.fp8_matmul(qa, sa, qb, sb, wide[:, 1:N + 1], bias=dev(bias))
    assert torch.equal(wide[:, 1:N + 1], out) and (wide[:, N + 1:] == 5).all() and (wide[:, 0] == 5).all()


@pytest.mark.parametrize("M,N,Kc,dtype", [(1, 64, 100, BF), (1, 4096, 4096, BF), (5, 333, 520, F32), (16, 1000, 2048, BF), (31, 96, 129, BF),
                                          (200, 300, 777, BF), (2, 128, 16384, F32)])
def test_fp8_linear_is_the_quantised_product(M, N, Kc, dtype):
    x = (rnd(M, Kc, seed=1) * torch.exp(rnd(1, Kc, seed=2))).to(dtype)
    (w, sw), wv = operand(N, Kc, "e4m3", True, 3)
    bias = rnd(N, seed=4)
    out = torch.full((M, N), float("nan"), device=DEV, dtype=dtype)
    ws = torch.full((K.fp8_linear_ws(M, N, Kc),), 0x7f, device=DEV, dtype=torch.uint8)
    K.fp8_linear(dev(x), w, sw, out, ws, bias=dev(bias))
    v, e = R.quantized(x, "e4m3", False)
    xv = v * R.power(e.repeat_interleave(128, 1))
    want = xv @ wv.t() + bias.double()
    within(out, want, product_bound(xv, wv, dtype, want), "linear")
    strided = torch.full((M, 2 * N), 3.0, device=DEV, dtype=dtype)
    K.fp8_linear(dev(x, 2), w, sw, strided[:, N:], ws, bias=dev(bias))
    assert torch.equal(strided[:, N:], out) and (strided[:, :N] == 3).all()


def test_fp8_empty_sums_and_empty_batches():
    """No rows: nothing is written; a weight gradient over no rows is zero (the bias, or what was there)."""
    e = torch.empty(0, 200, device=DEV)
    q, s, qt, st = K.fp8_alloc(0, 200, DEV, transposed=True)
    K.fp8_quantize(e, q, s, qt, st)
    (w, sw), _ = operand(50, 200, "e4m3", True, 3)
    K.fp8_matmul(q, s, w, sw, torch.empty(0, 50, device=DEV))
    K.fp8_linear(e, w, sw, torch.empty(0, 50, device=DEV), torch.empty(0, device=DEV, dtype=torch.uint8))
    out, bias = torch.full((200, 200), 9.0, device=DEV), dev(rnd(200, seed=1))
    K.fp8_matmul(qt, st, qt, st, out, bias=bias)
    assert torch.equal(out, bias.expand(200, 200))
    K.fp8_matmul(qt, st, qt, st, out, accumulate=True)
    assert torch.equal(out, bias.expand(200, 200))


def test_fp8_nan_and_infinity_stay_in_their_rows():
    x = rnd(40, 300, seed=1)
    x[3, 5], x[7, 200] = float("nan"), float("inf")
    (w, sw), wv = operand(150, 300, "e4m3", True, 3)
    out = torch.empty(40, 150, device=DEV)
    K.fp8_linear(dev(x), w, sw, out, torch.empty(K.fp8_linear_ws(40, 150, 300), device=DEV, dtype=torch.uint8))
    bad = torch.isnan(out.cpu()).any(1)
    assert bad.nonzero().flatten().tolist() == [3, 7] and torch.isnan(out[3]).all() and torch.isnan(out[7]).all()


# ---- gated scan ----------------------------------------------------------------------------------------------------------------
# B, T, D, dtype, floor, reset rate, lengths, h0, stride factor
SCAN_CASES = [
    (1, 1, 1, F32, False, 0.0, None, True, 1),
    (3, 1, 200, BF, True, 0.0, [1, 0, 1], True, 1),
    (2, 7, 130, F32, True, 0.3, None, True, 1),
    (2, 9, 33, BF, False, 0.0, [9, 4], False, 2),                     # odd: one channel a lane
    (2, 19, 64, F32, False, 0.0, None, True, 1),
    (1, 33, 256, BF, True, 0.1, None, False, 2),
    (3, 65, 70, F32, True, 0.05, [65, 0, 64], True, 1),               # a chunk of one step; an empty row
    (2, 500, 66, BF, False, 0.01, [500, 317], True, 2),
    (1, 1500, 40, F32, True, 0.0, None, False, 1),                    # many chunks
    (70, 70, 2048, BF, False, 0.02, None, True, 1),                   # enough channels for one chunk: two tiles
    (4, 1, 130, F32, False, 0.3, [1, 0, 1, 1], True, 2),              # single steps
    (300, 1, 258, BF, True, 0.2, None, False, 1),
    (2, 20, 130, BF, True, 0.1, [20, 11], True, 1),                   # three waves
    (3, 24, 258, F32, False, 0.05, None, True, 2),
    (2, 25, 130, BF, True, 0.1, [17, 25], False, 1),
]


def scan_inputs(case, seed=0):
    B, T, D, dt, floor, rate, lengths, has_h0, f = case
    gen = torch.Generator().manual_seed(seed + 77)
    return dict(x=rnd(B, T, D, seed=seed, dtype=dt), g=rnd(B, T, D, seed=seed + 1, dtype=dt, scale=2.0, mean=1.0),
                h0=rnd(B, D, seed=seed + 2) if has_h0 else None,
                floor=torch.rand(D, generator=gen) * 0.9 if floor else None,
                reset=(torch.rand(B, T, generator=gen) < rate).to(torch.uint8) if rate else None,
                lengths=torch.tensor(lengths, dtype=torch.int32) if lengths is not None else None)


def dev3(t, f=1):
    if t is None or f == 1:
        return None if t is None else t.to(DEV)
    B, T, D = t.shape
    wide = torch.full((B, T + 1, D * f), float("nan"), device=DEV, dtype=t.dtype)
    wide[:, 1:, D:2 * D] = t.to(DEV)
    return wide[:, 1:, D:2 * D]


def scan_reference(i, d_y=None, d_hT=None):
    """Outputs (and gradients) in fp64, with bounds: an error e of the state goes on as f e, and every step adds DELTA times the size
    of its terms."""
    B, T, D = i["x"].shape
    x, g = i["x"].double().requires_grad_(), i["g"].double().requires_grad_()
    h0 = (torch.zeros(B, D, dtype=torch.float64) if i["h0"] is None else i["h0"].double()).requires_grad_()
    low = (torch.zeros(D, dtype=torch.float64) if i["floor"] is None else i["floor"].double()).requires_grad_()
    ends = torch.full((B,), T) if i["lengths"] is None else i["lengths"].long()
    fresh = torch.zeros(B, T, dtype=torch.bool) if i["reset"] is None else i["reset"] != 0
    y, hT = R.scan_forward(x, g, h0, low, ends, fresh)
    out = dict(y=y, hT=hT)
    with torch.no_grad():
        runs = (torch.arange(T)[None] < ends[:, None])[..., None]
        up, down, k = torch.sigmoid(g), torch.sigmoid(-g), 1 - low
        f = low + k * up
        keep = torch.where(runs, torch.where(fresh[..., None], torch.zeros_like(f), f), torch.ones_like(f))
        a = torch.where(runs, k * down * x.abs(), torch.zeros_like(f))
        M, E, e_y, M_y = h0.abs(), torch.zeros(B, D, dtype=torch.float64), [], []
        before_M, before_E = [], []
        for t in range(T):
            cut = fresh[:, t, None] & runs[:, t]
            before_M.append(torch.where(cut, torch.zeros_like(M), M))
            before_E.append(torch.where(cut, torch.zeros_like(E), E))
            M = keep[:, t] * M + a[:, t]
            E = keep[:, t] * E + DELTA * M
            e_y.append(torch.where(runs[:, t], E, torch.zeros_like(E)))
        bound = dict(y=torch.stack(e_y, 1), hT=E)
    if d_y is None:
        return out, bound
    grads = torch.autograd.grad((y, hT), (x, g, h0, low), (d_y.double(), d_hT.double()))
    out.update(d_x=grads[0], d_g=grads[1], d_h0=grads[2], d_floor=grads[3])
    with torch.no_grad():
        Dm, De = d_hT.double().abs(), torch.zeros(B, D, dtype=torch.float64)
        ex, eg = torch.zeros(B, T, D, dtype=torch.float64), torch.zeros(B, T, D, dtype=torch.float64)
        e_low, m_low = torch.zeros(D, dtype=torch.float64), torch.zeros(D, dtype=torch.float64)
        for t in range(T - 1, -1, -1):
            live = runs[:, t]
            m = Dm + d_y[:, t].double().abs()
            e = De + DELTA * m
            s = before_M[t] + x[:, t].abs()                             # |h - x| at most
            ex[:, t] = torch.where(live, k * down[:, t] * (e + DELTA * m), 0.0)
            ef = e * s + m * (before_E[t] + DELTA * s)
            eg[:, t] = torch.where(live, k * up[:, t] * down[:, t] * (ef + DELTA * m * s), 0.0)
            e_low += torch.where(live, down[:, t] * (ef + DELTA * m * s), 0.0).sum(0)
            m_low += torch.where(live, down[:, t] * m * s, 0.0).sum(0)
            Dm = torch.where(live, keep[:, t] * m, Dm)
            De = torch.where(live, keep[:, t] * (e + DELTA * m), De)
        bound.update(d_x=ex, d_g=eg, d_h0=De, d_floor=e_low + (T + 64) * R.U32 * m_low)     # a lane adds up to T steps, then partial sums
    return out, bound


# a step's roundings: the gates (argument of the exponential up to 12: 18 units, reciprocal, three products), their product with the
# state, the sum; composed maps add their products' own
DELTA = 48 * 2.0 ** -24


def scan_how(i):
    return dict(h0=dev(i["h0"]), floor=dev(i["floor"]), lengths=dev(i["lengths"]), reset=dev(i["reset"]))


@pytest.mark.parametrize("case", SCAN_CASES)
def test_gated_scan_forward_and_backward(case):
    B, T, D, dt, floor, rate, lengths, has_h0, f = case
    i = scan_inputs(case)
    if lengths is not None:                                             # what is behind a row's length is not looked at
        for b, n in enumerate(lengths):
            i["x"][b, n:], i["g"][b, n:] = float("nan"), float("inf")
    d_y, d_hT = rnd(B, T, D, seed=5, dtype=dt), rnd(B, D, seed=6)
    clean = dict(i)
    if lengths is not None:
        clean["x"], clean["g"], d_y = i["x"].nan_to_num(0.0), i["g"].nan_to_num(0.0, posinf=0.0), d_y.clone()
        for b, n in enumerate(lengths):
            d_y[b, n:] = 0
    want, bound = scan_reference(clean, d_y, d_hT)
    for b, n in enumerate(lengths or []):
        d_y[b, n:] = float("nan")
    y, hT = dev3(torch.zeros(B, T, D, dtype=dt), f), torch.full((B, D), float("nan"), device=DEV)
    carry = torch.full((K.gated_scan_carry(B, T, D),), float("nan"), device=DEV)
    x, g, how = dev3(i["x"], f), dev3(i["g"], f), scan_how(i)
    K.gated_scan_forward(x, g, y, hT, carry, **how)
    within(y, want["y"], bound["y"] + 1.01 * R.HALF[dt] * want["y"].abs(), "y %s" % (case,))
    within(hT, want["hT"], bound["hT"] + R.U32 * want["hT"].abs(), "hT %s" % (case,))
    got = dict(d_x=dev3(torch.zeros(B, T, D, dtype=dt), f), d_g=dev3(torch.zeros(B, T, D, dtype=dt), f))
    if has_h0:
        got["d_h0"] = torch.full((B, D), float("nan"), device=DEV)
    if floor:
        got["d_floor"] = torch.full((D,), float("nan"), device=DEV)
    ws = torch.full((K.gated_scan_ws(B, T, D),), float("nan"), device=DEV)

    def backward():
        K.gated_scan_backward(x, g, dev3(d_y, f), dev(d_hT), carry, got["d_x"], got["d_g"], ws, d_h0=got.get("d_h0"),
                              d_floor=got.get("d_floor"), **how)
    backward()
    for n, v in got.items():
        within(v, want[n], bound[n] + 1.01 * R.HALF[v.dtype] * want[n].abs() + 1e-30, "%s %s" % (n, case))
    first = {n: v.clone() for n, v in got.items()}
    backward()
    assert all(torch.equal(v, first[n]) for n, v in got.items()), "the same inputs give other bits"


def test_gated_scan_step_by_step_is_the_sequence():
    """Serving: T single steps that hand on the state, in place, against one call; keep=False needs no carry for one step."""
    B, T, D = 3, 12, 96
    i = scan_inputs((B, T, D, F32, True, 0.0, None, True, 1))
    y, hT = torch.empty(B, T, D, device=DEV), torch.empty(B, D, device=DEV)
    K.gated_scan_forward(dev(i["x"]), dev(i["g"]), y, hT, None, h0=dev(i["h0"]), floor=dev(i["floor"]), keep=False)
    state, steps = dev(i["h0"]), torch.empty(B, T, D, device=DEV)
    x, g = dev(i["x"]), dev(i["g"])
    for t in range(T):
        K.gated_scan_forward(x[:, t:t + 1], g[:, t:t + 1], steps[:, t:t + 1], state, None, h0=state, floor=dev(i["floor"]), keep=False)
    want, bound = scan_reference(i)
    for got, ref, e in ((y, want["y"], bound["y"]), (steps, want["y"], bound["y"]), (hT, want["hT"], bound["hT"]), (state, want["hT"], bound["hT"])):
        within(got, ref, e + R.U32 * ref.abs(), "steps")


def test_gated_scan_long_sequence_in_place():
    """A sequence in chunks, more workgroups than run at once, its state handed on in place and y over x or g: as with tensors apart."""
    B, T, D = 1, 4096, 16384
    x, g = torch.randn(B, T, D, device=DEV).to(BF), torch.randn(B, T, D, device=DEV).to(BF) + 3
    h0 = torch.randn(B, D, device=DEV) * 1e6                       # still there after 4096 steps of gates near 1
    reset = torch.zeros(B, T, device=DEV, dtype=torch.uint8)
    carry = torch.empty(K.gated_scan_carry(B, T, D), device=DEV)
    y, hT = torch.empty_like(x), torch.empty(B, D, device=DEV)
    for low in (None, torch.full((D,), 0.999, device=DEV)):
        K.gated_scan_forward(x, g, y, hT, carry, h0=h0, floor=low, reset=reset, keep=False)
        for over in "xg":
            xc, gc, state = x.clone(), g.clone(), h0.clone()
            out = xc if over == "x" else gc
            K.gated_scan_forward(xc, gc, out, state, carry, h0=state, floor=low, reset=reset, keep=False)
            assert torch.equal(out, y) and torch.equal(state, hT)


def test_gated_scan_a_reset_stops_nan_and_a_zero_gate_is_kept_apart():
    B, T, D = 1, 200, 64
    x, g = rnd(B, T, D, seed=1), rnd(B, T, D, seed=2)
    x[0, 90] = float("nan")
    reset = torch.zeros(B, T, dtype=torch.uint8)
    reset[0, 150] = 1
    y, hT, carry = torch.empty(B, T, D, device=DEV), torch.empty(B, D, device=DEV), torch.empty(K.gated_scan_carry(B, T, D), device=DEV)
    K.gated_scan_forward(dev(x), dev(g), y, hT, carry, reset=dev(reset))
    bad = torch.isnan(y[0].cpu())
    assert bad[90:150].all() and not bad[:90].any() and not bad[150:].any() and not torch.isnan(hT).any()
    dx, dg = torch.empty(B, T, D, device=DEV), torch.empty(B, T, D, device=DEV)
    d_y = rnd(B, T, D, seed=3)
    d_y[0, 160] = float("nan")
    K.gated_scan_backward(dev(x), dev(g), dev(d_y), None, carry, dx, dg, torch.empty(K.gated_scan_ws(B, T, D), device=DEV), reset=dev(reset))
    bad = torch.isnan(dx[0].cpu())
    assert bad[150:161].all() and not bad[161:].any() and not bad[:150].any()


def test_gated_scan_directional_difference():
    case = (2, 70, 24, F32, True, 0.05, [70, 41], True, 1)
    i = scan_inputs(case)
    B, T, D = 2, 70, 24
    d_y, d_hT = rnd(B, T, D, seed=5), rnd(B, D, seed=6)
    y, hT, carry = torch.empty(B, T, D, device=DEV), torch.empty(B, D, device=DEV), torch.empty(K.gated_scan_carry(B, T, D), device=DEV)
    K.gated_scan_forward(dev(i["x"]), dev(i["g"]), y, hT, carry, **scan_how(i))
    got = dict(x=torch.empty(B, T, D, device=DEV), g=torch.empty(B, T, D, device=DEV), h0=torch.empty(B, D, device=DEV), floor=torch.empty(D, device=DEV))
    K.gated_scan_backward(dev(i["x"]), dev(i["g"]), dev(d_y), dev(d_hT), carry, got["x"], got["g"], torch.empty(K.gated_scan_ws(B, T, D), device=DEV),
                          d_h0=got["h0"], d_floor=got["floor"], **scan_how(i))
    a = {n: i[n].double() for n in ("x", "g", "h0", "floor")}
    ends, fresh, step = i["lengths"].long(), i["reset"] != 0, 1e-5
    for n in a:
        direction = rnd(*a[n].shape, seed=31).double()

        def loss(t):
            b = {m: v + t * direction if m == n else v for m, v in a.items()}
            yy, hh = R.scan_forward(b["x"], b["g"], b["h0"], b["floor"], ends, fresh)
            return ((yy * d_y.double()).sum() + (hh * d_hT.double()).sum()).item()
        want = (loss(step) - loss(-step)) / (2 * step)
        terms = got[n].double().cpu() * direction
        assert abs(terms.sum().item() - want) <= 3e-5 * terms.abs().sum().item(), (n, terms.sum().item(), want)


# ---- together, streams, graphs -------------------------------------------------------------------------------------------------
class Block:
    """Norm -> fp8 projection (to x and gate) -> recurrence -> fp8 projection -> gate, residual scale, next norm; both directions."""

    def __init__(self, B, T, C, D, seed=0):
        self.B, self.T, self.C, self.D = B, T, C, D
        n = B * T
        mk = lambda *s, dt=BF: torch.empty(*s, device=DEV, dtype=dt)  # noqa: E731
        self.w1, self.w2 = rnd(2 * D, C, seed=seed, scale=C ** -0.5), rnd(C, D, seed=seed + 1, scale=D ** -0.5)
        self.q1, self.q2 = K.fp8_alloc(2 * D, C, DEV, tile=True, transposed=True), K.fp8_alloc(C, D, DEV, tile=True, transposed=True)
        K.fp8_quantize(dev(self.w1), *self.q1, tile=True)
        K.fp8_quantize(dev(self.w2), *self.q2, tile=True)
        self.p = dict(scale=dev(rnd(C, seed=seed + 2, scale=0.3)), w_pre=dev(rnd(C, seed=seed + 3, scale=0.1, mean=1.0)))
        self.gate = dev(rnd(B, C, seed=seed + 4, dtype=BF))
        self.h, self.xg, self.y, self.o, self.out, self.h2 = mk(n, C), mk(n, 2 * D), mk(B, T, D), mk(n, C), mk(n, C), mk(n, C)
        self.hq, self.yq = K.fp8_alloc(n, C, DEV, transposed=True), K.fp8_alloc(n, D, DEV, transposed=True)
        self.doq, self.dxgq = K.fp8_alloc(n, C, DEV, "e5m2", transposed=True), K.fp8_alloc(n, 2 * D, DEV, "e5m2", transposed=True)
        self.carry, self.sws = mk(K.gated_scan_carry(B, T, D), dt=F32), mk(K.gated_scan_ws(B, T, D), dt=F32)
        self.nws = mk(K.gated_norm_ws(n, C, T), dt=F32)
        self.nws1 = mk(K.gated_norm_ws(n, C, 1), dt=F32)
        self.hT = mk(B, D, dt=F32)
        self.d = dict(x=mk(n, C), o=mk(n, C), gate=mk(B, C), y=mk(n, D), xg=mk(n, 2 * D), h=mk(n, C), x0=mk(n, C), w1=mk(2 * D, C, dt=F32),
                      w2=mk(C, D, dt=F32), scale=mk(C, dt=F32), w_pre=mk(C, dt=F32))

    def forward(self, x):
        n, D = self.B * self.T, self.D
        K.gated_norm_forward(x, None, None, None, self.h, w_pre=self.p["w_pre"])
        K.fp8_quantize(self.h, *self.hq)
        K.fp8_matmul(*self.hq[:2], *self.q1[:2], self.xg)
        xg = self.xg.view(self.B, self.T, 2 * D)
        K.gated_scan_forward(xg[..., :D], xg[..., D:], self.y, self.hT, self.carry)
        K.fp8_quantize(self.y.view(n, D), *self.yq)
        K.fp8_matmul(*self.yq[:2], *self.q2[:2], self.o)
        K.gated_norm_forward(x, self.o, self.gate, self.out, self.h2, post=K.NORM_RMS, pre=K.NORM_RMS, gate_act=K.ACT_SIGMOID,
                             rows_per_gate=self.T, alpha=0.5, scale=self.p["scale"])
        return self.out, self.h2

    def backward(self, x, d_out, d_h2):
        n, D, d = self.B * self.T, self.D, self.d
        K.gated_norm_backward(d_out, d_h2, self.out, self.o, self.gate, d["x"], d["o"], d["gate"], self.nws, post=K.NORM_RMS, pre=K.NORM_RMS,
                              gate_act=K.ACT_SIGMOID, rows_per_gate=self.T, alpha=0.5, scale=self.p["scale"], d_scale=d["scale"])
        K.fp8_quantize(d["o"], *self.doq)
        K.fp8_matmul(*self.doq[:2], *self.q2[2:], d["y"])
        K.fp8_matmul(*self.doq[2:], *self.yq[2:], d["w2"])
        xg, dxg = (t.view(self.B, self.T, 2 * D) for t in (self.xg, d["xg"]))
        K.gated_scan_backward(xg[..., :D], xg[..., D:], d["y"].view(self.B, self.T, D), None, self.carry, dxg[..., :D], dxg[..., D:], self.sws)
        K.fp8_quantize(d["xg"], *self.dxgq)
        K.fp8_matmul(*self.dxgq[:2], *self.q1[2:], d["h"])
        K.fp8_matmul(*self.dxgq[2:], *self.hq[2:], d["w1"])
        K.gated_norm_backward(d["x"], d["h"], x, None, None, d["x0"], None, None, self.nws1, w_pre=self.p["w_pre"], d_w_pre=d["w_pre"])
        return d


def stored(q, s):
    e = s.cpu()[:, :q.shape[1] // 128].long() - 127
    if e.shape[0] != q.shape[0]:
        e = e.repeat_interleave(128, 0)[:q.shape[0]]
    return values8(q) * R.power(e.repeat_interleave(128, 1))


def test_a_block_forward_and_backward_stage_by_stage():
    """Every stage against 64 bits from the stage's own inputs; the products from what is stored in 8 bits (exact, tested above)."""
    B, T, C, D = 2, 75, 200, 136
    m = Block(B, T, C, D)
    x, d_out, d_h2 = rnd(B * T, C, seed=20, dtype=BF), rnd(B * T, C, seed=21, dtype=BF), rnd(B * T, C, seed=22, dtype=BF)
    xd = dev(x)
    m.forward(xd)
    d = m.backward(xd, dev(d_out), dev(d_h2))
    n = B * T

    def near(got, a, b, what):
        want = a @ b.t()
        within(got, want, product_bound(a, b, got.dtype, want), what)
    near(m.xg, stored(*m.hq[:2]), stored(*m.q1[:2]), "first projection")
    near(m.o, stored(*m.yq[:2]), stored(*m.q2[:2]), "second projection")
    near(d["y"], stored(*m.doq[:2]), stored(*m.q2[2:]), "gradient of the second projection's input")
    near(d["w2"], stored(*m.doq[2:])[:C], stored(*m.yq[2:])[:D], "gradient of the second weight")
    near(d["h"], stored(*m.dxgq[:2]), stored(*m.q1[2:]), "gradient of the first projection's input")
    near(d["w1"], stored(*m.dxgq[2:])[:2 * D], stored(*m.hq[2:])[:C], "gradient of the first weight")
    xg = m.xg.cpu().view(B, T, 2 * D)
    i = dict(x=xg[..., :D].contiguous(), g=xg[..., D:].contiguous(), h0=None, floor=None, lengths=None, reset=None)
    want, bound = scan_reference(i, d["y"].cpu().view(B, T, D), torch.zeros(B, D))
    dxg = d["xg"].view(B, T, 2 * D)
    for got, key in ((m.y, "y"), (dxg[..., :D], "d_x"), (dxg[..., D:], "d_g")):
        within(got, want[key], bound[key] + 1.01 * R.HALF[BF] * want[key].abs() + 1e-30, key)
    case = (n, C, BF, BF, "rms", "rms", T, "sigmoid", True, 1)
    p = dict(w_post=None, b_post=None, scale=m.p["scale"].cpu(), w_pre=None, b_pre=None)
    wy, wh = R.norm_forward(x.double(), m.o.cpu().double(), m.gate.cpu().double(), d64(p), "rms", "rms", "sigmoid", T, 0.5, 1e-6)
    within(m.out, wy, 1.01 * R.HALF[BF] * wy.abs() + 1e-4, "y")                     # fp32 terms below 10: 160 * 2^-24 * 10
    within(m.h2, wh, 1.01 * R.HALF[BF] * wh.abs() + 2e-4, "h")
    want, mag = norm_gradients(case, dict(x=m.out.cpu(), o=m.o.cpu(), gate=m.gate.cpu()), p, d_out, d_h2, 0.5, 1e-6)
    for key in ("d_x", "d_o", "d_gate", "d_scale"):
        got = d[key[2:]]
        within(got, want[key], N_SUM * R.U32 * mag[key] + 1.01 * R.HALF[got.dtype] * want[key].abs(), key)


def test_a_block_captured_and_replayed_beside_eager_work():
    """A graph of forward and backward, replayed with new inputs and eager calls of another block (its own workspaces) in between."""
    B, T, C, D = 2, 140, 128, 96
    m, other = Block(B, T, C, D, seed=1), Block(B, T, C, D, seed=1)
    xs = [dev(rnd(B * T, C, seed=30 + k, dtype=BF)) for k in range(3)]
    gs = [dev(rnd(B * T, C, seed=40 + k, dtype=BF)) for k in range(3)]
    x, g = xs[0].clone(), gs[0].clone()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        m.forward(x)
        m.backward(x, g, g)
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        m.forward(x)
        m.backward(x, g, g)
    for k in (0, 1, 2, 1):
        x.copy_(xs[k])
        g.copy_(gs[k])
        graph.replay()
        want = [t.clone() for t in other.forward(xs[k])] + [t.clone() for t in other.backward(xs[k], gs[k], gs[k]).values()]
        torch.cuda.synchronize()
        got = [m.out, m.h2] + list(m.d.values())
        assert all(torch.equal(a, b) for a, b in zip(got, want)), k


def test_calls_go_to_the_current_stream():
    """On a side stream, behind a producer there: nothing runs on the default stream ahead of it."""
    s = torch.cuda.Stream()
    x = torch.zeros(4096, 1024, device=DEV)
    h = torch.empty_like(x)
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        for _ in range(20):
            x.add_(1.0)
        K.gated_norm_forward(x, None, None, None, h, pre=K.NORM_RMS, eps=1e-6)
    s.synchronize()
    assert torch.allclose(h, torch.full_like(h, 1.0), atol=1e-6) and (x == 20).all()


def test_refusals_on_the_device():
    x = torch.zeros(4, 64, device=DEV)
    with pytest.raises(TecoHipError, match="rows of 64"):
        K.gated_norm_forward(x, torch.zeros(3, 64, device=DEV), None, x, x)
    with pytest.raises(TecoHipError, match="y goes with the block output"):
        K.gated_norm_forward(x, x, None, None, x)
    with pytest.raises(TecoHipError, match="workspace"):
        K.gated_norm_backward(x, x, x, None, None, x, None, None, torch.empty(4, device=DEV))
    with pytest.raises(TecoHipError, match="types"):
        K.gated_norm_forward(x.bfloat16(), x, None, x.bfloat16(), x)
    q, s = K.fp8_alloc(4, 64, DEV)
    with pytest.raises(TecoHipError, match="padded columns"):
        K.fp8_matmul(q, s, *K.fp8_alloc(4, 200, DEV), torch.empty(4, 4, device=DEV))
    with pytest.raises(TecoHipError, match="accumulation"):
        K.fp8_matmul(q, s, q, s, torch.empty(4, 4, device=DEV, dtype=BF), accumulate=True)
    with pytest.raises(TecoHipError, match="workspace"):
        K.fp8_linear(x, *K.fp8_alloc(8, 64, DEV, tile=True), torch.empty(4, 8, device=DEV), torch.empty(16, device=DEV, dtype=torch.uint8))
    z = torch.zeros(2, 300, 64, device=DEV)
    with pytest.raises(TecoHipError, match="carry"):
        K.gated_scan_forward(z, z, z, None, None)
    with pytest.raises(TecoHipError, match="carry"):
        K.gated_scan_forward(z, z, z, None, torch.empty(8, device=DEV))
    with pytest.raises(TecoHipError, match="steps overlap"):
        K.gated_scan_forward(z, z, z[:, :1].expand(2, 300, 64), None, torch.empty(K.gated_scan_carry(2, 300, 64), device=DEV))


def test_offsets_beyond_32_bits():
    """A tensor of more than 2^32 values: the last rows of a norm, a scan and a quantisation."""
    rows, C = (1 << 19) + 8, 8200
    if torch.cuda.mem_get_info()[0] < 5 * rows * C * 2:
        pytest.skip("not enough free memory")
    big = torch.zeros(rows, C, device=DEV, dtype=BF)
    out = torch.zeros(rows, C, device=DEV, dtype=BF)
    tail = rnd(8, C, seed=1, dtype=BF)
    big[-8:] = dev(tail)
    K.gated_norm_forward(big, None, None, None, out)
    want = R.normed("rms", tail.double(), None, None, 1e-6)
    within(out[-8:], want, 1.01 * R.HALF[BF] * want.abs() + 1e-4, "norm")
    x3, y3 = big[:, :8192].unsqueeze(0), out[:, :8192].unsqueeze(0)
    carry = torch.empty(K.gated_scan_carry(1, rows, 8192), device=DEV)
    K.gated_scan_forward(x3, x3, y3, None, carry, keep=False)
    i = dict(x=tail[None, :, :8192], g=tail[None, :, :8192], h0=None, floor=None, lengths=None, reset=None)
    want, bound = scan_reference(i)
    within(y3[:, -8:], want["y"], bound["y"] + 1.01 * R.HALF[BF] * want["y"].abs() + 1e-30, "scan")
    del out, y3, carry
    q, s = K.fp8_alloc(rows, C, DEV)
    K.fp8_quantize(big, q, s)
    wq, e = R.quantized(tail, "e4m3", False)
    assert torch.equal(values8(q[-8:]), wq) and torch.equal(s[-8:].cpu()[:, :e.shape[1]].long() - 127, e)
    assert not q[:-8].view(torch.uint8).any()
    assert math.isfinite(float(s.float().mean()))
