"""The sequence-block operators on the paths and inputs that small cases do not reach: the tiles of large products, sums that cancel,
chunks of several tiles, several rows an item, gates far from zero.  References and bounds as in test_seqblock_gpu."""
import pytest
import torch

import seqblock_ref as R
import test_seqblock_gpu as S
from tecogan_amd import kernels as K

pytestmark = pytest.mark.gpu
DEV, BF, F32 = S.DEV, S.BF, S.F32
rnd, dev, within = S.rnd, S.dev, S.within


# ---- fp8 -----------------------------------------------------------------------------------------------------------------------
def cancelling(rows, cols):
    """Rows whose first two values are 256 and -256 (times 1 in the other operand: they cancel) beside six of 15 x 2^-9: all of them are
    e4m3 values at scale 1."""
    m = rnd(rows, cols, seed=3).clamp(-3, 3)
    m[:, 0], m[:, 1], m[:, 2:8] = 256.0, -256.0, 15 * 2.0 ** -9
    return m


@pytest.mark.parametrize("M,N,Kc", [(33, 64, 128), (40, 200, 100), (200, 333, 640), (2100, 2101, 128)])
@pytest.mark.parametrize("odt", [BF, F32])
def test_fp8_sums_are_whole_where_products_cancel(M, N, Kc, odt):
    """Whatever the output's type: products are added in fp32, so that what two large ones leave behind keeps its value.  The bound is one
    fp32 rounding for each k, relative to what has been added up (at most 2^-24 x 136 x 1000 in the first block), and the output's own."""
    x, w = cancelling(M, Kc), rnd(N, Kc, seed=4).clamp(-3, 3)
    w[:, :8] = 1.0
    q, s = K.fp8_alloc(M, Kc, DEV)
    K.fp8_quantize(dev(x), q, s)
    wq, ws = K.fp8_alloc(N, Kc, DEV, tile=True)
    K.fp8_quantize(dev(w), wq, ws, tile=True)
    a, b = S.stored(q, s), S.stored(wq, ws)
    want = a @ b.t()
    bound = (a.shape[1] + 8) * R.U32 * (a.abs() @ b.abs().t()) + 1.01 * R.HALF[odt] * want.abs()
    out = torch.full((M, N), float("nan"), device=DEV, dtype=odt)
    K.fp8_matmul(q, s, wq, ws, out)
    within(out, want, bound, "product")
    out.fill_(float("nan"))
    K.fp8_linear(dev(x), wq, ws, out, torch.empty(K.fp8_linear_ws(M, N, Kc), device=DEV, dtype=torch.uint8))
    within(out, want, bound, "linear")


def tile_of(M, N, Kc, fast):
    """The product kernel (fragments of 16 in each direction, stages, groups) that the launcher's rule takes, restated: a case below has to
    reach the one that it stands for."""
    cus = torch.cuda.get_device_properties(0).multi_processor_count

    def up(n, d):
        return -(-n // d)
    t256, t128, t64 = (up(M, t) * up(N, t) for t in (256, 128, 64))
    brief, whole = up(Kc, 128) * 128 <= 1024, not fast
    gain = 114 if brief else 125
    if t256 * 5 >= cus * 4 and gain * t256 * up(t128, 2 * cus) * 2 * cus >= 100 * t128 * up(t256, cus) * cus and not (whole and brief and t256 > cus):
        return 8, 8, 2, 1
    if whole:
        return (4, 4, 2, 1) if t128 * 5 >= cus * 4 else (2, 2, 4, 1) if t64 > 2 * cus else (2, 2, 2, 2) if t64 > cus else (2, 2, 2, 4)
    return (4, 4, 2, 1) if t128 > cus else (4, 4, 4, 1) if t128 * 5 >= cus * 4 else (2, 2, 4, 1) if t64 > cus else (2, 2, 4, 2)


TILES = [
    # kernel, fast, M, N, K, format and tile of a, of b, bias.  Odd N: the way out through LDS, rows wider than a wave at 8 fragments;
    # K: odd and even numbers of blocks, one block
    ((8, 8, 2, 1), False, 3700, 3701, 1300, "e5m2", False, "e4m3", True, True),
    ((8, 8, 2, 1), False, 3844, 3700, 100, "e4m3", True, "e5m2", False, False),
    ((4, 4, 2, 1), False, 2100, 2101, 700, "e4m3", False, "e4m3", True, True),
    ((4, 4, 2, 1), False, 1990, 2104, 1409, "e5m2", False, "e5m2", False, False),
    ((2, 2, 4, 1), False, 1500, 1501, 700, "e4m3", False, "e5m2", True, True),
    ((2, 2, 4, 1), False, 1501, 1500, 1200, "e5m2", True, "e4m3", False, False),
    ((2, 2, 2, 2), False, 1030, 1700, 900, "e5m2", False, "e4m3", True, True),
    ((2, 2, 2, 4), False, 130, 257, 1153, "e5m2", False, "e4m3", True, True),
    ((8, 8, 2, 1), True, 3700, 3701, 1300, "e5m2", False, "e4m3", True, True),
    ((8, 8, 2, 1), True, 3844, 3700, 100, "e4m3", True, "e5m2", False, False),
    ((4, 4, 2, 1), True, 2100, 2101, 700, "e5m2", False, "e4m3", True, True),
    ((4, 4, 2, 1), True, 2600, 2100, 1409, "e4m3", False, "e5m2", False, False),
    ((4, 4, 4, 1), True, 1920, 2041, 1100, "e5m2", False, "e5m2", True, True),
    ((4, 4, 4, 1), True, 2048, 2040, 500, "e4m3", True, "e4m3", False, False),
    ((2, 2, 4, 1), True, 1100, 1101, 700, "e5m2", False, "e4m3", True, True),
    ((2, 2, 4, 1), True, 1101, 1100, 1250, "e4m3", True, "e5m2", False, False),
    ((2, 2, 4, 2), True, 130, 257, 1153, "e5m2", False, "e4m3", True, True),
    ((2, 2, 4, 2), True, 64, 72, 128, "e4m3", False, "e4m3", True, False),
]


def cut_of(a, b):
    """What the 8-bit instruction may cut: 7 of 8 neighbouring products to 2^-13 of a power of two that is at most the largest of the 8."""
    total = torch.zeros(a.shape[0], b.shape[0], device=DEV)
    for k in range(0, a.shape[1], 8):
        most = torch.zeros_like(total)
        for j in range(k, k + 8):
            most = torch.maximum(most, a[:, j, None] * b[None, :, j])
        total += most
    return 7 * 2.0 ** -13 * 1.001 * total.double()


@pytest.mark.parametrize("case", TILES)
def test_fp8_matmul_in_each_tile(case):
    tile, fast, M, N, Kc, fa, ta, fb, tb, has_bias = case
    assert tile_of(M, N, Kc, fast) == tile
    (qa, sa), a = S.operand(M, Kc, fa, ta, 1)
    (qb, sb), b = S.operand(N, Kc, fb, tb, 2)
    bias = rnd(N, seed=9) if has_bias else None
    a, b = a.to(DEV), b.to(DEV)
    want = a @ b.t()
    if has_bias:
        want += bias.double().to(DEV)
    sums = (a.shape[1] + 8) * R.U32 * (a.abs() @ b.abs().t()) + 1e-30
    if fast:
        sums += cut_of(a.abs().float(), b.abs().float())
    for odt in ((BF,) if fast else (BF, F32)):
        bound = sums + 1.01 * R.HALF[odt] * want.abs()
        out = torch.full((M, N), float("nan"), device=DEV, dtype=odt)
        K.fp8_matmul(qa, sa, qb, sb, out, bias=dev(bias), fast=fast)
        within(out, want, bound, "product %s %s" % (case, odt))
        if odt == F32:
            prior = torch.randn(M, N, device=DEV)
            acc = prior.clone()
            K.fp8_matmul(qa, sa, qb, sb, acc, bias=dev(bias), accumulate=True)
            total = want + prior.double()
            within(acc, total, bound + R.U32 * (total.abs() + prior.double().abs()), "accumulated %s" % (case,))
        wide = torch.full((M + 1, 2 * N + 3), 5.0, device=DEV, dtype=odt)
        K.fp8_matmul(qa, sa, qb, sb, wide[:M, 1:N + 1], bias=dev(bias), fast=fast)
        assert torch.equal(wide[:M, 1:N + 1], out) and (wide[:, N + 1:] == 5).all() and (wide[:, 0] == 5).all() and (wide[M] == 5).all()


# ---- gated scan ----------------------------------------------------------------------------------------------------------------
def scan_both_ways(i, B, T, D, dt, f, what):
    """Forward and backward of `i` against 64 bits, twice (the same bits), with nothing but NaN in the scratch buffers before."""
    d_y, d_hT = rnd(B, T, D, seed=5, dtype=dt), rnd(B, D, seed=6)
    if i["lengths"] is not None:
        for b, n in enumerate(i["lengths"].tolist()):
            d_y[b, n:] = 0
    want, bound = R.scan_with_bounds(i, d_y, d_hT, S.DELTA)
    how = S.scan_how(i)
    x, g = S.dev3(i["x"], f), S.dev3(i["g"], f)
    got = dict(y=S.dev3(torch.zeros(B, T, D, dtype=dt), f), hT=torch.full((B, D), float("nan"), device=DEV))
    carry = torch.full((K.gated_scan_carry(B, T, D),), float("nan"), device=DEV)
    K.gated_scan_forward(x, g, got["y"], got["hT"], carry, **how)
    got.update(d_x=S.dev3(torch.zeros(B, T, D, dtype=dt), f), d_g=S.dev3(torch.zeros(B, T, D, dtype=dt), f))
    if i["h0"] is not None:
        got["d_h0"] = torch.full((B, D), float("nan"), device=DEV)
    if i["floor"] is not None:
        got["d_floor"] = torch.full((D,), float("nan"), device=DEV)
    ws = torch.full((K.gated_scan_ws(B, T, D),), float("nan"), device=DEV)
    for again in (False, True):
        first = {n: v.clone() for n, v in got.items()}
        K.gated_scan_backward(x, g, S.dev3(d_y, f), dev(d_hT), carry, got["d_x"], got["d_g"], ws, d_h0=got.get("d_h0"),
                              d_floor=got.get("d_floor"), **how)
        if again:
            assert all(torch.equal(v, first[n]) for n, v in got.items()), "the same inputs give other bits"
    for n, v in got.items():
        within(v, want[n], bound[n] + 1.01 * R.HALF[v.dtype] * want[n].abs() + 1e-30, "%s %s" % (n, what))


@pytest.mark.parametrize("B,T,D,dt,rate", [(2, 1, 70, F32, 0.3), (2, 9, 70, F32, 0.0), (3, 100, 66, BF, 0.05), (1, 700, 40, F32, 0.01),
                                           (2, 700, 130, BF, 0.0)])
def test_gated_scan_with_floors_outside_their_range(B, T, D, dt, rate):
    """A floor is a trained parameter: below 0 (the gate's value then is too where it closes) the formula still holds, however the steps are
    split over waves, tiles and chunks, and a reset still drops what came before."""
    case = (B, T, D, dt, True, rate, None, True, 1)
    i = S.scan_inputs(case)
    gen = torch.Generator().manual_seed(8)
    i["floor"] = torch.rand(D, generator=gen) * 1.6 - 0.6                # -0.6 .. 1
    i["g"] = (i["g"].float() - 3).to(dt)
    scan_both_ways(i, B, T, D, dt, 1, case)


# ---- gates far from zero -------------------------------------------------------------------------------------------------------
# Roundings of sigmoid(g) or sigmoid(-g) times one value, relative to the result, in units of 2^-24: the exponential 3 (its instruction one
# step, its argument's two parts), 1 + e one, the reciprocal two, the product of both one, two more factors and one sum at most four;
# one to spare
N_GATE = 12
FAR = torch.linspace(12.0, 80.0, 2048)


def test_gated_scan_gates_far_from_zero():
    """fp32, one step: a closed gate lets (1 - f) x through, an open one f h0; both keep their value to a few last bits, however small."""
    D = FAR.numel()
    one, zero = torch.ones(1, 1, D, device=DEV), torch.zeros(1, 1, D, device=DEV)
    y = torch.empty(1, 1, D, device=DEV)
    K.gated_scan_forward(one, dev(FAR)[None, None], y, None, None, keep=False)             # f near 1: y = sigmoid(-g)
    want = torch.sigmoid(-FAR.double())
    within(y[0, 0], want, N_GATE * R.U32 * want, "1 - f")
    K.gated_scan_forward(zero, -dev(FAR)[None, None], y, None, None, h0=one[0], keep=False)   # f near 0: y = sigmoid(g)
    within(y[0, 0], want, N_GATE * R.U32 * want, "f")
    carry = torch.empty(K.gated_scan_carry(1, 1, D), device=DEV)
    K.gated_scan_forward(zero, dev(FAR)[None, None], y, None, carry, h0=one[0])
    dx, dg = torch.empty_like(y), torch.empty_like(y)
    K.gated_scan_backward(zero, dev(FAR)[None, None], one, None, carry, dx, dg, torch.empty(K.gated_scan_ws(1, 1, D), device=DEV), h0=one[0])
    within(dx[0, 0], want, N_GATE * R.U32 * want, "d_x")
    slope = want * torch.sigmoid(FAR.double())
    within(dg[0, 0], slope, (N_GATE + 4) * R.U32 * slope, "d_g")                            # both sigmoids


@pytest.mark.parametrize("act", ["sigmoid", "silu"])
def test_gated_norm_gates_far_from_zero(act):
    """fp32, no norm in front: y = act(gate) o for closed gates, and the gate's gradient."""
    C = FAR.numel()
    gate, one = -dev(FAR)[None], torch.ones(1, C, device=DEV)
    y = torch.empty(1, C, device=DEV)
    K.gated_norm_forward(torch.zeros(1, C, device=DEV), one, gate, y, None, pre=K.NORM_NONE, gate_act=S.ACTS[act])
    g = -FAR.double()
    want = R.act(act, g)
    within(y[0], want, N_GATE * R.U32 * want.abs(), "y")
    d_gate, d_o = torch.empty(1, C, device=DEV), torch.empty(1, C, device=DEV)
    K.gated_norm_backward(one, None, y, one, gate, None, d_o, d_gate, torch.empty(K.gated_norm_ws(1, C), device=DEV), pre=K.NORM_NONE,
                          gate_act=S.ACTS[act])
    within(d_o[0], want, N_GATE * R.U32 * want.abs(), "d_o")
    slope = R.act_slope(act, g)
    within(d_gate[0], slope, (N_GATE + 8) * R.U32 * slope.abs(), "d_gate")                  # silu: s + g s (1 - s), terms 1 to 1 - g


def test_gated_norm_tanh_gates_far_from_zero():
    """The slope 1 - tanh^2 = 1 / cosh^2 keeps its value where tanh is 1 to the last bit."""
    v = FAR / 8
    C = v.numel()
    gate, one = dev(v)[None], torch.ones(1, C, device=DEV)
    y, d_gate, d_o = (torch.empty(1, C, device=DEV) for _ in range(3))
    K.gated_norm_forward(torch.zeros(1, C, device=DEV), one, gate, y, None, pre=K.NORM_NONE, gate_act=K.ACT_TANH)
    want = torch.tanh(v.double())
    within(y[0], want, N_GATE * R.U32 * want, "y")
    K.gated_norm_backward(one, None, y, one, gate, None, d_o, d_gate, torch.empty(K.gated_norm_ws(1, C), device=DEV), pre=K.NORM_NONE,
                          gate_act=K.ACT_TANH)
    slope = torch.cosh(v.double()) ** -2
    within(d_gate[0], slope, (N_GATE + 4) * R.U32 * slope, "d_gate")                        # the reciprocal squared


# ---- chunks of several tiles ---------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("B,T,D,dt,floor,rate,lengths,f", [
    (4, 1100, 1000, F32, True, 0.01, [1100, 0, 517, 1099], 1),           # 12 chunks of 3 tiles of 32 steps, the last of 2
    (4, 1100, 1000, BF, True, 0.0, None, 2),
    (4, 1100, 1000, BF, False, 0.05, [700, 1, 1100, 96], 1),             # ends inside a chunk, in its first step, at a chunk's end
    (40, 1000, 51, F32, True, 0.01, None, 1),                            # one channel a lane; 11 chunks of 3 tiles, the last of 2
])
def test_gated_scan_in_chunks_of_several_tiles(B, T, D, dt, floor, rate, lengths, f):
    tiles, chunks = -(-T // 32), K.gated_scan_ws(B, T, D) // (2 * B * D)
    assert chunks > 1 and -(-tiles // chunks) > 1                        # scratch for two values a chunk and channel: it is cut, into tiles
    case = (B, T, D, dt, floor, rate, lengths, True, f)
    scan_both_ways(S.scan_inputs(case), B, T, D, dt, f, case)


# ---- several rows an item ------------------------------------------------------------------------------------------------------
def item_of(rows, C, k):
    """Rows of an item of the norm's backward pass and (0: whole gate rows) pieces of a gate row, the split's rule restated."""
    lanes = 1
    while lanes < -(-C // 8) and lanes < 512:
        lanes *= 2
    m = -(-rows // (256 * (512 // lanes)))
    if 1 < k <= 2 * m:
        return (-(-m // k) * k if k <= m else k), 0
    if k > m:
        k = min(k, rows)
        pieces = -(-k // m)
        return -(-k // pieces), pieces
    return m, 0


# rows, C, dtype, res, post, pre, gate (None / rows per gate), act, scale, row stride factor; (rows an item, pieces)
ITEMS = [
    ((4999, 520, BF, F32, "rms", "layer", 3, "silu", True, 1), (6, 0)),       # two gate rows an item; the last item one row of a short one
    ((5000, 520, F32, F32, "layer", "rms", 1, "tanh", True, 1), (5, 0)),
    ((1501, 2104, BF, BF, "layer", "layer", 2, "sigmoid", True, 1), (6, 0)),   # a row over eight waves: sums through LDS row after row
    ((1500, 2104, F32, F32, "rms", "rms", 100, "silu", True, 1), (6, 17)),     # pieces of six rows, the last of four
    ((1499, 2104, BF, F32, "none", "layer", None, "none", True, 2), (6, 0)),
    ((1501, 4104, BF, BF, "rms", "layer", 3, "tanh", True, 1), (6, 0)),        # parameter sums in LDS over several rows
    ((1301, 8200, BF, F32, "layer", "rms", 2, "silu", True, 1), (6, 0)),
    ((70001, 24, F32, F32, "rms", "rms", 3, "sigmoid", True, 1), (3, 0)),      # 128 items a workgroup
    ((2999, 1003, BF, BF, "rms", "rms", 2, "silu", True, 1), (4, 0)),          # rows that begin at every alignment
]


@pytest.mark.parametrize("case,split", ITEMS)
def test_gated_norm_with_several_rows_an_item(case, split):
    assert item_of(case[0], case[1], case[6] or 1) == split
    S.test_gated_norm_forward(case)
    S.test_gated_norm_backward(case)


@pytest.mark.parametrize("B,T,D,dt", [(3, 70, 66, BF), (5, 300, 33, F32)])
def test_gated_scan_layouts(B, T, D, dt):
    """Steps outside the batch ([T, B, D] in memory), inputs as windows over one another, x beside g in one tensor: the same bits as with
    tensors of their own."""
    def time_major():
        return torch.zeros(T, B, D, device=DEV, dtype=dt).transpose(0, 1)
    both = dev(rnd(B + T, 2 * D, seed=1, dtype=dt))
    x, g = (torch.as_strided(both, (B, T, D), (2 * D, 2 * D, 1), at) for at in (0, D))      # batch row b begins one step later
    d_y, d_hT = dev(rnd(B, T, D, seed=2, dtype=dt)), dev(rnd(B, D, seed=3))
    carry, ws = torch.empty(K.gated_scan_carry(B, T, D), device=DEV), torch.empty(K.gated_scan_ws(B, T, D), device=DEV)

    def run(x, g, make):
        y, dx, dg, hT = make(), make(), make(), torch.empty(B, D, device=DEV)
        K.gated_scan_forward(x, g, y, hT, carry)
        K.gated_scan_backward(x, g, d_y, d_hT, carry, dx, dg, ws)
        return y, hT, dx, dg
    apart = run(x.contiguous(), g.contiguous(), lambda: torch.zeros(B, T, D, device=DEV, dtype=dt))
    for a, b in zip(apart, run(x, g, time_major)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("T", [20, 100, 700])
def test_gated_scan_a_reset_stops_a_gate_of_nan(T, dt):
    """A gate that is NaN makes the state NaN up to the next reset, and the gradients up to the one before, in one wave, tile or chunk and
    across them: the mark of a reset is not taken for it, nor it for a reset."""
    B, D, at, first, second = 2, 66, T // 2, T // 4, 3 * T // 4
    x, g = rnd(B, T, D, seed=1, dtype=dt), rnd(B, T, D, seed=2, dtype=dt)
    g[:, at] = float("nan")
    reset = torch.zeros(B, T, dtype=torch.uint8)
    reset[0, first] = reset[0, second] = 1                              # row 1 has none
    y, hT, carry = torch.empty(B, T, D, device=DEV, dtype=dt), torch.empty(B, D, device=DEV), torch.empty(K.gated_scan_carry(B, T, D), device=DEV)
    K.gated_scan_forward(dev(x), dev(g), y, hT, carry, reset=dev(reset))
    dx, dg = torch.empty_like(y), torch.empty_like(y)
    K.gated_scan_backward(dev(x), dev(g), torch.ones_like(y), None, carry, dx, dg, torch.empty(K.gated_scan_ws(B, T, D), device=DEV), reset=dev(reset))
    bad, steps = torch.isnan(y.cpu()), torch.arange(T)
    assert torch.equal(bad[0], ((steps >= at) & (steps < second))[:, None].expand(T, D)) and not torch.isnan(hT[0]).any()
    assert torch.equal(bad[1], (steps >= at)[:, None].expand(T, D)) and torch.isnan(hT[1]).all()
    bad = torch.isnan(dx.cpu())
    assert torch.equal(bad[0], ((steps >= first) & (steps <= at))[:, None].expand(T, D))
    assert torch.equal(bad[1], (steps <= at)[:, None].expand(T, D))


@pytest.mark.parametrize("dt", [BF, F32])
def test_gates_of_infinity(dt):
    """A gate of infinity keeps the state, one of minus infinity takes the input: exactly, and with gradients that are numbers."""
    x, h0 = rnd(1, 2, 130, seed=1, dtype=dt), rnd(1, 130, seed=2)
    g = torch.zeros(1, 2, 130, dtype=dt)
    g[:, 0], g[:, 1] = float("inf"), float("-inf")
    y, hT = torch.empty(1, 2, 130, device=DEV, dtype=dt), torch.empty(1, 130, device=DEV)
    carry, ws = torch.empty(K.gated_scan_carry(1, 2, 130), device=DEV), torch.empty(K.gated_scan_ws(1, 2, 130), device=DEV)
    K.gated_scan_forward(dev(x), dev(g), y, hT, carry, h0=dev(h0))
    assert torch.equal(y[0, 0].cpu(), h0[0].to(dt)) and torch.equal(y[0, 1].cpu(), x[0, 1]) and torch.equal(hT.cpu(), x[:, 1].float())
    dx, dg, dh0 = torch.empty_like(y), torch.empty_like(y), torch.empty(1, 130, device=DEV)
    K.gated_scan_backward(dev(x), dev(g), torch.ones_like(y), torch.ones(1, 130, device=DEV), carry, dx, dg, ws, h0=dev(h0), d_h0=dh0)
    assert (dx[0, 0] == 0).all() and (dx[0, 1] == 2).all() and (dg == 0).all() and (dh0 == 1).all()
