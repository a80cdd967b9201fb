"""The sequence-block operators from their definitions in 64 bits, with what bounds a 32-bit evaluation's error.

`norm_forward` / `scan_forward` are differentiable (gradients by torch's autograd in fp64).  The `*_error` functions restate the
formulas over absolute values: the size of what is added up, which times the unit roundoff and the number of roundings bounds the error
of any order of evaluation.
"""
import torch

U32 = 2.0 ** -24                                     # half a step of fp32, relative
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


def act(name, v):
    return {"none": lambda t: t, "sigmoid": torch.sigmoid, "tanh": torch.tanh, "silu": lambda t: t * torch.sigmoid(t)}[name](v)


def act_slope(name, v):
    p = torch.sigmoid(v)
    return {"none": torch.ones_like(v), "sigmoid": p * (1 - p), "tanh": 1 - torch.tanh(v) ** 2, "silu": p * (1 + v * (1 - p))}[name]


def moments(kind, z, eps):
    mu = z.mean(-1, keepdim=True) if kind == "layer" else torch.zeros_like(z[..., :1])
    return mu, ((z - mu) ** 2).mean(-1, keepdim=True).add(eps).rsqrt()


def normed(kind, z, w, b, eps):
    if kind == "none":
        return z
    mu, r = moments(kind, z, eps)
    n = (z - mu) * r
    n = n if w is None else n * w
    return n if b is None else n + b


def gate_rows(gate, k, rows):
    return gate[torch.arange(rows, device=gate.device) // k]


def norm_forward(x, o, gate, p, post, pre, gate_act, k, alpha, eps):
    """x, o [R, C], gate [ceil(R / k), C] or None, p: dict of parameters or None -> y, h."""
    y = x
    if o is not None:
        v = normed(post, o, p["w_post"], p["b_post"], eps) * alpha
        if gate is not None:
            v = v * act(gate_act, gate_rows(gate, k, x.shape[0]))
        if p["scale"] is not None:
            v = v * p["scale"]
        y = x + v
    return y, (normed(pre, y, p["w_pre"], p["b_pre"], eps) if pre != "none" else None)


def scan_forward(x, g, h0, low, ends, fresh):
    """x, g [B, T, D], h0 [B, D], low [D], ends [B], fresh [B, T] bool -> y, hT."""
    h, ys = h0, []
    for t in range(x.shape[1]):
        up, down = torch.sigmoid(g[:, t]), torch.sigmoid(-g[:, t])
        came = torch.where(fresh[:, t, None], torch.zeros_like(h), h)
        new = (low + (1 - low) * up) * came + (1 - low) * down * x[:, t]
        runs = (t < ends)[:, None]
        ys.append(torch.where(runs, new, torch.zeros_like(new)))
        h = torch.where(runs, new, h)
    return torch.stack(ys, 1), h


def power(e):
    """2^e in fp64 from its bits."""
    return ((e.long() + 1023) << 52).view(torch.float64)


LIMITS = {"e4m3": (448.0, 3, -6), "e5m2": (57344.0, 2, -14)}           # largest value, mantissa bits, lowest exponent


def exponent(top, fmt):
    """The smallest e in [-126, 127] with top <= largest * 2^e (0 for top = 0), by trying."""
    most = LIMITS[fmt][0]
    e = torch.full(top.shape, -126, dtype=torch.int64)
    for step in (128, 64, 32, 16, 8, 4, 2, 1):                          # the largest e whose predecessor is too small
        e = torch.where(top > most * power(e + step - 1), e + step, e)
    return torch.where(top > 0, e, torch.zeros_like(e))


def to8(v, fmt):
    """Round to nearest even in the type's grid (|v| <= largest), as values in fp64; NaN and infinities as the operator stores them."""
    most, bits, low = LIMITS[fmt]
    a = v.abs()
    fin = torch.isfinite(v)
    a = torch.where(fin, a, torch.zeros_like(a))
    m, p = torch.frexp(a)
    step = power(torch.clamp(p - 1, min=low) - bits)
    r = torch.round(v / step) * step
    if fmt == "e4m3":
        return torch.where(fin, r, torch.full_like(r, float("nan")))
    return torch.where(fin, r, v)


def quantized(x, fmt, tile):
    """(values that are stored, exponents): blocks of 128 along the last dimension of x [R, C]; tile: of 128 x 128."""
    R, Cc = x.shape
    pad = torch.nn.functional.pad(x.double(), (0, -Cc % 128, 0, -R % 128))
    t = pad.reshape(pad.shape[0] // 128, 128, pad.shape[1] // 128, 128)
    a = torch.where(torch.isfinite(t), t.abs(), torch.zeros_like(t))
    top = a.amax((1, 3), keepdim=True) if tile else a.amax(3, keepdim=True)
    e = exponent(top, fmt)
    q = to8(t * power(-e), fmt).reshape(pad.shape)[:R]
    code = e[:, 0, :, 0] if tile else e[..., 0].reshape(pad.shape[0], -1)[:R]
    return q, code


def scan_with_bounds(i, d_y, d_hT, delta):
    """Outputs and gradients of the recurrence for a dict of inputs (x, g, h0, floor, reset, lengths; None: not given), any floor, and what an
    evaluation may be off by: an error e of the state goes on as |f| e, and every step adds delta times the size of its terms, the
    gate's two among them (they cancel where the floor is negative)."""
    B, T, D = i["x"].shape
    x, g = i["x"].double().requires_grad_(), i["g"].double().requires_grad_()
    h0 = (torch.zeros(B, D, dtype=torch.float64) if i["h0"] is None else i["h0"].double()).requires_grad_()
    low = (torch.zeros(D, dtype=torch.float64) if i["floor"] is None else i["floor"].double()).requires_grad_()
    ends = torch.full((B,), T) if i["lengths"] is None else i["lengths"].long()
    fresh = torch.zeros(B, T, dtype=torch.bool) if i["reset"] is None else i["reset"] != 0
    y, hT = scan_forward(x, g, h0, low, ends, fresh)
    grads = torch.autograd.grad((y, hT), (x, g, h0, low), (d_y.double(), d_hT.double()))
    want = dict(y=y, hT=hT, d_x=grads[0], d_g=grads[1], d_h0=grads[2], d_floor=grads[3])
    with torch.no_grad():
        zero = torch.zeros((), dtype=torch.float64)
        runs = (torch.arange(T)[None] < ends[:, None])[..., None]
        cut = fresh[..., None] & runs
        up, down, k = torch.sigmoid(g), torch.sigmoid(-g), (1 - low).abs()
        f, terms = (low + (1 - low) * up).abs(), low.abs() + k * up
        f, terms = (torch.where(runs, torch.where(cut, zero, v), zero + 1) for v in (f, terms))
        a = torch.where(runs, k * down * x.abs(), zero)
        M, E, e_y, came_M, came_E = h0.abs(), torch.zeros(B, D, dtype=torch.float64), [], [], []
        for t in range(T):
            came_M.append(torch.where(cut[:, t], zero, M))
            came_E.append(torch.where(cut[:, t], zero, E))
            E = f[:, t] * E + delta * (terms[:, t] * M + a[:, t])
            M = f[:, t] * M + a[:, t]
            e_y.append(torch.where(runs[:, t], E, zero))
        bound = dict(y=torch.stack(e_y, 1), hT=E)
        Dm, De = d_hT.double().abs(), torch.zeros(B, D, dtype=torch.float64)
        ex, eg = torch.zeros(B, T, D, dtype=torch.float64), torch.zeros(B, T, D, dtype=torch.float64)
        e_low, m_low = torch.zeros(D, dtype=torch.float64), torch.zeros(D, dtype=torch.float64)
        for t in range(T - 1, -1, -1):
            live = runs[:, t]
            m = Dm + d_y[:, t].double().abs()
            e = De + delta * m
            s = came_M[t] + x[:, t].abs()                               # |h - x| at most
            ef = e * s + m * (came_E[t] + delta * s) + delta * m * s
            ex[:, t] = torch.where(live, k * down[:, t] * (e + delta * m), zero)
            eg[:, t] = torch.where(live, k * up[:, t] * down[:, t] * ef, zero)
            e_low += torch.where(live, down[:, t] * ef, zero).sum(0)
            m_low += torch.where(live, down[:, t] * m * s, zero).sum(0)
            De = torch.where(live, f[:, t] * e + delta * terms[:, t] * m, De)
            Dm = torch.where(live, f[:, t] * m, Dm)
        bound.update(d_x=ex, d_g=eg, d_h0=De, d_floor=e_low + (T + 64) * U32 * m_low)   # a lane adds up to T steps, then partial sums
    return want, bound
