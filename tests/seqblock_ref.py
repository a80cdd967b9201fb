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
