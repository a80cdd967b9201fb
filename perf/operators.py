"""Sequence-block operators: what is timed, their plain forms and their values in 64 bits.

Three operators that make up one block over rows of features (a frame's pixels, a sequence's steps):

  norm   y = x + alpha * scale * act(gate) * post(o),  h = pre(y): the boundary between two blocks -- the norm after the
         block that ends, its gate, the residual scale, the residual sum and the norm before the block that begins
  fp8    y = x W^T with 8-bit floating-point operands and one power-of-two scale for each block of 128 along the reduction
         (x: a scale per row and block; W: a scale per 128 x 128 tile), forward, and forward with both gradients
  scan   h[t] = f[t] h[t-1] + (1 - f[t]) x[t] with f = floor + (1 - floor) sigmoid(g): a gated linear recurrence along a
         sequence, a single step of it, and its backward pass

A case is a dict of plain values; its "op" names the operator and "pass" the direction.
"""
import math

import torch

own = False

DEV = "cuda"
BF16, F32 = torch.bfloat16, torch.float32
DTYPES = {"bf16": BF16, "f32": F32}
FP8 = {"e4m3": (torch.float8_e4m3fn, 8, 1.75), "e5m2": (torch.float8_e5m2, 15, 1.75)}   # largest value = 1.75 * 2^emax


# ---- the cases ---------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one step of eight streams through a block boundary: latency only
        dict(name="norm token", op="norm", **{"pass": "forward"}, rows=8, C=2048, dtype="bf16", res="bf16", post="rms", pre="rms",
             gate="row", act="none", rows_per_gate=1, alpha=0.2, scale=False),
        # a long batch of wide rows, the gate a sigmoid of a projection
        dict(name="norm wide", op="norm", **{"pass": "forward"}, rows=16384, C=4096, dtype="bf16", res="bf16", post="rms", pre="rms",
             gate="row", act="sigmoid", rows_per_gate=1, alpha=1.0, scale=True),
        # the generator's 64 features over 4 clips of 19 frames at 32 x 32, fp32 parity mode, per-channel residual scale
        dict(name="norm features backward", op="norm", **{"pass": "backward"}, rows=77824, C=64, dtype="f32", res="f32", post="none",
             pre="layer", gate="none", act="none", rows_per_gate=1, alpha=1.0, scale=True),
        # training: one modulation gate per sample of 1024 rows, the residual stream kept in fp32
        dict(name="norm gated backward", op="norm", **{"pass": "backward"}, rows=8192, C=2048, dtype="bf16", res="f32", post="rms",
             pre="layer", gate="sample", act="tanh", rows_per_gate=1024, alpha=0.2, scale=True),
        # a single token against a square weight: the weight's bytes count
        dict(name="fp8 token", op="fp8", **{"pass": "forward"}, M=1, N=4096, K=4096, fmt="e4m3", grad="e4m3", bias=True, dtype="bf16"),
        # nothing a multiple of a tile
        dict(name="fp8 ragged", op="fp8", **{"pass": "forward"}, M=1000, N=1111, K=1345, fmt="e4m3", grad="e4m3", bias=True, dtype="bf16"),
        # a prompt's batch through a wide projection
        dict(name="fp8 wide", op="fp8", **{"pass": "forward"}, M=8192, N=8192, K=4096, fmt="e4m3", grad="e4m3", bias=False, dtype="bf16"),
        # a training step of one projection: product, both gradients, gradients quantised with a wider exponent
        dict(name="fp8 train", op="fp8", **{"pass": "train"}, M=8192, N=4096, K=2048, fmt="e4m3", grad="e5m2", bias=True, dtype="bf16"),
        # serving: one step of 64 streams
        dict(name="scan step", op="scan", **{"pass": "forward"}, B=64, T=1, D=4096, dtype="bf16", floor=True, resets=0.0, lengths=False, h0=True),
        # one very long sequence
        dict(name="scan long", op="scan", **{"pass": "forward"}, B=1, T=65536, D=1024, dtype="bf16", floor=False, resets=0.0, lengths=False, h0=False),
        # training on a padded batch of packed sequences
        dict(name="scan train", op="scan", **{"pass": "train"}, B=8, T=4096, D=1536, dtype="bf16", floor=True, resets=0.002, lengths=True, h0=True),
        # 64 feature channels at 32 x 32 carried over the 19 frames of the ping-pong sequence, fp32 parity mode
        dict(name="scan frames train", op="scan", **{"pass": "train"}, B=4, T=19, D=65536, dtype="f32", floor=False, resets=0.0, lengths=False, h0=True),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("norm", "fp8", "scan"))
    if op == "norm":
        C = _log(rng, 24, 8192)
        C = C if rng.random() < 0.3 else max(8, C // 8 * 8)
        rows = _log(rng, 1, max(1, min(100000, (48 << 20) // C)))
        dtype = rng.choice(("bf16", "bf16", "f32"))
        gate = rng.choice(("none", "row", "sample"))
        return dict(op=op, **{"pass": rng.choice(("forward", "backward"))}, rows=rows, C=C, dtype=dtype,
                    res="f32" if dtype == "f32" else rng.choice(("bf16", "bf16", "f32")),
                    post=rng.choice(("none", "rms", "rms", "layer")), pre=rng.choice(("rms", "rms", "layer")), gate=gate,
                    act="none" if gate == "none" else rng.choice(("none", "sigmoid", "tanh", "silu")),
                    rows_per_gate=_log(rng, 1, rows) if gate == "sample" else 1, alpha=rng.choice((1.0, 0.2)), scale=rng.random() < 0.5)
    if op == "fp8":
        while True:
            M, N, K = _log(rng, 1, 8192), _log(rng, 64, 8192), _log(rng, 64, 8192)
            if rng.random() < 0.6:
                N, K = max(64, N // 64 * 64), max(64, K // 64 * 64)
            if rng.random() < 0.4:
                M = _log(rng, 1, 64)
            p = rng.choice(("forward", "forward", "train"))
            if (6 if p == "train" else 2) * M * N * K <= 2 * 8192 * 8192 * 4096 // 2:
                return dict(op=op, **{"pass": p}, M=M, N=N, K=K, fmt="e4m3", grad=rng.choice(("e4m3", "e5m2")), bias=rng.random() < 0.5,
                            dtype=rng.choice(("bf16", "bf16", "f32")))
    B, D = _log(rng, 1, 64), _log(rng, 32, 8192)
    D = D if rng.random() < 0.3 else max(8, D // 8 * 8)
    T = _log(rng, 1, max(1, min(65536, (40 << 20) // (B * D))))
    T = 1 if rng.random() < 0.1 else T
    return dict(op="scan", **{"pass": rng.choice(("forward", "train"))}, B=B, T=T, D=D, dtype=rng.choice(("bf16", "bf16", "f32")),
                floor=rng.random() < 0.5, resets=rng.choice((0.0, 0.002, 0.05)), lengths=rng.random() < 0.4, h0=rng.random() < 0.6)


def work(case):
    e = 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "norm":
        R, C = case["rows"], case["C"]
        r = 2 if case["res"] == "bf16" else 4
        gates = 0 if case["gate"] == "none" else R * C if case["gate"] == "row" else -(-R // case["rows_per_gate"]) * C
        if case["pass"] == "forward":                          # reads x, o, gate; writes y, h
            return dict(bytes=R * C * (2 * r + 2 * e) + gates * e + 20 * C, flops=14 * R * C)
        return dict(bytes=R * C * (3 * r + 3 * e) + 2 * gates * e + 40 * C, flops=40 * R * C)   # dy, dh, y, o, gate; dx, do, dgate
    if case["op"] == "fp8":
        M, N, K = case["M"], case["N"], case["K"]
        if case["pass"] == "forward":
            return dict(bytes=e * M * K + N * K + e * M * N + 4 * N * case["bias"], flops=2 * M * N * K)
        # reads x, dy, W in both orders; writes y, dx, dW
        return dict(bytes=e * (2 * M * K + 2 * M * N) + 2 * N * K + 4 * N * K + 4 * N * case["bias"], flops=6 * M * N * K)
    n = case["B"] * case["T"] * case["D"]
    s = 4 * case["B"] * case["D"]
    if case["pass"] == "forward":
        return dict(bytes=3 * e * n + s * (1 + case["h0"]), flops=14 * n)
    return dict(bytes=6 * e * n + s * 4, flops=50 * n)          # x, g, dy; y, dx, dg


# ---- inputs ------------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def normal(*shape, dtype=dt, mean=0.0, std=1.0):
        return torch.empty(*shape, device=DEV, dtype=F32).normal_(mean, std, generator=gen).to(dtype)

    def uniform(*shape, lo=0.0, hi=1.0):
        return torch.empty(*shape, device=DEV, dtype=F32).uniform_(lo, hi, generator=gen)

    s = dict(case=dict(case))
    if case["op"] == "norm":
        R, C, res = case["rows"], case["C"], DTYPES[case["res"]]
        s["o"] = normal(R, C, std=1.5)
        groups = -(-R // case["rows_per_gate"])
        s["gate"] = None if case["gate"] == "none" else normal(groups, C, std=0.7)
        s["w_pre"] = normal(C, dtype=F32, mean=1.0, std=0.1)
        s["b_pre"] = normal(C, dtype=F32, std=0.1) if case["pre"] == "layer" else None
        s["w_post"] = normal(C, dtype=F32, mean=1.0, std=0.1) if case["post"] != "none" else None
        s["b_post"] = normal(C, dtype=F32, std=0.1) if case["post"] == "layer" else None
        s["scale"] = uniform(C, lo=0.05, hi=0.5) if case["scale"] else None
        if case["pass"] == "forward":
            s["x"] = normal(R, C, dtype=res, std=2.0)
        else:
            s["y"] = normal(R, C, dtype=res, std=2.0)
            s["d_y"] = normal(R, C, dtype=res)
            s["d_h"] = normal(R, C)
        return s
    if case["op"] == "fp8":
        M, N, K = case["M"], case["N"], case["K"]
        outliers = torch.exp(normal(K, dtype=F32, std=0.8))                 # a few channels of large activations
        s["x"] = (normal(M, K, dtype=F32) * outliers).to(dt)
        w = normal(N, K, dtype=F32, std=K ** -0.5)
        s["w"], s["sw"] = _store_tiles(w)                                   # the layer's weight as it is kept, in both orders
        s["wt"], s["swt"] = _store_tiles(w.t())
        s["bias"] = normal(N, dtype=F32, std=0.1) if case["bias"] else None
        if case["pass"] == "train":
            s["d_y"] = normal(M, N, std=1e-3)
        return s
    B, T, D = case["B"], case["T"], case["D"]
    s["x"], s["g"] = normal(B, T, D), normal(B, T, D, mean=2.0, std=1.5)
    s["floor"] = uniform(D, hi=0.9) if case["floor"] else None
    s["h0"] = normal(B, D, dtype=F32) if case["h0"] else None
    s["reset"] = (uniform(B, T) < case["resets"]).to(torch.uint8) if case["resets"] else None
    s["lengths"] = (uniform(B, lo=0.5, hi=1.0) * T).ceil().to(torch.int32) if case["lengths"] else None
    if case["pass"] == "train":
        s["d_y"], s["d_hT"] = normal(B, T, D), normal(B, D, dtype=F32)
    return s


# ---- plain forms: norm -------------------------------------------------------------------------------------------------
EPS = 1e-6


def _act(name, v):
    return v if name == "none" else torch.sigmoid(v) if name == "sigmoid" else torch.tanh(v) if name == "tanh" else v * torch.sigmoid(v)


def _act_grad(name, v):
    if name == "none":
        return torch.ones_like(v)
    if name == "tanh":
        return 1 - torch.tanh(v) ** 2
    p = torch.sigmoid(v)
    return p * (1 - p) if name == "sigmoid" else p * (1 + v * (1 - p))


def _standard(kind, v):
    """(v - mean) / deviation and 1 / deviation, by row."""
    if kind == "layer":
        v = v - v.mean(-1, keepdim=True)
    r = torch.rsqrt((v * v).mean(-1, keepdim=True) + EPS)
    return v * r, r


def _standard_grad(kind, d, n, r):
    d = d - n * (d * n).mean(-1, keepdim=True) - (d.mean(-1, keepdim=True) if kind == "layer" else 0)
    return d * r


def _affine(n, w, b):
    n = n if w is None else n * w
    return n if b is None else n + b


def _norm_forward(s):
    c = s["case"]
    x, u = s["x"].float(), s["o"].float()
    if c["post"] != "none":
        u = _affine(_standard(c["post"], u)[0], s["w_post"], s["b_post"])
    if s["gate"] is not None:
        u = u * _act(c["act"], s["gate"].float()).repeat_interleave(c["rows_per_gate"], 0)[:c["rows"]]
    if s["scale"] is not None:
        u = u * s["scale"]
    y = x + c["alpha"] * u
    h = _affine(_standard(c["pre"], y)[0], s["w_pre"], s["b_pre"])
    return dict(y=y.to(s["x"].dtype), h=h.to(s["o"].dtype))


def _norm_backward(s):
    c, out = s["case"], {}
    y, o, d_h = s["y"].float(), s["o"].float(), s["d_h"].float()
    n, r = _standard(c["pre"], y)
    out["d_w_pre"] = (d_h * n).sum(0)
    if s["b_pre"] is not None:
        out["d_b_pre"] = d_h.sum(0)
    d = s["d_y"].float() + _standard_grad(c["pre"], d_h * s["w_pre"], n, r)
    out["d_x"] = d.to(s["y"].dtype)
    d = d * c["alpha"]
    if c["post"] != "none":
        n, r = _standard(c["post"], o)
        u = _affine(n, s["w_post"], s["b_post"])
    else:
        u = o
    k, v = c["rows_per_gate"], None
    if s["gate"] is not None:
        v = s["gate"].float().repeat_interleave(k, 0)[:c["rows"]]
        a = _act(c["act"], v)
    else:
        a = torch.ones_like(u)
    if s["scale"] is not None:
        out["d_scale"] = (d * a * u).sum(0)
        d = d * s["scale"]
    if v is not None:
        t = d * u * _act_grad(c["act"], v)
        if k > 1:
            short = -c["rows"] % k
            t = torch.nn.functional.pad(t, (0, 0, 0, short)).reshape(-1, k, c["C"]).sum(1)
        out["d_gate"] = t.to(s["o"].dtype)
        d = d * a
    if c["post"] != "none":
        out["d_w_post"] = (d * n).sum(0)
        if s["b_post"] is not None:
            out["d_b_post"] = d.sum(0)
        d = _standard_grad(c["post"], d * s["w_post"], n, r)
    out["d_o"] = d.to(s["o"].dtype)
    return out


# ---- plain forms: fp8 --------------------------------------------------------------------------------------------------
def _padded(v, rows):
    return torch.nn.functional.pad(v, (0, -v.shape[1] % 128, 0, -v.shape[0] % 128 if rows else 0))


def _power(e):
    """2^e in 32 bits, from its bits: exact."""
    return ((e + 127).to(torch.int32) << 23).view(F32)


def _exponent(top, fmt):
    """The smallest e in -126 .. 127 with top <= largest value of the type * 2^e; 0 where there is nothing to scale."""
    _, emax, most = FP8[fmt]
    m, p = torch.frexp(top)
    e = p - 1 - emax + (2 * m > most).to(p.dtype)
    return torch.where(top > 0, e.clamp(-126, 127), 0)


def _round8(v, e, fmt):
    return (v * _power(-e)).to(FP8[fmt][0])


def _blocks(v, fmt):
    """`v`'s values as 8-bit floating point holds them, one power of two for each row and 128 columns."""
    p = _padded(v.float(), False).reshape(v.shape[0], -1, 128)
    e = _exponent(p.abs().amax(-1, keepdim=True), fmt)
    return (_round8(p, e, fmt).float() * _power(e)).reshape(v.shape[0], -1)


def _store_tiles(w):
    """The 8-bit matrix [rows, columns padded to 128] and the biased exponents [row tiles, column tiles padded to 4]."""
    p = _padded(w, True)
    t = p.reshape(p.shape[0] // 128, 128, p.shape[1] // 128, 128)
    e = _exponent(t.abs().amax((1, 3), keepdim=True), "e4m3")
    q = _round8(t, e, "e4m3").reshape(p.shape)[:w.shape[0]].contiguous()
    code = (e[:, 0, :, 0] + 127).to(torch.uint8)
    return q, torch.nn.functional.pad(code, (0, -code.shape[1] % 4), value=127).contiguous()


def _load_tiles(q, code):
    e = code[:, :q.shape[1] // 128].int() - 127
    e = e.repeat_interleave(128, 0)[:q.shape[0]].repeat_interleave(128, 1)
    return q.float() * _power(e)


def _fp8_forward(s):
    y = _blocks(s["x"], "e4m3") @ _load_tiles(s["w"], s["sw"]).t()
    return (y if s["bias"] is None else y + s["bias"]).to(s["x"].dtype)


def _fp8_train(s):
    c, dt = s["case"], s["x"].dtype
    out = dict(y=_fp8_forward(s))
    out["d_x"] = (_blocks(s["d_y"], c["grad"]) @ _load_tiles(s["wt"], s["swt"]).t()).to(dt)
    # the weight's gradient sums over the rows: both operands have their blocks along them
    out["d_w"] = _blocks(s["d_y"].t(), c["grad"]) @ _blocks(s["x"].t(), c["fmt"]).t()
    return out


# ---- plain forms: scan -------------------------------------------------------------------------------------------------
def _running(a, b):
    """h[t] = a[t] h[t-1] + b[t] from h[-1] = 0, by doubling: after each turn an element covers twice the steps."""
    k, T = 1, a.shape[1]
    while k < T:
        b = torch.cat((b[:, :k], b[:, k:] + a[:, k:] * b[:, :-k]), 1)
        a = torch.cat((a[:, :k], a[:, k:] * a[:, :-k]), 1)
        k *= 2
    return b


def _gates(s):
    """Per step: what is kept of the state, the forget gate, the input gate, its sigmoids, and where the sequence still runs."""
    g = s["g"].float()
    up, down = torch.sigmoid(g), torch.sigmoid(-g)
    low = torch.zeros((), device=g.device) if s["floor"] is None else s["floor"]
    f, i = low + (1 - low) * up, (1 - low) * down
    keep = f
    if s["reset"] is not None:
        keep = torch.where(s["reset"][..., None] != 0, 0.0, f)
    live = None
    if s["lengths"] is not None:
        live = (torch.arange(g.shape[1], device=g.device) < s["lengths"][:, None])[..., None]
        keep, i = torch.where(live, keep, 1.0), torch.where(live, i, 0.0)
    return keep, f, i, up, down, low, live


def _scan_states(s, keep, i):
    b = i * s["x"].float()
    if s["h0"] is not None:
        b = torch.cat((b[:, :1] + keep[:, :1] * s["h0"][:, None], b[:, 1:]), 1)
    return _running(keep, b)


def _scan_forward(s):
    keep, _, i, _, _, _, live = _gates(s)
    h = _scan_states(s, keep, i)
    return dict(y=(h if live is None else torch.where(live, h, 0.0)).to(s["x"].dtype), hT=h[:, -1].clone())


def _scan_train(s):
    c = s["case"]
    keep, _, i, up, down, low, live = _gates(s)
    h = _scan_states(s, keep, i)
    out = dict(y=(h if live is None else torch.where(live, h, 0.0)).to(s["x"].dtype), hT=h[:, -1].clone())
    d = s["d_y"].float()
    d = d if live is None else torch.where(live, d, 0.0)
    d = torch.cat((d[:, :-1], d[:, -1:] + s["d_hT"][:, None]), 1)
    after = torch.cat((keep[:, 1:], torch.ones_like(keep[:, :1])), 1)      # what step t + 1 keeps of step t
    d = _running(after.flip(1), d.flip(1)).flip(1)
    first = torch.zeros_like(h[:, :1]) if s["h0"] is None else s["h0"][:, None]
    before = torch.cat((first, h[:, :-1]), 1)
    if s["reset"] is not None:
        before = torch.where(s["reset"][..., None] != 0, 0.0, before)
    d_f = d * (before - s["x"].float())
    if live is not None:
        d_f = torch.where(live, d_f, 0.0)
    out["d_x"] = (d * i).to(s["x"].dtype)
    out["d_g"] = (d_f * (1 - low) * up * down).to(s["g"].dtype)
    if c["floor"]:
        out["d_floor"] = (d_f * down).sum((0, 1))
    if c["h0"]:
        out["d_h0"] = keep[:, 0] * d[:, 0]
    return out


# ---- one pass ----------------------------------------------------------------------------------------------------------
def run(state):
    c = state["case"]
    if own:
        return _own(state)
    if c["op"] == "norm":
        return _norm_forward(state) if c["pass"] == "forward" else _norm_backward(state)
    if c["op"] == "fp8":
        return dict(y=_fp8_forward(state)) if c["pass"] == "forward" else _fp8_train(state)
    return _scan_forward(state) if c["pass"] == "forward" else _scan_train(state)


def _own(s):
    """The framework's operators.  Outputs and workspaces are made at the state's first pass and kept, as an engine keeps them."""
    from tecogan_amd import kernels as K
    c = s["case"]
    kept = s.setdefault("kept", {})
    if c["op"] == "norm":
        return _own_norm(K, s, c, kept)
    if c["op"] == "fp8":
        return _own_fp8(K, s, c, kept)
    return _own_scan(K, s, c, kept)


def _own_norm(K, s, c, kept):
    kinds = dict(none=K.NORM_NONE, rms=K.NORM_RMS, layer=K.NORM_LAYER)
    acts = dict(none=K.ACT_NONE, sigmoid=K.ACT_SIGMOID, tanh=K.ACT_TANH, silu=K.ACT_SILU)
    how = dict(post=kinds[c["post"]], pre=kinds[c["pre"]], w_post=s["w_post"], b_post=s["b_post"], scale=s["scale"], w_pre=s["w_pre"],
               b_pre=s["b_pre"], alpha=c["alpha"], gate_act=acts[c["act"]], rows_per_gate=c["rows_per_gate"], eps=EPS)
    if c["pass"] == "forward":
        if not kept:
            kept.update(y=torch.empty_like(s["x"]), h=torch.empty_like(s["o"]))
        K.gated_norm_forward(s["x"], s["o"], s["gate"], kept["y"], kept["h"], **how)
        return kept
    if not kept:
        kept.update(d_x=torch.empty_like(s["y"]), d_o=torch.empty_like(s["o"]))
        if s["gate"] is not None:
            kept["d_gate"] = torch.empty_like(s["gate"])
        for p in ("w_post", "b_post", "scale", "w_pre", "b_pre"):
            if s[p] is not None:
                kept["d_" + p] = torch.empty_like(s[p])
        s["ws"] = torch.empty(K.gated_norm_ws(c["rows"], c["C"], c["rows_per_gate"]), device=DEV, dtype=F32)
    K.gated_norm_backward(s["d_y"], s["d_h"], s["y"], s["o"], s["gate"], kept["d_x"], kept["d_o"], kept.get("d_gate"), s["ws"],
                          d_w_post=kept.get("d_w_post"), d_b_post=kept.get("d_b_post"), d_scale=kept.get("d_scale"),
                          d_w_pre=kept.get("d_w_pre"), d_b_pre=kept.get("d_b_pre"), **how)
    return kept


def _own_fp8(K, s, c, kept):
    M, N, Kd = c["M"], c["N"], c["K"]
    dt = s["x"].dtype
    if not kept:
        kept["y"] = torch.empty(M, N, device=DEV, dtype=dt)
        if c["pass"] == "train":
            kept.update(d_x=torch.empty(M, Kd, device=DEV, dtype=dt), d_w=torch.empty(N, Kd, device=DEV, dtype=F32))
            s["x8"], s["d8"] = K.fp8_alloc(M, Kd, DEV, c["fmt"], transposed=True), K.fp8_alloc(M, N, DEV, c["grad"], transposed=True)
        else:
            s["ws"] = torch.empty(K.fp8_linear_ws(M, N, Kd), device=DEV, dtype=torch.uint8)
    if c["pass"] == "forward":
        K.fp8_linear(s["x"], s["w"], s["sw"], kept["y"], s["ws"], bias=s["bias"])
        return kept
    (xq, xs, xqt, xst), (dq, ds, dqt, dst) = s["x8"], s["d8"]
    K.fp8_quantize(s["x"], xq, xs, xqt, xst)
    K.fp8_matmul(xq, xs, s["w"], s["sw"], kept["y"], bias=s["bias"])
    K.fp8_quantize(s["d_y"], dq, ds, dqt, dst)
    K.fp8_matmul(dq, ds, s["wt"], s["swt"], kept["d_x"])
    K.fp8_matmul(dqt, dst, xqt, xst, kept["d_w"])
    return kept


def _own_scan(K, s, c, kept):
    B, T, D = c["B"], c["T"], c["D"]
    train = c["pass"] == "train"
    if not kept:
        kept.update(y=torch.empty_like(s["x"]), hT=torch.empty(B, D, device=DEV, dtype=F32))
        s["carry"] = torch.empty(K.gated_scan_carry(B, T, D), device=DEV, dtype=F32)
        if train:
            kept.update(d_x=torch.empty_like(s["x"]), d_g=torch.empty_like(s["g"]))
            if c["floor"]:
                kept["d_floor"] = torch.empty(D, device=DEV, dtype=F32)
            if c["h0"]:
                kept["d_h0"] = torch.empty(B, D, device=DEV, dtype=F32)
            s["ws"] = torch.empty(K.gated_scan_ws(B, T, D), device=DEV, dtype=F32)
    how = dict(h0=s["h0"], floor=s["floor"], lengths=s["lengths"], reset=s["reset"])
    K.gated_scan_forward(s["x"], s["g"], kept["y"], kept["hT"], s["carry"], keep=train, **how)
    if train:
        K.gated_scan_backward(s["x"], s["g"], s["d_y"], s["d_hT"], s["carry"], kept["d_x"], kept["d_g"], s["ws"],
                              d_h0=kept.get("d_h0"), d_floor=kept.get("d_floor"), **how)
    return kept


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------------
def exact(case, seed):
    s = {k: v.double() if isinstance(v, torch.Tensor) and v.is_floating_point() and v.element_size() > 1 else v
         for k, v in prepare(case, seed).items()}
    if case["op"] == "norm":
        return _exact_norm(case, s)
    return _exact_fp8(case, s) if case["op"] == "fp8" else _exact_scan(case, s)


def _exact_norm(case, s):
    R, C, k = case["rows"], case["C"], case["rows_per_gate"]
    of = torch.arange(R, device=DEV) // k                                  # the gate row of each row

    def squash(v):                                                         # the activation and its derivative
        if case["act"] == "none":
            return v, torch.ones_like(v)
        if case["act"] == "tanh":
            t = torch.tanh(v)
            return t, 1 - t * t
        p = 1 / (1 + torch.exp(-v))
        return (p, p - p * p) if case["act"] == "sigmoid" else (v * p, p + v * (p - p * p))

    def stats(kind, v):
        mu = v.sum(1, keepdim=True) / C if kind == "layer" else torch.zeros(R, 1, device=DEV, dtype=v.dtype)
        return mu, 1 / torch.sqrt(((v - mu) ** 2).sum(1, keepdim=True) / C + EPS)

    post = case["post"] != "none"
    o, gain = s["o"], torch.full((C,), case["alpha"], device=DEV, dtype=torch.float64)
    if s["scale"] is not None:
        gain = gain * s["scale"]
    z, wz, bz = o, 1.0, 0.0
    if post:
        mu_o, r_o = stats(case["post"], o)
        z, wz, bz = (o - mu_o) * r_o, s["w_post"], 0.0 if s["b_post"] is None else s["b_post"]
    act, slope = (1.0, None) if s["gate"] is None else squash(s["gate"])
    act_rows = act if s["gate"] is None else act[of]
    branch = z * wz + bz
    if case["pass"] == "forward":
        y = s["x"] + gain * act_rows * branch
        mu, r = stats(case["pre"], y)
        h = (y - mu) * r * s["w_pre"]
        return dict(y=y, h=h if s["b_pre"] is None else h + s["b_pre"])
    y, dh = s["y"], s["d_h"]
    mu, r = stats(case["pre"], y)
    z_y = (y - mu) * r
    out = dict(d_w_pre=(dh * z_y).sum(0))
    if s["b_pre"] is not None:
        out["d_b_pre"] = dh.sum(0)
    t = dh * s["w_pre"]
    t = t - z_y * ((t * z_y).sum(1, keepdim=True) / C) - ((t.sum(1, keepdim=True) / C) if case["pre"] == "layer" else 0.0)
    dx = s["d_y"] + r * t
    out["d_x"] = dx
    if s["scale"] is not None:
        out["d_scale"] = case["alpha"] * (dx * act_rows * branch).sum(0)
    if s["gate"] is not None:
        groups = s["gate"].shape[0]
        total = torch.zeros(groups, C, device=DEV, dtype=torch.float64).index_add_(0, of, dx * branch * gain)
        out["d_gate"] = total * slope
    db = dx * gain * act_rows
    if post:
        out["d_w_post"] = (db * z).sum(0)
        if s["b_post"] is not None:
            out["d_b_post"] = db.sum(0)
        t = db * wz
        t = t - z * ((t * z).sum(1, keepdim=True) / C) - ((t.sum(1, keepdim=True) / C) if case["post"] == "layer" else 0.0)
        db = r_o * t
    out["d_o"] = db
    return out


def _exact_fp8(case, s):
    limits = dict(e4m3=(448.0, 3, -6), e5m2=(57344.0, 2, -14))             # largest value, mantissa bits, lowest exponent

    def two_to(e):
        return ((e.long() + 1023) << 52).view(torch.float64)

    def held(v, fmt):                                                      # rows x 128: a power of two each, round to nearest even
        most, bits, low = limits[fmt]
        n = v.shape[1]
        v = torch.cat((v, v.new_zeros(v.shape[0], -n % 128)), 1).view(v.shape[0], -1, 128)
        top = v.abs().amax(2, keepdim=True)
        e = torch.ceil(torch.log2(top / most))
        e = torch.where(top > 0, e.clamp(-126, 127), torch.zeros_like(e))
        e = torch.where((top > 0) & (top <= most * two_to(e - 1)), e - 1, torch.where(top > most * two_to(e), e + 1, e))   # log2 at a border
        unit = two_to(e.clamp(-126, 127))
        v = v / unit
        step = two_to(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** (low - 8)))).clamp(min=low) - bits)
        return (torch.round(v / step) * step * unit).reshape(v.shape[0], -1)

    def weight(q, code):
        rows, cols = torch.arange(q.shape[0], device=DEV) // 128, torch.arange(q.shape[1], device=DEV) // 128
        return q.float().double() * two_to(code[rows][:, cols].long() - 127)

    x = s["x"]
    y = held(x, "e4m3") @ weight(s["w"], s["sw"]).t()
    out = dict(y=y if s["bias"] is None else y + s["bias"])
    if case["pass"] == "train":
        out["d_x"] = held(s["d_y"], case["grad"]) @ weight(s["wt"], s["swt"]).t()
        out["d_w"] = held(s["d_y"].t().contiguous(), case["grad"]) @ held(x.t().contiguous(), case["fmt"]).t()
    return out


def _exact_scan(case, s):
    B, T, D = case["B"], case["T"], case["D"]
    low = torch.zeros(D, device=DEV, dtype=torch.float64) if s["floor"] is None else s["floor"]
    ends = torch.full((B, 1), T, device=DEV) if s["lengths"] is None else s["lengths"][:, None]
    fresh = torch.zeros(B, T, device=DEV, dtype=torch.bool) if s["reset"] is None else s["reset"] != 0
    x, g = s["x"], s["g"]
    h = torch.zeros(B, D, device=DEV, dtype=torch.float64) if s["h0"] is None else s["h0"].clone()
    first = h
    y = torch.zeros(B, T, D, device=DEV, dtype=torch.float64)
    states = torch.empty(B, T, D, device=DEV, dtype=torch.float64) if case["pass"] == "train" else None   # before each step
    for t in range(T):
        p = 1 / (1 + torch.exp(-g[:, t]))
        f = low + (1 - low) * p
        came = torch.where(fresh[:, t, None], 0.0, h)
        if states is not None:
            states[:, t] = came
        new = f * came + (1 - low) * (1 - p) * x[:, t]
        runs = t < ends
        y[:, t] = torch.where(runs, new, 0.0)
        h = torch.where(runs, new, h)
    out = dict(y=y, hT=h)
    if states is None:
        return out
    d, d_x, d_g = s["d_hT"].clone(), torch.zeros_like(x), torch.zeros_like(g)
    d_low = torch.zeros(D, device=DEV, dtype=torch.float64)
    for t in range(T - 1, -1, -1):
        p = 1 / (1 + torch.exp(-g[:, t]))
        runs = t < ends
        total = d + s["d_y"][:, t]
        to_f = torch.where(runs, total * (states[:, t] - x[:, t]), 0.0)
        d_x[:, t] = torch.where(runs, total * (1 - low) * (1 - p), 0.0)
        d_g[:, t] = to_f * (1 - low) * p * (1 - p)
        d_low += (to_f * (1 - p)).sum(0)
        d = torch.where(runs, torch.where(fresh[:, t, None], 0.0, total * (low + (1 - low) * p)), d)
    out["d_x"], out["d_g"] = d_x, d_g
    if case["floor"]:
        out["d_floor"] = d_low
    if case["h0"]:
        out["d_h0"] = d
    return out
