"""The sequence-block operators without a GPU: refusals (argument checks come before any launch), sizes, and the 64-bit references."""
import ctypes as C

import pytest
import torch

import seqblock_ref as R
from tecogan_amd import _lib as L
from tecogan_amd import kernels as K

P = C.c_void_p(4096)                                 # never read: the calls are refused


def norm_desc(**kw):
    d = L.GatedNormDesc()
    base = dict(rows=4, rows_per_gate=1, ldx=64, ldo=64, ldg=64, ldy=64, ldh=64, ld_dy=64, ld_do=64, ld_dg=64, C=64, dtype=L.TG_BF16,
                res_dtype=L.TG_BF16, post=L.NORM_RMS, pre=L.NORM_RMS, gate_act=0, alpha=1.0, eps=1e-6)
    for n, v in {**base, **kw}.items():
        setattr(d, n, v)
    return d


def refused(rc, *words):
    msg = L.lib().tg_last_error_string().decode()
    assert rc == -1 and all(w in msg for w in words), (rc, msg)


@pytest.mark.parametrize("kw,word", [(dict(C=0), "C in"), (dict(C=16385), "C in"), (dict(rows=-1), "rows"),
                                     (dict(rows=1 << 31), "rows"), (dict(rows_per_gate=0), "rows_per_gate"), (dict(eps=0.0), "eps"),
                                     (dict(eps=float("nan")), "eps"), (dict(post=3), "norm kind"), (dict(gate_act=1), "activation"),
                                     (dict(dtype=L.TG_F32), "types"), (dict(dtype=2), "types"), (dict(ldx=63), "stride"),
                                     (dict(ldg=10), "stride"), (dict(ldh=0), "stride")])
def test_gated_norm_forward_refuses(kw, word):
    refused(L.lib().tg_gated_norm_forward(C.byref(norm_desc(**kw)), P, P, P, None, None, None, None, None, P, P, None), word)


def test_gated_norm_refuses_what_does_not_fit_together():
    f, b = L.lib().tg_gated_norm_forward, L.lib().tg_gated_norm_backward
    none = [None] * 5
    refused(f(C.byref(norm_desc()), P, None, None, *none, None, P, None), "post norm")
    refused(f(C.byref(norm_desc()), P, P, None, *none, None, P, None), "y goes with")
    refused(f(C.byref(norm_desc(pre=0)), P, P, None, *none, P, P, None), "h with a pre norm")
    refused(f(C.byref(norm_desc(post=0, pre=0)), P, None, None, *none, None, None, None), "nothing to do")
    refused(f(C.byref(norm_desc()), None, P, None, *none, P, P, None), "x is missing")
    refused(f(None, P, P, None, *none, P, P, None), "descriptor")
    tail = [None] * 5
    refused(b(C.byref(norm_desc()), P, P, P, P, None, *none, P, P, P, *tail, P, 1 << 20, None), "d_gate without a gate")
    refused(b(C.byref(norm_desc(pre=0)), P, P, P, P, None, *none, P, P, None, *tail, P, 1 << 20, None), "without a pre norm")
    refused(b(C.byref(norm_desc(post=0)), P, P, P, P, None, *none, P, P, None, P, None, None, None, None, P, 1 << 20, None), "without a post norm")
    refused(b(C.byref(norm_desc()), P, P, P, P, None, *none, P, P, None, *tail, P, 3, None), "workspace")
    refused(b(C.byref(norm_desc()), P, P, P, P, None, *none, P, P, None, *tail, C.c_void_p(4100), 1 << 20, None), "workspace")


def test_gated_norm_workspace_sizes():
    for rows, Cn, k in ((0, 1, 1), (1, 1, 1), (1, 16384, 1), (100000, 64, 7), (100000, 64, 50000), (77824, 64, 1 << 30), (8192, 2048, 1024)):
        n = K.gated_norm_ws(rows, Cn, k)
        # partial sums of at most 512 + (gate rows' rounding) workgroups, a gate row's pieces
        assert 0 <= n <= 5 * Cn * 1100 + (2 * 512 * 256 * 8 if k > 1 else 0) + 4 * Cn * 520, (rows, Cn, k, n)
    with pytest.raises(L.TecoHipError):
        K.gated_norm_ws(4, 0)


def test_fp8_refuses():
    q, m, lin = L.lib().tg_fp8_quantize, L.lib().tg_fp8_matmul, L.lib().tg_fp8_linear
    refused(q(P, 7, 4, 4, 4, 2, 0, P, P, None, None, None), "dtype")
    refused(q(P, 0, 4, 4, 4, 1, 0, P, P, None, None, None), "8-bit type")
    refused(q(P, 0, -4, 4, 4, 2, 0, P, P, None, None, None), "rows and cols")
    refused(q(P, 0, 4, 4, 3, 2, 0, P, P, None, None, None), "stride")
    refused(q(P, 0, 4, 4, 4, 2, 0, None, None, None, None, None), "neither")
    refused(q(P, 0, 4, 4, 4, 2, 0, P, None, None, None, None), "scales")
    refused(q(P, 0, 4, 4, 4, 2, 0, C.c_void_p(4104), P, None, None, None), "aligned")

    def desc(**kw):
        d = L.Fp8MatmulDesc()
        for n, v in {**dict(M=4, N=4, K=128, ldo=4, a_fmt=2, b_fmt=2, a_tile=0, b_tile=1, out_dtype=1, accumulate=0), **kw}.items():
            setattr(d, n, v)
        return d
    for kw, word in ((dict(K=64), "multiple of 128"), (dict(K=-128), "multiple of 128"), (dict(M=-1), "M and N"), (dict(a_fmt=0), "8-bit type"),
                     (dict(out_dtype=2), "output type"), (dict(accumulate=1), "f32"), (dict(ldo=3), "stride")):
        refused(m(C.byref(desc(**kw)), P, P, P, P, None, P, None), word)
    refused(m(C.byref(desc()), P, None, P, P, None, P, None), "null")
    refused(m(C.byref(desc()), C.c_void_p(4104), P, P, P, None, P, None), "aligned")
    refused(lin(P, 1, 4, 100, 100, P, P, 8, 2, None, P, 1, 8, P, 4, None), "workspace")
    refused(lin(P, 1, 4, 100, 99, P, P, 8, 2, None, P, 1, 8, P, 1 << 20, None), "stride")
    refused(lin(P, 1, 4, 100, 100, P, P, 8, 2, None, P, 1, 7, P, 1 << 20, None), "output")
    refused(lin(P, 1, 4, 0, 100, P, P, 8, 2, None, P, 1, 8, P, 1 << 20, None), "K in")


def test_gated_scan_refuses():
    f, b, z = L.lib().tg_gated_scan_forward, L.lib().tg_gated_scan_backward, L.lib().tg_gated_scan_sizes
    n, m = C.c_int64(0), C.c_int64(0)

    def desc(**kw):
        d = L.GatedScanDesc()
        for k in ("x_t", "g_t", "y_t", "dy_t", "dx_t", "dg_t"):
            setattr(d, k, 64)
        for k, v in {**dict(B=2, T=300, D=64, dtype=0), **kw}.items():
            setattr(d, k, v)
        return d
    refused(z(1, 0, 4, C.byref(n), C.byref(m)), "T >= 1")
    refused(z(1 << 20, 1, 4, C.byref(n), C.byref(m)), "2^20")
    big = 1 << 30
    for kw, word in ((dict(T=0), "T >= 1"), (dict(B=-1), "B >= 0"), (dict(dtype=2), "dtype"), (dict(x_t=63), "stride"), (dict(y_t=0), "stride")):
        refused(f(C.byref(desc(**kw)), P, P, None, None, None, None, P, None, P, big, 1, None), word)
    refused(f(C.byref(desc(T=1 << 20)), P, P, None, None, None, None, P, None, None, 0, 0, None), "carry")
    refused(f(C.byref(desc(T=3)), P, P, None, None, None, None, P, None, None, 0, 1, None), "carry")
    refused(f(C.byref(desc()), P, None, None, None, None, None, P, None, P, big, 1, None), "missing")
    refused(b(C.byref(desc()), P, P, None, None, None, P, None, None, big, P, P, None, None, P, big, None), "carry")
    refused(b(C.byref(desc(T=1 << 20)), P, P, None, None, None, P, None, P, big, P, P, None, None, P, 8, None), "workspace")
    refused(b(C.byref(desc()), P, P, None, None, None, P, None, P, big, P, P, None, P, P, big, None), "floor")
    refused(b(C.byref(desc(dx_t=1)), P, P, None, None, None, P, None, P, big, P, P, None, None, P, big, None), "stride")


def test_wrappers_refuse_cpu_tensors_and_bad_layouts():
    t = torch.zeros(4, 64)
    with pytest.raises(L.TecoHipError, match="not on the GPU"):
        K.gated_norm_forward(t, t, None, t, t)
    with pytest.raises(L.TecoHipError, match="not on the GPU"):
        K.fp8_quantize(t, *K.fp8_alloc(4, 64, "cpu"))
    with pytest.raises(L.TecoHipError, match="not on the GPU"):
        K.gated_scan_forward(t[None], t[None], t[None], None, None)
    rows = K._rows
    assert rows(t[:, :16], 4, 16, torch.float32, "t")[1] == 64 and rows(torch.zeros(2, 3, 8), 6, 8, torch.float32, "t")[1] == 8
    assert rows(torch.zeros(2, 1, 3, 16)[..., :8], 6, 8, torch.float32, "t")[1] == 16
    assert rows(torch.zeros(1, 8).expand(1, 8), 1, 8, torch.float32, "t")[1] == 8
    for bad, word in ((torch.zeros(4, 8, 2)[..., 0], "contiguous"), (torch.zeros(4, 3, 8)[:, :2], "no common stride"), (torch.zeros(1, 8).expand(8, 8), "overlap"),
                      (torch.zeros(4, 8).double(), "expected")):
        with pytest.raises(L.TecoHipError, match=word):
            rows(bad, 8 if bad.shape[-1] == 8 and bad.numel() == 64 else 4, 8, torch.float32, "t")
    with pytest.raises(L.TecoHipError, match="channels"):
        K._steps(torch.zeros(2, 8, 4).transpose(1, 2), (2, 4, 8), torch.float32, "t")
    assert K._steps(torch.zeros(2, 1, 8).expand(2, 1, 8), (2, 1, 8), torch.float32, "t")[1:] == (8, 8)
    with pytest.raises(L.TecoHipError, match="contiguous uint8|contiguous"):
        K._fp8_operand(torch.zeros(4, 128).to(torch.float8_e4m3fn), torch.zeros(4, 1, dtype=torch.uint8), "a")
    assert [tuple(v.shape) for v in K.fp8_alloc(130, 700, "cpu", tile=True, transposed=True)] == [(130, 768), (2, 8), (700, 256), (6, 4)]


def test_reference_rounds_as_torch_does():
    """The 64-bit reference's 8-bit grid against torch's own conversion, over every bf16 value in range."""
    v = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    for fmt, dt in (("e4m3", torch.float8_e4m3fn), ("e5m2", torch.float8_e5m2)):
        w = v[torch.isfinite(v) & (v.abs() <= R.LIMITS[fmt][0])]
        assert torch.equal(R.to8(w.double(), fmt), w.float().to(dt).double())
    top = torch.tensor([0.0, 1e-45, 448.0, 448.1, 449 * 2.0 ** -140, 3e38, 2.0 ** -126, 224.0, 224.0001], dtype=torch.float64)
    e = R.exponent(top, "e4m3")
    assert e.tolist() == [0, -126, 0, 1, -126, 120, -126, -1, 0]


def test_reference_gradients_are_those_of_differences():
    g = torch.Generator().manual_seed(0)

    def rn(*s):
        return torch.randn(*s, generator=g, dtype=torch.float64, requires_grad=True)
    x, o, gate, w = rn(5, 6), rn(5, 6), rn(3, 6), rn(6)
    for post, pre, act in (("rms", "layer", "silu"), ("layer", "rms", "tanh"), ("none", "rms", "sigmoid")):
        assert torch.autograd.gradcheck(lambda *t: R.norm_forward(t[0], t[1], t[2], dict(w_post=t[3], b_post=None, scale=t[3], w_pre=t[3], b_pre=None),
                                                                  post, pre, act, 2, 0.5, 1e-3), (x, o, gate, w))
    xs, gs, h0, low = rn(2, 5, 3), rn(2, 5, 3), rn(2, 3), torch.rand(3, dtype=torch.float64, generator=g).mul(0.8).requires_grad_()
    ends, fresh = torch.tensor([5, 3]), torch.tensor([[0, 0, 1, 0, 0], [0, 1, 0, 0, 1]]) != 0
    assert torch.autograd.gradcheck(lambda *t: R.scan_forward(*t, ends, fresh), (xs, gs, h0, low))
