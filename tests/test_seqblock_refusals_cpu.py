"""Calls of the sequence-block operators that are refused before anything is launched (no GPU: a launch would report another error)."""
import ctypes as C

from tecogan_amd import _lib as L
from test_seqblock_cpu import P, refused


def test_fp8_linear_refuses_too_many_tiles_before_it_quantises():
    M, N, K = 1 << 21, 1 << 19, 128
    refused(L.lib().tg_fp8_linear(P, 1, M, K, K, P, P, N, 2, None, P, 1, N, P, 1 << 40, None), "too many output tiles")


def test_fp8_matmul_refuses_fast_sums_of_f32_outputs():
    d = L.Fp8MatmulDesc(M=64, N=64, K=128, ldo=64, a_fmt=2, b_fmt=2, a_tile=0, b_tile=1, out_dtype=L.TG_F32, accumulate=0, fast=1)
    refused(L.lib().tg_fp8_matmul(C.byref(d), P, P, P, P, None, P, None), "fast sums")


def test_gated_scan_refuses_outputs_whose_batch_rows_overlap():
    B, T, D, big = 3, 40, 64, 1 << 30

    def desc(**kw):
        d = L.GatedScanDesc(B=B, T=T, D=D, dtype=0)
        for n in ("x", "g", "y", "dy", "dx", "dg"):
            setattr(d, n + "_t", D)
            setattr(d, n + "_b", T * D)
        for n, v in kw.items():
            setattr(d, n, v)
        return C.byref(d)

    def forward(d):
        return L.lib().tg_gated_scan_forward(d, P, P, None, None, None, None, P, None, P, big, 1, None)

    def backward(d):
        return L.lib().tg_gated_scan_backward(d, P, P, None, None, None, P, None, P, big, P, P, None, None, P, big, None)
    for bad in (0, D - 1, D, (T - 1) * D + D - 1):
        refused(forward(desc(y_b=bad)), "overlap")
        refused(backward(desc(dx_b=bad)), "overlap")
        refused(backward(desc(dg_b=bad)), "overlap")
    refused(forward(desc(y_t=(B - 1) * D + D - 1, y_b=D)), "overlap")
