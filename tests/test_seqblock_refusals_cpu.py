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
