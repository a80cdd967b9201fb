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
