"""Tiles whose rows are no power of two: products with a scale for each 128 of K and products by expert on 128 x 96, against the definition in 64 bits."""
import pytest

from test_gpu_grouped import check_forward, run_forward, run_packed
from test_gpu_scaled_matmul import BLK, VEC, run
from zluda_amd import abi as K

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("k", [16, 128, 272, 512, 640, 784, 2048])
def test_forced(gpu_api, k):
    for m, n in ((256, 192), (130, 97), (300, 95), (520, 1), (128, 300)):
        for modes in ((BLK, VEC), (BLK, BLK), (VEC, VEC), (VEC, BLK)):
            assert run(gpu_api, m, n, k, *modes, kernel=K.ZLUDA_KERNEL_MFMA_BLK8, variant=6) == (K.ZLUDA_KERNEL_MFMA_BLK8, 6)
        run(gpu_api, m, n, k, row_major=True, out="f16", act="gelu", bias=1, kernel=K.ZLUDA_KERNEL_MFMA_BLK8, variant=6)
        run(gpu_api, m, n, k, beta=0.5, out="f16", kernel=K.ZLUDA_KERNEL_MFMA_BLK8, variant=6, workspace=0)


@pytest.mark.parametrize("counts,spare", [([300, 96, 97, 0, 191, 500], 3), ([96] * 10, 0), ([1001], 40)])
def test_by_expert(counts, spare):
    """sizes whose row tiles are around multiples of 96"""
    for f, d in ((2816, 1024), (640, 520)):
        check_forward(*run_forward("f16", counts, spare, f, d), f, "%dx%d" % (f, d))
        run_packed("bf16", counts, spare, f, d)
