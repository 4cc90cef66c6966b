"""cublasLtMatmul with a scale for each 128 of K, few tokens: the kernel that shares K out over a workgroup's waves, against the definition in 64 bits."""
import pytest

from test_gpu_scaled_matmul import BLK, VEC, run
from zluda_amd import abi as K

pytestmark = pytest.mark.gpu
FORCED = dict(kernel=K.ZLUDA_KERNEL_MFMA_BLK8, variant=7)


@pytest.mark.parametrize("k", [16, 112, 128, 272, 1024, 1040, 4096, 4112, 5200, 14336])
def test_lengths(gpu_api, k):
    """blocks of K around multiples of the waves and of what each has in flight"""
    for m, n in ((16, 1), (130, 3), (300, 16), (72, 17), (264, 32), (40, 33), (128, 70)):
        for modes in ((BLK, VEC), (BLK, BLK), (VEC, VEC), (VEC, BLK)):
            assert run(gpu_api, m, n, k, *modes, **FORCED) == (K.ZLUDA_KERNEL_MFMA_BLK8, 7)
        run(gpu_api, m, n, k, out="f32", **FORCED)
        run(gpu_api, m, n, k, VEC, VEC, out="f16", act="gelu", bias=1, pad=16, workspace=0, **FORCED)


@pytest.mark.parametrize("a,b", [("e4m3", "e4m3"), ("e4m3", "e5m2"), ("e5m2", "e4m3"), ("e5m2", "e5m2")])
@pytest.mark.parametrize("out", ["bf16", "f16", "f32"])
def test_types_and_epilogues(gpu_api, a, b, out):
    for m, n, k in ((136, 1, 272), (40, 30, 2064)):
        run(gpu_api, m, n, k, a=a, b=b, out=out, **FORCED)
        run(gpu_api, m, n, k, VEC, BLK, a=a, b=b, out=out, act="relu", bias=1, beta=0.5, alpha=-1.5, **FORCED)
        run(gpu_api, n, m, k, BLK, VEC, a=a, b=b, out=out, row_major=True, bias=1, **FORCED)
    run(gpu_api, 40, 9, 528, a=a, b=b, out=out, batch=3, **FORCED)


@pytest.mark.parametrize("m,n,k", [(1, 1, 16), (4096, 1, 14336), (2048, 1, 2048), (14336, 16, 4096), (1000, 32, 1008), (100, 5, 32768)])
def test_chosen(gpu_api, m, n, k):
    """whichever kernel the rule takes"""
    for modes in ((BLK, VEC), (VEC, VEC)):
        for out in ("bf16", "f32"):
            run(gpu_api, m, n, k, *modes, out=out)
            run(gpu_api, m, n, k, *modes, out=out, workspace=0)
