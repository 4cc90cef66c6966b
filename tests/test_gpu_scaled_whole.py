"""cublasLtMatmul with a scale for each 128 of K on every tile: whole numbers with scales of powers of two bit for bit, the norms of random products' errors, and operands of
E5M2 as either side of the tile."""
import pytest
import torch

import ffn_oracle as O
import packed_norms as N
import packed_oracle as P
import test_gpu_scaled_matmul as T
from test_gpu_ffn import DEV
from test_gpu_scaled_matmul import BLK, F8, VEC, run
from zluda_amd import abi as K

pytestmark = pytest.mark.gpu
TILES = [0, 1, 2, 3, 4, 5, 6]
WIDE_D = (2, 3, 4)                     # those with results in 32 bits
PAIRS = [(BLK, VEC), (BLK, BLK), (VEC, VEC), (VEC, BLK)]


def forced(variant):
    return dict(kernel=K.ZLUDA_KERNEL_MFMA_BLK8, variant=variant)


def modes_of(variant, row_major=False):
    """pairs of modes that the variant takes: the first one's P rows (D's unit stride) share their scales"""
    return [m for m in PAIRS if variant != 0 or m[1 if row_major else 0] == BLK]


class Whole(T.Operand):
    """codes -1, 0 and 1, of which about eight products of a sum are none of zeros; scales 1, 2 and 4: sums have a standard deviation of 16 sqrt(8) = 45 at most, the 256 up to
    which bf16 has all whole numbers is 5.7 of these"""

    def __init__(self, rows, k, typ, mode, seed, kc=True, pad=0, skip=0, batch=1):
        super().__init__(rows, k, typ, mode, seed, kc, pad, skip, batch)
        gen = torch.Generator(device=DEV)
        gen.manual_seed(seed + 77)
        pick, some = torch.rand((batch, rows, k), device=DEV, generator=gen), 0.5 * min(1.0, (8 / k) ** 0.5)
        self.codes = (pick < some).double() - (pick >= 1 - some).double()
        v = self.codes.float().to(F8[typ][0])
        for b in range(batch):
            at = 256 + skip + b * self.stride
            self.raw[at:at + rows * self.ld].view(rows, self.ld)[:, :k].copy_(v[b].view(torch.uint8))
        self.scales.copy_(torch.randint(0, 3, self.scales.shape, device=DEV, generator=gen).exp2())
        s = self.scales.double()
        if mode == VEC:
            s = s.transpose(1, 2).repeat_interleave(128, 2)
        else:
            s = s[:, :, :P.blocks(k)].repeat_interleave(128, 1)[:, :rows].repeat_interleave(128, 2)
        self.spread = s[:, :, :k]


@pytest.fixture
def whole(monkeypatch):
    monkeypatch.setattr(T, "Operand", Whole)
    monkeypatch.setattr(T.O, "check", N.exact_check)


@pytest.fixture
def norms(monkeypatch):
    monkeypatch.setattr(T.O, "check", N.both_checks(O.check))


@pytest.mark.parametrize("variant", TILES)
@pytest.mark.parametrize("k", [16, 128, 400, 640, 1040])
def test_whole_numbers(gpu_api, whole, variant, k):
    for m, n in ((256, 256), (300, 290), (520, 70), (130, 40)):
        for a_mode, b_mode in modes_of(variant):
            assert run(gpu_api, m, n, k, a_mode, b_mode, **forced(variant)) == (K.ZLUDA_KERNEL_MFMA_BLK8, variant)
        run(gpu_api, m, n, k, out="f16", workspace=0, pad=16, **forced(variant))
        for a_mode, b_mode in modes_of(variant, True):
            run(gpu_api, m, n, k, a_mode, b_mode, row_major=True, batch=2, **forced(variant))
        if variant in WIDE_D:
            run(gpu_api, m, n, k, VEC, VEC, out="f32", **forced(variant))


@pytest.mark.parametrize("variant", TILES)
@pytest.mark.parametrize("a,b", [("e4m3", "e5m2"), ("e5m2", "e4m3")])
def test_whole_numbers_of_two_formats(gpu_api, whole, variant, a, b):
    for m, n, k in ((256, 256, 512), (300, 290, 400)):
        for row_major in (False, True):
            for a_mode, b_mode in modes_of(variant, row_major):
                run(gpu_api, m, n, k, a_mode, b_mode, a=a, b=b, row_major=row_major, **forced(variant))
            run(gpu_api, m, n, k, BLK, BLK, a=a, b=b, row_major=row_major, out="f16", **forced(variant))


@pytest.mark.parametrize("variant", TILES)
@pytest.mark.parametrize("a,b", [("e4m3", "e5m2"), ("e5m2", "e4m3")])
def test_formats(gpu_api, variant, a, b):
    """E5M2 as P and as Q, whole tiles and ragged ones, shared out along K and not"""
    for m, n, k in ((256, 256, 512), (300, 290, 400), (520, 97, 2000)):
        for row_major in (False, True):
            for a_mode, b_mode in modes_of(variant, row_major):
                assert run(gpu_api, m, n, k, a_mode, b_mode, a=a, b=b, row_major=row_major, **forced(variant)) == (K.ZLUDA_KERNEL_MFMA_BLK8, variant)
            run(gpu_api, m, n, k, BLK, BLK, a=a, b=b, row_major=row_major, out="f16", workspace=0, alpha=2.0 ** -8, bias=1, **forced(variant))
            if variant in WIDE_D:
                for a_mode, b_mode in ((BLK, BLK), (VEC, VEC)):
                    run(gpu_api, m, n, k, a_mode, b_mode, a=a, b=b, row_major=row_major, out="f32", **forced(variant))


@pytest.mark.parametrize("variant", TILES)
@pytest.mark.parametrize("m,n,k", [(520, 390, 2048), (1000, 300, 4112), (256, 256, 14336)])
def test_norms(gpu_api, norms, variant, m, n, k):
    for a_mode, b_mode in modes_of(variant):
        run(gpu_api, m, n, k, a_mode, b_mode, out="f16", alpha=2.0 ** -8, **forced(variant))
    run(gpu_api, m, n, k, workspace=0, **forced(variant))
    run(gpu_api, m, n, k, BLK, BLK, a="e5m2", out="f16", alpha=2.0 ** -10, **forced(variant))
    if variant in WIDE_D:
        run(gpu_api, m, n, k, VEC, VEC, out="f32", **forced(variant))


@pytest.mark.parametrize("m,n,k", [(5632, 333, 2000), (4096, 1000, 1024), (2048, 2048, 2048), (8192, 16, 4096)])
def test_norms_of_what_is_chosen(gpu_api, norms, m, n, k):
    for a_mode in (BLK, VEC):
        run(gpu_api, m, n, k, a_mode, VEC, out="f16", alpha=2.0 ** -8)
        run(gpu_api, m, n, k, a_mode, VEC, out="f32")
