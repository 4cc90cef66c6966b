"""One row as wide as the entry points take it."""
import torch

import ffn_probe
import pytest
from test_gpu_ffn import DEV, stream
from zluda_amd import abi, ffn

pytestmark = pytest.mark.gpu


def test_checkpoint_of_the_widest_row(gpu_api):
    cols = ffn_probe.load().probe_max_side()
    # 1 .. 15: four significant bits, and a block of 32 holds a 15 and is scaled by 2^-4: what comes back is what went in
    x = (torch.arange(15 << 20, device=DEV) % 15 + 1).to(torch.bfloat16).repeat(-(-cols // (15 << 20)))[:cols]
    codes, scales = ffn.checkpoint_buffers(1, cols, DEV)
    back = torch.full((cols + 64,), -1.0, dtype=torch.bfloat16, device=DEV)
    c = ffn.Checkpoint(dict(type=abi.CUDA_R_16BF, rows=1, cols=cols))
    c.store(x=x.data_ptr(), codes=codes.data_ptr(), scales=scales.data_ptr(), stream=stream())
    c.load(codes=codes.data_ptr(), scales=scales.data_ptr(), x=back.data_ptr(), stream=stream())
    torch.cuda.synchronize()
    assert (scales == 127 - 4).all()        # 15 <= 448 * 2^-4, not 2^-5
    for a in range(0, cols, 1 << 28):
        b = min(cols, a + (1 << 28))
        assert torch.equal(back[a:b], x[a:b]), a
    assert (back[cols:] == -1.0).all()
