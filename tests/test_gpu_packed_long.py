"""RMS norms and packing of so many rows that workgroups go round: every kernel of the forward pass, rows shared out unevenly, and grids at their limit."""
import pytest
import torch

import packed_oracle as P
from test_gpu_ffn import DEV, TYPES, randn, stream
from test_gpu_packed import test_rms_backward as rms_backward, test_rms_forward as rms_forward
from zluda_amd import ffn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,cols", [(20011, 200), (9001, 1000), (5003, 2048), (3001, 4096), (1501, 8192), (8201, 4104), (1100, 16384)])
def test_forward(rows, cols):
    for typ in ("bf16", "f32"):
        rms_forward(typ, rows, cols)


@pytest.mark.parametrize("rows,cols", [(20011, 200), (2049, 512), (1791, 512), (1793, 512), (897, 1000), (3001, 4096), (1501, 8192)])
def test_backward(rows, cols):
    """around the row counts from which a workgroup takes a second round"""
    rms_backward("bf16", rows, cols)


@pytest.mark.parametrize("block_rows", [1, 128])
def test_more_rows_than_a_grid_has(block_rows):
    rows, cols = (300000, 40) if block_rows == 1 else (128 * 65540 + 5, 16)
    x = randn(1, rows, cols).to(torch.bfloat16)
    codes, scales = ffn.packed_buffers(rows, cols, DEV, block_rows)
    spec = dict(type=TYPES["bf16"][1], rows=rows, cols=cols, block_rows=block_rows)
    ffn.Activate(dict(spec, activation=ffn.COPY)).run(gate=x.data_ptr(), codes=codes.data_ptr(), scales=scales.data_ptr(), stream=stream())
    back = torch.empty_like(x)
    ffn.Unpack(spec).run(codes=codes.data_ptr(), scales=scales.data_ptr(), y=back.data_ptr(), stream=stream())
    torch.cuda.synchronize()
    rest = [slice(0, 1024), slice(rows - 256 - rows % 128, rows)]
    for r in rest:                                           # (whole blocks of 128 rows, whose scales are of all of them)
        value = x[r].double()
        s = scales[:, r].t() if block_rows == 1 else scales[r.start // 128:-(-r.stop // 128), :1]          # (the rest of a pitch of four is nobody's)
        P.check_packed(codes[r], s, value, torch.zeros_like(value), cols, block_rows)
    # each code is off by half a step at most: 2^-4 of its value, or of the smallest normal number 2^-6 times the scale; and what it stands for, at most that much larger
    # than the value, is rounded to y's type: 2^-8 of it
    scale = scales.t().repeat_interleave(128, 1)[:, :cols] if block_rows == 1 else scales[:, :1].repeat_interleave(128, 0)[:rows]
    step = 2.0 ** -4 * torch.maximum(x.float().abs(), 2.0 ** -6 * scale)
    assert ((back.float() - x.float()).abs() <= (step + 2.0 ** -8 * (x.float().abs() + step)) * 1.0001).all()
