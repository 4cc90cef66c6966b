"""Products by expert on every tile there is (test_expert_tile_choices.py has which sizes take which): random values element by element and by norms, whole numbers bit for bit;
ragged counts, experts without rows, rows without an expert, features and widths that are no multiples of a tile and some that are, a single stage of K and more."""
import pytest
import torch

import ffn_oracle as O
import packed_norms as N
import packed_oracle as P
import test_gpu_grouped as T
from test_gpu_ffn import DEV, Mat
from test_gpu_grouped import check_forward, run_forward, run_packed

pytestmark = pytest.mark.gpu

# tile: rows, experts, features, model
H16 = {0: [(5418, 6, 1504, 288), (5492, 2, 1536, 256), (5353, 6, 1480, 8)], 1: [(2985, 5, 2008, 272), (3427, 2, 1792, 256), (5274, 5, 1088, 8)],
       2: [(2106, 6, 208, 392), (2604, 2, 256, 256), (2277, 6, 256, 8)], 3: [(98, 5, 184, 496), (174, 2, 256, 320), (387, 9, 168, 8)],
       4: [(4251, 9, 208, 336), (2065, 2, 512, 256), (3688, 6, 264, 8)], 5: [(4569, 5, 728, 784), (3108, 1, 1024, 832)], 6: [(5696, 12, 336, 272), (4227, 2, 512, 320)]}
PACKED = {0: [(5500, 6, 1880, 528), (5074, 2, 2048, 512), (5819, 5, 1784, 16)], 1: [(5279, 5, 1032, 624), (4873, 2, 1280, 512), (4287, 6, 1328, 16)],
          2: [(1658, 5, 288, 688), (2123, 2, 256, 512), (1292, 6, 344, 16)], 3: [(365, 5, 200, 992), (363, 1, 256, 640), (756, 6, 176, 16)],
          4: [(4066, 9, 200, 656), (4208, 3, 256, 512), (4446, 5, 224, 16)], 5: [(4160, 5, 696, 6096), (6173, 2, 512, 6144)], 6: [(5533, 5, 344, 752), (2761, 2, 768, 768)]}
PACKED_F32 = {2: [(2060, 5, 216, 736), (2393, 3, 256, 512), (4092, 6, 168, 16)], 3: [(731, 6, 224, 544), (140, 1, 512, 512), (148, 6, 184, 32)],
              4: [(3257, 6, 288, 576), (4068, 3, 256, 512), (4006, 9, 224, 16)]}
KINDS = {"bf16": H16, "f16": H16, "packed bf16": PACKED, "packed f16": PACKED, "packed f32": PACKED_F32}
CASES = [(kind, tile, *size) for kind, tiles in KINDS.items() for tile, sizes in tiles.items() for size in sizes]


def counts_of(rows, experts):
    """uneven shares, an expert without rows and one with a single one where there are more than two; rows behind the last expert's"""
    spare = rows // 40 if experts > 2 else 0
    weight = [0 if experts > 2 and e == 1 else 2 + (5 * e) % 7 for e in range(experts)]
    counts = [(rows - spare) * w // sum(weight) for w in weight]
    if experts > 2:
        counts[-1] = 1
    counts[0] += rows - spare - sum(counts)
    return counts, spare


def run(kind, rows, experts, features, model):
    counts, spare = counts_of(rows, experts)
    assert sum(counts) + spare == rows and min(counts) >= 0
    print(kind, rows, experts, features, model, counts, flush=True)
    if kind.startswith("packed"):
        run_packed(kind.split()[1], counts, spare, features, model)
    else:
        check_forward(*run_forward(kind, counts, spare, features, model), features, kind)


def whole(seed, k, *shape):
    """-1, 0 and 1, of which about eight products of a sum over k are none of zeros"""
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    pick, some = torch.rand(shape, device=DEV, generator=gen), 0.5 * min(1.0, (8 / k) ** 0.5)
    return (pick < some).float() - (pick >= 1 - some).float()


def whole_pack(rows, cols, block_rows, seed, std=1.0, pad=0, skip=0, experts=1):
    """as test_gpu_grouped.pack(): codes of such numbers, scales 1, 2 and 4"""
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed + 77)
    codes = Mat(rows, cols, torch.uint8, -(-cols // 16) * 16, 0, whole(seed, cols, rows, cols).to(torch.float8_e4m3fn).view(torch.uint8))
    f = rows // experts
    lines, width = (P.blocks(cols), rows) if block_rows == 1 else (experts * P.blocks(f), P.blocks(cols))
    values = torch.randint(0, 3, (lines, width), device=DEV, generator=gen).exp2()
    scales = Mat(lines, width, torch.float32, None, 0, values)
    v = values.double()
    spread = P.spread(v.t(), rows, cols) if block_rows == 1 else torch.cat([P.spread(v[e * P.blocks(f):(e + 1) * P.blocks(f)], f, cols, 128) for e in range(experts)])
    return codes, scales, spread


@pytest.mark.parametrize("kind,tile,rows,experts,features,model", CASES)
def test_random_values(gpu_api, monkeypatch, kind, tile, rows, experts, features, model):
    monkeypatch.setattr(T.O, "check", N.both_checks(O.check))
    run(kind, rows, experts, features, model)


@pytest.mark.parametrize("kind,tile,rows,experts,features,model", CASES)
def test_whole_numbers(gpu_api, monkeypatch, kind, tile, rows, experts, features, model):
    monkeypatch.setattr(T.O, "check", N.exact_check)
    monkeypatch.setattr(T, "randn", lambda seed, *shape, std=1.0: whole(seed, shape[-1], *shape))
    monkeypatch.setattr(T, "pack", whole_pack)
    run(kind, rows, experts, features, model)
