"""What the gated feed-forward kernels' comments promise about the compiler's output and about their DMA counts, without a GPU:
the persistent kernel's instantiations obey the rules of test_w4_codegen.py, the tiles hold no spills, and every counted wait of the
tiles' ring lets a stage be read only after its instructions have retired."""
import os
import re

import pytest

import test_w4_codegen as w4

CSRC = os.path.join(w4.ROOT, "zluda_amd", "csrc")
FLAGS = {unit: ["-mllvm", "-amdgpu-mfma-vgpr-form=1"] for unit in ("ffn_small_bf16.hip", "ffn_products.hip")}


@pytest.mark.parametrize("unit", ["ffn_gated_bf16.hip", "ffn_gated_f16.hip"])
def test_persistent_kernel(unit, monkeypatch):
    text = w4.assembly(unit)
    monkeypatch.setattr(w4, "assembly", lambda _: text)
    w4.test_nothing_reads_an_accumulator_too_soon_after_an_mfma(unit)
    seen = []
    for m in re.finditer(r"^(_ZN9zluda_amd19gemm_mfma_w4_kernel\w+):\s*;.*?\n(.*?)^\s*s_endpgm", text, re.S | re.M):
        hot = w4.loop_body(m.group(2), m.group(1))
        seen.append((hot.count("v_mfma"), hot.count("ds_read_b128"), hot.count("buffer_load_dwordx4")))
        for bad in ("scratch_", "v_accvgpr_", "v_readlane", "v_writelane"):
            assert bad not in hot, "%s: %s inside the K loop" % (m.group(1), bad)
        assert hot.count("s_barrier") == 2 and hot.count("s_waitcnt vmcnt") == 2, m.group(1)
    # two stages of 128 x 128 and of 128 x 96 wave tiles: MFMAs, fragments, DMA instructions
    assert sorted(seen) == [(192, 56, 28), (256, 64, 32)]


def tiles():
    text = open(os.path.join(CSRC, "ffn_launch.hpp")).read()
    table = re.search(r"kGatedTiles\[\] = \{(.*?)\};", text, re.S).group(1)
    rows = [tuple(float(v.rstrip("f")) for v in r.split(",")) for r in re.findall(r"\{([^{}]*)\}", table)]
    first = int(re.search(r"kGatedPersistent = (\d+)", text).group(1))
    assert len(rows) == int(re.search(r"kGatedTileCount = (\d+)", text).group(1))
    return [tuple(int(v) for v in r[:5]) for r in rows[:first]]


@pytest.mark.parametrize("features,tokens,wp,wq,ring", tiles())
def test_a_stage_is_read_only_after_it_has_landed(features, tokens, wp, wq, ring):
    """replays a wave's issue order: all of a ring's stages, then a wait and the reads of the next stage in front of each refill;
    loads retire in order, so a wait for at most n outstanding has everything but the youngest n"""
    loads = (2 * features + tokens) // (8 * wp * wq)
    for stages in (1, 2, 3, 4, 5, 6, 7, 16, 17):
        issued = [s for s in range(min(ring, stages)) for _ in range(loads)]

        def landed(younger):
            """the wait of wait_for(younger): at most that many stages' instructions outstanding"""
            n = (ring - 1 if younger >= ring - 1 else ring - 2 if younger == ring - 2 else 1 if ring > 3 and younger == 1 else 0) * loads
            return issued[:len(issued) - n] if n else issued

        assert landed(stages - 1).count(0) == loads                         # the prologue's wait
        for kt in range(stages):
            done = landed(ring - 2 if kt + ring < stages else min(stages - kt, ring) - 2)
            if kt + 1 < stages:
                assert done.count(kt + 1) == loads                          # read behind this barrier
            if kt + ring < stages:
                issued += [kt + ring] * loads                               # into the slot of stage kt, whose fragments are in registers
        assert issued == [s for s in range(stages) for _ in range(loads)]
    assert (ring - 1) * loads < 64 and ring * (2 * features + tokens) * 128 <= 160 * 1024


def test_tiles_hold_no_spills(tmp_path):
    import subprocess
    out = str(tmp_path / "k.s")
    cmd = [w4.HIPCC, "--offload-arch=gfx950", "-O3", "-std=c++17", "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops", *FLAGS["ffn_small_bf16.hip"],
           "--cuda-device-only", "-S", os.path.join(CSRC, "ffn_small_bf16.hip"), "-o", out]
    res = subprocess.run(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    assert res.returncode == 0, res.stdout[-2000:]
    text = open(out).read()
    found = re.findall(r"\.name:\s+(\S*gated_(?:tile|any)_kernel\S*).*?\.vgpr_spill_count:\s+(\d+)", text, re.S)
    assert len(found) == len(tiles()) + 1 and all(n == "0" for _, n in found), found
    assert "scratch_" not in text and "v_pk_fma_f32" not in text and "v_pk_mul_f32" not in text and "v_pk_add_f32" not in text


def test_grad_products_stages(tmp_path):
    """two stages of the loops of dX and dW: 32 MFMAs and 8 DMA instructions each, one barrier with a wait for everything; registers and LDS of two
    workgroups a CU"""
    import subprocess
    out = str(tmp_path / "k.s")
    cmd = [w4.HIPCC, "--offload-arch=gfx950", "-O3", "-std=c++17", "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops", *FLAGS["ffn_products.hip"],
           "--cuda-device-only", "-S", os.path.join(CSRC, "ffn_products.hip"), "-o", out]
    res = subprocess.run(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    assert res.returncode == 0, res.stdout[-2000:]
    text = open(out).read()
    assert "scratch_" not in text and "v_accvgpr_" not in text and "v_pk_" not in re.sub(r"v_pk_(mov|lshl|or|and)", "", text)
    meta = re.findall(r"\.group_segment_fixed_size: (\d+).*?\.name:\s+\S*grad_products_kernel\S*.*?\.vgpr_count:\s+(\d+)", text, re.S)
    assert len(meta) == 2 and all(int(lds) * 2 <= 160 * 1024 and int(regs) <= 256 for lds, regs in meta), meta
    for m in re.finditer(r"^(_ZN9zluda_amd20grad_products_kernel\w+):\s*;.*?\n(.*?)^\.Lfunc_end", text, re.S | re.M):
        blocks = re.split(r"^\.LBB\d+_\d+:", m.group(2), flags=re.M)
        loops = [b for b in blocks if b.count("v_mfma") == 64]
        assert len(loops) == 2, m.group(1)
        for b in loops:
            assert len(re.findall(r"buffer_load_dwordx4.* lds", b)) == 16 and b.count("s_barrier") == 2 and b.count("s_waitcnt vmcnt(0)") == 2
        assert sorted((b.count("ds_read_b64_tr_b16"), b.count("ds_read_b128")) for b in loops) == [(32, 16), (64, 0)]
