"""The GPU tests of products by expert reach every tile that a call can take: the launches' rule over their sizes on a chip of 256 CUs, so that a new time or tile in the rule
cannot leave one without a test."""
import grouped_probe
import test_gpu_expert_tiles as T


def test_every_tile_has_a_test_for_every_kind_of_operands():
    for kind, tiles in T.KINDS.items():
        assert set(tiles) == (set(range(grouped_probe.tiles())) if kind != "packed f32" else {2, 3, 4})
        for tile, sizes in tiles.items():
            assert [grouped_probe.tile(kind, *s) for s in sizes] == [tile] * len(sizes), (kind, tile)


def test_the_sizes_are_whole_and_ragged():
    for kind, tiles in T.KINDS.items():
        piece = 16 if kind.startswith("packed") else 8
        for sizes in tiles.values():
            assert all(d % piece == 0 for _, _, _, d in sizes)          # (the tiles' operands lie on 16 bytes)
            assert any(f % 128 for _, _, f, _ in sizes) and any(f % 256 == 0 for _, _, f, _ in sizes)
            assert any(e > 2 and T.counts_of(r, e)[0][1] == 0 and T.counts_of(r, e)[1] for r, e, _, _ in sizes)


def test_wide_results_have_no_other_tiles():
    for rows in (1, 7, 64, 1000, 4000, 16000):
        for experts in (1, 8, 64):
            for features in (8, 256, 2816, 8192):
                for model in (16, 512, 4096, 14336):
                    assert grouped_probe.tile("packed f32", rows, experts, features, model) in (2, 3, 4)
