"""The GPU tests of the feed-forward operators reach every kernel that a call can take: the launches' rules replayed over the tests' sizes on a chip of 256
CUs, so that a new time or tile in the rules cannot leave one of them without a test."""
import test_gpu_ffn
import test_gpu_ffn_persistent
from ffn_probe import gated_tile, tile_shape


def sizes(test, names="t,d,f"):
    """what a test is parametrised with"""
    return next(m.args[1] for m in test.pytestmark if m.name == "parametrize" and m.args[0] == names)


def test_every_tile_of_the_gated_products_has_a_test():
    tests = [test_gpu_ffn.test_gated_forward_sizes, test_gpu_ffn.test_gated_forward_tiles, test_gpu_ffn.test_gated_forward_many_tiles, test_gpu_ffn.test_gated_forward_many_narrow_tiles,
             test_gpu_ffn_persistent.test_wide_tiles]
    reached = {gated_tile(t, d, f) for test in tests for t, d, f in sizes(test)}
    count = 0
    while tile_shape(count)[0]:
        count += 1
    assert count == 6 and reached == set(range(-1, count))
    assert {gated_tile(*s) for s in sizes(test_gpu_ffn.test_gated_forward_many_narrow_tiles)} == {4}
    assert {gated_tile(*s) for s in test_gpu_ffn_persistent.SIZES} == {5}


def test_the_wide_tiles_sizes_cover_their_loops():
    """one tile a workgroup and several, one to six stages of K, last tiles that are not full"""
    f0, t0, persistent = tile_shape(5)
    assert persistent
    tiles = [-(-f // f0) * -(-t // t0) for t, _, f in test_gpu_ffn_persistent.SIZES]
    assert any(n <= 256 for n in tiles) and any(n > 512 for n in tiles) and any(256 < n < 512 for n in tiles)
    assert {-(-d // 64) for _, d, _ in test_gpu_ffn_persistent.SIZES} == {1, 2, 3, 4, 6}
    assert all(t % t0 for t, _, _ in test_gpu_ffn_persistent.SIZES) and any(f % f0 and f % 2 for _, _, f in test_gpu_ffn_persistent.SIZES)
