"""The GPU tests of the feed-forward operators reach every kernel that a call can take: the launches' rules replayed over the tests' sizes on a chip of 256
CUs, so that a new time or tile in the rules cannot leave one of them without a test."""
import ffn_probe
import test_gpu_ffn
import test_gpu_ffn_large_tiles
import test_gpu_ffn_persistent
import test_gpu_ffn_products
from ffn_probe import gated_tile, grad_splits, tile_shape
from planner_probe import planned
from zluda_amd import abi as K


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


def test_the_launch_of_both_products_has_tests_of_its_loops():
    """stages of dW's K, shares of dX's K and stages of a share, tiles of tokens"""
    chosen = {s: grad_splits(*s) for s in test_gpu_ffn_products.SIZES}
    assert all(n > 0 for n, _ in chosen.values())
    assert {n for n, _ in chosen.values()} >= {1, 2, 3, 4, 5, 6, 10, 13, 16}
    assert {-(-t // 64) for t, _, _ in chosen} >= {3, 4, 5, 6, 7, 8, 10, 11, 16} and any(t % 64 == 1 for t, _, _ in chosen)
    assert {-(-t // 128) for (t, _, _), (n, _) in chosen.items() if n > 1} >= {2, 3, 4, 5, 8}
    # a last share that is shorter than the others, one of a single stage less, shares of 4 stages and of many
    stages = {s: -(-2 * s[2] // 64) for s in chosen}
    assert any(n > 1 and stages[s] % each for s, (n, each) in chosen.items()) and {each for _, each in chosen.values()} >= {4, 5, 6, 7, 8, 9, 16}
    for pad in (0, 8):
        for x_kept in (False, True):
            for s in chosen:
                for dz_ld in (None, 2 * s[2] + pad):
                    assert grad_splits(*s, pad=pad, skip=pad, dz_ld=dz_ld, x_kept=x_kept) == chosen[s]


def test_the_largest_tiles_have_tests_and_are_planned(api):
    """dx: A:N B:N, model x tokens, K 2 features; dw: A:N B:T, model x 2 features, K tokens"""
    for which, t, d, f, _ in test_gpu_ffn_large_tiles.CASES:
        m, n, k, tb = (d, t, 2 * f, 0) if which == "dx" else (d, 2 * f, t, 1)
        assert ffn_probe.load().probe_grad_largest_tiles(m, n, 256)
        status, _, plan, _ = planned(api, m, n, k, ta=0, tb=tb, workspace=16 << 20, family=K.ZLUDA_KERNEL_MFMA_TR16, variant=3)
        assert status == 0 and (plan.kernel, plan.variant) == (K.ZLUDA_KERNEL_MFMA_TR16, 3)
    assert not ffn_probe.load().probe_grad_largest_tiles(4096, 31 * 256, 256) and ffn_probe.load().probe_grad_largest_tiles(4096, 31 * 256 + 1, 256)
