"""Checks of whole results beside the element-wise bounds of packed_oracle.py, which allow the worst case of every sum and so hide what is wrong by a little everywhere.

norm_check    the error's 2-norm, and what of the error lies along the result (a factor that is off), against bounds of a random error:
  * rounding to the result's type is off by `unit` of a value at most, so by `unit` of the 2-norm, and by either sign: its part along the result is a sum of terms
    of at most unit v^2, 8 of whose standard deviations are 8 unit sqrt(sum v^4)
  * what the 8-bit instruction drops of eight neighbouring products: seven of them lose up to 2^-13 of the largest one's power of two each, spread over that
    range sqrt(7 / 3) 2^-13 of their 2-norm, 1.9e-4 (seen: 1.4e-5), and as much along the result
  * sums in 32 bits: 2^-24 of the terms, nothing beside these
exact_check   results that are whole numbers of no more bits than the type has, which every order of a sum in 32 bits gives bit for bit
"""
import torch

import ffn_oracle as O

DROPPED = 2e-4
WHOLE = {torch.bfloat16: 2 ** 8, torch.float16: 2 ** 11, torch.float32: 2 ** 24}      # whole numbers up to here are values of the type


def norm_check(got, ref, what="", dropped=DROPPED):
    v, g, unit = ref[0], got.double(), O.UNIT[got.dtype]
    n2 = v.square().sum().item()
    off = (g - v).norm().item() / n2 ** 0.5
    assert off <= unit + dropped, "%s: 2-norm of the error %.3g" % (what, off)
    along = abs(((g - v) * v).sum().item()) / n2
    allowed = 8 * unit * v.pow(4).sum().sqrt().item() / n2 + dropped
    assert along <= allowed, "%s: off by a factor of 1 %+.3g, %.3g allowed" % (what, along, allowed)


def exact_check(got, ref, what=""):
    v = ref[0]
    assert v.abs().max().item() <= WHOLE[got.dtype] and (v == v.round()).all(), what + ": no whole numbers of the type"
    wrong = (got.double() != v).sum().item()
    assert wrong == 0, "%s: %d of %d elements" % (what, wrong, v.numel())


def both_checks(check):
    """`check` (element by element), and the norms of what has enough elements for them"""
    def run(got, ref, what=""):
        check(got, ref, what)
        if got.numel() >= 4096:
            norm_check(got, ref, what)
    return run
