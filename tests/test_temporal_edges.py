"""Rotary positions, the paged K/V cache and the attention over it at their edges: what lies in places that no row
sees, pages that are given up or do not exist, rows of very different sizes, empty calls.  Plain forms, tolerances and
their derivation: test_temporal_ops.py."""
import math

import numpy as np
import pytest

from chestnut_b200 import _lib, kernels

torch = pytest.importorskip("torch")

import test_temporal_ops as ops  # noqa: E402

gpu = pytest.mark.gpu


ALTERNATING = [
    # dtype, dim, page, cache heads, group, (new, length) of each sequence: contexts in whole blocks of 128 keys
    ("f16", 128, 64, 8, 1, [(64, 640), (256, 512), (128, 256), (20, 384), (200, 1280), (64, 128), (128, 1024), (256, 256)] * 3),
    ("bf16", 64, 32, 8, 1, [(128, 1152), (40, 128), (129, 256), (64, 768), (17, 256), (255, 384), (100, 1408)] * 3),
    ("bf16", 128, 128, 5, 3, [(30, 640), (100, 256), (42, 384), (6, 128), (85, 512), (43, 896)] * 2),
    ("f16", 64, 16, 16, 1, [(64, 256 + 128 * (i * 7 % 5)) if i % 3 else (256, 256) for i in range(40)]),
]


@gpu
@pytest.mark.parametrize("shape", ALTERNATING, ids=lambda s: "-".join(map(str, s[:5])))
@pytest.mark.parametrize("causal", [False, True])
def test_tiles_of_one_and_of_two_halves_in_turn(shape, causal):
    """Tiles whose halves share the keys, followed by pieces of one block and by tiles of two halves."""
    dtype, dim, page, hk, group, seqs = shape
    ops.test_attention_over_long_contexts((dtype, dtype, dim, page, hk, group, [n for n, _ in seqs],
                                           [total - n for n, total in seqs], causal, 0))
