"""Every way the gated feed-forward block takes its products: columns of a tile, one CTA or two, sums split or whole. Oracle and
counted bounds of ``test_mlp.py``; sizes at which the library's own choice reaches each of them, none a multiple of 64."""

import ctypes
import importlib
import math
import random

import pytest

from test_mlp import check, inputs

lib = importlib.import_module("kalman-linear-attention_b200._lib")

SIZES = [(38, 40, 40, 48), (33, 130, 10594, 42), (12669, 80, 148, 238), (8488, 259, 394, 1535), (549, 333, 3942, 686), (25574, 134, 1225, 412),
         (20470, 2421, 143, 2845), (275, 1175, 10633, 3578), (1397, 950, 6606, 558), (14534, 3559, 41, 371), (6531, 149, 6760, 268),
         (1710, 386, 8712, 649), (12067, 138, 3267, 264), (20812, 45, 10383, 133)]
PRODUCTS = ("gate and up", "y", "gradients of gate and up", "dx", "dw3", "dw12")


def plans(rows, d, H, out):
    args, got = lib.MlpArgs(rows=rows, d=d, H=H, out=out), set()
    for i, name in enumerate(PRODUCTS):
        columns, ctas, splits = (ctypes.c_int() for _ in range(3))
        assert lib.load().kla_b200_mlp_plan(ctypes.byref(args), i, ctypes.byref(columns), ctypes.byref(ctas), ctypes.byref(splits)) == 0
        got.add((name, columns.value, ctas.value, splits.value > 1))
    return got


def test_the_sizes_reach_every_variant():
    reached = set().union(*(plans(*s) for s in SIZES))
    alone, paired = [(n, c, 1) for n in PRODUCTS for c in (64, 128, 192, 256)], [(n, c, 2) for n in PRODUCTS for c in (192, 256)]
    every = {(*v, split) for v in alone + paired for split in (False, True)
             if not (v[0] == "gate and up" and v[1] == 64) and not (split and v[0] in ("gate and up", "gradients of gate and up"))}
    assert reached == every
    rng = random.Random(0)
    size = lambda most: int(math.exp(rng.uniform(0, math.log(most))))  # noqa: E731
    for _ in range(4000):
        assert plans(size(40000), size(6000), size(12000), size(6000)) <= reached


def test_the_plans_arguments_are_checked():
    L, c = lib.load(), [ctypes.byref(ctypes.c_int()) for _ in range(3)]
    args = lambda **kw: ctypes.byref(lib.MlpArgs(**{**dict(rows=4, d=8, H=8, out=8), **kw}))  # noqa: E731
    assert L.kla_b200_mlp_plan(None, 0, *c) == 1 and L.kla_b200_mlp_plan(args(rows=0), 0, *c) == 1
    assert L.kla_b200_mlp_plan(args(), 6, *c) == 1 and L.kla_b200_mlp_plan(args(), -1, *c) == 1 and L.kla_b200_mlp_plan(args(), 0, None, *c[1:]) == 1
    assert L.kla_b200_mlp_plan(args(), 5, *c) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("i", range(len(SIZES)))
def test_forward_and_backward(i):
    check(*inputs(*SIZES[i], bias=True, residual=True), act=("silu", "gelu", "relu", None)[i % 4])
