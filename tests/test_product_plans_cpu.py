"""The plans of the 8-bit product: every kind is what the shapes of the GPU tests get, and
every plan is one that the kernel can run."""

import random

import pytest

import product_plans as P


@pytest.fixture(scope="module")
def plans(tmp_path_factory):
    return P.Planner(tmp_path_factory.mktemp("plans"))


def tiles(shape, plan):
    """(tiles, how many run at a time, stages of a CTA's part of one)."""
    t, k, n = shape
    wide = 256 if plan.pair else 128
    depth = -(-k // (128 * plan.chunks))
    return (-(-t // plan.tile_tokens) * -(-n // wide),
            plan.ctas // (2 if plan.pair else plan.split), -(-depth // plan.split))


@pytest.mark.parametrize("kind", P.SHAPES)
def test_shapes_have_the_plans_they_are_meant_for(plans, kind):
    shapes = P.SHAPES[kind]
    several = wraps = short = False
    for half in (True, False):
        for shape, plan in zip(shapes, plans([(*s, half) for s in shapes]), strict=True):
            assert plan.kind() == kind, (shape, plan)
            assert plan.pieces == (half and plan.split == 1)
            count, at_once, stages = tiles(shape, plan)
            several |= count > at_once
            wraps |= stages > plan.stages
            short |= shape[1] % 128 != 0
    assert several and wraps and short


def test_plans_fit_the_kernel(plans):
    """Over sizes of every order, and devices of fewer processors."""
    r = random.Random(1)

    def size(top):
        return max(1, round(2 ** r.uniform(0, top)))

    for sms in (148, 132, 20, 2, 1):
        shapes = [(size(17), size(15), size(16), r.random() < 0.5) for _ in range(400)]
        for shape, plan in zip(shapes, plans(shapes, sms), strict=True):
            t, k, n, half = shape
            count, at_once, _ = tiles(shape[:3], plan)
            assert 16 <= plan.tile_tokens <= 224 and plan.tile_tokens % 16 == 0
            assert plan.split in (1, 2, 4) and plan.split <= max(1, -(-k // 128))
            assert not plan.pair or (plan.split == 1 and plan.chunks == 2
                                     and plan.tile_tokens % 32 == 0)
            assert 1 <= at_once <= count and plan.ctas <= sms
            assert plan.stages >= 2 and 120 * 1024 <= plan.smem <= 227 * 1024
            assert -(-(-(-k // 128)) // plan.chunks) >= plan.split  # a stage for every CTA
