"""What the block-scaled e4m3 products plan from their sizes, on the CPU: the scratch queries refuse what the
calls refuse, and the sizes of the GPU tests reach every tile shape, by the rule of fp8_matmul.hip restated here."""
import math
import os
import random
import re

import numpy as np
import pytest
import torch

from eredu_amd import _native
from tests import test_gpu_fp8 as products
from tests import test_gpu_fp8_edges as edges
from tests import test_gpu_fp8_tiles as tiles

L = _native.lib()
P = 4096  # an address; nothing here gets as far as a launch
F32, BF16, E4M3 = 0, 2, 4


def grouped(x_rows, experts, routes, n, k, x_dtype):
    coded = x_dtype == E4M3
    return L.eq_fp8_grouped_matmul(P, P, k, P if coded else None, x_rows if coded else 0, x_rows, P, P, experts, P, P, routes, n, k,
                                   x_dtype, BF16, P + 16, 0, None)  # (scratch that no call takes)


@pytest.mark.parametrize("routes", [1, 64, 65, 5000])
@pytest.mark.parametrize("x_rows,k,x_dtype,words", [
    (0, 128, E4M3, "x must have a row"), (0, 128, BF16, "x must have a row"),
    (1 << 20, 3200, E4M3, "3 * 2^30"), (1 << 20, 3200, BF16, "3 * 2^30"), (1 << 12, 1 << 20, BF16, "3 * 2^30")])
def test_scratch_of_routes_is_refused_where_the_call_is(x_rows, k, x_dtype, words, routes):
    assert grouped(x_rows, 4, routes, 64, k, x_dtype) != 0
    assert words in L.eq_last_error().decode()
    assert L.eq_fp8_grouped_matmul_scratch(x_rows, 4, routes, 64, k, x_dtype, BF16) == -1
    assert words in L.eq_last_error().decode()


def test_scratch_of_routes_up_to_the_limit():
    """One row below 3 * 2^30 bytes is taken, and nothing is refused for an x that no route reads."""
    rows = (3 << 30) // 3200
    assert rows * 3200 < 3 << 30 <= (rows + 1) * 3200
    assert L.eq_fp8_grouped_matmul_scratch(rows, 4, 100, 64, 3200, BF16, BF16) >= rows * 3200
    assert L.eq_fp8_grouped_matmul_scratch(rows + 1, 4, 100, 64, 3200, BF16, BF16) == -1
    for routes, n in ((0, 64), (100, 0)):
        assert L.eq_fp8_grouped_matmul_scratch(0, 4, routes, n, 128, E4M3, BF16) >= 0
        assert grouped(0, 4, routes, n, 128, E4M3) == 0


# ------------------------------------------------------------ the rule that chooses tiles, restated

SOURCE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "eredu_amd", "csrc", "fp8_matmul.hip")
CUS, MOST_TILES = 256, (1 << 23) - 4096
BF, SF = torch.bfloat16, torch.float32
WIDE = 3  # the shapes that f32 results do not take


def shapes():
    """(columns, rows, fixed, one, two, routed) of kShapes."""
    table = re.search(r"kShapes\[\] = \{(.*?)\};", open(SOURCE).read(), re.S).group(1)
    rows = re.findall(r"\{([^{}]+)\}", table)
    return [[float(np.float32(v.strip().rstrip("f"))) for v in r.split(",")] for r in rows]


SHAPES = shapes()


def slots_of(s):
    return (2 if s[4] > 0 else 1) * CUS // 8 * 8


def passes(tiles, slots, most):
    """(whole tiles, tiles in parts, parts of each)."""
    left = tiles % slots
    if most < 2 or left == 0 or slots // left < 2:
        return tiles, 0, 1
    return tiles - left, left, min(slots // left, most)


def tiles_us(s, tiles, blocks, most, rate, read, routed):
    slots = slots_of(s)
    unit = s[0] * s[1] * 8 / 6e6

    def took(at_once, per):
        return s[2] + per * (s[4] if at_once > CUS else s[3]) * (s[5] if routed else 1)

    if routed and tiles > slots:
        us = tiles / slots * took(slots, blocks)
        us += took(CUS, blocks // min(most, 4)) + 8 + slots * unit if most > 1 else .5 * took(slots, blocks)
    else:
        whole, rest, parts = passes(tiles, slots, most)
        us = whole // slots * took(slots, blocks)
        if whole % slots:
            us += took(whole % slots, blocks)
        if rest:
            us += took(rest * parts, -(-blocks // parts)) + 8 + rest * parts * unit
    us = max(us, tiles * blocks * (s[0] + s[1]) * 128 / rate)
    return max(us, read / 6e6) + .25 * min(us, read / 6e6)


def choose(m, n, k, experts, dtype):
    """(shape, most parts, row tiles at the most, scratch for parts) of m rows or routes."""
    blocks, used = -(-k // 128), min(experts, m) if experts else 1
    best = None
    for i, s in enumerate(SHAPES):
        if dtype is SF and i < WIDE:
            continue
        cols, rows = int(s[0]), int(s[1])
        guess = max(used, m // rows + used * 5 // 8) + 1 if experts else -(-m // rows)
        tiles = min(guess * -(-n // cols), MOST_TILES)
        for most in range(1, 17):
            if most > 1 and blocks // most < 4:
                break
            us = tiles_us(s, tiles, blocks, most, 11e6 if experts else 17e6, used * float(n) * float(k), experts > 0)
            if best is None or us < best[0]:
                best = us, i, most
    _, i, most = best
    cols, rows = int(SHAPES[i][0]), int(SHAPES[i][1])
    mtiles = min(m, m // rows + experts + 1) if experts else -(-m // rows)
    scratch = 0
    if most > 1:
        tiles, slots = mtiles * -(-n // cols), slots_of(SHAPES[i])
        _, rest, parts = passes(tiles, slots, most)
        scratch = (min(slots, tiles * most) if experts else rest * parts) * cols * rows * 4
    return i, most, mtiles, scratch


def up256(n):
    return -(-n // 256) * 256


def test_the_restated_rule_is_the_one():
    """By the scratch that products of rows in codes take: of parts of tiles, and of routes lists of tiles and routes."""
    rng = random.Random(3)
    for _ in range(600):
        m, n, k = (int(math.exp(rng.uniform(math.log(lo), math.log(hi)))) for lo, hi in ((65, 12000), (16, 20000), (1, 1000)))
        k *= 16
        for dtype, code in ((BF, BF16), (SF, F32)):
            assert L.eq_fp8_matmul_scratch(m, n, k, E4M3, code) == up256(choose(m, n, k, 0, dtype)[3]), (m, n, k, dtype)
            for experts in (1, 3, 8, 128):
                _, _, mtiles, part = choose(m, n, k, experts, dtype)
                want = up256(16 * (mtiles + 1)) + up256(8 * m) + up256(part)
                assert L.eq_fp8_grouped_matmul_scratch(m, experts, m, n, k, E4M3, code) == want, (m, experts, n, k, dtype)


def table(test):
    return [mark for mark in test.pytestmark if mark.name == "parametrize"][0].args[1]


def taken(m, n, k, dtype):
    """(shape, parts of the last pass's tiles, whether whole passes are before it) of a product."""
    i, most, mtiles, _ = choose(m, n, k, 0, dtype)
    whole, rest, parts = passes(mtiles * -(-n // int(SHAPES[i][0])), slots_of(SHAPES[i]), most)
    return i, parts, rest > 0 and whole > 0


def taken_by_routes(routes, experts, n, k, dtype):
    """The same of the routes that the GPU tests draw, whose tiles the device counts."""
    i, most, _, _ = choose(routes, n, k, experts, dtype)
    ids = edges.drawn_ids(np.random.default_rng(routes), routes, experts)
    counts = np.bincount(ids + 1, minlength=experts + 1)
    used = sum(-(-int(c) // int(SHAPES[i][1])) for c in counts)
    whole, rest, parts = passes(used * -(-n // int(SHAPES[i][0])), slots_of(SHAPES[i]), most)
    return i, parts, rest > 0 and whole > 0


def ways(cases, f32):
    """{"whole", "parts", "behind"}: shapes taken whole, in parts of K, and in parts behind whole passes."""
    found = {"whole": set(), "parts": set(), "behind": set()}
    for (shape, parts, behind), wide in cases:
        if wide == f32:
            found["behind" if behind else "parts" if parts > 1 else "whole"].add(shape)
    return found


def test_the_gpu_tests_take_every_shape():
    """Of one weight and of routes, of 16-bit and of f32 results, what random sizes were found to reach (256 x 192 is not
    taken in parts by routes, 128 x 32 not behind whole passes)."""
    dense = [(taken(*c), c[-1] is SF) for t in (tiles.test_shapes, tiles.test_parts_of_the_last_pass, edges.test_more_shapes) for c in table(t)]
    routed = [(taken_by_routes(*c), c[-1] is SF)
              for t in (tiles.test_shapes_of_routes, tiles.test_parts_of_the_last_pass_of_routes, edges.test_more_shapes_of_routes)
              for c in table(t)]
    assert len(SHAPES) == 7 and SHAPES[WIDE][0] < SHAPES[WIDE - 1][0]
    # (128 x 32 whole of f32 results: sizes of test_gpu_fp8)
    dense += [(taken(*c, SF), True) for c in products.SIZES if c[0] > 16]
    every, narrow = set(range(7)), set(range(WIDE, 7))
    found = ways(dense, False)
    assert found["whole"] == every and found["parts"] == every and found["behind"] == every - {6}
    found = ways(dense, True)
    assert found["whole"] == narrow and found["parts"] == narrow and found["behind"] == {3, 5}
    found = ways(routed, False)
    assert found["whole"] == every and found["parts"] == every - {1} and found["behind"] == {0, 2, 3, 4}
    found = ways(routed, True)
    assert found["whole"] == narrow and found["parts"] == narrow and found["behind"] == {3, 4}
