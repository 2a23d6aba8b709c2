"""Where the callers' tensors of the operators lie (katago_b200/csrc/kb_box.h, compiled here; no GPU needed): tensors that are said to be
apart share no element, whatever their strides, and a dimension that repeats (stride 0) is as good as any other."""
import ctypes
import os
import random
import subprocess
from itertools import product

import pytest

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BASE = 1 << 20


@pytest.fixture(scope="module")
def box(tmp_path_factory):
    d = tmp_path_factory.mktemp("boxes")
    (d / "b.cpp").write_text(
        '#include "kb_box.h"\n'
        "static kb::Box of(const int64_t* v) { return kb::Box{\"x\", (const void*)v[0], {v[1], v[2], v[3]}, {v[4], v[5], v[6]}, v[7], (size_t)v[8]}; }\n"
        'extern "C" int apart(const int64_t* a, const int64_t* b) { return !kb::mayOverlap(of(a), of(b)); }\n'
        'extern "C" int distinct(const int64_t* a) { return !kb::overlapsItself(of(a)); }\n')
    subprocess.run(["g++", "-std=c++17", "-shared", "-fPIC", "-I", os.path.join(_ROOT, "katago_b200", "csrc"), "-o", str(d / "b.so"), str(d / "b.cpp")], check=True)
    return ctypes.CDLL(str(d / "b.so"))


def _record(at, n, s, width, elem=4):
    """Address in elements, counts and strides of the three outer dimensions, channels."""
    return (ctypes.c_int64 * 9)(BASE + at * elem, *n, *s, width, elem)


def _elements(at, n, s, width):
    return [at + sum(i * j for i, j in zip(place, s)) + c for place in product(*(range(x) for x in n)) for c in range(width)]


# a query that all tokens of a sequence share, beside the output in one buffer; what repeats is the tokens, the sequences, both
@pytest.mark.parametrize("a,b,apart", [
    ((0, (2, 8, 1), (576, 0, 64), 64), (64, (2, 8, 1), (576, 64, 64), 64), False),   # cannot be told apart: rows of other strides
    ((0, (2, 3, 1), (64, 0, 16), 16), (16, (2, 3, 1), (64, 16, 16), 16), False),
    ((0, (2, 8, 1), (128, 0, 64), 64), (64, (2, 1, 1), (128, 0, 64), 64), True),     # a row per sequence, halves of the same rows
    ((0, (2, 8, 1), (128, 0, 64), 64), (32, (2, 1, 1), (128, 0, 64), 64), False),
    ((0, (2, 8, 1), (0, 0, 64), 64), (64, (2, 8, 1), (1024, 128, 64), 64), True),    # one row for everything in the gap of the output's rows
    ((0, (2, 8, 1), (0, 0, 64), 64), (0, (2, 8, 1), (1024, 128, 64), 64), False),
    ((0, (2, 8, 4), (1024, 128, 0), 64), (64, (2, 8, 1), (1024, 128, 64), 64), True),  # heads that repeat
    ((0, (2, 8, 1), (0, 128, 64), 64), (64, (2, 8, 1), (1024, 128, 64), 64), True),  # sequences that repeat
    ((0, (3, 5, 1), (100, 0, 0), 10), (50, (3, 5, 2), (300, 60, 10), 10), False),
])
def test_tensors_that_repeat(a, b, apart, box):
    assert bool(box.apart(_record(*a), _record(*b))) == apart
    assert bool(box.apart(_record(*b), _record(*a))) == apart
    if apart:
        assert not set(_elements(*a)) & set(_elements(*b))


def test_tensors_said_to_be_apart_share_nothing(box):
    """Small tensors of every kind of stride, half of them in rows of one buffer."""
    rng = random.Random(7)
    told = {True: 0, False: 0}
    for _ in range(60000):
        row = rng.randint(1, 16)
        pair = []
        for _ in range(2):
            n = [rng.randint(0 if rng.random() < 0.02 else 1, 4) for _ in range(3)]
            width = rng.randint(1, 5)
            s = [rng.choice((0, 1, rng.randint(0, 24), row, row * rng.randint(1, 6))) for _ in range(3)]
            if rng.random() < 0.5:
                s[1], s[0] = rng.choice((row, row, 0)), rng.choice((row * n[1], row * rng.randint(0, 6), 0))
            pair.append((rng.randint(0, 40), tuple(n), tuple(s), width))
        a, b = pair
        apart = bool(box.apart(_record(*a), _record(*b)))
        assert apart == bool(box.apart(_record(*b), _record(*a))), pair
        told[apart] += 1
        if apart:
            assert not set(_elements(*a)) & set(_elements(*b)), pair
        if box.distinct(_record(*a)):
            places = _elements(*a)
            assert len(set(places)) == len(places), a
    assert min(told.values()) > 5000  # both answers are tested
