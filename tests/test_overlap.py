"""Whether strided views share memory (csrc/overlap.h), on the CPU against sets of bytes: no overlap is missed, and views
of the same strides are told apart exactly, as is one that lies between the other's runs."""
import ctypes
import random
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "inferno_amd" / "csrc"


@pytest.fixture(scope="module")
def over(tmp_path_factory):
    d = tmp_path_factory.mktemp("overlap")
    (d / "o.cpp").write_text(
        '#include "overlap.h"\n'
        'static inf::Memory m(const int64_t* a) { return inf::Memory((const void*)a[0], a[1], a[2], a[3], a[4], a[5], a[6],'
        ' a[7]); }\n'
        'extern "C" int over(const int64_t* a, const int64_t* b) { return m(a).over(m(b)); }\n')
    subprocess.run(["g++", "-std=c++17", "-O1", "-fsanitize=undefined", "-fno-sanitize-recover", "-shared", "-fPIC",
                    f"-I{CSRC}", str(d / "o.cpp"), "-o", str(d / "o.so")], check=True)
    f = ctypes.CDLL(str(d / "o.so")).over
    view = ctypes.c_int64 * 8
    return lambda a, b: bool(f(view(*a), view(*b)))


def memory(v):
    at, B, sb, H, sh, T, st, run = v
    return {at + b * sb + h * sh + t * st + i for b in range(B) for h in range(H) for t in range(T) for i in range(run)}


def nested(rng):
    """Dims of a view that does not overlap itself, in any order."""
    run = rng.randint(1, 6)
    span, dims = run, []
    for _ in range(3):
        n = rng.randint(1, 4)
        stride = span + rng.choice([0, 0, 1, 3, 7, 20])
        span = stride * (n - 1) + span
        dims.append((n, stride))
    rng.shuffle(dims)
    return [x for d in dims for x in d] + [run]


def test_same_strides_are_exact(over):
    rng = random.Random(1)
    both = [0, 0]
    for _ in range(4000):
        a = nested(rng)
        b = list(a)
        b[6] = rng.randint(1, a[6])  # a narrower run
        for i in (0, 2, 4):
            b[i] = rng.choice([a[i], max(1, a[i] - 1)]) if a[i] > 2 else a[i]
        x, y = [1000, *a], [1000 + rng.randint(-80, 80), *b]
        want = bool(memory(x) & memory(y))
        both[want] += 1
        assert over(x, y) == over(y, x) == want, (x, y)
    assert min(both) > 500


def test_no_overlap_is_missed(over):
    rng = random.Random(2)
    told = 0
    for _ in range(6000):
        x, y = [1000, *nested(rng)], [1000 + rng.randint(-100, 100), *nested(rng)]
        for v in (x, y):  # what is only read may repeat itself
            if rng.random() < 0.3:
                v[rng.choice([2, 4, 6])] = rng.choice([0, 1, 5])
        want = bool(memory(x) & memory(y))
        if want:
            assert over(x, y) and over(y, x), (x, y)
        elif max(memory(x)) >= min(memory(y)) and max(memory(y)) >= min(memory(x)):
            told += not over(x, y)
    assert told


def test_between_the_runs(over):
    """A dense vector in a gap of a matrix, and over one of its runs."""
    for at in range(0, 300):
        x, y = [4096, 1, 0, 8, 32, 1, 0, 20], [4000 + at, 1, 0, 1, 0, 1, 0, 12]
        assert over(x, y) == over(y, x) == bool(memory(x) & memory(y))


def test_nothing_and_far(over):
    a = [4096, 2, 64, 2, 32, 2, 16, 16]
    assert not over([0, *a[1:]], a) and not over(a, [*a[:7], 0])
    assert over(a, [4096, 4, 1 << 62, 1, 0, 1, 0, 4]) and over(a, [100, 4, 1 << 62, 1, 0, 1 << 40, 1 << 40, 1 << 60])
    assert not over(a, [1 << 62, 1, 0, 1, 0, 1, 0, 4])
