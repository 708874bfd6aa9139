"""The check of a sequence's numbers (csrc/paged_seq.h), compiled for the host:
whatever the device arrays hold, what passes lies inside the token buffers and the
cache, and nothing wraps around."""
import ctypes as C
import itertools
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LOW, HIGH = -2 ** 31, 2 ** 31 - 1


@pytest.fixture(scope="module")
def numbers(tmp_path_factory):
    d = tmp_path_factory.mktemp("seq")
    src = d / "seq.cpp"
    src.write_text("""#include "paged_seq.h"
extern "C" int seq(int row0, int end, int kv, int n_tokens, int max_new, int max_kv, int* n, int* pos0) {
    const tvb::SeqView v = tvb::seq_numbers(row0, end, kv, n_tokens, max_new, max_kv);
    *n = v.n;
    *pos0 = v.pos0;
    return v.ok;
}
""")
    so = d / "seq.so"
    subprocess.run(["g++", "-std=c++17", "-shared", "-fPIC", "-fwrapv", "-I", os.path.join(ROOT, "ternative_b200", "csrc"),
                    str(src), "-o", str(so)], check=True)
    f = C.CDLL(str(so)).seq

    def call(*a):
        n, p = C.c_int(), C.c_int()
        return bool(f(*a, C.byref(n), C.byref(p))), n.value, p.value
    return call


def test_what_fits(numbers):
    assert numbers(3, 8, 20, 10, 5, 20) == (True, 5, 15)
    assert numbers(3, 3, 0, 10, 5, 20) == (True, 0, 0)
    assert numbers(0, 5, 5, 5, 5, 5) == (True, 5, 0)


@pytest.mark.parametrize("kv", [LOW, LOW + 1, LOW + 4, LOW + 5, -1, 0, 4, 21, HIGH])
def test_lengths_that_cannot_be(numbers, kv):
    """Shorter than its new tokens (near the lowest int, where a difference would wrap to a large position, too) or longer
    than max_kv."""
    assert numbers(3, 8, kv, 10, 5, 20) == (False, 0, 0)


def test_any_numbers(numbers):
    """Against the same conditions on integers of any size."""
    some = [LOW, LOW + 1, -7, -1, 0, 1, 5, 6, HIGH - 1, HIGH]
    for row0, end, kv, n_tokens, max_new, max_kv in itertools.product(some, some, some, [0, 6, HIGH], [0, 1, 5, HIGH],
                                                                      [0, 6, HIGH]):
        n = end - row0
        ok = row0 >= 0 and end <= n_tokens and 0 <= n <= max_new and n <= kv <= max_kv
        assert numbers(row0, end, kv, n_tokens, max_new, max_kv) == ((True, n, kv - n) if ok else (False, 0, 0))
