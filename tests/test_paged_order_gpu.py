"""Row starts that go back (cu_tokens not in order): a sequence that starts before
the end of an earlier one is left out with those whose own numbers do not fit, and
reported; all the others are computed, by the rotary append and by attention alike,
and nothing else is written."""
import math

import pytest
import torch

from paged_util import Batch, rope, rope_frequencies
from test_paged_gpu import status_word

pytestmark = pytest.mark.gpu

F32, F16 = torch.float32, torch.float16


@pytest.fixture(scope="module")
def be(cuda):
    from ternative_b200 import CUDABackend
    return CUDABackend()


def in_use(cu, kv, n_tokens, max_new, max_kv):
    """The rows of each sequence that counts: {sequence: (first row, rows)}."""
    used, ends = {}, 0
    for b, (r, e) in enumerate(zip(cu[:-1], cu[1:])):
        n = e - r
        if not (r >= 0 and 0 <= n <= max_new and e <= n_tokens and n <= kv[b] <= max_kv):
            continue
        if r >= ends:
            used[b] = (r, n)
        if n:
            ends = max(ends, e)
    return used


def run(be, b, cu, max_new, dtype):
    """(used, status words) after the rotary append and attention over the batch with these starts; checks every row."""
    from ternative_b200 import PagedBatch, RopeConfig
    max_kv = max(b.kv)
    batch = PagedBatch(torch.tensor(cu, dtype=torch.int32).cuda(), b.kv_len.cuda(), b.table.cuda(), b.T, max_new, max_kv)
    used = in_use(cu, b.kv, b.T, max_new, max_kv)
    words = [status_word(), status_word()]
    guard = 64   # rows before and behind the buffers
    def buffer(heads):
        whole = torch.full((b.T + 2 * guard, heads, b.hd), 7.0, device="cuda")
        return whole, whole[guard:guard + b.T]
    qw, q = buffer(b.nh)
    ow, out = buffer(b.nh)
    lw = torch.full((b.T + 2 * guard, b.nh), 7.0, device="cuda")
    k0, v0 = b.k.clone(), b.v.clone()
    be.rope_append_paged_d(q, b.dq, b.dkn, b.dvn, b.cache(), batch, RopeConfig(b.hd), b.nh, b.nkv, b.hd, status=words[0])
    appended = (b.k.clone(), b.v.clone())
    b.k.copy_(k0), b.v.copy_(v0)
    be.attention_paged_d(out, b.dq, b.cache(), batch, b.nh, b.nkv, b.hd, 0.125, lse=lw[guard:guard + b.T], status=words[1])
    torch.cuda.synchronize()
    f, m = rope_frequencies(b.hd, 500000.0, "none", 1.0, 0)
    mine = torch.zeros(b.T, dtype=torch.bool)
    g = b.nh // b.nkv
    touched = torch.zeros(b.k.shape[:2], dtype=torch.bool)
    for i, (r, n) in used.items():
        if not n:
            continue
        assert not mine[r:r + n].any()
        mine[r:r + n] = True
        pos = torch.arange(b.kv[i] - n, b.kv[i])
        touched[b.where[i][0][pos], b.where[i][1][pos]] = True
        assert float((q[r:r + n].cpu().double() - rope(b.q[r:r + n], pos, b.hd, "half", f, m)).abs().max()) < 1e-5
        kk, vv = b.hk[b.where[i]].double(), b.hv[b.where[i]].double()
        for j in range(0, n, max(1, n // 3)):
            p = b.kv[i] - n + j
            for h in range(b.nh):
                w = torch.softmax(kk[:p + 1, h // g] @ b.q[r + j, h].double() * 0.125, 0)
                # 2 max |v| ((hd + 4) U S + 2^-20 + n U) with S < 64, n < 1200, max |v| < 6
                assert float((out[r + j, h].cpu().double() - w @ vv[:p + 1, h // g]).abs().max()) < 5e-3
    assert torch.equal((qw[guard:guard + b.T] == 7).all(-1).all(-1).cpu(), ~mine)
    assert torch.equal((out == 7).all(-1).all(-1).cpu(), ~mine)
    assert torch.equal((lw[guard:guard + b.T] == 7).all(-1).cpu(), ~mine)
    for w in (qw, ow, lw):
        assert (w[:guard] == 7).all() and (w[guard + b.T:] == 7).all()
    for a, old in ((appended[0], k0), (appended[1], v0)):
        changed = (a != old).flatten(2).any(-1).cpu()
        assert not (changed & ~touched).any() and (changed | ~touched).all()
    return used, [int(w.item()) for w in words]


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("new,before", [([1] * 40, 60), ([1] * 40, 900), ([3] * 30, 60), ([3] * 30, 900),
                                        ([45, 1, 80, 30, 60, 7, 64], 60), ([45, 1, 80, 30, 60, 7, 64], 900)])
@pytest.mark.parametrize("heads", [(2, 2), (16, 2)])
@pytest.mark.parametrize("value", [0, 2, "end", -5, 2 ** 31 - 1, -2 ** 31])
def test_one_start_is_wrong(be, dtype, new, before, heads, value):
    b = Batch(new, [n + before + i % 7 for i, n in enumerate(new)], *heads, 64, 16, dtype, seed=len(new), junk=0.0, tail=2)
    cu = b.cu.tolist()
    at = len(new) // 2
    cu[at] = b.used if value == "end" else value
    used, words = run(be, b, cu, max(new), dtype)
    assert len(used) >= len(new) - 3
    assert words == [2, 2]


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("before", [60, 900])
def test_starts_that_go_back(be, dtype, before):
    """[0, 180, 40, 200]: the first has its rows, the second fewer than none, the third starts inside the first."""
    b = Batch([180, 10, 10], [180 + before, 180 + before, 180 + before], 4, 2, 64, 16, dtype, seed=1, junk=0.0)
    used, words = run(be, b, [0, 180, 40, 200], 180, dtype)
    assert used == {0: (0, 180)} and words == [2, 2]


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("new", [1, 30])
def test_starts_that_go_back_among_many(be, dtype, new):
    """More sequences than a balanced grid keeps, a wrong start early, late and in both."""
    n = 600
    for wrong in ([3], [590], [2, 300, 599]):
        b = Batch([new] * n, [new + 5 + i % 9 for i in range(n)], 2, 1, 64, 16, dtype, seed=2, junk=0.0)
        cu = b.cu.tolist()
        for i in wrong:
            cu[i] = 1
        used, words = run(be, b, cu, new, dtype)
        assert len(used) >= n - 3 * len(wrong) and words == [2, 2]


def test_empty_sequences_in_order(be):
    """What is in order stays so: empty sequences at the ends and in runs are no fault."""
    new = [0, 0, 3, 0, 1, 0, 0, 5, 0]
    b = Batch(new, [n + 20 for n in new], 4, 2, 64, 16, F16, seed=3, junk=0.0, tail=1)
    used, words = run(be, b, b.cu.tolist(), 5, F16)
    assert len(used) == len(new) and words == [0, 0]
