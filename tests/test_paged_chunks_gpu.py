"""Attention of prompt chunks large enough for the tensor cores (tvb_attention_paged),
against a plain form in 64 bits: heads enough that the call does not fall to the
few-rows kernels, at the sizes, masks and values where chunks can go wrong."""
import math

import pytest
import torch

from paged_util import Batch
from test_paged_gpu import attend, check_attention

pytestmark = pytest.mark.gpu

F32, F16 = torch.float32, torch.float16
HEADS = (32, 8)   # 32 heads x 80 tokens: more row blocks than SMs


@pytest.fixture(scope="module")
def be(cuda):
    from ternative_b200 import CUDABackend
    return CUDABackend()


CASES = [
    # new, kv, heads, hd, page, order, window
    ([100], [100], HEADS, 128, 16, "rows", 0),
    ([65, 1, 50], [300, 257, 50], HEADS, 128, 64, "heads", 0),
    ([70, 33], [400, 33], (48, 8), 64, 24, "rows", 50),
    ([129, 40, 0, 3], [129, 300, 7, 3], HEADS, 64, 5, "heads", 0),
    ([90, 90], [700, 1500], HEADS, 128, 128, "rows", 0),
    ([257], [257], (16, 16), 64, 1, "rows", 1),
    ([200, 13], [900, 900], (24, 2), 128, 16, "rows", 333),
    ([170], [640], (15, 5), 64, 1000, "rows", 0),
]


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{c[0][:3]}-{c[1][:3]}-{c[2]}-{c[3]}-p{c[4]}-{c[5]}-w{c[6]}")
def test_chunks(be, case, dtype):
    new, kv, heads, hd, page, order, window = case
    b = Batch(new, kv, *heads, hd, page, dtype, order, seed=len(new) + hd, tail=2, interleave=order == "rows")
    out, lse, st = attend(be, b, window=window)
    assert st == 0
    check_attention(b, out, lse, window=window)


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("kv", [90, 200, 900])
def test_values_of_unseen_keys(be, dtype, kv):
    """Keys and values that a row does not see may hold anything: rows before them are as without them."""
    b = Batch([90, 5], [kv, 50], *HEADS, 64, 16, dtype, seed=1)
    want, wlse, _ = attend(be, b)
    pg, at = (t[kv - 30:].cuda() for t in b.where[0])
    for pool, bad in ((b.v, math.nan), (b.k, math.nan), (b.v, math.inf)):
        keep = pool[pg, at].clone()
        pool[pg, at] = bad
        out, lse, st = attend(be, b)
        assert st == 0
        # rows 0..59 see none of the thirty; their sums may be taken key by key, in another order
        ref, rlse, tol = b.attention()
        assert ((out[:60].double() - ref[:60]).abs().amax(-1) <= tol[:60]).all()
        assert float((out[:60] - want[:60]).abs().max()) < 1e-4
        assert not torch.isfinite(out[60:90]).any()
        assert torch.equal(out[90:], want[90:]) and torch.equal(lse[90:], wlse[90:])
        pool[pg, at] = keep


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("size", [1e-6, 1.0, 1e3])
def test_magnitudes(be, dtype, size):
    """Queries of any size (scores stay of order one) and values of 1000: relative precision holds."""
    b = Batch([90], [300], *HEADS, 64, 16, dtype, seed=2, junk=0.0)
    b.q.mul_(size)
    b.dq.mul_(size)
    b.hv.mul_(1000.0)
    b.v.mul_(1000.0)
    scale = 0.125 / size
    out, lse, st = attend(be, b, scale=scale)
    assert st == 0
    check_attention(b, out, lse, scale=scale)


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("kv", [300, 1300])
def test_a_page_that_does_not_exist(be, dtype, kv):
    b = Batch([90, 4], [kv, 40], *HEADS, 64, 16, dtype, seed=3)
    want, _, _ = attend(be, b)
    b.table[0, -(-(kv - 95) // 16) - 1:] = -1   # behind the cache's older part
    first = (-(-(kv - 95) // 16) - 1) * 16
    out, lse, st = attend(be, b)
    assert st == 2
    ref, rlse, tol = b.attention(limit=[first, 40])
    assert ((out.double() - ref).abs().amax(-1) <= tol).all()
    assert torch.equal(out[90:], want[90:])


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("kv", [100, 1300])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_a_query_that_is_not_finite_stays_alone(be, dtype, kv, bad):
    b = Batch([90], [kv], *HEADS, 64, 16, dtype, seed=4)
    want, wlse, _ = attend(be, b)
    b.dq[7, 3, 11] = bad
    out, lse, st = attend(be, b)
    assert st == 0 and torch.isnan(out[7, 3]).all() and torch.isnan(lse[7, 3])
    out[7, 3], lse[7, 3] = want[7, 3], wlse[7, 3]
    assert torch.equal(out, want) and torch.equal(lse, wlse)


@pytest.mark.parametrize("dtype", [F32, F16])
def test_many_short_sequences(be, dtype):
    """More sequences than a balanced grid keeps, empty ones and single tokens among them."""
    n = 600
    lens = [0 if i % 7 == 3 else 1 + i * 31 % 40 for i in range(n)]
    kv = [t + i * 37 % 200 if t else 0 for i, t in enumerate(lens)]
    b = Batch(lens, kv, 2, 1, 64, 16, dtype, seed=2, tail=3)
    out, lse, st = attend(be, b)
    assert st == 0
    check_attention(b, out, lse)


def test_captured_and_other_streams(be):
    """Two captured chunks with workspaces, replayed on two streams at once with new queries, against eager calls."""
    runs = []
    for seed, dtype in enumerate((F16, F32)):
        b = Batch([90, 30], [1300, 700], *HEADS, 64, 16, dtype, seed=seed)
        cache, batch, out = b.cache(), b.batch(), torch.empty_like(b.dq)

        def call(o, stream, b=b, cache=cache, batch=batch):
            be.attention_paged_d(o, b.dq, cache, batch, b.nh, b.nkv, b.hd, 0.125, stream=stream)
        s, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(g, stream=s):
            call(out, torch.cuda.current_stream().cuda_stream)
        runs.append((b, out, call, s, g))
    for turn in range(3):
        for b, out, call, s, g in runs:
            b.dq.mul_(-0.7)
        torch.cuda.synchronize()
        for b, out, call, s, g in runs:
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for b, out, call, s, g in runs:
            want = torch.empty_like(out)
            call(want, torch.cuda.current_stream().cuda_stream)
            torch.cuda.synchronize()
            assert torch.equal(out, want)
