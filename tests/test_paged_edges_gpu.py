"""The paged operators at the calls that are rare but allowed: rows that are not
finite, more sequences than a balanced grid keeps, empty sequences among them,
sequences out of order, pages shared by sequences, pools past 32-bit offsets,
a first call inside a capture."""
import math
import os
import subprocess
import sys

import pytest
import torch

from paged_util import Batch, rope, rope_frequencies
from test_paged_gpu import attend, check_attention, status_word

pytestmark = pytest.mark.gpu

F32, F16 = torch.float32, torch.float16


@pytest.fixture(scope="module")
def be(cuda):
    from ternative_b200 import CUDABackend
    return CUDABackend()


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("new,kv,heads", [
    ([2, 1], [40, 9], (2, 2)), ([2, 1], [900, 50], (2, 2)),        # one or two rows
    ([2, 1], [40, 9], (8, 2)), ([2, 1], [900, 50], (8, 2)),        # four to eight
    ([3, 1], [40, 9], (8, 2)), ([3, 1], [900, 50], (8, 2)),        # to sixteen
    ([50, 20], [100, 60], (4, 2)), ([50, 20], [900, 300], (4, 2)),   # tensor cores
])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_a_query_that_is_not_finite_stays_alone(be, dtype, new, kv, heads, bad):
    """Its row is NaN, with the log of its sum, as in the formula; every other row is as without it."""
    b = Batch(new, kv, *heads, 64, 16, dtype, seed=5)
    want, wlse, _ = attend(be, b)
    b.dq[1, 0, 3] = bad
    out, lse, st = attend(be, b)
    assert st == 0
    assert torch.isnan(out[1, 0]).all() and torch.isnan(lse[1, 0])
    out[1, 0], lse[1, 0] = want[1, 0], wlse[1, 0]
    assert torch.equal(out, want) and torch.equal(lse, wlse)


@pytest.mark.parametrize("dtype,new", [(F16, 1), (F32, 1), (F16, 3), (F16, 40), (F32, 70)])
def test_more_sequences_than_a_balanced_grid_keeps(be, dtype, new):
    n = 600
    lens = [0 if i % 7 == 3 else 1 + i * 31 % new for i in range(n)]
    kv = [t + i * 37 % 300 if t else 0 for i, t in enumerate(lens)]
    b = Batch(lens, kv, 2, 1, 64, 16, dtype, seed=2, tail=3)
    out, lse, st = attend(be, b)
    assert st == 0
    check_attention(b, out, lse)


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("scale", [1, 20])
@pytest.mark.parametrize("before", [50, 300])
def test_sequences_out_of_order_are_reported(be, dtype, scale, before):
    """Starts that go back: what has no rows of its own is reported and left out, nothing is read or written outside."""
    from ternative_b200 import RopeConfig
    for lens in ([5, 1, 4], [9, 30, 40]):
        lens = [x * scale for x in lens]
        b = Batch(lens, [x + before for x in lens], 4, 2, 64, 16, dtype, seed=3)
        total = b.T
        b.cu[1], b.cu[2] = total - scale, 2 * scale   # then the second has fewer than no rows
        out, lse, st = attend(be, b, batch=b.batch(max_new=total, max_kv=max(b.kv)))
        assert st == 2
        word = status_word()
        be.rope_append_paged_d(torch.empty_like(b.dq), b.dq, b.dkn, b.dvn, b.cache(), b.batch(max_new=total),
                               RopeConfig(64), b.nh, b.nkv, b.hd, status=word)
        torch.cuda.synchronize()
        assert int(word.item()) == 2


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("new,kv", [([1, 1, 1], [70, 90, 400]), ([60, 33, 100], [170, 90, 400])])
def test_sequences_that_share_pages(be, dtype, new, kv):
    """A prefix that several requests have in common lies in the pool once."""
    b = Batch(new, kv, 4, 2, 64, 16, dtype, seed=4)
    shared = (min(x - n for x, n in zip(kv, new))) // 16
    for i in (1, 2):
        b.table[i, :shared] = b.table[0, :shared]
        t = torch.arange(kv[i])
        b.where[i] = (b.table[i].long()[t // 16], t % 16)
    out, lse, st = attend(be, b)
    assert st == 0
    check_attention(b, out, lse)


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("page", [100, 1000, 4096])
@pytest.mark.parametrize("new", [1, 90])
def test_large_pages(be, dtype, page, new):
    b = Batch([new, 1], [777, 1030], 4, 2, 64, page, dtype, seed=6)
    out, lse, st = attend(be, b, window=500)
    assert st == 0
    check_attention(b, out, lse, window=500)


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("new,kv", [([1, 1], [40, 300]), ([40, 20], [40, 300])])
def test_pools_past_32_bit_offsets(be, dtype, new, kv):
    """Pages 700 MB apart: rotary append and attention over rows beyond 4 GB of a pool."""
    from ternative_b200 import PagedCache, RopeConfig
    b = Batch(new, kv, 4, 2, 64, 64, dtype, seed=7, junk=0.0)
    n, page, nkv, hd = b.k.shape
    stride = 700 * 1000 * 1000 // b.k.element_size() // 64 * 64
    assert (n - 1) * stride * b.k.element_size() > 2 ** 32
    pools = []
    for p in (b.k, b.v):
        far = torch.empty((n - 1) * stride + page * nkv * hd, dtype=dtype, device="cuda")
        view = far.as_strided((n, page, nkv, hd), (stride, nkv * hd, hd, 1))
        view.copy_(p)
        pools.append(view)
    near = b.cache()
    f, m = rope_frequencies(64, 500000.0, "none", 1.0, 0)
    outs = []
    for cache in (near, PagedCache(*pools)):
        q = torch.empty_like(b.dq)
        st = status_word()
        be.rope_append_paged_d(q, b.dq, b.dkn, b.dvn, cache, b.batch(), RopeConfig(64), b.nh, b.nkv, b.hd, status=st)
        out = torch.empty_like(b.dq)
        be.attention_paged_d(out, q, cache, b.batch(), b.nh, b.nkv, b.hd, 0.125, status=st)
        torch.cuda.synchronize()
        assert int(st.item()) == 0
        outs.append((q.cpu(), out.cpu()))
    assert torch.equal(pools[0], b.k) and torch.equal(pools[1], b.v)
    assert torch.equal(outs[0][0], outs[1][0]) and torch.equal(outs[0][1], outs[1][1])
    pos = torch.cat([torch.arange(x - t, x) for t, x in zip(new, kv)])
    assert float((outs[0][0].double() - rope(b.q, pos, 64, "half", f, m)).abs().max()) < 1e-5


@pytest.mark.parametrize("new,kv,heads", [(1, 40, 4), (1, 900, 4), (3, 900, 4), (80, 900, 4)])
@pytest.mark.parametrize("dtype", ["float16", "float32"])
def test_first_call_inside_a_capture(new, kv, heads, dtype):
    """No call before the capture: one-time set-up comes inside it, in a process of its own; the graph then follows new
    queries."""
    code = f"""
import math, sys, torch
sys.path.insert(0, 'tests')
from paged_util import Batch
from ternative_b200 import CUDABackend, RopeConfig
be = CUDABackend()
b = Batch([{new}], [{kv}], {heads}, 2, 64, 16, torch.{dtype}, seed=1)
cache, batch = b.cache(), b.batch()
out, q = torch.empty_like(b.dq), torch.empty_like(b.dq)
s, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
torch.cuda.synchronize()
with torch.cuda.graph(g, stream=s):
    st = torch.cuda.current_stream().cuda_stream
    be.attention_paged_d(out, b.dq, cache, batch, b.nh, b.nkv, b.hd, 0.125, stream=st)
    be.rope_append_paged_d(q, b.dq, b.dkn, b.dvn, cache, batch, RopeConfig(64), b.nh, b.nkv, b.hd, stream=st)
b.q.mul_(-0.5)
b.dq.copy_(b.q)
g.replay()
torch.cuda.synchronize()
ref, _, tol = b.attention(0.125)
assert ((out.cpu().double() - ref).abs().amax(-1) <= tol).all()
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    subprocess.run([sys.executable, "-c", code], check=True, cwd=root, timeout=300)


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("new,kv,heads,hd,page,window", [
    ([300, 40], [1500, 700], (4, 2), 128, 16, 0),
    ([300, 40, 0, 1], [1500, 700, 9, 2000], (6, 2), 64, 24, 0),
    ([129, 600], [129, 2100], (2, 2), 128, 5, 900),
    ([700], [700], (8, 2), 64, 64, 0),
    ([33, 1, 50], [3000, 40, 50], (3, 1), 128, 128, 0),
    ([9, 3], [1700, 900], (4, 2), 128, 16, 0),
    ([5, 3], [1700, 900], (4, 2), 64, 7, 600),
    ([1, 1], [5000, 700], (2, 2), 128, 16, 0),
])
def test_attention_cut_into_runs(be, dtype, new, kv, heads, hd, page, window):
    """Caches long enough that blocks are cut over several CTAs and joined."""
    b = Batch(new, kv, *heads, hd, page, dtype, seed=11, tail=2)
    out, lse, st = attend(be, b, window=window)
    assert st == 0
    check_attention(b, out, lse, window=window)


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("new", [1, 3, 9, 200])
def test_attention_cut_into_runs_with_odd_values(be, dtype, new):
    """Values that some rows do not see are not finite, a page in the middle does not exist: the other keys count, run
    by run."""
    b = Batch([new, new], [1500, 1300], 4, 2, 64, 16, dtype, seed=12)
    out, lse, _ = attend(be, b)
    limit = 1500 - new   # keys of the new tokens: seen by the later ones only
    want = out[:1].clone()
    if new > 1:
        pg, at = b.where[0]
        b.v[pg[limit + 1:].cuda(), at[limit + 1:].cuda()] = math.inf
        out2, _, st = attend(be, b)
        assert st == 0
        # (the first row's keys are as they were; its sum may be taken in another order)
        assert float((out2[:1] - want).abs().max()) < 1e-5 * float(b.v[torch.isfinite(b.v)].abs().max())
        assert not torch.isfinite(out2[1:new]).any()
        assert torch.equal(out2[new:], out[new:])
    b = Batch([new, new], [1500, 1300], 4, 2, 64, 16, dtype, seed=12)
    b.table[0, 40] = 1 << 30
    out3, lse3, st = attend(be, b)
    assert st == 2
    assert torch.equal(out3[new:], out[new:])
    keep = torch.ones(1500, dtype=torch.bool)
    keep[640:656] = False
    k, v = b.hk[b.where[0]].double(), b.hv[b.where[0]].double()
    for j in range(0, new, max(1, new // 5)):
        seen = keep & (torch.arange(1500) <= 1500 - new + j)
        for h in range(4):
            z = k[seen, h // 2] @ b.q[j, h].double() * 0.125
            ref = torch.softmax(z, 0) @ v[seen, h // 2]
            # (hd + 4) U S + n U with S < 64 and n = 1500, twice max |v| < 6: below 6e-5
            assert float((out3[j, h].double() - ref).abs().max()) < 6e-5
