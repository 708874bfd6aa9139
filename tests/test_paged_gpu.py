"""Rotary append and attention over the paged cache (tvb_rope_append_paged,
tvb_attention_paged) against plain forms in 64 bits, at the sizes, page sizes,
orders, masks and lengths where they can go wrong; unused rows of the pool hold
NaN throughout."""
import math

import pytest
import torch

from paged_util import U, Batch, rope, rope_frequencies

pytestmark = pytest.mark.gpu

F32, F16 = torch.float32, torch.float16


@pytest.fixture(scope="module")
def be(cuda):
    from ternative_b200 import CUDABackend
    return CUDABackend()


def status_word():
    return torch.zeros(1, dtype=torch.int32, device="cuda")


def attend(be, b, window=0, scale=None, batch=None, with_lse=True, **kw):
    out = torch.full((b.T, b.nh, b.hd), 7.0, device="cuda")
    lse = torch.full((b.T, b.nh), 7.0, device="cuda") if with_lse else None
    st = status_word()
    be.attention_paged_d(out, b.dq, b.cache(), batch or b.batch(), b.nh, b.nkv, b.hd,
                         1 / math.sqrt(b.hd) if scale is None else scale, window=window, lse=lse, status=st, **kw)
    torch.cuda.synchronize()
    return out.cpu(), None if lse is None else lse.cpu(), int(st.item())


def check_attention(b, out, lse, window=0, scale=None, limit=None):
    ref, rlse, tol = b.attention(scale, window, limit)
    err = (out[:b.used].double() - ref).abs().amax(-1)
    assert torch.isfinite(out[:b.used]).all()
    assert (err <= tol).all(), float((err - tol).max())
    # together far closer than each row's bound: rounding errors do not line up
    rel = float((out[:b.used].double() - ref).norm() / ref.norm().clamp_min(1e-30))
    assert rel < 4e-6, rel
    if lse is not None:
        empty = rlse == -math.inf
        assert torch.equal(lse[:b.used] == -math.inf, empty)
        # scores within (hd + 4) U S, the sum within (n + 16) U of itself; S below 64 here
        d = (lse[:b.used].double() - rlse)[~empty].abs()
        assert not d.numel() or float(d.max()) < (b.hd + 4) * U * 64 + (max(b.kv) + 16) * U + 2.0 ** -20
    assert (out[b.used:] == 7.0).all()   # rows behind the last sequence


CASES = [
    # new, kv, heads, hd, page, dtype, order, window
    ([1], [1], (4, 2), 128, 16, F32, "rows", 0),
    ([1], [130], (20, 5), 128, 16, F32, "rows", 0),
    ([1, 1, 1], [1, 64, 65], (4, 1), 64, 16, F16, "heads", 0),
    ([1] * 9, [3, 700, 15, 16, 17, 1, 333, 128, 129], (8, 8), 128, 5, F16, "rows", 0),
    ([1, 1], [2000, 1999], (32, 8), 128, 64, F16, "heads", 0),
    ([1, 1], [1500, 40], (16, 2), 64, 1, F32, "rows", 0),
    ([1, 1, 1], [900, 31, 257], (12, 2), 128, 24, F16, "rows", 100),
    ([2, 1, 5], [2, 600, 77], (4, 2), 128, 16, F16, "rows", 0),
    ([4, 3], [300, 1000], (5, 5), 64, 7, F32, "heads", 33),
    ([7, 0, 13], [7, 50, 500], (4, 2), 128, 16, F32, "rows", 0),
    ([130], [130], (2, 1), 128, 16, F16, "rows", 0),
    ([65, 1, 200], [300, 257, 200], (4, 2), 128, 64, F16, "heads", 0),
    ([70, 33], [400, 33], (6, 2), 64, 24, F16, "rows", 50),
    ([129, 40], [129, 300], (8, 2), 128, 16, F32, "rows", 0),
    ([100, 31], [411, 31], (3, 1), 64, 5, F32, "heads", 64),
    ([257], [257], (3, 3), 128, 128, F16, "rows", 1),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{c[0][:3]}-{c[1][:3]}-{c[2]}-{c[3]}-p{c[4]}-{c[6]}-w{c[7]}")
def test_attention(be, case):
    new, kv, heads, hd, page, dtype, order, window = case
    b = Batch(new, kv, heads[0], heads[1], hd, page, dtype, order, seed=sum(kv), tail=3)
    out, lse, st = attend(be, b, window)
    assert st == 0
    check_attention(b, out, lse, window)


def test_attention_strided_buffers_and_pools(be):
    """q and out are slices of wider rows, k and v of a page share one pool, no lse."""
    b = Batch([1, 40, 2], [100, 200, 9], 4, 2, 128, 16, F16, seed=5, interleave=True, tail=1)
    wide = torch.zeros(b.T, 4 * 128 + 96, device="cuda")
    wide[:, 64:64 + 512] = b.dq.flatten(1)
    obuf = torch.full((b.T, 700), 7.0, device="cuda")
    be.attention_paged_d(obuf[:, 100:612], wide[:, 64:576], b.cache(), b.batch(), 4, 2, 128, 1 / math.sqrt(128))
    torch.cuda.synchronize()
    check_attention(b, obuf[:, 100:612].reshape(b.T, 4, 128).cpu(), None)
    assert (obuf[:, :100] == 7).all() and (obuf[:, 612:] == 7).all()


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("new,kv", [(3, 20), (40, 200), (150, 150)])
def test_attention_values_of_unseen_keys(be, dtype, new, kv):
    """The last token's key and value are infinite and NaN: no earlier row sees them."""
    b = Batch([new, 5], [kv, 50], 4, 2, 128, 16, dtype, seed=1)
    at = (b.where[0][0][-1], b.where[0][1][-1])
    for h, d, x in ((b.hk, b.k, math.inf), (b.hv, b.v, math.nan)):
        h[at] = x
        d[int(at[0]), int(at[1])] = x
    out, lse, _ = attend(be, b)
    ref, _, tol = b.attention()
    rows = [i for i in range(b.used) if i != new - 1]
    assert torch.isfinite(out[rows]).all()
    assert ((out[rows].double() - ref[rows]).abs().amax(-1) <= tol[rows]).all()


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("size", [1e-6, 1.0, 3e4])
def test_attention_magnitudes(be, dtype, size):
    """Values of any magnitude the type holds keep their relative precision.  (F16 ends at 65504 = 2.18 x 30000, so 3% of
    normal values times 30000 would be infinite inputs; times 12000 the largest of 77,000 values, below 5, fit.)"""
    if dtype == F16:
        size = min(max(size, 1e-4), 1.2e4)
    for new, kv in ((1, 300), (200, 300)):
        b = Batch([new], [kv], 4, 2, 128, 16, dtype, seed=2, junk=0.0)
        b.hv.mul_(size), b.v.mul_(size)
        q = 1.0 / size if dtype == F32 else 1.0
        if dtype == F32:
            b.hk.mul_(size), b.k.mul_(size)
            b.q.mul_(q), b.dq.mul_(q)
        out, lse, _ = attend(be, b)
        check_attention(b, out, lse)


def test_attention_large_scores(be):
    """Scores in the thousands: one key takes everything, nothing overflows."""
    b = Batch([1, 130], [500, 300], 4, 2, 128, 16, F16, seed=3)
    b.q.mul_(300), b.dq.mul_(300)
    out, lse, _ = attend(be, b)
    ref, rlse, tol = b.attention()
    assert torch.isfinite(out).all()
    # S is about 82 * 300 / sqrt(128): a score is off by up to 132 U S = 0.02, so close keys may trade weight
    assert ((out[:b.used].double() - ref).abs().amax(-1) <= tol).all()
    assert float((lse[:b.used].double() - rlse).abs().max()) < 0.04


def test_attention_zero_length_and_empty_batches(be):
    b = Batch([0, 1, 0], [0, 5, 0], 4, 2, 64, 16, F32, seed=4, tail=2)
    out, lse, st = attend(be, b)
    assert st == 0
    check_attention(b, out, lse)
    from ternative_b200 import PagedBatch
    z = torch.zeros(1, dtype=torch.int32, device="cuda")
    e = PagedBatch(z, z[:0], b.table.cuda()[:0], 0, 0, 0)
    be.attention_paged_d(torch.empty(0, 256, device="cuda"), torch.empty(0, 256, device="cuda"), b.cache(), e, 4, 2, 64, 1.0)


@pytest.mark.parametrize("new,kv", [([1, 1, 1], [40, 300, 60]), ([70, 40, 3], [90, 300, 60])])
def test_attention_bad_pages_and_sequences(be, new, kv):
    """A page out of range is reported and its keys are not read; a sequence whose length is above max_kv is skipped."""
    b = Batch(new, kv, 4, 2, 128, 16, F16, seed=6)
    b.table[1, 290 // 16] = b.n_pages
    lim = [kv[0], 288, kv[2]]
    out, lse, st = attend(be, b)
    assert st == 2
    check_attention(b, out, lse, limit=lim)
    b2 = Batch(new, kv, 4, 2, 128, 16, F16, seed=6)
    out, lse, st = attend(be, b2, batch=b2.batch(max_kv=299))
    assert st == 2
    ref, _, tol = b2.attention()
    at = sum(new[:2])
    assert (out[new[0]:at] == 7).all()
    for rows in (slice(0, new[0]), slice(at, b2.used)):
        assert ((out[rows].double() - ref[rows]).abs().amax(-1) <= tol[rows]).all()


ROPES = [
    # new, kv, heads, hd, rot, pairs, scaling, page, dtype, order
    ([1] * 8, [1, 5, 16, 17, 300, 4000, 31, 2], (20, 5), 128, 128, "half", "none", 16, F32, "rows"),
    ([5, 0, 70], [5, 9, 1000], (4, 2), 64, 64, "interleaved", "linear", 5, F16, "heads"),
    ([33], [33], (3, 1), 128, 64, "half", "bands", 1, F16, "rows"),
    ([2, 300], [200000, 300], (2, 2), 256, 32, "interleaved", "yarn", 64, F32, "heads"),
    ([9], [70000], (2, 1), 72, 8, "half", "bands", 24, F32, "rows"),
    ([4], [40], (2, 1), 40, 0, "half", "none", 24, F32, "rows"),
    ([700], [900], (20, 5), 128, 128, "interleaved", "yarn", 16, F16, "rows"),
]


@pytest.mark.parametrize("case", ROPES, ids=lambda c: f"{c[0][:3]}-{c[3]}-{c[4]}-{c[5]}-{c[6]}-p{c[7]}-{c[9]}")
@pytest.mark.parametrize("in_place", [False, True])
def test_rope_append(be, case, in_place):
    from ternative_b200 import RopeConfig
    new, kv, heads, hd, rot, pairs, scaling, page, dtype, order = case
    b = Batch(new, kv, heads[0], heads[1], hd, page, dtype, order, seed=sum(kv), tail=2, junk=3.0)
    cfg = RopeConfig(rot, 10000.0, pairs, scaling, factor=4.0, original_len=4096)
    before = (b.k.clone(), b.v.clone())
    q_out = b.dq.clone() if in_place else torch.full_like(b.dq, 7.0)
    st = status_word()
    be.rope_append_paged_d(q_out, q_out if in_place else b.dq, b.dkn, b.dvn, b.cache(), b.batch(), cfg, b.nh, b.nkv, hd,
                           status=st)
    torch.cuda.synchronize()
    assert int(st.item()) == 0
    f, m = rope_frequencies(rot, 10000.0, scaling, 4.0, 4096)
    # cosine and sine: the angle within 2 pi 2^-26 and 2 pi 2^-25, sincospi 2 steps; three roundings of the result
    e = m * 7e-7
    half = 2.0 ** -11 if dtype == F16 else 0.0
    k, v = before[0].cpu().double(), before[1].cpu().double()
    r = 0
    kt = torch.zeros_like(k)
    for i, n in enumerate(new):
        pos = torch.arange(kv[i] - n, kv[i])
        rows = slice(r, r + n)
        want = rope(b.q[rows], pos, rot, pairs, f, m)
        mag = rope(b.q[rows].abs(), pos * 0, rot, pairs, f * 0, 1.0).amax(-1, keepdim=True)
        assert ((q_out[rows].cpu().double() - want).abs() <= 2 * e * mag).all()
        w = (b.where[i][0][kv[i] - n:], b.where[i][1][kv[i] - n:])
        k[w] = rope(b.kn[rows], pos, rot, pairs, f, m)
        kt[w] = 2 * e * b.kn[rows].double().abs().amax(-1, keepdim=True) + half * k[w].abs() + 2.0 ** -25 * (half > 0)
        v[w] = b.vn[rows].to(dtype).double()
        r += n
    assert ((b.k.cpu().double() - k).abs() <= kt).all()   # untouched rows exactly as before
    assert torch.equal(b.v.cpu().double(), v)
    assert (q_out[b.used:].cpu() == (b.q[b.used:] if in_place else 7.0)).all()


def test_rope_append_bad_data(be):
    """A page out of range, a length below the new tokens: skipped and reported, the others done."""
    from ternative_b200 import RopeConfig
    b = Batch([1, 2, 1, 1], [20, 40, 30, 8], 4, 2, 64, 16, F32, seed=9, junk=0.0)
    b.table[0, 1] = -1
    b.kv_len[1] = 1
    before = b.k.clone()
    q = torch.full_like(b.dq, 7.0)
    st = status_word()
    be.rope_append_paged_d(q, b.dq, b.dkn, b.dvn, b.cache(), b.batch(), RopeConfig(64), 4, 2, 64, status=st)
    assert int(st.item()) == 2
    assert (q[:3] == 7).all() and not (q[3:] == 7).all(-1).any()
    changed = (b.k != before).flatten(1).any(1).nonzero().flatten().tolist()
    assert sorted(changed) == sorted(int(b.where[i][0][-1]) for i in (2, 3))


def test_captured_calls_replay_with_new_lengths_and_other_streams(be):
    """Two captured graphs with workspaces, replayed in turn on two streams with rewritten lengths, against eager
    calls on a third."""
    from ternative_b200 import PagedBatch, RopeConfig
    cases = []
    for seed, n in enumerate([2, 3]):
        b = Batch([1] * n, [1024] * n, 8, 2, 128, 16, F16, seed=seed, junk=0.0)   # pages for the longest
        kvl = b.kv_len.cuda()
        batch = PagedBatch(b.cu.cuda(), kvl, b.table.cuda(), b.T, 1, 1024)
        cache, rc = b.cache(), RopeConfig(128)
        qr, out = torch.empty_like(b.dq), torch.empty_like(b.dq)
        cases.append((b, kvl, batch, cache, rc, qr, out, torch.cuda.Stream(), torch.cuda.CUDAGraph()))

    def step(c, stream):
        b, kvl, batch, cache, rc, qr, out = c[:7]
        be.rope_append_paged_d(qr, b.dq, b.dkn, b.dvn, cache, batch, rc, 8, 2, 128, stream=stream)
        be.attention_paged_d(out, qr, cache, batch, 8, 2, 128, 0.09, stream=stream)

    for c in cases:
        step(c, torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        with torch.cuda.graph(c[8], stream=c[7]):
            step(c, torch.cuda.current_stream().cuda_stream)
    for lens in ([(700, 40), (900, 1024, 5)], [(3, 512), (1, 600, 800)]):
        for c, n in zip(cases, lens):
            c[1].copy_(torch.tensor(n, dtype=torch.int32))
        torch.cuda.synchronize()
        for _ in range(3):
            for c in cases:
                with torch.cuda.stream(c[7]):
                    c[8].replay()
        torch.cuda.synchronize()
        for c in cases:
            got = c[6].clone()
            other = torch.cuda.Stream()
            c[6].zero_()
            torch.cuda.synchronize()
            with torch.cuda.stream(other):
                step(c, other.cuda_stream)
            torch.cuda.synchronize()
            assert torch.equal(got, c[6]) and torch.isfinite(got).all()
