"""Keys and values that are not finite and that rows do see (tvb_attention_paged):
every kernel gives what the formula gives, whatever the number of rows."""
import math

import pytest
import torch

from paged_util import Batch
from test_paged_gpu import attend

pytestmark = pytest.mark.gpu

F32, F16 = torch.float32, torch.float16
CALLS = [
    (1, (2, 2), 40), (1, (2, 2), 900), (1, (4, 2), 900),     # one or two rows
    (2, (8, 2), 40), (2, (8, 2), 900),                       # up to eight
    (4, (8, 2), 40), (4, (8, 2), 900),                       # up to sixteen
    (90, (32, 8), 100), (90, (32, 8), 1300),                 # tensor cores
]


@pytest.fixture(scope="module")
def be(cuda):
    from ternative_b200 import CUDABackend
    return CUDABackend()


def case(new, heads, kv, dtype):
    b = Batch([new, 1], [kv, 30], *heads, 64, 16, dtype, seed=kv + new)
    at = 20   # seen by every row of the first sequence, or by none but the last few
    at = at if kv - new >= at else kv - new // 2
    return b, at, (int(b.where[0][0][at]), int(b.where[0][1][at]))


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("new,heads,kv", CALLS)
@pytest.mark.parametrize("bad", [math.inf, -math.inf])
def test_an_infinite_key(be, dtype, new, heads, kv, bad):
    """A score of -infinity weighs nothing and leaves the rest as they are; one of +infinity makes its row NaN."""
    b, at, pg = case(new, heads, kv, dtype)
    b.k[pg[0], pg[1], :, 5] = bad
    out, lse, st = attend(be, b)
    assert st == 0
    b.hk[pg[0], pg[1], :, 5] = 0.0
    g = b.nh // b.nkv
    for j in range(new):
        for h in range(0, b.nh, max(1, b.nh // 8)):
            seen = at <= kv - new + j
            if seen and float(b.q[j, h, 5]) * bad > 0:
                assert torch.isnan(out[j, h]).all() and torch.isnan(lse[j, h])
                continue
            keep = torch.arange(kv) <= kv - new + j
            keep[at] = False if seen else keep[at]
            k, v = b.hk[b.where[0]][keep, h // g].double(), b.hv[b.where[0]][keep, h // g].double()
            z = k @ b.q[j, h].double() / 8.0
            # scores below 8 in magnitudes' sum S < 64: 2 max |v| ((hd + 4) U S + 2^-20 + n U) < 2 x 6 x 4e-4
            assert float((out[j, h].double() - torch.softmax(z, 0) @ v).abs().max()) < 5e-3
            rel = float((out[j, h].double() - torch.softmax(z, 0) @ v).norm() / (torch.softmax(z, 0) @ v).norm())
            assert rel < 2e-5, rel
            assert abs(float(lse[j, h]) - float(torch.logsumexp(z, 0))) < 1e-3
    other, olse, _ = b.attention()
    assert float((out[new:].double() - other[new:]).abs().max()) < 5e-3 and torch.isfinite(lse[new:]).all()


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("new,heads,kv", CALLS)
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_a_value_that_is_not_finite(be, dtype, new, heads, kv, bad):
    """It is what its dimension becomes in every row that sees it; the other dimensions are as they were."""
    b, at, pg = case(new, heads, kv, dtype)
    want, wlse, _ = b.attention()
    b.v[pg[0], pg[1], :, 7] = bad
    out, lse, st = attend(be, b)
    assert st == 0
    for j in range(new):
        o = out[j].double()
        if at <= kv - new + j:
            assert (torch.isnan(o[:, 7]) if math.isnan(bad) else o[:, 7] == bad).all()
        else:
            assert torch.isfinite(o[:, 7]).all()
        rest = [d for d in range(64) if d != 7]
        assert float((o[:, rest] - want[j][:, rest]).norm() / want[j][:, rest].norm()) < 2e-5
    assert float((lse.double() - wlse).abs().max()) < 1e-3
    assert float((out[new:].double() - want[new:]).abs().max()) < 5e-3
