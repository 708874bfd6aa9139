"""Queries near the largest float (tvb_attention_paged): one key takes everything, in
every kernel."""
import pytest
import torch

from paged_util import Batch
from test_paged_gpu import attend

pytestmark = pytest.mark.gpu

F32, F16 = torch.float32, torch.float16


@pytest.fixture(scope="module")
def be(cuda):
    from ternative_b200 import CUDABackend
    return CUDABackend()


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("new,heads,kv", [(1, (2, 2), 900), (2, (8, 2), 900), (4, (8, 2), 40), (90, (32, 8), 100), (90, (32, 8), 900)])
@pytest.mark.parametrize("size", [2.0 ** 110, 2.0 ** 120])
def test_queries_near_the_largest_float(be, dtype, new, heads, kv, size):
    b = Batch([new], [kv], *heads, 64, 16, dtype, seed=kv)
    b.dq.mul_(size)
    out, lse, st = attend(be, b, scale=0.125)
    assert st == 0
    g = b.nh // b.nkv
    k, v = b.hk[b.where[0]].double(), b.hv[b.where[0]]
    for j in range(0, new, max(1, new // 5)):
        for h in range(b.nh):
            z = k[:kv - new + j + 1, h // g] @ b.q[j, h].double()
            top = z.topk(2)[0]
            # the largest by more than what F32 sums of 64 products (magnitudes below 128) lose: its key alone counts
            if top[0] - top[1] > 64 * 128 * 2.0 ** -23:
                assert torch.equal(out[j, h], v[z.argmax(), h // g].float())
                assert abs(float(lse[j, h]) / (float(top[0]) * size * 0.125) - 1) < 1e-4
