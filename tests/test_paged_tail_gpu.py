"""Attention where one key takes nearly all the weight and the output is what the
others leave (tvb_attention_paged): small probabilities keep their precision beside
a large one, in the sum and in the weighted values alike."""
import math

import pytest
import torch

from paged_util import U, Batch
from test_paged_gpu import attend

pytestmark = pytest.mark.gpu

F32, F16 = torch.float32, torch.float16


@pytest.fixture(scope="module")
def be(cuda):
    from ternative_b200 import CUDABackend
    return CUDABackend()


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("new,heads,kv,hd", [
    (1, (4, 4), 300, 128), (1, (4, 4), 5000, 64), (1, (4, 2), 3000, 64),          # one or two rows
    (1, (8, 2), 300, 64), (1, (8, 2), 5000, 128), (2, (8, 2), 700, 64),           # up to eight
    (3, (8, 2), 300, 128), (4, (8, 2), 5000, 64),                                 # up to sixteen
    (90, (32, 8), 200, 128), (90, (32, 8), 3000, 64), (90, (32, 8), 3000, 128),   # tensor cores
])
@pytest.mark.parametrize("nats", [12.0, 15.0, 17.5, 20.0])
@pytest.mark.parametrize("sink", [0.0, 1.0])
def test_tail_beside_one_key(be, dtype, new, heads, kv, hd, nats, sink):
    nh, nkv = heads
    b = Batch([new], [kv], nh, nkv, hd, 16, dtype, seed=kv + new)
    g = torch.Generator().manual_seed(int(nats) + kv)
    # scores of the tail: four products of N(0, 1/4) keys with +-8 at scale 1/8; of the sink: one product, `nats`
    q = torch.zeros(b.T, nh, hd)
    q[..., :4] = 8.0 * (torch.randint(0, 2, (b.T, nh, 4), generator=g) * 2 - 1)
    q[..., 4] = 8.0
    k = torch.zeros(kv, nkv, hd)
    k[..., :4] = torch.randn(kv, nkv, 4, generator=g) * 0.5
    k[0] = 0.0
    k[0, :, 4] = nats
    v = 1.0 + 0.1 * torch.randn(kv, nkv, hd, generator=g)
    v[0] = sink * math.exp(-nats) * kv   # of the tail's size, or nothing
    k, v = k.to(dtype), v.to(dtype)
    b.dq.copy_(q)
    b.k[b.where[0][0].cuda(), b.where[0][1].cuda()] = k.cuda()
    b.v[b.where[0][0].cuda(), b.where[0][1].cuda()] = v.cuda()
    out, lse, st = attend(be, b, scale=0.125)
    assert st == 0

    S = nats + 1.0   # a score's sum of magnitudes: the sink's, and no tail score lies above nats / 2 + 1
    e = 2 * ((5 + 4) * U * S + 2.0 ** -20 + kv * U)
    for h in range(nh):
        z = q[:, h].double() @ k[:, h * nkv // nh].double().T * 0.125
        z[torch.arange(kv)[None] > torch.arange(kv - new, kv)[:, None]] = -math.inf
        w = torch.softmax(z, 1)
        vv = v[:, h * nkv // nh].double()
        want = w @ vv
        # a relative error of every probability, each counted with its own value: the tail has no share of the sink's error
        assert ((out[:, h].double() - want).abs() <= e * (w @ vv.abs())).all(), \
            float(((out[:, h].double() - want).abs() / (w @ vv.abs())).max())
        assert float((lse[:, h].double() - torch.logsumexp(z, 1)).abs().max()) <= e * (1 + S)
