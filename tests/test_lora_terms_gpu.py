"""tvb_matmul_lora, one term at a time: the adapters' products alone over long rows
and large ranks, and rows up to the largest float."""
import math

import pytest
import torch

from paged_util import U

pytestmark = pytest.mark.gpu

F32, F16 = torch.float32, torch.float16


@pytest.fixture(scope="module")
def be(cuda):
    from ternative_b200 import CUDABackend
    return CUDABackend()


def project(be, x, w, A, B, ids):
    from ternative_b200 import DeviceWeight, LoraTable, TVB_F16
    r = torch.tensor([a.shape[0] for a in A], dtype=torch.int32, device="cuda")
    table = LoraTable([a.cuda() for a in A], [b.cuda() for b in B], r, torch.ones(len(A), device="cuda"), max_rank=int(r.max()))
    dw = w.cuda()
    y = torch.empty(x.shape[0], w.shape[0], device="cuda")
    be.matmul_lora_d(y, x.cuda(), x.shape[0], x.shape[1], DeviceWeight(dw.data_ptr(), TVB_F16), w.shape[0], table, ids.cuda())
    return y.cpu().double()


@pytest.mark.parametrize("M,K,rank", [(5, 16384, 16), (300, 6912, 24), (300, 16384, 250), (520, 6912, 256), (520, 16384, 256),
                                      (3600, 16384, 32), (520, 64, 256)])
def test_adapters_of_one_sign(be, M, K, rank):
    """A zero weight leaves the adapter's term alone; with everything positive, what each step of a sum loses adds up.

    Tensor cores truncate to 24 bits, at most 30 products before the sum goes to F32: together 30 x 2^-26 to 2^-25 of it
    in each of the two products; the planes 2^-22 each; and 2^-24 at most an addition: K / 640 + 16 of them in the first
    where a CTA's eight warps cut K, 8 in the second.  (The CUDA-core kernels add K / 2048 + 14 and rank values.)"""
    g = torch.Generator().manual_seed(M + K)
    x = torch.rand(M, K, generator=g) + 0.5
    A = [torch.rand(rank, K, generator=g) + 0.5]
    B = [torch.rand(40, rank, generator=g) + 0.5]
    y = project(be, x, torch.zeros(40, K, dtype=F16), A, B, torch.zeros(M, dtype=torch.int32))
    want = (x.double() @ A[0].double().T) @ B[0].double().T
    rel = (y - want) / want
    # what the additions lose is of either sign: their root mean square; the rest in full
    adds = math.sqrt(K / 640 + 24 + rank) * U
    assert float(rel.mean().abs()) < 2 * 30 * 2.0 ** -26 + 2 * 2.0 ** -22 + adds, float(rel.mean())
    assert float(rel.abs().max()) < 2 * 30 * 2.0 ** -25 + 2 * 2.0 ** -22 + 4 * adds, float(rel.abs().max())


@pytest.mark.parametrize("M", [1, 12, 40, 300])
@pytest.mark.parametrize("size", [2.0 ** -110, 2.0 ** 112, 2.0 ** 118, 2.0 ** 121])
def test_rows_up_to_the_largest_float(be, M, size):
    g = torch.Generator().manual_seed(M)
    x = torch.randn(M, 512, generator=g) * size
    w = (torch.randn(96, 512, generator=g) * 0.02).half()
    y = project(be, x, w, [torch.zeros(4, 512)], [torch.zeros(96, 4)], torch.zeros(M, dtype=torch.int32))
    want = x.double() @ w.double().T
    # planes scaled by 2^-100 at least: below 2^-24 of the smallest row's largest value; F32's normal range ends at 2^-126
    tol = (x.double().abs() @ w.double().abs().T) * ((512 + 4) * U + 2.0 ** -21) + 512 * 2.0 ** -140
    assert torch.isfinite(y).all()
    assert ((y - want).abs() <= tol).all()


@pytest.mark.parametrize("M", [1, 12, 40, 300])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_what_is_not_finite_reaches_its_own_row_and_column(be, M, bad):
    g = torch.Generator().manual_seed(M)
    x = torch.randn(M, 512, generator=g)
    w = (torch.randn(96, 512, generator=g) * 0.02).half()
    A, B = [torch.randn(4, 512, generator=g)], [torch.randn(96, 4, generator=g)]
    ids = torch.zeros(M, dtype=torch.int32)
    want = project(be, x, w, A, B, ids)
    xb, wb = x.clone(), w.clone()
    xb[M // 2, 77] = bad
    wb[50, 300] = bad
    y = project(be, xb, w, A, B, ids)
    assert not torch.isfinite(y[M // 2]).any()
    rest = [m for m in range(M) if m != M // 2]
    assert torch.equal(y[rest], want[rest])
    y = project(be, x, wb, A, B, ids)
    assert not torch.isfinite(y[:, 50]).any()
    rest = [n for n in range(96) if n != 50]
    assert torch.equal(y[:, rest], want[:, rest])
