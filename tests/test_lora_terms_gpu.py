"""tvb_matmul_lora, one term at a time: the projection of rows up to the largest float."""
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
