"""The workspaces' pool: what a large call took goes back to the device."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_a_large_workspace_is_given_back(cuda):
    from ternative_b200 import CUDABackend, DeviceWeight, LoraTable, TVB_F16
    be = CUDABackend()
    M, K, N = 60000, 16384, 64
    w = (torch.randn(N, K, device="cuda") * 0.02).half()
    table = LoraTable([], [], torch.zeros(0, dtype=torch.int32, device="cuda"), torch.zeros(0, device="cuda"), 0)
    x = torch.randn(M, K, device="cuda")
    y = torch.empty(M, N, device="cuda")

    def call(rows):
        be.matmul_lora_d(y, x, rows, K, DeviceWeight(w.data_ptr(), TVB_F16), N, table, None)
        torch.cuda.synchronize()

    call(300)
    free = torch.cuda.mem_get_info()[0]
    call(M)   # two planes of x: 3.9 GB
    torch.cuda.synchronize()
    assert free - torch.cuda.mem_get_info()[0] < 2100 << 20
    want = x[:8].double() @ w.double().T
    assert float((y[:8].double() - want).norm() / want.norm()) < 4e-6
