"""A projection with an adapter for each row (tvb_matmul_lora) against a plain
form in 64 bits: weight types, adapter types, ranks, rows from one to many, ids
in runs, mixed, absent or out of range; and the operators of a layer together."""
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


class Projection:
    def __init__(self, K, N, kind, ranks, dtype, seed=0, size=1.0):
        from ternative_b200 import TVB_F16, TVB_I8_ROW, TVB_I8_TENSOR, DeviceWeight, LoraTable
        g = torch.Generator().manual_seed(seed)
        self.K, self.N, self.ranks = K, N, ranks
        if kind == "f16":
            w = (torch.randn(N, K, generator=g) * 0.02).half()
            self.w = w.double()
            self.dw = w.cuda()
            self.weight = DeviceWeight(self.dw.data_ptr(), TVB_F16)
        else:
            w = torch.randint(-127, 128, (N, K), generator=g, dtype=torch.int8)
            self.dw = w.cuda()
            if kind == "i8row":
                s = torch.rand(N, generator=g) * 3e-4 + 1e-5
                self.ds = s.cuda()
                self.weight = DeviceWeight(self.dw.data_ptr(), TVB_I8_ROW, self.ds.data_ptr())
                self.w = w.double() * s.double()[:, None]
            else:
                self.weight = DeviceWeight(self.dw.data_ptr(), TVB_I8_TENSOR, None, 2e-4)
                self.w = w.double() * float(torch.tensor(2e-4))
        self.A = [(torch.randn(r, K, generator=g) / math.sqrt(K) * size).to(dtype) for r in ranks]
        self.B = [(torch.randn(N, r, generator=g) * 0.05).to(dtype) for r in ranks]
        self.scale = torch.rand(len(ranks), generator=g) * 2 + 0.1
        self.table = LoraTable([a.cuda() for a in self.A], [b.cuda() for b in self.B],
                               torch.tensor(ranks, dtype=torch.int32).cuda(), self.scale.cuda(),
                               max_rank=max(ranks + [1]))

    def __call__(self, x, ids):
        y = x.double() @ self.w.T
        e = (x.double().abs() @ self.w.abs().T) * ((self.K + 4) * U + 2.0 ** -21)
        for i, r in enumerate(self.ranks):
            at = (ids == i).nonzero().flatten()
            xs, a, b, s = x[at].double(), self.A[i].double(), self.B[i].double(), self.scale[i].double()
            y[at] += s * ((xs @ a.T) @ b.T)
            e[at] += s * ((xs.abs() @ a.abs().T) @ b.abs().T) * ((self.K + r + 8) * U + 2.0 ** -20)
        return y, e + y.abs() * 2 * U


def project(be, p, x, ids, status=None, stream=None):
    y = torch.full((x.shape[0], p.N), 7.0, device="cuda")
    be.matmul_lora_d(y, x, x.shape[0], p.K, p.weight, p.N, p.table, ids, status=status, stream=stream)
    return y


CASES = [
    # M, K, N, weight, ranks, adapter type
    (1, 256, 64, "f16", [16], F32),
    (1, 2560, 2560, "f16", [16], F16),
    (2, 264, 37, "f16", [1, 3], F32),
    (3, 272, 100, "i8row", [5], F16),
    (7, 4096, 640, "f16", [64, 8, 16], F32),
    (8, 2560, 6912, "i8row", [16] * 8, F32),
    (15, 6912, 512, "i8tensor", [64, 33, 2], F16),
    (16, 512, 1000, "f16", [200, 7], F32),
    (17, 512, 130, "f16", [12, 64], F32),
    (40, 640, 1025, "i8row", [8, 8, 8, 8], F16),
    (129, 256, 300, "f16", [64, 1], F32),
    (300, 2560, 640, "f16", [16, 32, 64, 100], F32),
    (257, 320, 512, "i8tensor", [256, 65], F16),
    (64, 24, 40, "f16", [4], F32),
    (520, 1024, 2560, "i8row", [40] * 20, F16),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{c[0]}x{c[1]}x{c[2]}-{c[3]}-r{c[4][0]}x{len(c[4])}")
@pytest.mark.parametrize("order", ["mixed", "runs"])
def test_matmul_lora(be, case, order):
    M, K, N, kind, ranks, dtype = case
    p = Projection(K, N, kind, ranks, dtype, seed=M + N)
    g = torch.Generator().manual_seed(M)
    x = torch.randn(M, K, generator=g) * 2
    ids = torch.randint(-1 if M > 1 else 0, len(ranks), (M,), generator=g)
    if order == "runs":
        ids = ids.sort()[0]
    ref, tol = p(x, ids)
    st = torch.zeros(1, dtype=torch.int32, device="cuda")
    y = project(be, p, x.cuda(), ids.to(torch.int32).cuda(), st).cpu().double()
    assert int(st.item()) == 0
    assert ((y - ref).abs() <= tol).all(), float(((y - ref).abs() / tol).max())
    assert float((y - ref).norm() / ref.norm()) < 4e-6


@pytest.mark.parametrize("M", [4, 40])
def test_rows_of_any_magnitude(be, M):
    """Rows from 1e-6 to 1e6 and adapters that outweigh the projection keep their relative precision."""
    p = Projection(512, 256, "f16", [16, 8], F32, seed=3, size=200.0)
    g = torch.Generator().manual_seed(M)
    x = torch.randn(M, 512, generator=g) * torch.logspace(-6, 6, M)[:, None]
    ids = torch.arange(M) % 3 - 1
    ref, tol = p(x, ids)
    y = project(be, p, x.cuda(), ids.to(torch.int32).cuda()).cpu().double()
    assert ((y - ref).abs() <= tol).all()
    rel = (y - ref).norm(dim=1) / ref.norm(dim=1)
    assert float(rel.max()) < 8e-6, rel


@pytest.mark.parametrize("M", [3, 33])
def test_ids_out_of_range_and_no_adapters(be, M):
    p = Projection(256, 96, "f16", [8, 8], F32)
    x = torch.randn(M, 256, generator=torch.Generator().manual_seed(1))
    ids = torch.zeros(M, dtype=torch.long)
    ids[1], ids[2] = 2, -5
    st = torch.zeros(1, dtype=torch.int32, device="cuda")
    y = project(be, p, x.cuda(), ids.to(torch.int32).cuda(), st).cpu().double()
    assert int(st.item()) == 2
    ids[1:3] = -1
    ref, tol = p(x, ids)
    assert ((y - ref).abs() <= tol).all()
    none = Projection(256, 96, "f16", [], F32)
    y = project(be, none, x.cuda(), torch.full((M,), -1, dtype=torch.int32).cuda()).cpu().double()
    ref, tol = none(x, torch.full((M,), -1))
    assert ((y - ref).abs() <= tol).all()


@pytest.mark.parametrize("M", [2, 20])
def test_a_row_that_is_not_finite_stays_alone(be, M):
    p = Projection(512, 64, "f16", [16, 8], F32, seed=8)
    x = torch.randn(M, 512, generator=torch.Generator().manual_seed(2))
    ids = (torch.arange(M) % 2).to(torch.int32)
    bad = x.clone()
    bad[1, 5] = math.nan
    y, z = project(be, p, x.cuda(), ids.cuda()).cpu(), project(be, p, bad.cuda(), ids.cuda()).cpu()
    rest = [i for i in range(M) if i != 1]
    assert torch.equal(y[rest], z[rest]) and torch.isnan(z[1]).all()


def test_captured_graphs_and_streams(be):
    p = Projection(512, 384, "f16", [16, 8, 4], F32, seed=4)
    runs = []
    for M in (5, 70):
        x = torch.randn(M, 512, device="cuda")
        ids = torch.zeros(M, dtype=torch.int32, device="cuda")
        y = torch.empty(M, 384, device="cuda")
        s, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        be.matmul_lora_d(y, x, M, 512, p.weight, 384, p.table, ids, stream=torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        with torch.cuda.graph(g, stream=s):
            be.matmul_lora_d(y, x, M, 512, p.weight, 384, p.table, ids, stream=torch.cuda.current_stream().cuda_stream)
        runs.append((M, x, ids, y, s, g))
    for turn in range(3):
        for M, x, ids, y, s, g in runs:
            ids.copy_((torch.arange(M) * (turn + 1)) % 4 - 1)
        torch.cuda.synchronize()
        for _ in range(2):
            for M, x, ids, y, s, g in runs:
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        for M, x, ids, y, s, g in runs:
            assert torch.equal(y, project(be, p, x, ids))


@pytest.mark.parametrize("new,kv", [([1, 1, 1], [9, 200, 33]), ([20, 1, 40], [20, 77, 90])])
def test_a_layers_serving_step(be, new, kv):
    """q, k and v projections with each request's adapters, rotary append, attention over the cache and the output
    projection: one fused q/k/v buffer, every operator on one stream, against 64 bits."""
    from ternative_b200 import RopeConfig
    nh, nkv, hd, H = 4, 2, 64, 256
    b = Batch(new, kv, nh, nkv, hd, 16, F32, seed=12)
    T = b.T
    g = torch.Generator().manual_seed(5)
    x = torch.randn(T, H, generator=g)
    ids = torch.repeat_interleave(torch.tensor([0, -1, 1]), torch.tensor(new))
    qkv = Projection(H, (nh + 2 * nkv) * hd, "f16", [8, 16], F32, seed=20)
    o = Projection(nh * hd, H, "i8row", [8, 16], F32, seed=21)
    st = torch.zeros(1, dtype=torch.int32, device="cuda")
    d = ids.to(torch.int32).cuda()
    y = project(be, qkv, x.cuda(), d, st)
    q, k, v = y.split([nh * hd, nkv * hd, nkv * hd], 1)
    cache, batch = b.cache(), b.batch()
    be.rope_append_paged_d(q, q, k, v, cache, batch, RopeConfig(hd, 10000.0), nh, nkv, hd, status=st)
    att = torch.empty(T, nh * hd, device="cuda")
    be.attention_paged_d(att, q, cache, batch, nh, nkv, hd, 1 / math.sqrt(hd), status=st)
    z = project(be, o, att, d, st).cpu().double()
    assert int(st.item()) == 0

    ref, _ = qkv(x, ids)
    rq, rk, rv = [t.reshape(T, -1, hd) for t in ref.split([nh * hd, nkv * hd, nkv * hd], 1)]
    f, m = rope_frequencies(hd, 10000.0, "none", 1.0, 0)
    b.hk, b.hv = b.hk.double(), b.hv.double()
    r = 0
    turned = []
    for i, n in enumerate(new):
        pos = torch.arange(kv[i] - n, kv[i])
        w = (b.where[i][0][kv[i] - n:], b.where[i][1][kv[i] - n:])
        b.hk[w], b.hv[w] = rope(rk[r:r + n], pos, hd, "half", f, m), rv[r:r + n]
        turned.append(rope(rq[r:r + n], pos, hd, "half", f, m))
        r += n
    b.q = torch.cat(turned)
    out, _, _ = b.attention()
    want, _ = o(out.reshape(T, -1), ids)
    # four operators of relative error below 4e-6 each (and a softmax that passes its inputs' on): 2e-5
    assert float((z - want).norm() / want.norm()) < 2e-5


# Around the rows where the kernels change over, and several blocks of rows at once.
MORE = [
    (63, 1008, 333, "i8tensor", [16, 3], F32),
    (64, 2560, 2560, "f16", [16] * 8, F32),
    (65, 640, 1025, "i8row", [8, 8, 8, 8], F16),
    (70, 512, 130, "f16", [12, 64], F32),
    (100, 264, 700, "f16", [200, 7, 1], F16),
    (33, 6912, 2560, "i8row", [64, 8], F32),
    (3, 14336, 96, "f16", [16, 4], F32),
    (16, 14336, 64, "i8row", [8], F32),
    (49, 20000, 40, "f16", [4, 9], F32),
    (1500, 128, 520, "f16", [16, 1], F16),
]


@pytest.mark.parametrize("case", MORE, ids=lambda c: f"{c[0]}x{c[1]}x{c[2]}-{c[3]}-r{c[4][0]}x{len(c[4])}")
@pytest.mark.parametrize("order", ["mixed", "runs"])
def test_matmul_lora_rows_in_blocks(be, case, order):
    test_matmul_lora(be, case, order)


def test_many_rows_of_any_magnitude(be):
    test_rows_of_any_magnitude(be, 100)


def test_many_rows_ids_out_of_range_and_no_adapters(be):
    test_ids_out_of_range_and_no_adapters(be, 80)


@pytest.mark.parametrize("M", [40, 90])
def test_one_bad_row_of_many(be, M):
    test_a_row_that_is_not_finite_stays_alone(be, M)


@pytest.mark.parametrize("M", [2, 16, 40, 200])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_an_adapter_that_is_not_finite_stays_alone(be, M, bad):
    """A request's broken adapter spoils its own rows and no other's."""
    p = Projection(256, 300, "f16", [16, 8, 4], F32, seed=5)
    x = torch.randn(M, 256, generator=torch.Generator().manual_seed(M)).cuda()
    ids = (torch.arange(M) % 4 - 1).to(torch.int32)
    from ternative_b200 import LoraTable
    want = project(be, p, x, ids.cuda()).cpu()
    for which in ("A", "B"):
        A, B = [a.clone().cuda() for a in p.A], [b.clone().cuda() for b in p.B]
        (A if which == "A" else B)[0].fill_(bad)
        keep = p.table
        p.table = LoraTable(A, B, torch.tensor(p.ranks, dtype=torch.int32).cuda(), p.scale.cuda(), max_rank=16)
        y = project(be, p, x, ids.cuda()).cpu()
        p.table = keep
        assert torch.equal(y[ids != 0], want[ids != 0])
        assert not torch.isfinite(y[ids == 0]).any()


@pytest.mark.parametrize("M", [3, 30, 90])
def test_output_at_any_address(be, M):
    p = Projection(256, 512, "f16", [8], F32, seed=6)
    x = torch.randn(M, 256, device="cuda")
    ids = torch.zeros(M, dtype=torch.int32, device="cuda")
    want = project(be, p, x, ids)
    buf = torch.full((M * 512 + 8,), 7.0, device="cuda")
    y = buf[1:1 + M * 512].view(M, 512)
    be.matmul_lora_d(y, x, M, 256, p.weight, 512, p.table, ids)
    torch.cuda.synchronize()
    assert torch.equal(y, want) and float(buf[0]) == 7.0 and (buf[1 + M * 512:] == 7.0).all()


@pytest.mark.parametrize("M", [4, 40, 100])
def test_an_adapter_of_misaligned_rows_is_reported(be, M):
    """Pointers that the kernels could not load from are reported and left out."""
    from ternative_b200 import LoraTable
    p = Projection(256, 64, "f16", [8, 8], F32, seed=7)
    x = torch.randn(M, 256, device="cuda")
    ids = torch.arange(M) % 2
    odd = torch.zeros(8 * 256 + 1, device="cuda")
    p.table = LoraTable([p.A[0].cuda(), odd[1:].view(8, 256)], [b.cuda() for b in p.B],
                        torch.tensor(p.ranks, dtype=torch.int32).cuda(), p.scale.cuda(), max_rank=8)
    st = torch.zeros(1, dtype=torch.int32, device="cuda")
    y = project(be, p, x, ids.to(torch.int32).cuda(), st).cpu().double()
    assert int(st.item()) == 2
    ref, tol = p(x.cpu(), torch.where(ids == 1, -1, ids))
    assert ((y - ref).abs() <= tol).all()


@pytest.mark.parametrize("M", [2, 100])
def test_first_call_inside_a_capture(M):
    """No call before the capture: one-time set-up comes inside it, in a process of its own."""
    import os
    import subprocess
    import sys
    code = f"""
import torch
from ternative_b200 import CUDABackend, DeviceWeight, LoraTable, TVB_F16
be = CUDABackend()
w = torch.randn(200, 256, device='cuda').half()
x = torch.randn({M}, 256, device='cuda')
A, B = [torch.randn(8, 256, device='cuda')], [torch.randn(200, 8, device='cuda')]
tab = LoraTable(A, B, torch.full((1,), 8, dtype=torch.int32, device='cuda'), torch.ones(1, device='cuda'), 8)
ids = torch.zeros({M}, dtype=torch.int32, device='cuda')
y = torch.empty({M}, 200, device='cuda')
s, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
torch.cuda.synchronize()
with torch.cuda.graph(g, stream=s):
    be.matmul_lora_d(y, x, {M}, 256, DeviceWeight(w.data_ptr(), TVB_F16), 200, tab, ids,
                     stream=torch.cuda.current_stream().cuda_stream)
g.replay()
torch.cuda.synchronize()
ref = x.double() @ w.double().T + (x.double() @ A[0].double().T) @ B[0].double().T
assert float((y - ref).norm() / ref.norm()) < 4e-6
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    subprocess.run([sys.executable, "-c", code], check=True, cwd=root, timeout=300)


# More than 256 rows, or weights too large to come several times from L2: the two ways of adding the adapters, few
# values of t (rows x largest rank) and many.
MANY = [
    (257, 320, 512, "f16", [16, 3, 8], F32),
    (400, 264, 333, "f16", [20, 7], F16),
    (300, 128, 1000, "i8tensor", [1, 2, 5], F32),
    (1000, 64, 70, "i8row", [8, 4], F16),
    (48, 6144, 8000, "f16", [40, 100], F32),
    (600, 320, 512, "f16", [16, 3, 8], F32),
    (300, 272, 333, "i8row", [30, 7], F16),
    (1000, 64, 70, "i8tensor", [9, 4], F32),
    (40, 6144, 8000, "f16", [256, 33], F16),
]


@pytest.mark.parametrize("case", MANY, ids=lambda c: f"{c[0]}x{c[1]}x{c[2]}-{c[3]}-r{c[4][0]}x{len(c[4])}")
@pytest.mark.parametrize("order", ["mixed", "runs"])
def test_matmul_lora_many_rows(be, case, order):
    test_matmul_lora(be, case, order)


@pytest.mark.parametrize("M", [300, 600])
def test_many_rows_each_way(be, M):
    test_rows_of_any_magnitude(be, M)
    test_ids_out_of_range_and_no_adapters(be, M)
    test_a_row_that_is_not_finite_stays_alone(be, M)
    for bad in (math.nan, math.inf):
        test_an_adapter_that_is_not_finite_stays_alone(be, M, bad)
    test_output_at_any_address(be, M)
    test_an_adapter_of_misaligned_rows_is_reported(be, M)
    test_first_call_inside_a_capture(M)


def test_long_rows_of_few_and_many(be):
    """K above what the many-rows kernels take: the few-rows ones up to 256 rows, a refusal behind."""
    from ternative_b200 import TvbError
    p = Projection(16400, 3000, "f16", [4], F32, seed=9)
    x = torch.randn(40, 16400, generator=torch.Generator().manual_seed(1))
    ids = torch.zeros(40, dtype=torch.long)
    ref, tol = p(x, ids)
    y = project(be, p, x.cuda(), ids.to(torch.int32).cuda()).cpu().double()
    assert ((y - ref).abs() <= tol).all()
    with pytest.raises(TvbError, match="16384"):
        project(be, p, torch.zeros(257, 16400, device="cuda"), torch.zeros(257, dtype=torch.int32, device="cuda"))
