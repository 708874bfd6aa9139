"""CPU tests of the paged operators' refusals: every bad argument is turned away
with a status and a message before any device work."""
import ctypes as C

import pytest

P = 4096   # a 16-byte aligned address that nothing reads


def desc(cls, **kw):
    d = cls()
    for k, v in kw.items():
        setattr(d, k, v)
    return d


@pytest.fixture(scope="module")
def lib():
    from ternative_b200 import load
    return load()


def cache(**kw):
    from ternative_b200._lib import KvPages
    return desc(KvPages, **(dict(k=P, v=P, dtype=1, n_pages=10, page_size=16, page_stride=16 * 2 * 128,
                                 row_stride=2 * 128, head_stride=128) | kw))


def batch(**kw):
    from ternative_b200._lib import PagedBatchDesc
    return desc(PagedBatchDesc, **(dict(n_seqs=2, n_tokens=2, max_new=1, max_kv=100, cu_tokens=P, kv_len=P, block_table=P,
                                        table_ld=7) | kw))


def rope(**kw):
    from ternative_b200._lib import RopeDesc
    return desc(RopeDesc, **(dict(rot_dim=128, pairs=0, scaling=0, theta=1e4, factor=2.0, original_len=4096, low_turns=1.0,
                                  high_turns=4.0, fast_turns=32.0, slow_turns=1.0) | kw))


def attention(lib, kv=None, bt=None, **kw):
    a = dict(out=P, ldo=512, lse=None, q=P, ldq=512, nh=4, nkv=2, hd=128, scale=0.1, window=0) | kw
    st = lib.tvb_attention_paged(a["out"], a["ldo"], a["lse"], a["q"], a["ldq"], C.byref(kv or cache()),
                                 C.byref(bt or batch()), a["nh"], a["nkv"], a["hd"], a["scale"], a["window"], None, None)
    return st, lib.tvb_last_error()


def append(lib, kv=None, bt=None, rp=None, **kw):
    a = dict(qo=P, ldqo=512, q=P, ldq=512, k=P, ldk=256, v=P, ldv=256, nh=4, nkv=2, hd=128) | kw
    st = lib.tvb_rope_append_paged(a["qo"], a["ldqo"], a["q"], a["ldq"], a["k"], a["ldk"], a["v"], a["ldv"],
                                   C.byref(kv or cache()), C.byref(bt or batch()), C.byref(rp or rope()), a["nh"], a["nkv"],
                                   a["hd"], None, None)
    return st, lib.tvb_last_error()


BOTH = [
    (dict(kv=dict(k=None)), b"null"), (dict(kv=dict(dtype=2)), b"dtype"), (dict(kv=dict(n_pages=0)), b"pages"),
    (dict(kv=dict(page_size=0)), b"pages"), (dict(kv=dict(row_stride=120)), b"stride"),
    (dict(kv=dict(head_stride=64)), b"stride"), (dict(kv=dict(page_stride=-1)), b"stride"),
    (dict(kv=dict(row_stride=2 * 128 + 4)), b"16 bytes"), (dict(kv=dict(v=P + 8)), b"16 bytes"),
    (dict(bt=dict(cu_tokens=None)), b"null"), (dict(bt=dict(n_seqs=-1)), b"sequences"),
    (dict(bt=dict(n_seqs=70000)), b"sequences"), (dict(bt=dict(max_kv=-1)), b"max_kv"),
    (dict(bt=dict(max_kv=113)), b"max_kv"), (dict(bt=dict(max_new=-2)), b"max_new"),
    (dict(q=None), b"null"), (dict(q=P + 4), b"aligned"), (dict(ldq=508), b"leading"), (dict(ldq=514), b"leading"),
    (dict(nh=0), b"heads"), (dict(nkv=0), b"heads"),
]


@pytest.mark.parametrize("bad,word", BOTH, ids=str)
@pytest.mark.parametrize("call", [attention, append])
def test_refusals_of_both(lib, call, bad, word):
    kw = dict(bad)
    if "kv" in kw:
        kw["kv"] = cache(**kw["kv"])
    if "bt" in kw:
        kw["bt"] = batch(**kw["bt"])
    st, msg = call(lib, **kw)
    assert st == 1 and word in msg, msg


@pytest.mark.parametrize("bad,word", [
    (dict(out=None), b"null"), (dict(ldo=500), b"leading"), (dict(hd=96), b"head_dim"), (dict(nh=5), b"heads"),
    (dict(window=-1), b"window"), (dict(scale=float("nan")), b"scale"),
], ids=str)
def test_attention_refusals(lib, bad, word):
    st, msg = attention(lib, **bad)
    assert st == 1 and word in msg, msg


@pytest.mark.parametrize("bad,word", [
    (dict(hd=132), b"head_dim"), (dict(hd=264), b"head_dim"), (dict(ldk=252), b"leading"), (dict(v=P + 4), b"aligned"),
    (dict(ldqo=516), b"in place"),
    (dict(rp=dict(rot_dim=136)), b"rot_dim"), (dict(rp=dict(rot_dim=12)), b"rot_dim"), (dict(rp=dict(pairs=2)), b"pairs"),
    (dict(rp=dict(scaling=4)), b"scaling"), (dict(rp=dict(theta=1.0)), b"theta"),
    (dict(rp=dict(theta=float("inf"))), b"theta"), (dict(rp=dict(scaling=1, factor=0.5)), b"factor"),
    (dict(rp=dict(scaling=2, original_len=0)), b"original_len"), (dict(rp=dict(scaling=2, high_turns=1.0)), b"turns"),
    (dict(rp=dict(scaling=3, fast_turns=0.5)), b"turns"),
], ids=str)
def test_rope_refusals(lib, bad, word):
    kw = dict(bad)
    if "rp" in kw:
        kw["rp"] = rope(**kw["rp"])
    st, msg = append(lib, **kw)
    assert st == 1 and word in msg, msg


def lora(lib, t=None, w=None, **kw):
    from ternative_b200._lib import LoraTableDesc, Weight
    a = dict(y=P, x=P, M=2, K=256, N=64, adapter=P) | kw
    table = desc(LoraTableDesc, **(dict(n=1, max_rank=16, dtype=0, A=P, B=P, rank=P, scale=P) | (t or {})))
    weight = desc(Weight, **(dict(w=P, dtype=1) | (w or {})))
    st = lib.tvb_matmul_lora(a["y"], a["x"], a["M"], a["K"], C.byref(weight), a["N"], C.byref(table), a["adapter"],
                             None, None)
    return st, lib.tvb_last_error()


@pytest.mark.parametrize("bad,word", [
    (dict(y=None), b"null"), (dict(x=P + 4), b"aligned"), (dict(w=dict(w=P + 8)), b"aligned"), (dict(w=dict(w=None)), b"null"),
    (dict(w=dict(dtype=0)), b"dtype"), (dict(w=dict(dtype=2)), b"row_scales"), (dict(K=252), b"multiple of 8"),
    (dict(K=264, w=dict(dtype=3, tensor_scale=1.0)), b"multiple of 16"), (dict(M=-1), b"shape"), (dict(N=0), b"shape"),
    (dict(M=70000), b"rows"), (dict(adapter=None), b"null"), (dict(t=dict(A=None)), b"null"), (dict(t=dict(n=-1)), b"adapters"),
    (dict(t=dict(max_rank=257)), b"max_rank"), (dict(t=dict(max_rank=-1)), b"max_rank"), (dict(t=dict(dtype=2)), b"dtype"),
], ids=str)
def test_lora_refusals(lib, bad, word):
    st, msg = lora(lib, **bad)
    assert st == 1 and word in msg, msg


def test_nothing_to_do(lib):
    """Empty calls succeed without a GPU."""
    assert attention(lib, bt=batch(n_tokens=0))[0] == 0
    assert attention(lib, bt=batch(n_seqs=0, cu_tokens=None, kv_len=None, block_table=None))[0] == 0
    assert append(lib, bt=batch(n_tokens=0))[0] == 0
    assert lora(lib, M=0)[0] == 0


def test_python_checks():
    """The Python layer's own checks of types, shapes and devices."""
    import torch
    from ternative_b200 import LoraTable, PagedBatch, PagedCache, RopeConfig
    z = torch.zeros(4, 16, 2, 64)
    with pytest.raises(ValueError, match="current CUDA device"):
        PagedCache(z, z)
    with pytest.raises(ValueError, match="cache type"):
        PagedCache(z.double(), z.double())
    i = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(ValueError, match="current CUDA device"):
        PagedBatch(i, i[:2], i[:2, None], 1, 1, 1)
    with pytest.raises(ValueError, match="pairs"):
        RopeConfig(64, pairs="quarter")
    with pytest.raises(ValueError, match="2 A and 1 B"):
        LoraTable([z, z], [z], i, i, 4)
    with pytest.raises(ValueError, match="adapter type"):
        LoraTable([z.double()], [z.double()], i, i, 4)


def test_lora_long_rows_of_many_are_refused(lib):
    st, msg = lora(lib, M=257, K=16400)
    assert st == 1 and b"16384" in msg, msg
