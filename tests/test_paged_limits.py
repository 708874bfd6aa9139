"""Sizes of the paged operators at which a position would leave 32 bits are refused,
before any device work."""
import pytest

from test_paged import append, attention, batch, cache, lib   # noqa: F401  (lib: the fixture)


@pytest.mark.parametrize("call", [attention, append])
@pytest.mark.parametrize("max_kv,ok", [(2 ** 30 + 1, False), (2 ** 31 - 1, False), (2 ** 30, True)])
def test_positions_stay_in_32_bits(lib, call, max_kv, ok):   # noqa: F811
    """The kernels step from key to key behind the longest sequence before they stop.  (A refusal of the heads tells
    that the length passed.)"""
    kv, bt = cache(page_size=1 << 20), batch(max_kv=max_kv, table_ld=1 << 11)
    st, msg = call(lib, kv, bt, **({"ldq": 8} if ok else {}))
    assert st == 1 and (b"leading" in msg if ok else b"max_kv" in msg), msg
