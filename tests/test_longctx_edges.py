"""What the long-context entry points and the host functions over them refuse or promise, beyond test_longctx_refusals.py:
no GPU is needed, the addresses are never used."""
import ctypes as C

import pytest

from deusridet_amd import cabi, host
from tests.test_longctx_refusals import P, code, lay, rope_code


# ---- what the attention takes ------------------------------------------------------------------
def test_the_check_says_what_the_attention_would():
    def check(g=None, T=1, keep=64, io=cabi.BF16):
        return code("drk_paged_sparse_check", g or lay(), T, keep, io)

    assert check() == check(lay(dtype=cabi.INT8), io=cabi.F16) == check(keep=32768) == cabi.OK
    for g in (lay(D=64), lay(bs=8), lay(QH=136), lay(NB=2 ** 21)):
        assert check(g) == cabi.ERR_UNSUPPORTED
    assert check(keep=32769) == check(lay(bs=256), keep=2049) == check(T=2 ** 30) == cabi.ERR_UNSUPPORTED
    assert check(T=-1) == check(keep=0) == check(io=cabi.F16) == check(io=cabi.INT8) == cabi.ERR_INVALID


def host_bytes(rows, length, keep, nb=8192, bs=256):
    return host.lib().drkh_paged_sparse_workspace_bytes(rows, length, keep, nb, bs)


@pytest.mark.parametrize("rows", [1, 4, 600])
def test_no_workspace_for_lists_that_the_attention_refuses(rows):
    """A budget of more than 524 288 tokens a row: 0, although the selection by itself would have its bytes."""
    assert host.set_attention_geometry(2, 24, 4, 256, cabi.BF16)
    g = cabi.layout(2, 4, 24, 256, 256, 8192, cabi.BF16)
    assert host_bytes(rows, 262144, 2048) >= cabi.lib().drk_block_select_workspace_bytes(C.byref(g), rows, 262144) > 0
    assert host_bytes(rows, 262144, 2049) == host_bytes(rows, 262144, 2 ** 20) == 0
    assert host_bytes(rows, 1, 2049) == 0                               # the context's length does not matter
    assert host_bytes(rows, 262144, 2048, nb=2 ** 19) == 0              # a layer of more than 64 GiB
    assert host_bytes(rows, 262144, 0) == host_bytes(0, 262144, 64) == host_bytes(rows, 0, 64) == 0


def test_16_bit_pages_of_another_type_than_the_queries_are_not_supported():
    assert host.set_attention_geometry(2, 32, 8, 128, cabi.BF16, cabi.F16)
    assert not host.lib().drkh_paged_sparse_attention_supported(16) and host_bytes(1, 4096, 64, 512, 16) == 0
    for kv, io in ((cabi.BF16, cabi.BF16), (cabi.F16, cabi.F16), (cabi.INT8, cabi.F16), (cabi.FP8_E4M3, cabi.BF16)):
        assert host.set_attention_geometry(2, 32, 8, 128, kv, io)
        assert host.lib().drkh_paged_sparse_attention_supported(16) and host_bytes(1, 4096, 64, 512, 16) > 0
        assert not any(host.lib().drkh_paged_sparse_attention_supported(b) for b in (0, 8, 24, -16))


# ---- rotary positions ----------------------------------------------------------------------------
def test_rope_refuses_tensors_of_which_one_reads_what_another_writes():
    row = lambda x, out: (x * P, out * P, 8, 1024, 128, 1024, 128)
    for rows in ([row(1, 2), row(2, 3)], [row(2, 3), row(1, 2)], [row(1, 2), row(2, 1)], [row(1, 1), row(1, 2)], [row(1, 2), row(1, 1)],
                 [row(1, 2), row(3, 4), row(5, 1)]):
        assert rope_code(rows=rows) == cabi.ERR_INVALID, rows
        assert b"reads what" in cabi.lib().drk_last_error()
    none = (P, 2 * P, 0, 1024, 128, 1024, 128)                              # without heads nothing is read or written
    assert rope_code(rows=[none, (2 * P, 2 * P, 0, 0, 0, 0, 0)]) == cabi.OK
    assert rope_code(rows=[row(1, 2), row(1, 3)], T=0) == cabi.OK           # two readers of one tensor


def test_the_host_functions_take_no_missing_description():
    """NULL for a description: refused (an uninitialised driver and no tensors: nothing is launched either way)."""
    h = host.lib()
    h.drkh_apply_rope_scaled(None, P, P, P, 1, 8, 2, 128, None, 0, 0, None)
    assert host.KvStream().set_scaled_rope(None) is False
