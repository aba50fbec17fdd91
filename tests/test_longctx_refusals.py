"""What the long-context entry points refuse, before anything is launched: no GPU is needed and the addresses are
never used.  Also the byte counts, and the definitions' own edge cases in the plain statements the GPU tests use."""
import ctypes as C

import numpy as np
import pytest

from deusridet_amd import cabi
from tests import longctx_ref as R

P = 0x10000                                                    # 16-byte aligned, never dereferenced
G = dict(L=2, KVH=8, QH=32, D=128, bs=16, NB=64, dtype=cabi.BF16)


def lay(**kw):
    d = dict(G, **kw)
    return cabi.layout(d["L"], d["KVH"], d["QH"], d["D"], d["bs"], d["NB"], d["dtype"])


def code(name, *args):
    rc = getattr(cabi.lib(), name)(*args)
    if rc:
        assert cabi.lib().drk_last_error(), name
    return rc


def rope_code(r=None, freqs=P, rows=None, n=None, T=4, D=128, pos=None, start=0, inverse=0, dtype=cabi.BF16):
    rows = rows if rows is not None else [(P, P, 8, 1024, 128, 1024, 128)]
    return code("drk_rope_apply", r or cabi.rope(64), freqs, cabi.rope_rows(rows), len(rows) if n is None else n, T, D, pos, start, inverse,
                dtype, None)


def test_rope_refusals():
    ok = cabi.rope(64)
    for bad in (cabi.rope(8), cabi.rope(24), cabi.rope(0)):
        assert rope_code(bad) == cabi.ERR_UNSUPPORTED
    assert rope_code(cabi.rope(144)) == cabi.ERR_UNSUPPORTED                   # longer than the head
    inf, nan = float("inf"), float("nan")
    for bad in (cabi.rope(64, theta=0.0), cabi.rope(64, theta=nan), cabi.rope(64, theta=inf), cabi.rope(64, factor=0.0),
                cabi.rope(64, factor=-2.0), cabi.rope(64, factor=inf), cabi.rope(64, magnitude=nan), cabi.Rope(64, 2, 1e4, 1, 0, 1, 32, 1),
                cabi.rope(64, factor=2.0, low_turns=4.0, high_turns=4.0), cabi.rope(64, factor=2.0, low_turns=-1.0),
                cabi.rope(64, factor=2.0, original_positions=nan), cabi.rope(64, factor=2.0, high_turns=inf)):
        assert rope_code(bad) == cabi.ERR_INVALID
        assert code("drk_rope_freqs_fill", bad, P, None) == cabi.ERR_INVALID
        assert code("drk_rope_table_fill_scaled", bad, P, 5, None) == cabi.ERR_INVALID
    assert rope_code(ok, D=120) == rope_code(ok, D=1040) == rope_code(ok, D=0) == cabi.ERR_UNSUPPORTED
    assert rope_code(ok, dtype=cabi.INT8) == rope_code(ok, freqs=None) == rope_code(ok, n=0) == rope_code(ok, n=5) == cabi.ERR_INVALID
    assert rope_code(ok, T=-1) == rope_code(ok, start=-1) == cabi.ERR_INVALID
    for rows in ([(P + 8, P, 8, 1024, 128, 1024, 128)], [(P, P + 2, 8, 1024, 128, 1024, 128)], [(P, P, 8, 1024, 132, 1024, 132)],
                 [(P, P, 8, 1024, 128, 2048, 128)], [(P, 2 * P, 8, 1024, 128, 1024, 64)], [(None, P, 8, 1024, 128, 1024, 128)],
                 [(P, None, 1, 128, 128, 128, 128)], [(P, P, -1, 0, 0, 0, 0)]):
        assert rope_code(ok, rows=rows) == cabi.ERR_INVALID, rows
    assert rope_code(ok, T=0) == cabi.OK and rope_code(ok, rows=[(None, None, 0, 0, 0, 0, 0)]) == cabi.OK
    assert code("drk_rope_freqs_fill", ok, None, None) == cabi.ERR_INVALID
    assert code("drk_rope_table_fill_scaled", ok, P, 0, None) == cabi.ERR_INVALID
    assert code("drk_rope_table_fill_scaled", cabi.rope(64, True), P, 5, None) == cabi.ERR_UNSUPPORTED


def test_rope_refuses_rows_that_two_threads_would_write():
    ok = cabi.rope(64)
    for rows in ([(P, 2 * P, 8, 1024, 128, 512, 128)],                         # tokens inside one another's heads
                 [(P, 2 * P, 1, 128, 128, 0, 0)], [(P, 2 * P, 1, 128, 128, 120, 128)],
                 [(P, 2 * P, 8, 128, 512, 128, 384)],                          # heads inside one another's tokens
                 [(P, P, 8, 1024, 128, 1024, 128), (P, P, 8, 1024, 128, 1024, 128)],
                 [(P, 2 * P, 8, 1024, 128, 1024, 128), (3 * P, 2 * P, 2, 256, 128, 256, 128)]):
        assert rope_code(ok, rows=rows) == cabi.ERR_INVALID, rows


def test_bounds_refusals_and_bytes():
    L = cabi.lib()
    for kw in (dict(), dict(D=512, dtype=cabi.INT8), dict(D=64, bs=7, KVH=3, QH=3)):
        g = lay(**kw)
        n = g.num_layers * g.max_phys_blocks * g.num_kv_heads
        assert L.drk_kv_bounds_bytes(C.byref(g)) == (n * (2 * g.head_dim + 1) + 15) // 16 * 16
    for D in (32, 96, 192, 1024):
        assert L.drk_kv_bounds_bytes(C.byref(lay(D=D))) == 0

    def up(g=None, pool=P, tab=P, stride=64, pos=None, start=0, n=5, layer=0, count=1, bounds=P):
        return code("drk_kv_bounds_update", g or lay(), pool, tab, stride, pos, start, n, layer, count, bounds, None)

    assert up(lay(D=96)) == cabi.ERR_UNSUPPORTED
    assert up(pool=None) == up(tab=None) == up(bounds=None) == up(pool=P + 4) == up(bounds=P + 8) == cabi.ERR_INVALID
    assert up(n=-1) == up(start=-1) == up(stride=-1) == up(start=2 ** 31 - 2) == cabi.ERR_INVALID
    assert up(layer=2) == up(layer=-1) == up(layer=1, count=2) == up(count=-1) == cabi.ERR_INVALID
    assert up(n=0) == up(count=0) == cabi.OK

    def ex(g=None, dst=P, bounds=P, blocks=P, n=3, layer=0, count=1):
        return code("drk_kv_bounds_extract", g or lay(), dst, bounds, blocks, n, layer, count, None)

    assert ex(lay(D=80)) == cabi.ERR_UNSUPPORTED
    assert ex(dst=None) == ex(bounds=None) == ex(blocks=None) == ex(dst=P + 2) == ex(n=-1) == ex(layer=2) == ex(count=3) == cabi.ERR_INVALID
    assert ex(n=0) == cabi.OK


def test_select_refusals_and_bytes():
    L = cabi.lib()
    need = L.drk_block_select_workspace_bytes(C.byref(lay()), 3, 1000)
    assert need == 3 * 8 * 64 * 4                                              # 63 blocks, a multiple of four
    assert L.drk_block_select_workspace_bytes(C.byref(lay(D=96)), 3, 1000) == 0

    def sel(g=None, bounds=P, layer=0, q=P, io=cabi.BF16, tab=P, stride=64, lens=P, start=0, T=3, most=1000, keep=8, sink=1, recent=2,
            out=P, ws=P, wsb=need):
        return code("drk_block_select", g or lay(), bounds, layer, q, io, tab, stride, lens, start, T, most, keep, sink, recent, out, ws, wsb, None)

    assert sel(lay(D=96)) == sel(lay(QH=136)) == cabi.ERR_UNSUPPORTED
    assert sel(io=cabi.INT8) == sel(layer=2) == sel(layer=-1) == sel(T=-1) == sel(most=-1) == sel(stride=-1) == sel(start=-1) == cabi.ERR_INVALID
    assert sel(lens=None, start=2 ** 31 - 2) == cabi.ERR_INVALID
    assert sel(keep=0) == sel(sink=-1) == sel(recent=-1) == sel(sink=6, recent=3) == sel(sink=9) == cabi.ERR_INVALID
    assert sel(sink=2 ** 31 - 1, recent=2 ** 31 - 1) == cabi.ERR_INVALID
    assert sel(bounds=None) == sel(q=None) == sel(tab=None) == sel(out=None) == sel(q=P + 8) == sel(bounds=P + 1) == sel(ws=P + 4) == cabi.ERR_INVALID
    assert sel(wsb=need - 1) == sel(ws=None) == cabi.ERR_WORKSPACE
    assert sel(T=0) == cabi.OK


def test_attention_refusals_and_bytes():
    L = cabi.lib()

    def ws(g, T, keep):
        return L.drk_paged_sparse_workspace_bytes(C.byref(g), T, keep)

    need = ws(lay(), 1, 64)
    assert need and need % (32 * 130 * 4) == 0 and ws(lay(), 4096, 64) == 0
    assert ws(lay(), 0, 64) == ws(lay(D=64), 1, 64) == ws(lay(), 1, 0) == 0

    def at(g=None, q=P, pool=P, tab=P, stride=64, lens=P, start=0, T=1, s=P, keep=64, out=P, layer=0, scale=0.1, io=cabi.BF16, gate=None,
           gst=0, w=P, wsb=need):
        return code("drk_paged_sparse_attention", g or lay(), q, pool, tab, stride, lens, start, T, s, keep, out, layer, scale, io, gate, gst,
                    w, wsb, None)

    for g in (lay(D=64), lay(bs=8), lay(bs=24), lay(QH=136), lay(D=512)):
        assert at(g) == cabi.ERR_UNSUPPORTED
    assert at(lay(NB=2 ** 21)) == cabi.ERR_UNSUPPORTED                         # a layer of 128 GiB
    assert at(keep=2 ** 20) == cabi.ERR_UNSUPPORTED
    assert at(io=cabi.F16) == at(io=cabi.INT8) == at(layer=2) == at(layer=-1) == at(scale=0.0) == at(scale=float("nan")) == cabi.ERR_INVALID
    assert at(T=-1) == at(keep=0) == at(stride=-1) == at(start=-1) == at(lens=None, start=2 ** 31 - 1) == cabi.ERR_INVALID
    assert at(q=None) == at(pool=None) == at(tab=None) == at(s=None) == at(out=None) == cabi.ERR_INVALID
    assert at(q=P + 2) == at(out=P + 2) == at(pool=P + 8) == at(w=P + 4) == cabi.ERR_INVALID
    assert at(gate=P, gst=64) == at(gate=P, gst=132) == at(gate=P + 8, gst=128) == cabi.ERR_INVALID
    assert at(wsb=need - 1) == at(w=None) == cabi.ERR_WORKSPACE
    assert at(T=0) == cabi.OK


@pytest.mark.parametrize("amax,e", [(0.0, -40), (127.0, 0), (127.0000001, 1), (128.0, 1), (254.0, 1), (255.0, 2), (0.5, -7), (1e-30, -40), (1e30, 40),
                                    (float("inf"), 40)])
def test_the_exponent_of_a_bound(amax, e):
    assert R.exponent(amax) == e


def test_the_score_is_an_upper_bound_of_the_dot_product():
    """Without the query's rounding, every key of a block scores at most the block's bound."""
    rng = np.random.default_rng(0)
    k = rng.standard_normal((16, 64)) * rng.random(64) * 3
    lo, hi, e = R.bounds(k)
    for _ in range(20):
        q = rng.integers(-127, 128, 64).astype(np.float64)
        assert (k @ q).max() <= np.maximum(q * lo, q * hi).sum() * 2.0 ** e
