"""GPU: calls of the long-context operators at the edges of what their definitions allow."""
import ctypes as C
import math

import numpy as np
import pytest

from deusridet_amd import cabi, host
from tests import longctx_ref as R
from tests import test_gpu_longctx as G
from tests import test_gpu_stream as S
from tests import test_gpu_stream_sparse as SP
from tests import util as U
from tests.test_gpu_stream import eight_bit_pages  # noqa: F401 (a fixture: it changes the pages' type of S)

pytestmark = pytest.mark.gpu


# ---- bounds -----------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [cabi.BF16, cabi.INT8])
@pytest.mark.parametrize("bs", [16, 48])
def test_bounds_of_branches_over_one_table(dev, dtype, bs):
    """Positions of one table (stride 0): every one's block gets its bounds; a negative position and a hole are skipped."""
    rng = np.random.default_rng(bs)
    NBL = 9
    p = R.Pool(rng, 2, 2, 4, 128, bs, NBL + 2, dtype)
    table = U.shuffled_table(rng, p.NB, NBL)
    table[5] = -1
    pos = np.array([3, 2 * bs - 1, -1, 5 * bs + 2, 8 * bs], np.int32)
    db, dp, dt, dpos = G.bounds_dev(p), U.dev_bytes(p.raw), U.dev_i32(table), U.dev_i32(pos)
    db.fill_(0x55)
    cabi.call("drk_kv_bounds_update", p.g, U.p(dp), U.p(dt), 0, U.p(dpos), 0, len(pos), 0, 2, U.p(db), U.stream_ptr())
    U.sync()
    codes, exps = G.bounds_host(p, db)
    written = {int(table[x // bs]): x % bs + 1 for x in map(int, pos) if x >= 0 and table[x // bs] >= 0}
    assert len(written) == 3
    for blk in range(p.NB):
        for layer in range(2):
            if blk in written:
                G.check_block(p, codes, exps, layer, blk, written[blk])
            else:
                assert (codes[layer, blk] == 0x55).all() and (exps[layer, blk] == 0x55).all()


@pytest.mark.parametrize("start", [0, 37, 6 * 16, 19 * 16])
@pytest.mark.parametrize("bs", [16, 48])
def test_bounds_of_a_chunk_end_with_its_table(dev, start, bs):
    """With a table length, entries behind it are not read: their blocks keep what the buffer held."""
    rng = np.random.default_rng(start + bs)
    NBL, stride = 20, 6
    p = R.Pool(rng, 1, 2, 4, 128, bs, NBL, cabi.BF16)
    table = U.shuffled_table(rng, NBL, NBL)
    db, dp, dt = G.bounds_dev(p), U.dev_bytes(p.raw), U.dev_i32(table)
    db.fill_(0x55)
    cabi.call("drk_kv_bounds_update", p.g, U.p(dp), U.p(dt), stride, None, start, 20 * bs - start - 3, 0, 1, U.p(db), U.stream_ptr())
    U.sync()
    codes, exps = G.bounds_host(p, db)
    for lb in range(NBL):
        if start // bs <= lb < stride:
            G.check_block(p, codes, exps, 0, table[lb], bs)
        else:
            assert (codes[0, table[lb]] == 0x55).all() and (exps[0, table[lb]] == 0x55).all()


@pytest.mark.parametrize("dtype", G.DTYPES)
@pytest.mark.parametrize("D,bs,NBL", [(64, 48, 150), (128, 64, 180), (64, 256, 280), (256, 40, 240)])
def test_bounds_of_many_long_blocks(dev, dtype, D, bs, NBL):
    """Blocks above 32 tokens in such numbers that a thread walks every row of its columns; the last one is cut."""
    rng = np.random.default_rng(D + bs)
    p = R.Pool(rng, 2, 4, 4, D, bs, NBL, dtype)
    assert 2 * 4 * NBL * 16 > bs * D * (1 if dtype in (cabi.INT8, cabi.FP8_E4M3) else 2)
    table = U.shuffled_table(rng, NBL, NBL)
    last = bs - 5
    for layer in range(2):
        p.poison(layer, table[-1], last)
    db, dp, dt = G.bounds_dev(p), U.dev_bytes(p.raw), U.dev_i32(table)
    cabi.call("drk_kv_bounds_update", p.g, U.p(dp), U.p(dt), NBL, None, 0, NBL * bs - 5, 0, 2, U.p(db), U.stream_ptr())
    U.sync()
    codes, exps = G.bounds_host(p, db)
    for lb in (0, 1, 2, 37, NBL // 2, NBL - 2, NBL - 1):
        for layer in range(2):
            G.check_block(p, codes, exps, layer, table[lb], bs if lb < NBL - 1 else last)


# ---- attention --------------------------------------------------------------------------------
class SinkPages:
    """Pages of one kv head in which the first token's key leads every other score by about `lead`, with a value of the
    other sign: k, v float64 [NB, bs, D] of the stored numbers, vs [NB, bs] the V scales (int8), raw bytes."""

    def __init__(self, rng, dtype, lead, vmag, NB=9, bs=256, D=128, QH=4):
        self.dtype, self.NB, self.bs, self.D, self.QH = dtype, NB, bs, D, QH
        self.io = dtype if dtype in (cabi.F16, cabi.BF16) else cabi.F16
        base = rng.standard_normal(D)
        self.q = U.to_bits((base * (1 - 0.02 * np.arange(QH)[:, None])).astype(np.float32), self.io)
        k = rng.standard_normal((NB, bs, D)) * 0.05
        k[0, 0] = base * lead * math.sqrt(D) / (base ** 2).sum()
        if vmag == "mixed":                                    # scales over 2^20 within one list
            vmag = 2.0 ** rng.uniform(-20, 0, (NB, bs, 1)) * 127
            vmag[0, 0] = 2.0 ** -10 * 127
        v = (0.5 + 0.5 * rng.random((NB, bs, D))) * vmag
        v[0, 0] *= -1
        self.vs = np.ones((NB, bs))
        kv = np.stack([k, v], 1)                               # [NB, 2, bs, D]
        if dtype in (cabi.F16, cabi.BF16):
            bits = U.to_bits(kv.astype(np.float32), dtype)
            kv, raw = U.from_bits(bits, dtype).astype(np.float64), bits.view(np.uint8)
        elif dtype == cabi.INT8:
            sc = (np.abs(kv).max(3) / 127).astype(np.float16)
            scale = sc.astype(np.float64)
            codes = np.clip(np.rint(kv / scale[..., None]), -127, 127).astype(np.int8)
            kv, self.vs = codes * scale[..., None], scale[:, 1]
            raw = np.concatenate([codes.view(np.uint8).reshape(NB, -1), sc.view(np.uint8).reshape(NB, -1)], 1)
        else:
            import torch
            t = torch.from_numpy(kv.astype(np.float32)).to(torch.float8_e4m3fn)
            kv, raw = t.double().numpy(), t.view(torch.uint8).numpy()
        self.k, self.v, self.raw = kv[:, 0], kv[:, 1], np.ascontiguousarray(raw)
        self.g = cabi.layout(1, 1, QH, D, bs, NB, dtype)

    def want(self, sel, chain):
        """Every listed token counted as often as its block is listed -> (out [QH, D], bound on what a kernel may be off by
        before its last rounding): the weights' rounding to 16 bits, u (A + |out|) as in longctx_ref.attend; what a weight
        below fp16's normal range loses, 2^-25 where the largest is 2^14; the scores' fp32 sums (int8: twenty times, as
        there) and 2^-20 of the exponential, twice; `chain` dependent fp32 additions of the output."""
        cnt = np.bincount(sel, minlength=self.NB).astype(np.float64)[:, None]
        scale = 1 / math.sqrt(self.D)
        out, tol = np.zeros((self.QH, self.D)), np.zeros((self.QH, self.D))
        u = R.HALF_STEP[cabi.BF16 if self.dtype == cabi.BF16 else cabi.F16]
        for i, q in enumerate(U.from_bits(self.q, self.io).astype(np.float64)):
            s = self.k @ q * scale
            p = cnt * np.exp(s - s[cnt[:, 0] > 0].max())
            L = p.sum()
            mean = lambda x: np.tensordot(p, x, 2) / L
            o, A = mean(self.v), mean(np.abs(self.v))
            one = np.exp(s - s[cnt[:, 0] > 0].max())
            ds = (self.D + 8) * 2.0 ** -24 * (np.abs(self.k) @ np.abs(q))[cnt[:, 0] > 0].max() * scale
            if self.dtype == cabi.INT8:
                ds *= 20
                wide = mean(self.vs)[None] * 1279
                lost = (one * self.vs)[cnt[:, 0] > 0].max() * 127
            else:
                wide, lost = A, np.abs(self.v).max() + np.abs(o)
            tail = 0.0 if self.dtype == cabi.BF16 else 1.01 * 2.0 ** -39 * cnt.sum() * self.bs * lost / L
            out[i], tol[i] = o, u * (A + np.abs(o)) + tail + 2 * (ds + 2.0 ** -20) * A + chain * 2.0 ** -24 * wide
        return out, tol


@pytest.mark.parametrize("dtype,vmag,lead,keep,T", [
    (cabi.INT8, 0.01, 8, 16, 1), (cabi.INT8, 0.002, 8, 16, 1), (cabi.INT8, 0.01, 8, 16, 1100),
    (cabi.INT8, 0.002, 8, 16, 1100), (cabi.INT8, 30.0, 8, 16, 1),
    (cabi.INT8, "mixed", 8, 16, 1), (cabi.INT8, "mixed", 8, 16, 1100), (cabi.F16, 1.0, 18, 2048, 1), (cabi.F16, 1.0, 18, 128, 1100),
    (cabi.FP8_E4M3, 1.0, 18, 2048, 1), (cabi.BF16, 1.0, 18, 2048, 1)])
def test_small_weights_beside_a_dominating_token_count(dev, dtype, vmag, lead, keep, T):
    """A token that leads by many nats, and thousands whose weights -- int8: weight times V scale -- lie where fp16 ends:
    together they hold a share of the output, and must not vanish in the product while the sum counts them."""
    rng = np.random.default_rng(keep + T)
    p = SinkPages(rng, dtype, lead, vmag)
    sel = rng.integers(1, p.NB, keep).astype(np.int32)
    sel[keep // 3] = 0
    sels, q = np.tile(sel, (T, 1, 1)), np.tile(p.q, (T, 1, 1))
    need = cabi.lib().drk_paged_sparse_workspace_bytes(C.byref(p.g), T, keep)
    pieces = need // (T * p.QH * (p.D + 2) * 4) or 1
    groups = keep * (p.bs // 16)
    chain = 16 * math.ceil(groups / pieces / (8 if T == 1 else 1)) + 8 + pieces
    want, tol = p.want(sel, chain)
    do, dq, dp, dt, ds = U.dev_zeros(q.nbytes), U.dev_bytes(q), U.dev_bytes(p.raw), U.dev_i32(np.arange(p.NB)), U.dev_i32(sels)
    ws = U.dev_zeros(need + 16)
    cabi.call("drk_paged_sparse_attention", p.g, U.p(dq), U.p(dp), U.p(dt), 0, None, p.NB * p.bs - 1, T, U.p(ds), keep, U.p(do), 0,
              1 / math.sqrt(p.D), p.io, None, 0, U.p(ws), need, U.stream_ptr())
    U.sync()
    got = U.from_bits(U.host(do, np.uint16, q.shape), p.io)
    for t in {0, T // 2, T - 1}:
        ok, r = R.attend_ok(got[t], want, tol, p.io)
        assert ok, (t, r)


# ---- through the host functions and the stream driver --------------------------------------------
def test_the_driver_refuses_a_budget_that_the_attention_refuses(dev):
    """More than 524 288 tokens a row: refused, and the policy in force stays as it is."""
    s = S.Session(2)
    st = U.stream_ptr()
    most = 524288 // S.BS
    assert not s.ks.set_sparse_decode(0, most + 1, 1, 2, st) and not s.ks.set_sparse_decode(0, 2 ** 30, 1, 2, st)
    rng = np.random.default_rng(3)
    s.set_weights(U.normal_bits(rng, (S.D,), S.DT), U.normal_bits(rng, (S.D,), S.DT))
    assert s.ks.set_sparse_decode(0, 3, 1, 1, st)
    SP.prefill(s, rng, (64, 50))
    assert s.ks.open_branches(2) == 2
    ids = [s.ks.branch_id(i) for i in range(2)]
    for step in range(2):
        assert not s.ks.set_sparse_decode(0, most + 1, 0, 0, st)
        assert s.ks.begin_decode_step(st)
        pos = [s.ks.branch_pos(i) for i in range(2)]
        for layer, x in enumerate(SP.step_inputs(rng, 2)):
            s.load(*x)
            s.ks.decode_layer(layer, s.io(), st)
            SP.check_step(s, layer, ids, pos, x[0], s.out(2), 3, 1, 1)
        s.ks.end_decode_step(st)
    assert s.ks.set_sparse_decode(0, most, 1, 2, st)


@pytest.mark.parametrize("what", ["bounds", "selection", "attention"])
def test_a_chunk_whose_call_is_refused_says_so(dev, what):
    """drkh_paged_prefill_sparse is 0 where one of its three calls is refused, and those behind it are not made."""
    D, QH, KVH, bs, start, M, keep = 128, 8, 2, 16, 60, 9, 3
    assert host.set_attention_geometry(1, QH, KVH, D, cabi.BF16, cabi.BF16)
    rng = np.random.default_rng(1)
    p = R.Pool(rng, 1, KVH, QH, D, bs, 8, cabi.BF16)
    q = U.normal_bits(rng, (M, QH, D), cabi.BF16)
    dq, dp, dt, db = U.dev_bytes(q), U.dev_bytes(p.raw), U.dev_i32(np.arange(8)), U.dev_zeros(cabi.lib().drk_kv_bounds_bytes(C.byref(p.g)) + 16)
    dsel, do = U.dev_i32(np.full((M, KVH, keep), 77)), U.dev_bytes(np.full(q.shape, 0x1234, np.uint16))

    def call(refused):
        bounds = db.data_ptr() + (8 if refused and what == "bounds" else 0)
        sink = keep + 1 if refused and what == "selection" else 1
        gate, stride = (U.p(dq), D // 2) if refused and what == "attention" else (None, 0)
        return host.lib().drkh_paged_prefill_sparse(U.p(dq), U.p(dp), bounds, U.p(dt), start, M, keep, sink, 1, U.p(dsel), gate, stride, U.p(do),
                                                    0, 8, bs, 1 / math.sqrt(D), U.stream_ptr())

    assert call(True) == 0
    assert (U.host(do, np.uint16) == 0x1234).all()
    assert (U.host(dsel, np.int32) == 77).all() == (what != "attention") and U.host(db, np.uint8).any() == (what != "bounds")
    assert call(False) == 1
    sel = U.host(dsel, np.int32, (M, KVH, keep))
    G.check_attend(p, U.host(do, np.uint16, q.shape), q, np.arange(8), start + 1 + np.arange(M), sel, cabi.BF16)


# ---- selection ----------------------------------------------------------------------------------
@pytest.mark.parametrize("T,mode", [(1, "branches"), (2, "branches"), (3, "one table"), (70, "one table")])
def test_select_from_more_than_a_million_blocks(dev, T, mode):
    """1.1 million blocks of one token (the pages repeat): every row's best ones, by the lower index among equals."""
    rng = np.random.default_rng(T)
    D, QH, KVH, bs, NB, n, keep, sink, recent, io = 64, 4, 1, 1, 5000, 1_100_003, 40, 2, 3, cabi.BF16
    g = cabi.layout(1, KVH, QH, D, bs, NB, io)
    codes, exps = R.bounds_buffers(1, NB, KVH, D, rng)
    rows = T if mode == "branches" else 1
    tables = rng.integers(0, NB, (rows, n)).astype(np.int32)
    tables[:, 7] = -1
    lens = n - rng.integers(0, 90000, T).astype(np.int32)
    q = U.normal_bits(rng, (T, QH, D), io)
    got = G.run_select(g, R.bounds_bytes(codes, exps), q, tables, n if mode == "branches" else 0, lens, 0, T, n, keep, sink, recent, io)
    lo, hi = codes[0, :, 0].astype(np.int64).transpose(1, 0, 2)
    for t in range(T) if T < 8 else (0, 33, T - 1):
        score = np.full(NB, -np.inf)
        for x in U.from_bits(q[t], io).astype(np.float64):
            c, e = R.query_codes(x)
            score = np.maximum(score, np.maximum(c * lo, c * hi).sum(1) * 2.0 ** (exps[0, :, 0].astype(np.float64) + e))
        tab = tables[t if mode == "branches" else 0][:lens[t]]
        s = np.where(tab >= 0, score[tab], -np.inf)
        s[:sink], s[lens[t] - recent:] = np.inf, np.inf
        want = np.sort(np.lexsort((np.arange(len(s)), -s))[:keep])
        assert np.array_equal(got[t, 0], want), t


def test_the_driver_stretches_every_position_of_its_context(dev):
    """set_scaled_rope: keys, queries and outputs are those of a table that covers the whole context, bit for bit, on both
    sides of where init's own table ends; a refused description changes nothing."""
    import torch
    r = cabi.rope(S.RD, False, S.THETA, 8.0, 128.0, 1.0, 32.0, 1.2)

    def session(own):
        s = S.Session(2)
        st = U.stream_ptr()
        full = torch.zeros(S.NPOS * S.RD, dtype=torch.float32, device="cuda")
        cabi.call("drk_rope_table_fill_scaled", r, U.p(full), S.NPOS, st)
        assert s.ks.init(s.cm, S.NPOS, None, U.p(full), 48 if own else S.NPOS)
        if own:
            assert s.ks.set_scaled_rope(r, st)
            for bad in (cabi.rope(2 * S.RD), cabi.rope(S.RD, True), cabi.rope(S.RD, factor=-1.0)):
                assert not s.ks.set_scaled_rope(bad, st)
        rng = np.random.default_rng(4)
        s.set_weights(U.normal_bits(rng, (S.D,), S.DT), U.normal_bits(rng, (S.D,), S.DT))
        SP.prefill(s, rng, (40, 20))
        assert s.ks.open_branches(2) == 2
        outs = []
        for step in range(2):
            assert s.ks.begin_decode_step(st)
            for layer, x in enumerate(SP.step_inputs(rng, 2)):
                s.load(*x)
                s.ks.decode_layer(layer, s.io(), st)
                outs.append(s.out(2))
            s.ks.end_decode_step(st)
        s.full = full
        return s, outs

    a, want = session(False)
    b, got = session(True)
    assert np.array_equal(a.pool(), b.pool())
    assert all(np.array_equal(x, y) for x, y in zip(want, got))
    assert not host.KvStream().set_scaled_rope(r)                        # not initialised


class View8:
    """A session's pool bytes as float64 keys and values (8-bit pages), as longctx_ref's attention reads them."""

    def __init__(self, s):
        import torch
        self.L, self.KVH, self.QH, self.D, self.bs, self.NB, self.dtype = S.L, S.KVH, S.QH, S.D, S.BS, s.NB, S.KVDT
        raw = s.pool().reshape(S.L, s.NB, -1)
        n = S.KVH * S.BS * S.D
        codes = np.ascontiguousarray(raw[:, :, :2 * n])
        if S.KVDT == cabi.INT8:
            sc = np.ascontiguousarray(raw[:, :, 2 * n:2 * n + 4 * S.KVH * S.BS]).view(np.float16).astype(np.float64)
            v = codes.view(np.int8).astype(np.float64).reshape(S.L, s.NB, 2, S.KVH, S.BS, S.D) * sc.reshape(S.L, s.NB, 2, S.KVH, S.BS, 1)
        else:
            v = torch.from_numpy(codes).view(torch.float8_e4m3fn).double().numpy().reshape(S.L, s.NB, 2, S.KVH, S.BS, S.D)
        self.k, self.v = v[:, :, 0], v[:, :, 1]


def test_the_driver_chooses_among_8_bit_pages(dev, eight_bit_pages, monkeypatch):
    """Four of twelve blocks over int8 and fp8 pages: bounds, choice and attention of every step against the definitions."""
    monkeypatch.setattr(SP, "View", View8)
    s = S.Session(2)
    st = U.stream_ptr()
    rng = np.random.default_rng(14)
    s.set_weights(U.normal_bits(rng, (S.D,), S.DT), U.normal_bits(rng, (S.D,), S.DT))
    assert s.ks.set_sparse_decode(0, 4, 1, 1, st)
    SP.prefill(s, rng, (64, 64, 50))
    assert s.ks.open_branches(2) == 2
    ids = [s.ks.branch_id(i) for i in range(2)]
    for step in range(3):
        assert s.ks.begin_decode_step(st)
        pos = [s.ks.branch_pos(i) for i in range(2)]
        for layer, x in enumerate(SP.step_inputs(rng, 2)):
            s.load(*x)
            s.ks.decode_layer(layer, s.io(), st)
            SP.check_step(s, layer, ids, pos, x[0], s.out(2), 4, 1, 1)
        s.ks.end_decode_step(st)
