"""GPU tests of the long-context operators against their definitions in 64 bits: stretched rotary
positions, key bounds, block selection, attention over selected blocks, and all of them in a row."""
import ctypes as C
import math

import numpy as np
import pytest

from deusridet_amd import cabi, host
from tests import longctx_ref as R
from tests import util as U

pytestmark = pytest.mark.gpu


# ---- rotary positions -------------------------------------------------------------------------
def dev_f64(n):
    import torch
    return torch.zeros(n, dtype=torch.float64, device="cuda")


def freqs_of(r):
    f = dev_f64(r.rotary_dim // 2)
    cabi.call("drk_rope_freqs_fill", r, U.p(f), U.stream_ptr())
    return f


# an error of 2^-18 in the hardware's cos and sin (turns rounded to 2^-25 among it), and four fp32 roundings
ROPE_DELTA = 2.0 ** -18 + 4 * 2.0 ** -24


def rope_ok(got, x, want, mag, dtype, rotated):
    lim = ROPE_DELTA * mag + R.HALF_STEP[dtype] * (np.abs(want) + ROPE_DELTA * mag) + (2.0 ** -25 if dtype == cabi.F16 else 0)
    lim[..., ~rotated] = 0
    err = np.abs(got - want)
    assert (err <= lim).all(), (float((err - lim).max()), np.argwhere(err > lim)[:4])


ROPES = [cabi.rope(64), cabi.rope(128, True, 1e4), cabi.rope(48, True, 5e5, 8.0, 8192.0, 1.0, 4.0, 1.2079),
         cabi.rope(16, False, 1e4, 32.0), cabi.rope(128, False, 1e6, 2.5, 32768.0, 1.0, 32.0, 0.75)]


@pytest.mark.parametrize("i", range(len(ROPES)))
def test_rope_freqs_and_scaled_table(dev, i):
    import torch
    r = ROPES[i]
    f = freqs_of(r)
    want = R.rope_turns(r)
    U.sync()
    assert (np.abs(f.cpu().numpy() - want) <= 1e-14 * want).all()
    if r.interleaved:
        return
    n = 3001
    t = torch.zeros(n * r.rotary_dim, dtype=torch.float32, device="cuda")
    cabi.call("drk_rope_table_fill_scaled", r, U.p(t), n, U.stream_ptr())
    U.sync()
    w = 2 * math.pi * np.arange(n)[:, None] * want[None]
    got = t.cpu().numpy().reshape(n, -1, 2)
    tol = abs(r.magnitude) * (2.0 ** -24 + 1e-10)            # one rounding of values up to the magnitude; the angle to 64 bits
    assert np.abs(got[..., 0] - r.magnitude * np.cos(w)).max() <= tol
    assert np.abs(got[..., 1] - r.magnitude * np.sin(w)).max() <= tol


@pytest.mark.parametrize("dtype", [cabi.F16, cabi.BF16])
@pytest.mark.parametrize("i", range(len(ROPES)))
@pytest.mark.parametrize("T,mode", [(1, "chunk"), (1, "branches"), (37, "branches"), (130, "chunk")])
def test_rope_apply(dev, dtype, i, T, mode):
    r = ROPES[i]
    rng = np.random.default_rng(i * 10 + T)
    D, QH, KVH = max(r.rotary_dim, 48 if i == 3 else 64) if i != 1 else 256, 6, 2
    qg = U.normal_bits(rng, (T, QH, 2 * D), dtype)
    k = U.normal_bits(rng, (T, KVH, D), dtype)
    start = 2 ** 31 - 1 - T if i == 0 else 123457
    pos = rng.integers(0, 1 << 21, T).astype(np.int32) if mode == "branches" else start + np.arange(T)
    dpos = U.dev_i32(pos) if mode == "branches" else None
    dq, dk, qo, ko = U.dev_bytes(qg), U.dev_bytes(k), U.dev_zeros(T * QH * D * 2), U.dev_zeros(k.nbytes)
    f = freqs_of(r)
    rotated = np.arange(D) < r.rotary_dim
    for inverse in (0, 1):
        rows = cabi.rope_rows([(dq.data_ptr(), qo.data_ptr(), QH, QH * 2 * D, 2 * D, QH * D, D),
                               (dk.data_ptr(), ko.data_ptr(), KVH, KVH * D, D, KVH * D, D)])
        cabi.call("drk_rope_apply", r, U.p(f), rows, 2, T, D, U.p(dpos), 0 if dpos is not None else int(pos[0]), inverse, dtype, U.stream_ptr())
        U.sync()
        for buf, x in ((qo, qg[..., :D]), (ko, k)):
            xf = U.from_bits(x, dtype).astype(np.float64)
            want, mag = R.rope(r, xf, pos, bool(inverse))
            rope_ok(U.from_bits(U.host(buf, np.uint16, x.shape), dtype).astype(np.float64), xf, want, mag, dtype, rotated)
    assert np.array_equal(U.host(dq, np.uint16, qg.shape), qg)          # the gate half and the source are untouched


@pytest.mark.parametrize("interleaved", [False, True])
def test_rope_apply_in_place_three_tensors_and_head_major(dev, interleaved):
    """In place over head-major rows (the token stride below the head stride), three tensors, one of them without heads;
    equals the out-of-place call bit for bit."""
    rng = np.random.default_rng(5)
    T, D, dtype = 29, 96, cabi.BF16
    r = cabi.rope(64, interleaved, 1e4, 4.0, 4096.0)
    f = freqs_of(r)
    q, k = U.normal_bits(rng, (5, T, D), dtype), U.normal_bits(rng, (T, 3, D), dtype)
    dq, dk, oq, ok_ = U.dev_bytes(q), U.dev_bytes(k), U.dev_zeros(q.nbytes), U.dev_zeros(k.nbytes)
    call = lambda rows: cabi.call("drk_rope_apply", r, U.p(f), rows, 3, T, D, None, 777, 0, dtype, U.stream_ptr())
    call(cabi.rope_rows([(dq.data_ptr(), oq.data_ptr(), 5, D, T * D, D, T * D), (0, 0, 0, 0, 0, 0, 0),
                         (dk.data_ptr(), ok_.data_ptr(), 3, 3 * D, D, 3 * D, D)]))
    call(cabi.rope_rows([(dq.data_ptr(), dq.data_ptr(), 5, D, T * D, D, T * D), (0, 0, 0, 0, 0, 0, 0),
                         (dk.data_ptr(), dk.data_ptr(), 3, 3 * D, D, 3 * D, D)]))
    U.sync()
    assert np.array_equal(U.host(oq, np.uint16), U.host(dq, np.uint16))
    assert np.array_equal(U.host(ok_, np.uint16), U.host(dk, np.uint16))
    want, mag = R.rope(r, U.from_bits(q, dtype).transpose(1, 0, 2), 777 + np.arange(T))
    got = U.from_bits(U.host(oq, np.uint16, q.shape), dtype).astype(np.float64).transpose(1, 0, 2)
    rope_ok(got, None, want, mag, dtype, np.arange(D) < 64)


@pytest.mark.parametrize("dtype", [cabi.F16, cabi.BF16])
def test_scaled_table_in_the_fused_layer_step(dev, dtype):
    """The fused norm + rotation + append reads a table of stretched angles: its keys in the pages and its queries equal the
    norm followed by the rotation that forms the angles itself, but for the two roundings in between."""
    import torch
    rng = np.random.default_rng(8)
    D, QH, KVH, bs, T, start = 128, 4, 2, 16, 21, 4000
    r = cabi.rope(64, False, 1e6, 8.0, 1024.0, 1.0, 32.0, 1.2)
    g = cabi.layout(1, KVH, QH, D, bs, 300, dtype)
    pool = U.dev_zeros(cabi.lib().drk_kv_pool_bytes(C.byref(g)))
    table = U.dev_i32(np.arange(300))
    npos = start + T
    tab = torch.zeros(npos * 64, dtype=torch.float32, device="cuda")
    cabi.call("drk_rope_table_fill_scaled", r, U.p(tab), npos, U.stream_ptr())
    qg, k, v, w = (U.normal_bits(rng, s, dtype) for s in ((T, QH, 2 * D), (T, KVH, D), (T, KVH, D), (D,)))
    dqg, dk, dv, dw, dq = U.dev_bytes(qg), U.dev_bytes(k), U.dev_bytes(v), U.dev_bytes(w), U.dev_zeros(T * QH * D * 2)
    cabi.call("drk_qk_norm_rope_append", g, U.p(pool), U.p(table), 300, None, start, T, 0, U.p(dqg), U.p(dk), U.p(dv), U.p(dw), U.p(dw), 1e-6, 64,
              r.theta, U.p(tab), npos, U.p(dq), dtype, U.stream_ptr())
    U.sync()
    pages = U.from_bits(U.host(pool, np.uint16, (300, 2, KVH, bs, D)), dtype).astype(np.float64)
    got_k = np.stack([pages[p // bs, 0, :, p % bs] for p in range(start, npos)])
    got_q = U.from_bits(U.host(dq, np.uint16, (T, QH, D)), dtype).astype(np.float64)
    for got, x in ((got_q, qg[..., :D]), (got_k, k)):
        xf, wf = U.from_bits(x, dtype).astype(np.float64), U.from_bits(w, dtype).astype(np.float64)
        n = xf / np.sqrt((xf ** 2).mean(-1, keepdims=True) + 1e-6) * wf
        want, mag = R.rope(r, n, start + np.arange(T))
        mag[..., 64:] = np.abs(n[..., 64:])
        h = R.HALF_STEP[dtype]
        lim = h * 1.01 * mag + h * (np.abs(want) + 2 * h * mag) + 2.0 ** -20 * mag + (2.0 ** -23 if dtype == cabi.F16 else 0)
        assert (np.abs(got - want) <= lim).all()


def test_rope_through_the_host_class_in_place(dev):
    rng = np.random.default_rng(31)
    T, D, dtype = 5, 128, cabi.BF16
    assert host.set_attention_geometry(1, 8, 2, D, dtype, dtype)
    r = cabi.rope(96, True, 1e4, 16.0, 4096.0, 1.0, 32.0, 1.1)
    f = freqs_of(r)
    q, k = U.normal_bits(rng, (T, 8, D), dtype), U.normal_bits(rng, (T, 2, D), dtype)
    dq, dk = U.dev_bytes(q), U.dev_bytes(k)
    host.lib().drkh_apply_rope_scaled(r, U.p(f), U.p(dq), U.p(dk), T, 8, 2, D, None, 70000, 1, U.stream_ptr())
    U.sync()
    for buf, x in ((dq, q), (dk, k)):
        xf = U.from_bits(x, dtype).astype(np.float64)
        want, mag = R.rope(r, xf, 70000 + np.arange(T), True)
        rope_ok(U.from_bits(U.host(buf, np.uint16, x.shape), dtype).astype(np.float64), xf, want, mag, dtype, np.arange(D) < 96)


def test_rope_inverse_is_the_gradient(dev):
    """<g, R x> = <R^T g, x>, and a central difference of <g, R x> along a direction."""
    rng = np.random.default_rng(6)
    T, H, D, dtype = 17, 4, 128, cabi.F16
    r = cabi.rope(96, True, 1e4, 8.0, 4096.0, 1.0, 32.0, 1.1)
    f, pos = freqs_of(r), U.dev_i32(rng.integers(0, 100000, T))

    def rot(x, inverse):
        dx, do = U.dev_bytes(U.to_bits(x.astype(np.float32), dtype)), U.dev_zeros(x.size * 2)
        rows = cabi.rope_rows([(dx.data_ptr(), do.data_ptr(), H, H * D, D, H * D, D)])
        cabi.call("drk_rope_apply", r, U.p(f), rows, 1, T, D, U.p(pos), 0, inverse, dtype, U.stream_ptr())
        U.sync()
        return U.from_bits(U.host(do, np.uint16, x.shape), dtype).astype(np.float64)

    x, g, v = (U.from_bits(U.normal_bits(rng, (T, H, D), dtype), dtype).astype(np.float64) for _ in range(3))
    grad = rot(g, 1)
    # every product's two factors: one exact, one off by half a step (and the angles' error); |element| < 6
    tol = (2.0 ** -11 + 2 * ROPE_DELTA) * 1.1 * 2
    lhs, rhs = (g * rot(x, 0)).sum(), (grad * x).sum()
    assert abs(lhs - rhs) <= tol * (np.abs(g) * np.abs(x)).sum() * 2
    h = 0.5                                                            # linear in x: the step's size costs no accuracy
    up, down = (U.from_bits(U.to_bits((x + s * h * v).astype(np.float32), dtype), dtype).astype(np.float64) for s in (1, -1))
    diff = (g * (rot(up, 0) - rot(down, 0))).sum()
    assert abs(diff - (grad * (up - down)).sum()) <= tol * (np.abs(g) * (np.abs(up) + np.abs(down))).sum() * 2


# ---- bounds -----------------------------------------------------------------------------------
def bounds_dev(p):
    return U.dev_zeros(cabi.lib().drk_kv_bounds_bytes(C.byref(p.g)))


def bounds_host(p, dbounds):
    b = U.host(dbounds, np.int8)
    n = p.L * p.NB * p.KVH
    return b[:n * 2 * p.D].reshape(p.L, p.NB, p.KVH, 2, p.D), b[n * 2 * p.D:n * (2 * p.D + 1)].reshape(p.L, p.NB, p.KVH)


def check_block(p, codes, exps, layer, blk, n):
    for h in range(p.KVH):
        lo, hi, e = R.bounds(p.k[layer, blk, h, :n])
        assert exps[layer, blk, h] == e and np.array_equal(codes[layer, blk, h, 0], lo) and np.array_equal(codes[layer, blk, h, 1], hi), (layer, blk, h)


DTYPES = [cabi.F16, cabi.BF16, cabi.INT8, cabi.FP8_E4M3]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D,bs", [(128, 16), (64, 1), (64, 5), (256, 48), (512, 16), (128, 256)])
@pytest.mark.parametrize("start,n", [(0, 1), (37, 61), (0, 301)])
def test_bounds_update_chunk(dev, dtype, D, bs, start, n):
    rng = np.random.default_rng(D + bs + n)
    NBL = -(-(start + n) // bs)
    p = R.Pool(rng, 2, 3, 6, D, bs, NBL + 3, dtype)
    table = U.shuffled_table(rng, p.NB, NBL)
    if NBL > 3:
        table[-2] = -1
    if bs > 1 and (start + n) % bs and table[-1] >= 0:
        for layer in range(2):
            p.poison(layer, table[-1], (start + n) % bs)                # stale tokens behind the last one
    db, dp, dt = bounds_dev(p), U.dev_bytes(p.raw), U.dev_i32(table)
    db.fill_(0x55)
    cabi.call("drk_kv_bounds_update", p.g, U.p(dp), U.p(dt), 0, None, start, n, 0, 2, U.p(db), U.stream_ptr())
    U.sync()
    codes, exps = bounds_host(p, db)
    touched = set()
    for lb in range(start // bs, NBL):
        if table[lb] >= 0:
            touched.add(int(table[lb]))
            for layer in range(2):
                check_block(p, codes, exps, layer, table[lb], min(bs, start + n - lb * bs))
    for blk in set(range(p.NB)) - touched:                              # everything else is as it was
        assert (codes[:, blk] == 0x55).all() and (exps[:, blk] == 0x55).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_bounds_update_branches_and_extract(dev, dtype):
    import torch
    rng = np.random.default_rng(9)
    B, bs, D, NBL = 7, 16, 128, 9
    p = R.Pool(rng, 3, 2, 8, D, bs, B * NBL, dtype)
    tables = rng.permutation(p.NB).astype(np.int32).reshape(B, NBL)
    pos = np.array([0, 15, 16, 143, -1, 100, 9 * 16], np.int32)         # a branch without a position, one behind its table
    tables[5, 100 // bs] = -1
    db, dp, dt, dpos = bounds_dev(p), U.dev_bytes(p.raw), U.dev_i32(tables), U.dev_i32(pos)
    cabi.call("drk_kv_bounds_update", p.g, U.p(dp), U.p(dt), NBL, U.p(dpos), 0, B, 1, 2, U.p(db), U.stream_ptr())
    U.sync()
    codes, exps = bounds_host(p, db)
    written = {}
    for b in range(4):
        written[int(tables[b, pos[b] // bs])] = pos[b] % bs + 1
    for blk in range(p.NB):
        assert not codes[0, blk].any()
        for layer in (1, 2):
            if blk in written:
                check_block(p, codes, exps, layer, blk, written[blk])
            else:
                assert not codes[layer, blk].any()
    # the values, in the order of a table with a hole and a page that does not exist
    blocks = np.array(list(written) + [-1, p.NB], np.int32)
    out = torch.full((2, len(blocks), p.KVH, 2, D), 7.0, dtype=torch.bfloat16, device="cuda")
    cabi.call("drk_kv_bounds_extract", p.g, U.p(out), U.p(db), U.p(U.dev_i32(blocks)), len(blocks), 1, 2, U.stream_ptr())
    U.sync()
    got = out.double().cpu().numpy()
    want = codes[1:].astype(np.float64) * 2.0 ** exps[1:].astype(np.float64)[..., None, None]
    assert np.array_equal(got[:, :4], want[:, list(written)]) and not got[:, 4:].any()


@pytest.mark.parametrize("dtype", [cabi.F16, cabi.BF16])
def test_bounds_of_extreme_keys(dev, dtype):
    """Zeros, NaN, infinities, subnormals and exact powers of two; 127 * 2^e sits at the border between two exponents."""
    rng = np.random.default_rng(10)
    p = R.Pool(rng, 1, 1, 1, 64, 4, 9, dtype)
    k = p.raw[0].view(np.uint16).reshape(9, 2, 4, 64)[:, 0]             # [block, token, dim]
    k[0] = 0
    k[1] = U.to_bits(np.array([127.0], np.float32), dtype)
    k[2] = U.to_bits(np.array([128.0], np.float32), dtype)
    k[3] = U.to_bits(np.array([-127.5], np.float32), dtype)
    k[4] = 0x7FFF                                                       # NaN everywhere
    k[5, :, 3] = 0xFFFF                                                 # one dimension of NaN
    k[6, 2, 5] = U.to_bits(np.array([np.inf], np.float32), dtype)[0]
    k[7] = 1                                                            # the smallest subnormal
    k[8, 0] = U.to_bits(np.array([3e38 if dtype == cabi.BF16 else 65504], np.float32), dtype)
    p.k = U.from_bits(k, dtype).astype(np.float64)[None, :, None]
    db, dp, dt = bounds_dev(p), U.dev_bytes(p.raw), U.dev_i32(np.arange(9))
    cabi.call("drk_kv_bounds_update", p.g, U.p(dp), U.p(dt), 0, None, 0, 36, 0, 1, U.p(db), U.stream_ptr())
    U.sync()
    codes, exps = bounds_host(p, db)
    assert exps[0, 1, 0] == 0 and exps[0, 2, 0] == 1 and exps[0, 0, 0] == -40
    for blk in range(9):
        check_block(p, codes, exps, 0, blk, 4)


def test_bounds_of_int8_tokens_without_a_finite_scale(dev):
    rng = np.random.default_rng(11)
    p = R.Pool(rng, 1, 2, 2, 128, 16, 3, cabi.INT8)
    sc = p.raw[0][:, 2 * 2 * 16 * 128:].view(np.uint16).reshape(3, 2, 2, 16)
    sc[1, 0, 0, [2, 5, 7]] = [0x7FFF, 0x7C00, 0xFC00]                   # NaN, infinities
    sc[2, 0, 1] = 0x7E00                                                # nothing else
    sc[1, 0, 1, 4] = 0x7BFF                                             # the largest finite one
    p.k = p.raw[0][:, :2 * 2 * 16 * 128].view(np.int8).reshape(3, 2, 2, 16, 128)[:, 0].astype(np.float64)
    with np.errstate(invalid="ignore"):
        s = sc[:, 0].view(np.float16).astype(np.float64)
        p.k = (p.k * np.where(np.isfinite(s), s, np.nan)[..., None])[None]
    db, dp, dt = bounds_dev(p), U.dev_bytes(p.raw), U.dev_i32(np.arange(3))
    cabi.call("drk_kv_bounds_update", p.g, U.p(dp), U.p(dt), 0, None, 0, 48, 0, 1, U.p(db), U.stream_ptr())
    U.sync()
    codes, exps = bounds_host(p, db)
    for blk in range(3):
        check_block(p, codes, exps, 0, blk, 16)


# ---- selection --------------------------------------------------------------------------------
def run_select(g, raw, q, tables, stride, lens, start, T, max_len, keep, sink, recent, io, layer=0, shift=0):
    dsel = U.dev_i32(np.full(T * g.num_kv_heads * keep + 4, 77, np.int32))
    need = cabi.lib().drk_block_select_workspace_bytes(C.byref(g), T, max_len)
    ws = U.dev_zeros(need + 16)
    ws.fill_(0xA5)
    db, dq, dt = U.dev_bytes(raw), U.dev_bytes(q), U.dev_i32(tables)
    dl = U.dev_i32(lens) if lens is not None else None
    cabi.call("drk_block_select", g, U.p(db), layer, U.p(dq), io, U.p(dt), stride, U.p(dl), start, T, max_len, keep, sink, recent,
              U.p(dsel), U.p(ws), need, U.stream_ptr())
    U.sync()
    out = U.host(dsel, np.int32)
    assert (out[-4:] == 77).all()
    return out[:-4].reshape(T, g.num_kv_heads, keep)


@pytest.mark.parametrize("io", [cabi.F16, cabi.BF16])
@pytest.mark.parametrize("D,QH,KVH", [(128, 8, 2), (256, 6, 1), (64, 3, 3), (512, 5, 1), (128, 16, 1)])
@pytest.mark.parametrize("bs,keep,sink,recent", [(16, 9, 1, 2), (5, 1, 0, 0), (256, 70, 0, 3)])
def test_select_branches(dev, io, D, QH, KVH, bs, keep, sink, recent):
    rng = np.random.default_rng(D + QH + bs)
    lens = np.array([0, 1, bs, bs + 1, 37 * bs + 3, 20 * bs, -4], np.int32)
    n = 38
    tables = rng.permutation(len(lens) * n).astype(np.int32).reshape(-1, n)
    tables[rng.random(tables.shape) < 0.1] = -1
    tables[4, 5], tables[5, 7] = len(lens) * n + 2, 2 ** 30
    NB = len(lens) * n
    g = cabi.layout(2, KVH, QH, D, bs, NB, io)
    codes, exps = R.bounds_buffers(2, NB, KVH, D, rng)
    q = U.normal_bits(rng, (len(lens), QH, D), io)
    got = run_select(g, R.bounds_bytes(codes, exps), q, tables, n, lens, 0, len(lens), 38 * bs, keep, sink, recent, io, layer=1)
    qf = U.from_bits(q, io).astype(np.float64)
    for t, ln in enumerate(lens):
        assert np.array_equal(got[t], R.select(qf[t], codes[1], exps[1], tables[t], int(ln), bs, keep, sink, recent)), t


@pytest.mark.parametrize("D,QH,KVH", [(128, 8, 2), (256, 6, 1), (64, 2, 2), (512, 4, 2), (128, 16, 1)])
@pytest.mark.parametrize("T,start", [(1, 0), (5, 0), (41, 333)])
def test_select_chunk(dev, D, QH, KVH, T, start):
    rng = np.random.default_rng(D + T)
    bs, keep, sink, recent, io = 8, 11, 2, 1, cabi.BF16
    n = -(-(start + T) // bs)
    table = U.shuffled_table(rng, n + 2, n)
    if n > 20:
        table[[3, 17]] = -1
    g = cabi.layout(1, KVH, QH, D, bs, n + 2, cabi.INT8)
    codes, exps = R.bounds_buffers(1, n + 2, KVH, D, rng)
    q = U.normal_bits(rng, (T, QH, D), io)
    got = run_select(g, R.bounds_bytes(codes, exps), q, table, 0, None, start, T, start + T, keep, sink, recent, io)
    qf = U.from_bits(q, io).astype(np.float64)
    for t in range(T):
        assert np.array_equal(got[t], R.select(qf[t], codes[0], exps[0], table, start + t + 1, bs, keep, sink, recent)), t


@pytest.mark.parametrize("D,QH,KVH,T", [(128, 8, 2, 70), (256, 6, 1, 37), (64, 2, 2, 21), (128, 16, 1, 9), (512, 3, 3, 11)])
def test_select_rows_of_any_length_over_one_table(dev, D, QH, KVH, T):
    """One table, a length per row (none, one, ragged, beyond max_seq_len); more blocks than one workgroup selects from."""
    rng = np.random.default_rng(D * T)
    bs, n, keep, sink, recent, io = 4, 1400, 19, 1, 3, cabi.F16
    table = U.shuffled_table(rng, n, n)
    table[rng.random(n) < 0.05] = -1
    lens = rng.integers(-1, n * bs + 1, T).astype(np.int32)
    lens[:6] = [0, 1, n * bs, 5000, 4097, 4096]
    g = cabi.layout(1, KVH, QH, D, bs, n, cabi.INT8)
    codes, exps = R.bounds_buffers(1, n, KVH, D, rng)
    q = U.normal_bits(rng, (T, QH, D), io)
    qf = U.from_bits(q, io).astype(np.float64)
    for most in (n * bs, 4500):
        got = run_select(g, R.bounds_bytes(codes, exps), q, table, 0, lens, 0, T, most, keep, sink, recent, io)
        for t in range(T):
            want = R.select(qf[t], codes[0], exps[0], table, min(int(lens[t]), most), bs, keep, sink, recent)
            assert np.array_equal(got[t], want), (most, t)


@pytest.mark.parametrize("kind", ["equal", "few", "extreme"])
@pytest.mark.parametrize("n", [700, 2051, 9001])
def test_select_ties_and_spread(dev, kind, n):
    """Equal scores go to the lower index; scores at both ends of the range; more blocks than one pass of a workgroup."""
    rng = np.random.default_rng(n)
    D, io, bs = 64, cabi.F16, 16
    g = cabi.layout(1, 1, 2, D, bs, n, io)
    codes, exps = R.bounds_buffers(1, n, 1, D, rng)
    if kind == "equal":
        codes[:], exps[:] = codes[0, 0], exps[0, 0]
    elif kind == "few":
        pick = rng.integers(0, 3, n)
        codes[0], exps[0] = codes[0, pick], exps[0, pick]
    else:
        exps[0] = rng.choice([-40, 40, 0], (n, 1))
        codes[0, ::7] = 0
    q = U.normal_bits(rng, (1, 2, D), io)
    table = rng.permutation(n).astype(np.int32)
    qf = U.from_bits(q, io).astype(np.float64)
    for keep, sink, recent in ((1, 0, 0), (64, 1, 3), (n // 2, 0, 0), (n + 5, 2, 2)):
        got = run_select(g, R.bounds_bytes(codes, exps), q, table, n, np.array([n * bs - 3]), 0, 1, n * bs, keep, sink, recent, io)
        assert np.array_equal(got[0], R.select(qf[0], codes[0], exps[0], table, n * bs - 3, bs, keep, sink, recent)), keep


def test_select_odd_queries(dev):
    """Queries of zeros, NaN, infinities and subnormals."""
    rng = np.random.default_rng(3)
    D, bs, n, io = 128, 16, 40, cabi.BF16
    g = cabi.layout(1, 1, 1, D, bs, n, io)
    codes, exps = R.bounds_buffers(1, n, 1, D, rng)
    q = U.normal_bits(rng, (6, 1, D), io)
    q[0] = 0
    q[1, 0, 3] = 0x7FC1
    q[2, 0, 9], q[2, 0, 10] = 0x7F80, 0xFF80
    q[3] = 0x0003
    q[4] = 0x7FC0
    q[5, 0, 0] = U.to_bits(np.array([3e38], np.float32), io)[0]
    tables = np.tile(rng.permutation(n).astype(np.int32), (6, 1))
    lens = np.full(6, n * bs, np.int32)
    got = run_select(g, R.bounds_bytes(codes, exps), q, tables, n, lens, 0, 6, n * bs, 7, 0, 0, io)
    qf = U.from_bits(q, io).astype(np.float64)
    for t in range(6):
        assert np.array_equal(got[t], R.select(qf[t], codes[0], exps[0], tables[t], n * bs, bs, 7, 0, 0)), t


@pytest.mark.parametrize("n", [1500, 2100, 4200, 8300])
def test_select_many_rows_of_many_blocks(dev, n):
    """More (row, kv head) pairs than workgroups are wanted: the selection's other shapes, with ties among coarse bounds."""
    rng = np.random.default_rng(n)
    D, KVH, T, io = 64, 8, 66, cabi.BF16
    g = cabi.layout(1, KVH, KVH, D, 1, n, io)
    codes, exps = R.bounds_buffers(1, n, KVH, D, rng)
    codes[:, n // 2:] = np.sort(np.sign(codes[:, n // 2:]), 3)              # -1, 0, 1, low <= high: many equal scores
    exps[:, n // 2:] = 3
    q = U.normal_bits(rng, (T, KVH, D), io)
    table = rng.permutation(n).astype(np.int32)
    got = run_select(g, R.bounds_bytes(codes, exps), q, table, 0, None, n - T, T, n, 40, 1, 3, io)
    qf = U.from_bits(q, io).astype(np.float64)
    for t in (0, 1, 30, 31, 64, 65):
        assert np.array_equal(got[t], R.select(qf[t], codes[0], exps[0], table, n - T + t + 1, 1, 40, 1, 3)), t


@pytest.mark.parametrize("n", [6, 300, 2500])
def test_select_never_reads_past_a_table_row(dev, n):
    """Lengths beyond the table's blocks are cut to it, whichever kernels the size calls for."""
    rng = np.random.default_rng(n)
    D, QH, KVH, bs, io = 128, 8, 2, 4, cabi.F16
    tables = np.stack([rng.permutation(n).astype(np.int32) for _ in range(3)])
    g = cabi.layout(1, KVH, QH, D, bs, n, io)
    codes, exps = R.bounds_buffers(1, n, KVH, D, rng)
    q = U.normal_bits(rng, (3, QH, D), io)
    lens = np.array([n * bs + 50, n * bs - 3, 2 ** 31 - 1], np.int32)
    got = run_select(g, R.bounds_bytes(codes, exps), q, tables, n, lens, 0, 3, n * bs + 200, 5, 1, 2, io)
    qf = U.from_bits(q, io).astype(np.float64)
    for t in range(3):
        assert np.array_equal(got[t], R.select(qf[t], codes[0], exps[0], tables[t], min(int(lens[t]), n * bs), bs, 5, 1, 2)), t


# ---- attention --------------------------------------------------------------------------------
def run_attend(p, q, tables, stride, lens, start, sel, io, layer=0, gate=None, gate_stride=0, scale=None):
    T, keep = q.shape[0], sel.shape[2]
    out = np.full((T, p.QH, p.D), 0x1234, np.uint16)
    do, dq, dp, dt, ds = U.dev_bytes(out), U.dev_bytes(q), U.dev_bytes(p.raw), U.dev_i32(tables), U.dev_i32(sel)
    dl = U.dev_i32(lens) if lens is not None else None
    dg = U.dev_bytes(gate) if gate is not None else None
    need = cabi.lib().drk_paged_sparse_workspace_bytes(C.byref(p.g), T, keep)
    ws = U.dev_zeros(need + 16)
    ws.fill_(0xFF)
    cabi.call("drk_paged_sparse_attention", p.g, U.p(dq), U.p(dp), U.p(dt), stride, U.p(dl), start, T, U.p(ds), keep, U.p(do), layer,
              scale or 1 / math.sqrt(p.D), io, U.p(dg), gate_stride, U.p(ws), need, U.stream_ptr())
    U.sync()
    return U.host(do, np.uint16, out.shape)


def check_attend(p, got, q, tables, lens, sel, io, layer=0, gate=None, scale=None, rows=None):
    worst = 0.0
    for t in range(q.shape[0]) if rows is None else rows:
        tab = tables[t] if tables.ndim == 2 else tables
        want, tol = R.attend(p, layer, U.from_bits(q[t], io).astype(np.float64), tab, int(lens[t]), sel[t], scale or 1 / math.sqrt(p.D),
                             None if gate is None else U.from_bits(gate[t], io).astype(np.float64))
        for h in range(p.KVH):                                       # heads whose list holds nothing are left as they were
            some = any(b >= 0 and b * p.bs < lens[t] and 0 <= tab[b] < p.NB for b in map(int, sel[t, h]))
            G = p.QH // p.KVH
            mine = got[t, h * G:(h + 1) * G]
            if not some:
                assert (mine == 0x1234).all(), (t, h)
                continue
            ok, r = R.attend_ok(U.from_bits(mine, io), want[h * G:(h + 1) * G], tol[h * G:(h + 1) * G], io)
            assert ok, (t, h, r)
            worst = max(worst, r)
    return worst


GEOS = [(128, 32, 8, 16), (128, 5, 5, 48), (256, 6, 1, 16), (128, 16, 1, 32), (256, 24, 4, 256)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("geo", range(len(GEOS)))
@pytest.mark.parametrize("gated", [False, True])
def test_attend_branches(dev, dtype, geo, gated):
    D, QH, KVH, bs = GEOS[geo]
    rng = np.random.default_rng(geo)
    io = dtype if dtype < cabi.INT8 else (cabi.F16 if geo % 2 else cabi.BF16)
    n = 7
    lens = np.array([1, 0, bs, 3 * bs + 5, 7 * bs, 2 * bs + 16, -1, 6 * bs - 1], np.int32)
    B = len(lens)
    p = R.Pool(rng, 2, KVH, QH, D, bs, B * n, dtype)
    tables = rng.permutation(p.NB).astype(np.int32).reshape(B, n)
    tables[4, 3], tables[7, 2] = -1, p.NB + 1
    keep = 9
    sel = np.full((B, KVH, keep), -1, np.int32)
    for t in range(B):
        for h in range(KVH):
            m = rng.integers(0, n + 1)
            sel[t, h, :m] = np.sort(rng.permutation(n)[:m])
    sel[3, 0] = [3, 0, -1, 2, n - 1, 1, -7, 100000, 2 ** 31 - 1]            # any order, entries that hold nothing
    sel[4, 0] = [5, 5, 1, -1, -1, -1, -1, -1, -1]                           # listed twice: counted twice
    used = {(t, int(b)) for t in range(B) for h in range(KVH) for b in map(int, sel[t, h]) if 0 <= b * bs < lens[t]}
    for t in range(B):                                                      # stale tokens and unlisted blocks hold NaN
        for b in range(n):
            blk = tables[t, b]
            if 0 <= blk < p.NB:
                first = min(bs, max(0, int(lens[t]) - b * bs)) if (t, b) in used else 0
                if first < bs:
                    p.poison(1, blk, first)
    q = U.normal_bits(rng, (B, QH, D), io)
    gate = U.normal_bits(rng, (B, QH, 2 * D), io) if gated else None
    half = np.ascontiguousarray(gate[..., D:]) if gated else None
    got = run_attend(p, q, tables, n, lens, 0, sel, io, 1, half, D)
    check_attend(p, got, q, tables, lens, sel, io, 1, half)
    if gated:                                                               # the gate as a half of the projection
        dgate = U.dev_bytes(gate)
        out2 = U.dev_bytes(np.full((B, QH, D), 0x1234, np.uint16))
        need = cabi.lib().drk_paged_sparse_workspace_bytes(C.byref(p.g), B, keep)
        ws = U.dev_zeros(need + 16)
        dq, dp, dt, ds, dl = U.dev_bytes(q), U.dev_bytes(p.raw), U.dev_i32(tables), U.dev_i32(sel), U.dev_i32(lens)
        cabi.call("drk_paged_sparse_attention", p.g, U.p(dq), U.p(dp), U.p(dt), n, U.p(dl), 0, B, U.p(ds), keep, U.p(out2), 1,
                  1 / math.sqrt(D), io, dgate.data_ptr() + 2 * D, 2 * D, U.p(ws), need, U.stream_ptr())
        U.sync()
        assert np.array_equal(U.host(out2, np.uint16, got.shape), got)


def test_attend_passes_over_entries_behind_the_table(dev):
    rng = np.random.default_rng(5)
    D, QH, KVH, bs, n, io = 128, 8, 2, 16, 3, cabi.BF16
    p = R.Pool(rng, 1, KVH, QH, D, bs, 4 * n, io)
    tables = rng.permutation(4 * n).astype(np.int32).reshape(4, n)
    lens = np.full(4, 100 * bs, np.int32)                                   # longer than the tables
    sel = np.tile(np.array([0, 2, n, n + 1, 99, -1], np.int32), (4, KVH, 1))
    sel[2] = [n, n + 7, 50, -1, 99, 98]                                     # nothing of it is in the table
    q = U.normal_bits(rng, (4, QH, D), io)
    got = run_attend(p, q, tables, n, lens, 0, sel, io)
    inside = np.where(sel < n, sel, -1)
    check_attend(p, got, q, tables, np.full(4, n * bs, np.int32), inside, io)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,keep", [(1, 1), (1, 120), (3, 40), (70, 5)])
def test_attend_chunk(dev, dtype, T, keep):
    """Rows of a chunk over one table; few rows are cut into pieces, many are not."""
    rng = np.random.default_rng(T + keep)
    D, QH, KVH, bs, start = 128, 8, 2, 16, 1900
    io = dtype if dtype < cabi.INT8 else cabi.F16
    n = -(-(start + T) // bs)
    p = R.Pool(rng, 1, KVH, QH, D, bs, n + 1, dtype, 2.0)
    table = U.shuffled_table(rng, n + 1, n)
    sel = np.full((T, KVH, keep), -1, np.int32)
    for t in range(T):
        for h in range(KVH):
            m = min(keep, n)
            sel[t, h, :m] = np.sort(rng.permutation(n)[:m])
    q = U.normal_bits(rng, (T, QH, D), io, 1.5)
    got = run_attend(p, q, table, 0, None, start, sel, io)
    check_attend(p, got, q, table, start + 1 + np.arange(T), sel, io)


@pytest.mark.parametrize("dtype", [cabi.BF16, cabi.INT8])
@pytest.mark.parametrize("D,T", [(128, 130), (128, 261), (128, 515), (256, 131), (256, 300)])
@pytest.mark.parametrize("mode", ["chunk", "branches"])
def test_attend_many_rows(dev, dtype, D, T, mode):
    """Row counts from which a workgroup takes two, four or eight rows instead of one; the last workgroup is not full."""
    rng = np.random.default_rng(T)
    QH, KVH, bs, n, keep, start = 16, 8, 16, 12, 5, 40
    io = dtype if dtype < cabi.INT8 else cabi.F16
    chunk = mode == "chunk"
    n = -(-(start + T) // bs) if chunk else n
    NB = n + 3 if chunk else 40
    p = R.Pool(rng, 1, KVH, QH, D, bs, NB, dtype)
    tables = U.shuffled_table(rng, NB, n) if chunk else rng.integers(0, NB, (T, n)).astype(np.int32)
    lens = start + 1 + np.arange(T) if chunk else rng.integers(0, n * bs + 1, T)
    sel = np.sort(rng.integers(-1, n, (T, KVH, keep)).astype(np.int32), axis=2)
    sel[3], sel[T - 1, 2:] = -1, -1
    q = U.normal_bits(rng, (T, QH, D), io)
    gate = U.normal_bits(rng, (T, QH, D), io)
    got = run_attend(p, q, tables, 0 if chunk else n, None if chunk else lens.astype(np.int32), start if chunk else 0, sel, io, 0, gate, D)
    check_attend(p, got, q, tables, lens, sel, io, 0, gate)


@pytest.mark.parametrize("D,KVH,T,dtype", [(256, 1, 2100, cabi.INT8), (128, 1, 4100, cabi.INT8), (128, 2, 4096, cabi.BF16)])
def test_attend_many_rows_of_long_lists(dev, D, KVH, T, dtype):
    """16 query heads per kv head and 512 groups per row: what a workgroup keeps in LDS limits the rows it takes."""
    rng = np.random.default_rng(D + T)
    bs, n, keep, G = 256, 40, 32, 16
    io = dtype if dtype < cabi.INT8 else cabi.BF16
    p = R.Pool(rng, 1, KVH, KVH * G, D, bs, n, dtype)
    table = rng.permutation(n).astype(np.int32)
    sel = np.argsort(rng.random((T, KVH, n)), axis=2)[..., :keep].astype(np.int32)
    start = n * bs - T - 5
    q = U.normal_bits(rng, (T, KVH * G, D), io)
    got = run_attend(p, q, table, 0, None, start, sel, io)
    check_attend(p, got, q, table, start + 1 + np.arange(T), sel, io, rows=[0, 1, 7, 8, T // 2 + 1, T - 9, T - 1])


def test_attend_everything_equals_dense_decode(dev):
    """All blocks selected: the decode kernel's result, up to the order of summation and its two roundings."""
    rng = np.random.default_rng(12)
    D, QH, KVH, bs, B, n = 128, 32, 8, 16, 3, 40
    p = R.Pool(rng, 1, KVH, QH, D, bs, B * n, cabi.BF16)
    tables = rng.permutation(p.NB).astype(np.int32).reshape(B, n)
    lens = np.array([640, 17, 333], np.int32)
    sel = np.broadcast_to(np.arange(n, dtype=np.int32), (B, KVH, n)).copy()
    q = U.normal_bits(rng, (B, QH, D), cabi.BF16)
    got = run_attend(p, q, tables, n, lens, 0, sel, cabi.BF16)
    need = cabi.lib().drk_decode_workspace_bytes(C.byref(p.g), B, 640)
    ws, do = U.dev_zeros(need), U.dev_zeros(q.nbytes)
    dq, dp, dt, dl = U.dev_bytes(q), U.dev_bytes(p.raw), U.dev_i32(tables), U.dev_i32(lens)
    cabi.call("drk_paged_decode_attention_branches", p.g, U.p(dq), U.p(dp), U.p(dt), n, U.p(dl), B, 640, U.p(do), 0, 1 / math.sqrt(D),
              cabi.BF16, 0, U.p(ws), need, U.stream_ptr())
    U.sync()
    check_attend(p, got, q, tables, lens, sel, cabi.BF16)
    check_attend(p, U.host(do, np.uint16, q.shape), q, tables, lens, sel, cabi.BF16)


def test_attend_nan_and_infinities_in_listed_tokens(dev):
    """A NaN score makes the row NaN however the row is cut; a key of -inf takes weight nought; others are unharmed."""
    rng = np.random.default_rng(13)
    D, QH, KVH, bs, n = 128, 4, 1, 16, 64
    p = R.Pool(rng, 1, KVH, QH, D, bs, 2 * n, cabi.F16)
    tables = np.arange(2 * n, dtype=np.int32).reshape(2, n)
    k = p.raw[0].view(np.uint16).reshape(2 * n, 2, KVH, bs, D)
    k[40, 0, 0, 7] = 0x7FFF                                                 # row 0: one token of NaN
    q = np.abs(U.from_bits(U.normal_bits(rng, (2, QH, D), cabi.F16), cabi.F16))
    q = U.to_bits(np.maximum(q, 0.01), cabi.F16)
    k[n + 3, 0, 0, 2] = 0xFC00                                              # row 1: a key of -inf against positive queries
    p.k[0, n + 3, 0, 2] = -np.inf
    lens = np.array([n * bs, n * bs], np.int32)
    sel = np.broadcast_to(np.arange(n, dtype=np.int32), (2, KVH, n)).copy()
    got = run_attend(p, q, tables, n, lens, 0, sel, cabi.F16)
    assert np.isnan(U.f16_bits_to_f32(got[0])).all()
    want, _ = R.attend(p, 0, U.from_bits(q[1], cabi.F16).astype(np.float64), tables[1], n * bs, sel[1], 1 / math.sqrt(D))
    # the tolerance of the row without that token, whose weight is nought
    less = sel[1].copy()
    less[0, 3] = -1
    _, tol = R.attend(p, 0, U.from_bits(q[1], cabi.F16).astype(np.float64), tables[1], n * bs, less, 1 / math.sqrt(D))
    ok, r = R.attend_ok(U.from_bits(got[1], cabi.F16), want, 2 * tol, cabi.F16)
    assert ok, r


@pytest.mark.parametrize("dtype", [cabi.BF16, cabi.FP8_E4M3])
def test_chunk_over_selected_blocks_through_the_host_functions(dev, dtype):
    """Bounds of the context, selection and attention of a chunk's rows, as a model's prefill would call them."""
    rng = np.random.default_rng(40)
    D, QH, KVH, bs, start, M, keep, sink, recent = 128, 8, 2, 16, 411, 45, 7, 1, 2
    io = cabi.BF16
    assert host.set_attention_geometry(2, QH, KVH, D, dtype, io)
    n = -(-(start + M) // bs)
    p = R.Pool(rng, 2, KVH, QH, D, bs, n + 4, dtype, 1.5)
    table = U.shuffled_table(rng, n + 4, n)
    table[9] = -1
    q, gate = U.normal_bits(rng, (M, QH, D), io), U.normal_bits(rng, (M, QH, D), io)
    dq, dp, dt, dg, db = U.dev_bytes(q), U.dev_bytes(p.raw), U.dev_i32(table), U.dev_bytes(gate), bounds_dev(p)
    dsel, do = U.dev_i32(np.zeros((M, KVH, keep))), U.dev_zeros(q.nbytes)
    assert host.lib().drkh_paged_prefill_sparse(U.p(dq), U.p(dp), U.p(db), U.p(dt), start, M, keep, sink, recent, U.p(dsel), U.p(dg), D, U.p(do),
                                                1, n + 4, bs, 1 / math.sqrt(D), U.stream_ptr())
    codes, exps = bounds_host(p, db)
    sel = U.host(dsel, np.int32, (M, KVH, keep))
    qf = U.from_bits(q, io).astype(np.float64)
    for lb in range(n):
        if table[lb] >= 0:
            check_block(p, codes, exps, 1, table[lb], min(bs, start + M - lb * bs))
    for t in range(M):
        assert np.array_equal(sel[t], R.select(qf[t], codes[1], exps[1], table, start + t + 1, bs, keep, sink, recent)), t
    check_attend(p, U.host(do, np.uint16, q.shape), q, table, start + 1 + np.arange(M), sel, io, 1, gate)


# ---- together ---------------------------------------------------------------------------------
@pytest.mark.parametrize("D,bs,dtype", [(128, 16, cabi.BF16), (256, 64, cabi.INT8)])
def test_pages_and_bounds_beyond_32_bit_offsets(dev, D, bs, dtype):
    """The last pages of a layer of more than 4 GiB, the second of the pool, and bounds behind 4 GiB of others: what comes
    out is what the same pages give in a small pool, bit for bit."""
    import torch
    KVH, QH, io, T, keep = 4, 8, cabi.BF16, 3, 5
    rng = np.random.default_rng(bs)
    p = R.Pool(rng, 1, KVH, QH, D, bs, 40, dtype)
    L = cabi.lib()
    block = L.drk_kv_block_stride_bytes(C.byref(p.g))
    NB = (5 << 30) // block
    layers = -(-(9 << 29) // (NB * KVH * 2 * D)) + 1                        # so many that the last one's bounds lie beyond 4 GiB
    small_in_big = cabi.layout(2, KVH, QH, D, bs, NB, dtype)
    many = cabi.layout(layers, KVH, QH, D, bs, NB, dtype)
    big = torch.empty(L.drk_kv_pool_bytes(C.byref(small_in_big)), dtype=torch.uint8, device="cuda")
    at = big.numel() // 2 + (NB - 40) * block
    assert at - big.numel() // 2 > 1 << 32
    big[at:at + 40 * block].copy_(U.dev_bytes(p.raw))
    tables = rng.permutation(40)[:36].astype(np.int32).reshape(T, 12)
    lens = np.array([12 * bs - 3, 5 * bs + 1, 7 * bs], np.int32)
    q = U.dev_bytes(U.normal_bits(rng, (T, QH, D), io))
    dl = U.dev_i32(lens)

    def run(g, pool, layer, bg, blayer, tab):
        """bounds of `layer` of the pool into that layer of a buffer, then moved to layer `blayer` of the selection's layout"""
        db = torch.zeros(L.drk_kv_bounds_bytes(C.byref(g)), dtype=torch.uint8, device="cuda")
        dt = U.dev_i32(tab)
        for t in range(T):
            cabi.call("drk_kv_bounds_update", g, U.p(pool), dt.data_ptr() + 48 * t, 0, None, 0, int(lens[t]), layer, 1, U.p(db), U.stream_ptr())
        if bg is not g:
            n, n1 = NB * KVH * 2 * D, NB * KVH
            wide = torch.empty(L.drk_kv_bounds_bytes(C.byref(bg)), dtype=torch.uint8, device="cuda")
            wide[blayer * n:(blayer + 1) * n].copy_(db[layer * n:(layer + 1) * n])
            wide[layers * n + blayer * n1:layers * n + (blayer + 1) * n1].copy_(db[2 * n + layer * n1:2 * n + (layer + 1) * n1])
            db = wide
        ids = U.dev_i32(tab.reshape(-1))
        values = torch.empty(36 * KVH * 2 * D, dtype=torch.int16, device="cuda")
        cabi.call("drk_kv_bounds_extract", bg, U.p(values), U.p(db), U.p(ids), 36, blayer, 1, U.stream_ptr())
        sel = U.dev_i32(np.zeros((T, KVH, keep)))
        ws = U.dev_zeros(max(L.drk_block_select_workspace_bytes(C.byref(bg), T, 12 * bs), L.drk_paged_sparse_workspace_bytes(C.byref(g), T, keep)))
        cabi.call("drk_block_select", bg, U.p(db), blayer, U.p(q), io, U.p(dt), 12, U.p(dl), 0, T, 12 * bs, keep, 1, 1, U.p(sel), U.p(ws),
                  ws.numel(), U.stream_ptr())
        out = U.dev_zeros(T * QH * D * 2)
        cabi.call("drk_paged_sparse_attention", g, U.p(q), U.p(pool), U.p(dt), 12, U.p(dl), 0, T, U.p(sel), keep, U.p(out), layer,
                  1 / math.sqrt(D), io if dtype == cabi.INT8 else dtype, None, 0, U.p(ws), ws.numel(), U.stream_ptr())
        U.sync()
        return U.host(values, np.int16), U.host(sel, np.int32), U.host(out, np.uint16)

    dp = U.dev_bytes(p.raw)
    near = run(p.g, dp, 0, p.g, 0, tables)
    far = run(small_in_big, big, 1, many, layers - 1, (tables + (NB - 40)).astype(np.int32))
    for a, b in zip(near, far):
        assert np.array_equal(a, b)
    assert near[2].any()


def test_a_decode_step_of_all_four_eager_and_captured(dev):
    """Rotation out of the Q | gate projection, append, bounds, selection, attention: three branches, three steps; then the
    same steps from a captured graph, with eager work between the replays."""
    import torch
    rng = np.random.default_rng(21)
    D, QH, KVH, bs, B, n, steps = 128, 8, 2, 16, 3, 30, 3
    p = R.Pool(rng, 1, KVH, QH, D, bs, B * n, cabi.BF16)
    tables = rng.permutation(p.NB).astype(np.int32).reshape(B, n)
    pos = np.array([100, 250, 31], np.int32)
    r = cabi.rope(64, False, 1e6, 16.0, 4096.0, 1.0, 32.0, 1.277)
    f = freqs_of(r)
    keep, sink, recent, scale = 6, 1, 2, 1 / math.sqrt(D)
    qg = [U.normal_bits(rng, (B, QH, 2 * D), cabi.BF16) for _ in range(steps)]
    kn = [U.normal_bits(rng, (B, KVH, D), cabi.BF16) for _ in range(steps)]
    vn = [U.normal_bits(rng, (B, KVH, D), cabi.BF16) for _ in range(steps)]
    raw0 = p.raw.copy()

    dp, dt = U.dev_bytes(p.raw), U.dev_i32(tables)
    db = bounds_dev(p)
    dpos, dlen = U.dev_i32(pos), U.dev_i32(pos + 1)
    dqg, dk, dv = U.dev_zeros(qg[0].nbytes), U.dev_zeros(kn[0].nbytes), U.dev_zeros(vn[0].nbytes)
    dq, dkr, do = U.dev_zeros(B * QH * D * 2), U.dev_zeros(kn[0].nbytes), U.dev_zeros(B * QH * D * 2)
    dsel = U.dev_i32(np.zeros((B, KVH, keep)))
    L = cabi.lib()
    w1 = U.dev_zeros(L.drk_block_select_workspace_bytes(C.byref(p.g), B, n * bs))
    w2 = U.dev_zeros(max(16, L.drk_paged_sparse_workspace_bytes(C.byref(p.g), B, keep)))

    def step(st):
        rows = cabi.rope_rows([(dqg.data_ptr(), dq.data_ptr(), QH, QH * 2 * D, 2 * D, QH * D, D),
                               (dk.data_ptr(), dkr.data_ptr(), KVH, KVH * D, D, KVH * D, D)])
        cabi.call("drk_rope_apply", r, U.p(f), rows, 2, B, D, U.p(dpos), 0, 0, cabi.BF16, st)
        cabi.call("drk_kv_append_branches", p.g, U.p(dp), U.p(dt), n, U.p(dpos), B, 0, 1, U.p(dkr), U.p(dv), cabi.BF16, st)
        cabi.call("drk_kv_bounds_update", p.g, U.p(dp), U.p(dt), n, U.p(dpos), 0, B, 0, 1, U.p(db), st)
        cabi.call("drk_block_select", p.g, U.p(db), 0, U.p(dq), cabi.BF16, U.p(dt), n, U.p(dlen), 0, B, n * bs, keep, sink, recent,
                  U.p(dsel), U.p(w1), w1.numel(), st)
        cabi.call("drk_paged_sparse_attention", p.g, U.p(dq), U.p(dp), U.p(dt), n, U.p(dlen), 0, B, U.p(dsel), keep, U.p(do), 0, scale,
                  cabi.BF16, dqg.data_ptr() + 2 * D, 2 * D, U.p(w2), w2.numel(), st)
        cabi.call("drk_positions_advance", U.p(dpos), U.p(dlen), B, 1, st)

    def reset():
        dp.copy_(torch.from_numpy(raw0.reshape(-1)))
        dpos.copy_(torch.from_numpy(pos))
        dlen.copy_(torch.from_numpy(pos + 1))
        for b in range(B):
            cabi.call("drk_kv_bounds_update", p.g, U.p(dp), dt.data_ptr() + 4 * n * b, n, None, 0, int(pos[b]), 0, 1, U.p(db), U.stream_ptr())

    def feed(i):
        for buf, x in ((dqg, qg[i]), (dk, kn[i]), (dv, vn[i])):
            buf.copy_(torch.from_numpy(x.view(np.uint8).reshape(-1)))

    reset()
    eager = []
    for i in range(steps):
        feed(i)
        step(U.stream_ptr())
        U.sync()
        eager.append((U.host(dsel, np.int32, (B, KVH, keep)).copy(), U.host(do, np.uint16, (B, QH, D)).copy()))
        # every stage against its definition, on what the stage before it left on the device
        now = pos + i
        q = U.host(dq, np.uint16, (B, QH, D))
        kr = U.host(dkr, np.uint16, (B, KVH, D))
        want, mag = R.rope(r, U.from_bits(qg[i][..., :D], cabi.BF16), now)
        rope_ok(U.from_bits(q, cabi.BF16).astype(np.float64), None, want, mag, cabi.BF16, np.arange(D) < 64)
        vals = U.host(dp, np.uint16, (p.NB, 2, KVH, bs, D))
        for b in range(B):
            blk, at = tables[b, now[b] // bs], now[b] % bs
            assert np.array_equal(vals[blk, 0, :, at], kr[b]) and np.array_equal(vals[blk, 1, :, at], vn[i][b])
        f64 = U.from_bits(vals, cabi.BF16).astype(np.float64)
        p.k, p.v = f64[None, :, 0], f64[None, :, 1]
        codes, exps = bounds_host(p, db)
        for b in range(B):
            for lb in range(now[b] // bs + 1):
                check_block(p, codes, exps, 0, tables[b, lb], min(bs, now[b] + 1 - lb * bs))
            sel = R.select(U.from_bits(q[b], cabi.BF16).astype(np.float64), codes[0], exps[0], tables[b], int(now[b]) + 1, bs, keep, sink, recent)
            assert np.array_equal(eager[-1][0][b], sel)
        check_attend(p, eager[-1][1], q, tables, now + 1, eager[-1][0], cabi.BF16, 0, np.ascontiguousarray(qg[i][..., D:]))
    reset()
    st = C.c_void_p()
    cabi.call("drk_stream_create", C.byref(st))
    U.sync()
    cabi.call("drk_graph_begin_capture", st)
    step(st)
    ge = C.c_void_p()
    cabi.call("drk_graph_end_capture", st, C.byref(ge))
    for rep in range(2):
        if rep:
            reset()
        for i in range(steps):
            feed(i)
            U.sync()
            cabi.call("drk_graph_launch", ge, st)
            cabi.call("drk_stream_synchronize", st)
            assert np.array_equal(U.host(dsel, np.int32, (B, KVH, keep)), eager[i][0]), (rep, i)
            assert np.array_equal(U.host(do, np.uint16, (B, QH, D)), eager[i][1]), (rep, i)
    cabi.call("drk_graph_destroy", ge)
    cabi.call("drk_stream_destroy", st)
