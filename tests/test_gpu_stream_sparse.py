"""GPU: the stream driver decoding over selected blocks.  Every step is checked against the definitions in 64 bits
(bounds from the pool's bytes, selection, attention over the selected blocks, gate), a captured step against the
eager one bit for bit, and a selection of everything against the whole-context path."""
import ctypes as C

import numpy as np
import pytest

from deusridet_amd import cabi, host
from tests import longctx_ref as R
from tests import test_gpu_stream as S
from tests import util as U
from tests.test_gpu_stream import eight_bit_pages, reference_model_shape  # noqa: F401 (fixtures: they change the shapes of S)

pytestmark = pytest.mark.gpu


class View:
    """The pool's bytes as float64 keys and values, as longctx_ref's attention reads them (16-bit pages)."""

    def __init__(self, s):
        self.L, self.KVH, self.QH, self.D, self.bs, self.NB, self.dtype = S.L, S.KVH, S.QH, S.D, S.BS, s.NB, S.KVDT
        v = U.from_bits(s.pool().view(np.uint16).reshape(S.L, s.NB, 2, S.KVH, S.BS, S.D), S.KVDT).astype(np.float64)
        self.k, self.v = v[:, :, 0], v[:, :, 1]


def prefill(s, rng, chunks):
    st = U.stream_ptr()
    for M in chunks:
        assert s.ks.begin_prefill(M, st)
        for layer in range(S.L):
            s.load(*(U.normal_bits(rng, sh, S.DT, m) for sh, m in (((M, S.QH, 2 * S.D), 1.0), ((M, S.KVH, S.D), 0.7), ((M, S.KVH, S.D), 0.5))))
            s.ks.prefill_layer(layer, s.io(), M, st)
            U.sync()
        s.ks.end_prefill(M, st)


def step_inputs(rng, n):
    return [tuple(U.normal_bits(rng, sh, S.DT, m) for sh, m in (((n, S.QH, 2 * S.D), 1.0), ((n, S.KVH, S.D), 0.7), ((n, S.KVH, S.D), 0.5)))
            for _ in range(S.L)]


def check_step(s, layer, ids, pos, qg, got, keep, sink, recent):
    view = View(s)
    q = U.from_bits(U.host(s.bufs["q"], np.uint16)[:len(ids) * S.QH * S.D].reshape(len(ids), S.QH, S.D), S.DT).astype(np.float64)
    gate = U.from_bits(np.ascontiguousarray(qg[..., S.D:]), S.DT).astype(np.float64)
    codes, exps = np.zeros((view.NB, S.KVH, 2, S.D), np.int8), np.zeros((view.NB, S.KVH), np.int8)
    for i, b in enumerate(ids):
        table, length = s.cm.h_block_table(b), int(pos[i]) + 1
        for lb in range(-(-length // S.BS)):
            blk = table[lb]
            if blk < 0:
                continue
            for h in range(S.KVH):                          # a shared block holds whole stretches only, so min() serves every branch
                codes[blk, h, 0], codes[blk, h, 1], exps[blk, h] = R.bounds(view.k[layer, blk, h, :min(S.BS, length - lb * S.BS)])
        sel = R.select(q[i], codes, exps, table, length, S.BS, keep, sink, recent)
        want, tol = R.attend(view, layer, q[i], table, length, sel, 1 / np.sqrt(S.D), gate[i])
        ok, r = R.attend_ok(U.from_bits(got[i], S.DT), want, tol, S.DT)
        assert ok, (layer, i, r)


def session(nbranch, when, keep, sink, recent, mode, steps=4, seed=9, chunks=(64, 64, 37)):
    s = S.Session(nbranch)
    rng = np.random.default_rng(seed)
    s.set_weights(U.normal_bits(rng, (S.D,), S.DT), U.normal_bits(rng, (S.D,), S.DT))
    st = U.stream_ptr()
    policy = lambda: keep == 0 or s.ks.set_sparse_decode(0, keep, sink, recent, st)
    if when == "first":
        assert policy()
    prefill(s, rng, chunks)
    if when == "filled":
        assert policy()
    assert s.ks.open_branches(nbranch) == nbranch
    if when == "open":
        assert policy()
    ids = [s.ks.branch_id(i) for i in range(nbranch)]
    outs = []
    if mode == "graph":
        import torch
        lay = [dict(qg=U.dev_zeros(nbranch * S.QH * 2 * S.D * 2), k=U.dev_zeros(nbranch * S.KVH * S.D * 2), v=U.dev_zeros(nbranch * S.KVH * S.D * 2),
                    q=U.dev_zeros(nbranch * S.QH * S.D * 2), out=U.dev_zeros(nbranch * S.QH * S.D * 2)) for _ in range(S.L)]

        def layers(stream):
            for i, b in enumerate(lay):
                s.ks.decode_layer(i, (U.p(b["qg"]), U.p(b["k"]), U.p(b["v"]), U.p(s.dqw), U.p(s.dkw), U.p(b["q"]), U.p(b["out"])), stream)

        side = torch.cuda.Stream()
        sp = C.c_void_p(side.cuda_stream)
        assert s.ks.capture_decode_step(layers, sp)
    for step in range(steps):
        inputs = step_inputs(rng, nbranch)
        if mode == "graph":
            for b, (qg, k, v) in zip(lay, inputs):
                for name, a in (("qg", qg), ("k", k), ("v", v)):
                    b[name].copy_(torch.from_numpy(a.view(np.uint8).reshape(-1)))
            torch.cuda.synchronize()
            assert s.ks.replay_decode_step(sp)
            side.synchronize()
            outs.append([U.host(b["out"], np.uint16).reshape(nbranch, S.QH, S.D).copy() for b in lay])
            continue
        assert s.ks.begin_decode_step(st)
        pos = [s.ks.branch_pos(i) for i in range(nbranch)]
        row = []
        for layer, x in enumerate(inputs):
            s.load(*x)
            s.ks.decode_layer(layer, s.io(), st)
            row.append(s.out(nbranch))
            if keep and S.KVDT in (cabi.F16, cabi.BF16):
                check_step(s, layer, ids, pos, x[0], row[-1], keep, sink, recent)
        s.ks.end_decode_step(st)
        outs.append(row)
    return s, outs


@pytest.mark.parametrize("when", ["first", "filled", "open"])
@pytest.mark.parametrize("nbranch", [1, 3])
def test_decode_over_selected_blocks(dev, when, nbranch):
    session(nbranch, when, 5, 1, 2, "eager")


def test_captured_step_equals_eager(dev):
    _, eager = session(3, "filled", 4, 1, 1, "eager")
    _, graph = session(3, "filled", 4, 1, 1, "graph")
    assert all(np.array_equal(a, b) for x, y in zip(eager, graph) for a, b in zip(x, y))


def test_reference_model_shape(dev, reference_model_shape):
    session(2, "open", 1, 0, 0, "eager", steps=2, chunks=(64,) * 5)


def test_a_selection_of_everything_equals_the_whole_context(dev):
    a, sparse = session(3, "first", 40, 0, 0, "eager")
    pool = a.pool()
    b, dense = session(3, "first", 0, 0, 0, "eager")
    assert np.array_equal(pool, b.pool())
    for x, y in zip(sparse, dense):
        for p, q in zip(x, y):
            ok, mx, _ = U.rel_abs_ok(U.from_bits(p, S.DT), U.from_bits(q, S.DT))
            assert ok, mx


def test_eight_bit_pages(dev, eight_bit_pages):
    a, sparse = session(2, "filled", 40, 0, 0, "eager", steps=2)
    b, dense = session(2, "filled", 0, 0, 0, "eager", steps=2)
    for x, y in zip(sparse, dense):
        for p, q in zip(x, y):
            ok, mx, _ = U.rel_abs_ok(U.from_bits(p, S.DT), U.from_bits(q, S.DT))
            assert ok, mx


def test_short_contexts_stay_on_the_whole_path_and_policy_can_change(dev):
    s = S.Session(2)
    rng = np.random.default_rng(2)
    s.set_weights(U.normal_bits(rng, (S.D,), S.DT), U.normal_bits(rng, (S.D,), S.DT))
    st = U.stream_ptr()
    assert s.ks.set_sparse_decode(104, 3, 1, 1, st)                  # from 104 tokens on
    prefill(s, rng, (64, 36))
    assert s.ks.open_branches(2) == 2
    ids = [s.ks.branch_id(i) for i in range(2)]
    for step in range(8):
        assert s.ks.begin_decode_step(st)
        pos = [s.ks.branch_pos(i) for i in range(2)]
        if step == 6:
            assert s.ks.set_sparse_decode(0, 2, 0, 1, st)            # another budget between steps
        for layer, x in enumerate(step_inputs(rng, 2)):
            s.load(*x)
            s.ks.decode_layer(layer, s.io(), st)
            got = s.out(2)
            keep, sink, recent = (7, 0, 0) if pos[0] + 1 < 104 else ((3, 1, 1) if step < 6 else (2, 0, 1))   # 7 blocks: all
            check_step(s, layer, ids, pos, x[0], got, keep, sink, recent)
        s.ks.end_decode_step(st)
    assert s.ks.set_sparse_decode(0, 0, 0, 0, st) and s.ks.set_sparse_decode(0, 0, 0, 0, st)


def test_refusals(dev, tmp_path):
    s = S.Session(1)
    for bad in ((-1, 4, 1, 1), (0, -4, 0, 0), (0, 4, 3, 2), (0, 4, -1, 0), (0, 4, 0, 5)):
        assert not s.ks.set_sparse_decode(*bad)
    scored = S.Session(1, scorer=True)
    assert not scored.ks.set_sparse_decode(0, 4, 1, 1)
    assert not host.KvStream().set_sparse_decode(0, 4, 1, 1)         # not initialised


def test_a_scorer_that_is_not_ready_yet_is_refused_too(dev):
    s = S.Session(1)
    sc, ks = host.ImportanceScorer(), host.KvStream()
    assert ks.init(s.cm, S.NPOS, sc, U.p(s.dtab), S.NPOS)
    assert not ks.set_sparse_decode(0, 4, 1, 1)
