"""GPU: calls of the long-context operators at the edges of what their definitions allow."""
import ctypes as C
import math

import numpy as np
import pytest

from deusridet_amd import cabi, host
from tests import longctx_ref as R
from tests import test_gpu_longctx as G
from tests import util as U

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
