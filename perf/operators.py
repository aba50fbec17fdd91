"""Cases of the long-context operators: rotary positions with stretched frequencies, the per-block
bounds of the cached keys, the selection of blocks by a score against those bounds, and paged
attention over the selected blocks.

`run` computes a case in elementary torch operations, or -- with the module's `own` set -- through
the library's entry points on the same inputs.  A pool, a bounds buffer and a block table are laid
out as include/drk_kv.h states."""
import math

import torch

own = False

F16, BF16, INT8, FP8 = 0, 1, 2, 3
KINDS = {"f16": (F16, torch.float16, 2), "bf16": (BF16, torch.bfloat16, 2),
         "int8": (INT8, torch.int8, 1), "fp8": (FP8, torch.float8_e4m3fn, 1)}
# (query heads, kv heads, head_dim): the benchmark's shape, the reference model's, and the unit tests' neighbours of
# the two (one query head per kv head, sixteen, and the smallest of the fixtures)
SHAPES = [(32, 8, 128), (24, 4, 256), (16, 4, 128), (8, 8, 128), (16, 1, 128)]


def listed():
    flag = {"bf16": dict(QH=32, KVH=8, D=128, bs=16), "ref": dict(QH=24, KVH=4, D=256, bs=256)}
    return [
        # one decode step of 64 branches far into a context that is 32 times the trained one: the reference model's
        # quarter of a head, rotated straight out of its Q | gate projection
        dict(name="rope 64 branches", op="rope", mode="branches", T=64, ctx=1 << 20, rotary=64, interleaved=True, factor=32.0,
             inverse=False, gated=True, io="f16", **flag["ref"]),
        # a long perception chunk, whole heads
        dict(name="rope chunk 8192", op="rope", mode="chunk", T=8192, ctx=120001, rotary=128, interleaved=False, factor=8.0,
             inverse=False, gated=False, io="bf16", **flag["bf16"]),
        # what a decode step adds to the bounds: one token for each of 8 branches
        dict(name="bounds 8 branches", op="bounds", mode="branches", T=8, ctx=32768, layers=1, store="bf16", **flag["bf16"]),
        # a 2048-token chunk of the reference model that begins inside a page, all 16 layers at once
        dict(name="bounds chunk 2048", op="bounds", mode="chunk", T=2048, ctx=10007, layers=16, store="f16", **flag["ref"]),
        # the bounds of a whole 128k context over quantised pages, built after it was loaded
        dict(name="bounds 128k int8", op="bounds", mode="chunk", T=131072, ctx=0, layers=1, store="int8", **flag["bf16"]),
        # one branch at 32k: the latency case
        dict(name="select 1x32k", op="select", mode="branches", T=1, ctx=32768, keep=64, sink=1, recent=4, holes=0, io="bf16",
             **flag["bf16"]),
        # 16 branches up to 64k, ragged, a few pages evicted
        dict(name="select 16x64k", op="select", mode="branches", T=16, ctx=65536, keep=128, sink=1, recent=8, holes=3, io="bf16",
             **flag["bf16"]),
        # every token of a perception chunk selects for itself; small pages under the reference model's heads
        dict(name="select chunk 512", op="select", mode="chunk", T=512, ctx=31007, keep=64, sink=1, recent=4, holes=0, io="f16",
             QH=24, KVH=4, D=256, bs=16),
        # attention of the latency case: 1024 of 32k tokens
        dict(name="attend 1x64", op="attend", mode="branches", T=1, ctx=32768, keep=64, store="bf16", io="bf16", gated=False,
             **flag["bf16"]),
        # 16 branches up to 128k over quantised pages, gate folded in as the layer has it
        dict(name="attend 16x128 int8", op="attend", mode="branches", T=16, ctx=131072, keep=128, store="int8", io="bf16",
             gated=True, **flag["bf16"]),
        # the largest decode step: 64 branches, 4096 tokens each
        dict(name="attend 64x256", op="attend", mode="branches", T=64, ctx=32768, keep=256, store="bf16", io="bf16", gated=False,
             **flag["bf16"]),
        # a perception chunk whose tokens each read their own blocks
        dict(name="attend chunk 512", op="attend", mode="chunk", T=512, ctx=31007, keep=64, store="bf16", io="bf16", gated=False,
             **flag["bf16"]),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    QH, KVH, D = rng.choice(SHAPES)
    bs = rng.choice([16, 16, 32, 48, 64, 256])
    op = rng.choice(["rope", "bounds", "select", "attend"])
    mode = rng.choice(["branches", "chunk"])
    c = dict(op=op, mode=mode, QH=QH, KVH=KVH, D=D, bs=bs)
    if op == "rope":
        T = _log(rng, 1, 64) if mode == "branches" else _log(rng, 1, 8192 * 40 * 128 // ((QH + KVH) * D))
        c.update(T=T, ctx=_log(rng, 1, 1 << 20), rotary=rng.choice([D, D // 2, D // 4, 48]), interleaved=rng.random() < 0.5,
                 factor=rng.choice([1.0, 2.5, 8.0, 32.0]), inverse=rng.random() < 0.4, gated=rng.random() < 0.4,
                 io=rng.choice(["bf16", "f16"]))
    elif op == "bounds":
        T = _log(rng, 1, 64) if mode == "branches" else _log(rng, 1, 131072)
        ctx = _log(rng, 1, 32768)
        most = min(16, 131072 * 1024 // (T * KVH * D * 2)) if mode == "chunk" else min(8, 64 * 32768 // (T * ctx))
        layers = _log(rng, 1, max(1, most))
        c.update(T=T, ctx=ctx, layers=layers, store=rng.choice(["bf16", "f16", "int8", "fp8"]))
    elif op == "select":
        T = _log(rng, 1, 16) if mode == "branches" else _log(rng, 1, 512)
        sink, recent = rng.randint(0, 2), rng.randint(0, 8)
        c.update(T=T, ctx=_log(rng, 1, 65536 if mode == "branches" else 31007), keep=rng.randint(sink + recent + 1, 160), sink=sink,
                 recent=recent, holes=rng.choice([0, 0, 3, 20]), io=rng.choice(["bf16", "f16"]))
    else:
        T = _log(rng, 1, 64) if mode == "branches" else _log(rng, 1, 512)
        most = 64 * 256 * 8 * 128 * 16 // (T * KVH * D * bs)
        store = rng.choice(["bf16", "f16", "int8", "fp8"])
        c.update(T=T, ctx=_log(rng, 1, 32768), keep=_log(rng, 1, max(1, min(512, most, 65536 // bs))), store=store,
                 io=store if store in ("bf16", "f16") else rng.choice(["bf16", "f16"]), gated=rng.random() < 0.5)
    return c


# ---- inputs ----------------------------------------------------------------------------------------------------
def _lengths(c, gen):
    """Tokens each row sees: a chunk's rows follow its start, branches are ragged up to ctx."""
    if c["mode"] == "chunk":
        return c["ctx"] + 1 + torch.arange(c["T"], device="cuda", dtype=torch.int32)
    if c["T"] == 1:
        return torch.full((1,), c["ctx"], device="cuda", dtype=torch.int32)
    lens = torch.randint(max(1, c["ctx"] // 2), c["ctx"] + 1, (c["T"],), generator=gen, device="cuda", dtype=torch.int32)
    lens[0] = c["ctx"]
    return lens


def _tables(c, gen, lens):
    """(table [rows, stride], pages): shuffled pages, -1 behind each row's last block; one table for a chunk."""
    rows = 1 if c["mode"] == "chunk" else c["T"]
    longest = c["ctx"] + (c["T"] if c["mode"] == "chunk" else 0)
    n = -(-longest // c["bs"])
    nb = (lens[-1:] if c["mode"] == "chunk" else lens).add(c["bs"] - 1).div(c["bs"], rounding_mode="floor")
    pages = rows * n + 5
    table = torch.randperm(pages, generator=gen, device="cuda")[:rows * n].view(rows, n).to(torch.int32)
    at = torch.arange(n, device="cuda")
    table = torch.where(at[None] < nb[:, None], table, torch.full_like(table, -1))
    if c.get("holes"):                                    # evicted pages, never the ones the row writes to
        gone = torch.rand((rows, n), generator=gen, device="cuda") * 100 < c["holes"]
        table = torch.where(gone & (at[None] + 2 < nb[:, None]), torch.full_like(table, -1), table)
    table = torch.cat([table, torch.full((rows, 3), -1, device="cuda", dtype=torch.int32)], 1)
    return table.contiguous(), pages


def _normal(shape, gen, dtype):
    return torch.randn(shape, generator=gen, device="cuda", dtype=dtype)


def _pool(c, gen, layers, pages):
    """Pages of random keys and values as bytes; keys have a mean of their own per (layer, head, dim)."""
    _, dt, E = KINDS[c["store"]]
    KVH, bs, D = c["KVH"], c["bs"], c["D"]
    vals = (layers * pages, 2, KVH, bs, D)
    if c["store"] == "int8":
        x = torch.randint(-127, 128, vals, generator=gen, device="cuda", dtype=torch.int8)
        s = (torch.rand((layers * pages, 2, KVH, bs), generator=gen, device="cuda") * 0.02 + 0.004).to(torch.float16)
        parts = [x.view(layers * pages, -1).view(torch.uint8), s.view(layers * pages, -1).view(torch.uint8)]
        return torch.cat(parts, 1).reshape(-1)
    if c["store"] == "fp8":
        x = _normal(vals, gen, torch.float16).to(dt)
    else:
        x = _normal(vals, gen, dt)
        x[:, 0] += _normal((KVH, 1, D), gen, dt)
    return x.view(torch.uint8).reshape(-1)


def prepare(case, seed):
    c = dict(case)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    T, QH, KVH, D = c["T"], c["QH"], c["KVH"], c["D"]
    s = dict(c=c)
    if c["op"] == "rope":
        io = KINDS[c["io"]][1]
        s["q"] = _normal((T, QH, 2 * D if c["gated"] else D), gen, io)       # gated: the query half of a Q | gate projection
        s["k"] = _normal((T, KVH, D), gen, io)
        s["pos"] = None
        if c["mode"] == "branches":
            s["pos"] = torch.randint(0, c["ctx"], (T,), generator=gen, device="cuda", dtype=torch.int32)
            s["pos"][0] = c["ctx"] - 1
        s["q_out"] = torch.empty((T, QH, D), device="cuda", dtype=io)
        s["k_out"] = torch.empty((T, KVH, D), device="cuda", dtype=io)
        s["freqs"] = _turns(c).cuda()
        return s
    if c["op"] == "bounds":
        lens = _lengths(c, gen)
        table, pages = _tables(c, gen, lens)
        s.update(table=table, pages=pages, pool=_pool(c, gen, c["layers"], pages))
        if c["mode"] == "branches":
            s["pos"] = lens - 1
            s["blocks"] = table.gather(1, (s["pos"] // c["bs"]).long()[:, None]).reshape(-1).contiguous()
        else:
            s["pos"] = None
            first, last = c["ctx"] // c["bs"], (c["ctx"] + T - 1) // c["bs"]
            s["blocks"] = table[0, first:last + 1].contiguous()
        s["bounds"] = torch.zeros(_bounds_bytes(c["layers"], pages, KVH, D), device="cuda", dtype=torch.uint8)
        s["out"] = torch.empty((c["layers"], s["blocks"].numel(), KVH, 2, D), device="cuda", dtype=torch.bfloat16)
        return s
    lens = _lengths(c, gen)
    table, pages = _tables(c, gen, lens)
    s.update(table=table, pages=pages, lens=lens if c["mode"] == "branches" else None)
    io = KINDS[c["io"]][1]
    s["q"] = _normal((T, QH, D), gen, io)
    if c["op"] == "select":
        # bounds as blocks of keys with a mean have them: low and high around a common centre, codes within 7 bits
        mid = torch.randn((1, KVH, 1, D), generator=gen, device="cuda") * 25
        half = torch.rand((pages, KVH, 2, D), generator=gen, device="cuda") * 40 + 20
        half[:, :, 0].neg_()
        codes = (mid + half).round().clamp(-127, 127).to(torch.int8)
        exps = torch.randint(-6, -3, (pages, KVH), generator=gen, device="cuda", dtype=torch.int8)
        flat = torch.zeros(_bounds_bytes(1, pages, KVH, D), device="cuda", dtype=torch.uint8)
        flat[:codes.numel()] = codes.view(torch.uint8).reshape(-1)
        flat[codes.numel():codes.numel() + exps.numel()] = exps.view(torch.uint8).reshape(-1)
        s["bounds"] = flat
        s["out"] = torch.empty((T, KVH, c["keep"]), device="cuda", dtype=torch.int32)
        s["ws"] = torch.empty(4 * T * KVH * (table.shape[1]) + 64, device="cuda", dtype=torch.uint8)
        return s
    s["pool"] = _pool(c, gen, 1, pages)
    n = -(-lens.long() // c["bs"])                           # blocks each row may choose from
    rank = torch.rand((T, KVH, int(n.max())), generator=gen, device="cuda")
    at = torch.arange(rank.shape[2], device="cuda")[None, None]
    rank = torch.where((at < 1) | (at + 4 >= n[:, None, None]), rank + 2, rank)         # the first block and the last four
    rank = torch.where(at < n[:, None, None], rank, torch.full_like(rank, -1))
    if rank.shape[2] < c["keep"]:
        rank = torch.cat([rank, torch.full((T, KVH, c["keep"] - rank.shape[2]), -1.0, device="cuda")], 2)
    top, idx = rank.topk(c["keep"], dim=2)
    idx = torch.where(top >= 0, idx, torch.full_like(idx, 1 << 30)).sort(dim=2).values
    s["sel"] = torch.where(idx < 1 << 30, idx, torch.full_like(idx, -1)).to(torch.int32).contiguous()
    s["gate"] = _normal((T, QH, 2 * D), gen, io) if c["gated"] else None    # the gate half of a Q | gate projection
    s["out"] = torch.zeros((T, QH, D), device="cuda", dtype=io)
    s["ws"] = torch.empty(32 << 20, device="cuda", dtype=torch.uint8)
    return s


# ---- definitions both sides read ---------------------------------------------------------------------------------
THETA, TRAINED, LOW, HIGH = 1.0e7, 32768.0, 1.0, 32.0


def _magnitude(c):
    return 1.0 if c["factor"] == 1.0 else 0.1 * math.log(c["factor"]) + 1.0


def _turns(c):
    """Turns per position of every pair, 64 bits: pairs that turn HIGH times or more over the trained context keep their
    frequency, those below LOW turns are stretched by the factor, linear in between."""
    f = THETA ** (-2.0 * torch.arange(c["rotary"] // 2, dtype=torch.float64) / c["rotary"]) / (2 * math.pi)
    keep = ((f * TRAINED - LOW) / (HIGH - LOW)).clamp(0, 1)
    return f * (keep + (1 - keep) / c["factor"])


def _bounds_bytes(layers, pages, KVH, D):
    return -(-layers * pages * KVH * (2 * D + 1) // 16) * 16


# ---- one pass -----------------------------------------------------------------------------------------------------
def run(s):
    c = s["c"]
    return (_own if own else _plain)[c["op"]](s, c)


def _pow2(e):
    """2^e in float32 for whole e within +-126, exactly"""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _scale_exponent(amax):
    """Smallest e with amax <= 127 * 2^e, kept within +-40; amax as float32."""
    m, x = torch.frexp(amax)
    e = torch.where(m * 128 <= 127, x - 7, x - 6)
    return torch.where(amax > 0, e, torch.full_like(e, -40)).clamp(-40, 40)


def _rope(s, c):
    pos = s["pos"].double() if s["pos"] is not None else c["ctx"] + torch.arange(c["T"], device="cuda", dtype=torch.float64)
    ang = pos[:, None] * s["freqs"][None]
    ang = (ang - ang.floor()) * (2 * math.pi)
    cos = (torch.cos(ang) * _magnitude(c)).float()[:, None]
    sin = (torch.sin(ang) * (-_magnitude(c) if c["inverse"] else _magnitude(c))).float()[:, None]
    outs = []
    for x in (s["q"][:, :, :c["D"]], s["k"]):
        y, half = x.float(), c["rotary"] // 2
        a, b = (y[..., 0:c["rotary"]:2], y[..., 1:c["rotary"]:2]) if c["interleaved"] else (y[..., :half], y[..., half:c["rotary"]])
        ra, rb = a * cos - b * sin, b * cos + a * sin
        rot = torch.stack([ra, rb], -1).flatten(-2) if c["interleaved"] else torch.cat([ra, rb], -1)
        outs.append(torch.cat([rot, y[..., c["rotary"]:]], -1).to(x.dtype))
    return outs


def _rope_own(s, c):
    from deusridet_amd import cabi
    T, QH, KVH, D = c["T"], c["QH"], c["KVH"], c["D"]
    q, k = s["q"], s["k"]
    d = cabi.rope(c["rotary"], c["interleaved"], THETA, c["factor"], TRAINED, LOW, HIGH, _magnitude(c))
    rows = cabi.rope_rows([(q.data_ptr(), s["q_out"].data_ptr(), QH, q.stride(0), q.stride(1), QH * D, D),
                           (k.data_ptr(), s["k_out"].data_ptr(), KVH, KVH * D, D, KVH * D, D)])
    cabi.call("drk_rope_apply", d, s["freqs"].data_ptr(), rows, 2, T, D, cabi.p(s["pos"]),
              0 if c["mode"] == "branches" else c["ctx"], c["inverse"], KINDS[c["io"]][0], cabi.stream_ptr())
    return [s["q_out"], s["k_out"]]


def _page_values(s, c, pages, layers, kv):
    """Keys (kv = 0) or values of physical pages [n] of every layer as float32 [layers, n, KVH, bs, D]."""
    KVH, bs, D = c["KVH"], c["bs"], c["D"]
    _, dt, E = KINDS[c["store"]]
    plane = KVH * bs * D * E
    blocks = s["pool"].view(layers, s["pages"], -1)[:, pages]
    x = blocks[..., kv * plane:(kv + 1) * plane].contiguous().view(dt).view(*blocks.shape[:2], KVH, bs, D).float()
    if c["store"] == "int8":
        at = 2 * plane + kv * KVH * bs * 2
        sc = blocks[..., at:at + KVH * bs * 2].contiguous().view(torch.float16).view(*blocks.shape[:2], KVH, bs, 1)
        x = x * sc.float()
    return x


def _bounds_tokens(s, c):
    """(physical pages [n], tokens of each that count [n])"""
    if s["pos"] is not None:
        lb = s["pos"] // c["bs"]
        return s["table"].gather(1, lb.long()[:, None]).reshape(-1).long(), s["pos"] - lb * c["bs"] + 1
    first, end = c["ctx"] // c["bs"], c["ctx"] + c["T"]
    lb = torch.arange(first, (end - 1) // c["bs"] + 1, device="cuda")
    return s["table"][0, lb].long(), (end - lb * c["bs"]).clamp(max=c["bs"])


def _bounds(s, c):
    pages, cnt = _bounds_tokens(s, c)
    x = _page_values(s, c, pages, c["layers"], 0)
    live = (torch.arange(c["bs"], device="cuda")[None] < cnt[:, None])[None, :, None, :, None]
    lo = torch.where(live, x, torch.full_like(x, math.inf)).amin(3)
    hi = torch.where(live, x, torch.full_like(x, -math.inf)).amax(3)
    e = _scale_exponent(torch.maximum(lo.abs(), hi.abs()).amax(3, keepdim=True))
    return torch.stack([torch.floor(lo * _pow2(-e)) * _pow2(e), torch.ceil(hi * _pow2(-e)) * _pow2(e)], 3).to(torch.bfloat16)


def _layout(s, c, layers, kind):
    from deusridet_amd import cabi
    return cabi.layout(layers, c["KVH"], c["QH"], c["D"], c["bs"], s["pages"], KINDS[kind][0])


def _bounds_own(s, c):
    from deusridet_amd import cabi
    g, st, t = _layout(s, c, c["layers"], c["store"]), cabi.stream_ptr(), s["table"]
    cabi.call("drk_kv_bounds_update", g, s["pool"].data_ptr(), t.data_ptr(), t.stride(0), cabi.p(s["pos"]),
              0 if s["pos"] is not None else c["ctx"], c["T"], 0, c["layers"], s["bounds"].data_ptr(), st)
    cabi.call("drk_kv_bounds_extract", g, s["out"].data_ptr(), s["bounds"].data_ptr(), s["blocks"].data_ptr(), s["blocks"].numel(), 0,
              c["layers"], st)
    return s["out"]


def _bound_codes(s, c, pages):
    """(low and high codes, exponents) of physical pages of any shape, as float32"""
    n = s["pages"] * c["KVH"]
    codes = s["bounds"][:n * 2 * c["D"]].view(torch.int8).view(s["pages"], c["KVH"], 2, c["D"])
    exps = s["bounds"][n * 2 * c["D"]:n * (2 * c["D"] + 1)].view(torch.int8).view(s["pages"], c["KVH"])
    return codes[pages].float(), exps[pages].int()


def _select(s, c):
    T, QH, KVH, D, keep, bs = c["T"], c["QH"], c["KVH"], c["D"], c["keep"], c["bs"]
    lens = s["lens"].long() if s["lens"] is not None else c["ctx"] + 1 + torch.arange(T, device="cuda")
    table = s["table"].long()                                                  # [T or 1, n]
    codes, eb = _bound_codes(s, c, table.clamp(min=0))                         # [T or 1, n, KVH, 2, D], [T or 1, n, KVH]
    q = s["q"].float().view(T, KVH, QH // KVH, D)
    eq = _scale_exponent(q.abs().amax(3, keepdim=True))                        # [T, KVH, G, 1]
    qc = torch.round(q * _pow2(-eq))
    two = torch.cat([qc.clamp(max=0), qc.clamp(min=0)], 3)                     # against [low, high]: sum of max(q lo, q hi)
    flat = codes.flatten(3).permute(0, 2, 3, 1).contiguous()   # [T or 1, KVH, 2D, n]
    if table.shape[0] == 1:
        dots = torch.matmul(two.permute(1, 0, 2, 3).reshape(KVH, -1, 2 * D), flat[0]).view(KVH, T, QH // KVH, -1).transpose(0, 1)
    else:
        dots = torch.matmul(two, flat)                                         # [T, KVH, G, n], whole numbers below 2^24
    score = (dots * _pow2(eb.permute(0, 2, 1)[:, :, None] + eq)).amax(2)   # [T, KVH, n]
    nb = (-(-lens // bs))[:, None, None]
    at = torch.arange(table.shape[1], device="cuda")[None, None]
    here = (at < nb) & (table >= 0)[:, None]
    score = torch.where((at < c["sink"]) | (at >= nb - c["recent"]), torch.full_like(score, math.inf), score)
    score = torch.where(here, score, torch.full_like(score, -math.inf))
    if score.shape[2] < keep:
        score = torch.cat([score, torch.full((T, KVH, keep - score.shape[2]), -math.inf, device="cuda")], 2)
    top, idx = score.sort(dim=2, descending=True, stable=True)
    idx = torch.where(top[..., :keep] > -math.inf, idx[..., :keep], torch.full_like(idx[..., :keep], 1 << 30)).sort(dim=2).values
    return torch.where(idx < 1 << 30, idx, torch.full_like(idx, -1)).to(torch.int32)


def _select_own(s, c):
    from deusridet_amd import cabi
    t, T = s["table"], c["T"]
    chunk = c["mode"] == "chunk"
    cabi.call("drk_block_select", _layout(s, c, 1, "bf16"), s["bounds"].data_ptr(), 0, s["q"].data_ptr(), KINDS[c["io"]][0], t.data_ptr(),
              0 if chunk else t.stride(0), cabi.p(s["lens"]), c["ctx"] if chunk else 0, T, c["ctx"] + (T if chunk else 0), c["keep"],
              c["sink"], c["recent"], s["out"].data_ptr(), s["ws"].data_ptr(), s["ws"].numel(), cabi.stream_ptr())
    return s["out"]


def _attend(s, c):
    T, QH, KVH, D, bs = c["T"], c["QH"], c["KVH"], c["D"], c["bs"]
    lens = s["lens"].long() if s["lens"] is not None else c["ctx"] + 1 + torch.arange(T, device="cuda")
    sel = s["sel"].long()
    _, dt, E = KINDS[c["store"]]
    plane = KVH * bs * D * E
    table = s["table"].long().expand(T, -1)
    page = table[:, None].expand(T, KVH, -1).gather(2, sel.clamp(min=0))       # [T, KVH, keep]
    head = torch.arange(KVH, device="cuda")[None, :, None]
    blocks = s["pool"].view(s["pages"], -1)
    tok = sel[..., None] * bs + torch.arange(bs, device="cuda")
    live = ((sel >= 0) & (page >= 0))[..., None] & (tok < lens[:, None, None, None])       # [T, KVH, keep, bs]
    got = []
    for kv in (0, 1):
        x = blocks[:, kv * plane:(kv + 1) * plane].view(dt).view(-1, KVH, bs, D)[page.clamp(min=0), head].float()
        if c["store"] == "int8":
            at = 2 * plane + kv * KVH * bs * 2
            x = x * blocks[:, at:at + KVH * bs * 2].view(torch.float16).view(-1, KVH, bs)[page.clamp(min=0), head].float()[..., None]
        got.append(x.view(T, KVH, -1, D))
    q = s["q"].float().view(T, KVH, QH // KVH, D)
    score = torch.matmul(q, got[0].transpose(2, 3)) / math.sqrt(D)             # [T, KVH, G, keep * bs]
    score = torch.where(live.view(T, KVH, 1, -1), score, torch.full_like(score, -math.inf))
    p = torch.exp(score - score.amax(3, keepdim=True))
    out = torch.matmul(p, got[1]) / p.sum(3, keepdim=True)
    out = out.reshape(T, QH, D)
    if s["gate"] is not None:
        out = out / (1 + torch.exp(-s["gate"][..., D:].float()))
    return out.to(s["q"].dtype)


def _attend_own(s, c):
    from deusridet_amd import cabi
    t, T, D, gate = s["table"], c["T"], c["D"], s["gate"]
    chunk = c["mode"] == "chunk"
    cabi.call("drk_paged_sparse_attention", _layout(s, c, 1, c["store"]), s["q"].data_ptr(), s["pool"].data_ptr(), t.data_ptr(),
              0 if chunk else t.stride(0), cabi.p(s["lens"]), c["ctx"] if chunk else 0, T, s["sel"].data_ptr(), c["keep"],
              s["out"].data_ptr(), 0, 1 / math.sqrt(D), KINDS[c["io"]][0], None if gate is None else gate.data_ptr() + 2 * D,
              0 if gate is None else 2 * D, s["ws"].data_ptr(), s["ws"].numel(), cabi.stream_ptr())
    return s["out"]


_plain = {"rope": _rope, "bounds": _bounds, "select": _select, "attend": _attend}
_own = {"rope": _rope_own, "bounds": _bounds_own, "select": _select_own, "attend": _attend_own}


# ---- what a pass cannot do without ----------------------------------------------------------------------------------
def work(case):
    c = case
    T, QH, KVH, D, bs = c["T"], c["QH"], c["KVH"], c["D"], c["bs"]
    longest = c["ctx"] + (T if c["mode"] == "chunk" else 0)
    n = -(-longest // bs)
    if c["op"] == "rope":
        return {"bytes": T * (QH + KVH) * D * 2 * 2, "flops": 3 * T * (QH + KVH) * c["rotary"]}
    if c["op"] == "bounds":
        row = KVH * D * KINDS[c["store"]][2] + (KVH * 2 if c["store"] == "int8" else 0)
        blocks = T if c["mode"] == "branches" else (longest - 1) // bs - c["ctx"] // bs + 1
        tokens = min(blocks * bs, T * bs if c["mode"] == "branches" else longest)
        return {"bytes": c["layers"] * (tokens * row + blocks * KVH * (2 * D + 1 + 4 * D)), "flops": 2 * c["layers"] * tokens * KVH * D}
    if c["op"] == "select":
        rows = T if c["mode"] == "branches" else 1
        mean = n if rows == 1 else 0.75 * n                                  # branches are ragged between half and all of ctx
        return {"bytes": rows * mean * (KVH * (2 * D + 1) + 4) + T * (QH * D * 2 + KVH * c["keep"] * 4), "flops": 2 * T * QH * mean * 2 * D}
    keep = min(c["keep"], n)
    row = 2 * (D * KINDS[c["store"]][2] + (2 if c["store"] == "int8" else 0))
    tokens = T * keep * bs if c["mode"] == "branches" else min(T * keep * bs, longest)
    return {"bytes": tokens * KVH * row + T * (QH * D * 2 * (3 if c["gated"] else 2) + KVH * c["keep"] * 4),
            "flops": 4 * T * QH * keep * bs * D}


# ---- the definitions in 64 bits --------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    c = s["c"]
    T, QH, KVH, D, bs = c["T"], c["QH"], c["KVH"], c["D"], c["bs"]
    if c["op"] == "select":
        return None                                                          # indices: there is nothing to round
    if c["op"] == "rope":                                                    # a pair is a complex number times m e^(i angle)
        f = torch.tensor([THETA ** (-2 * i / c["rotary"]) for i in range(c["rotary"] // 2)], dtype=torch.float64, device="cuda")
        ramp = (f * TRAINED / (2 * math.pi) - LOW) / (HIGH - LOW)
        ramp = torch.minimum(torch.maximum(ramp, torch.zeros_like(ramp)), torch.ones_like(ramp))
        f = f * ramp + f / c["factor"] * (1 - ramp)
        pos = torch.arange(c["ctx"], c["ctx"] + T, device="cuda") if s["pos"] is None else s["pos"]
        turn = torch.polar(torch.full((T, 1, f.numel()), _magnitude(c), dtype=torch.float64, device="cuda"),
                           (pos.double()[:, None] * f)[:, None] * (-1 if c["inverse"] else 1))
        outs = []
        for x in (s["q"][..., :D].double(), s["k"].double()):
            h = c["rotary"] // 2
            pick = torch.arange(c["rotary"], device="cuda").view(-1, 2).T if c["interleaved"] else torch.arange(2 * h, device="cuda").view(2, h)
            z = torch.complex(x[..., pick[0]], x[..., pick[1]]) * turn
            y = x.clone()
            y[..., pick[0]], y[..., pick[1]] = z.real, z.imag
            outs.append(y)
        return outs
    if c["op"] == "bounds":
        out = []
        pages, cnt = _bounds_tokens(s, c)
        largest = torch.tensor([127 * 2.0 ** e for e in range(-40, 41)], dtype=torch.float64, device="cuda")    # by exponent
        for part in s["pool"].view(c["layers"], -1):
            x = _page_values(dict(s, pool=part), c, pages, 1, 0)[0].double()
            dead = (torch.arange(bs, device="cuda")[None] >= cnt[:, None])[:, None, :, None]
            lo, hi = x.masked_fill(dead, math.inf).min(2).values, x.masked_fill(dead, -math.inf).max(2).values
            step = largest[torch.searchsorted(largest, torch.maximum(lo.abs(), hi.abs()).amax(2)).clamp(max=80)][..., None] / 127
            out.append(torch.stack([torch.floor(lo / step) * step, torch.ceil(hi / step) * step], 2))
        return torch.stack(out)
    outs = []
    lens = c["ctx"] + 1 + torch.arange(T, device="cuda") if s["lens"] is None else s["lens"].long()
    _, dt, E = KINDS[c["store"]]
    for t in range(T):                                                        # row by row: softmax over a concatenation of blocks
        table = s["table"][t if s["table"].shape[0] > 1 else 0].long()
        sel = s["sel"][t].long()                                              # [KVH, keep]
        page = table[sel.clamp(min=0)]
        raw = s["pool"].view(s["pages"], -1)
        h = torch.arange(KVH, device="cuda")[:, None]
        plane = KVH * bs * D * E
        k, v = (raw[:, i * plane:(i + 1) * plane].view(dt).view(-1, KVH, bs, D)[page.clamp(min=0), h].double() for i in (0, 1))
        if c["store"] == "int8":
            sc = raw[:, 2 * plane:].view(torch.float16).view(-1, 2, KVH, bs)
            k, v = k * sc[page.clamp(min=0), 0, h].double()[..., None], v * sc[page.clamp(min=0), 1, h].double()[..., None]
        seen = ((sel * bs)[..., None] + torch.arange(bs, device="cuda") < lens[t]) & ((sel >= 0) & (page >= 0))[..., None]
        w = torch.matmul(s["q"][t].double().view(KVH, -1, D), k.view(KVH, -1, D).mT) * D ** -0.5
        w = torch.softmax(w.masked_fill(~seen.view(KVH, 1, -1), -math.inf), -1)
        y = torch.matmul(w, v.view(KVH, -1, D)).view(QH, D)
        outs.append(y if s["gate"] is None else y * torch.sigmoid(s["gate"][t, :, D:].double()))
    return torch.stack(outs)
