"""The operators of a paged KV cache, as a serving program calls them, with their plain forms.

Three operators on the framework's raw int16 words (power-of-two exponents):

* ``prep``: the q / k / v rows of a packed batch of sequences (any lengths, any positions) -> an optional RMS norm of
  every q and k head, the rotation at each row's position, the K / V rows written into the pages of a block table
  (16-bit words or 8-bit codes with a shift per row and head) — and the written rows read back;
* ``attn``: the causal grouped-head attention of the packed rows over the pages, with the softmax unit's integers;
* ``read``: cached rows back as int16 words.

``step`` is a decode step's prep followed by its attention.  Every output is a whole number.

``run`` takes the plain form (torch products, sums, shifts, comparisons and indexing; float64 products are exact
integers here, every sum stays below 2^53) or, with ``own``, the calls of ``cormorant_b200.ops``.
"""
import math
import random

import numpy as np
import torch

own = False

RB, F = 40, 12          # the softmax unit: R = floor(2^40 / S); its table has 2^12 entries an octave
ROPE_BITS, P1_BITS, RM_BITS = 23, 24, 47
FQ0, FN, FQ, FV0, FV = 13, 12, 10, 13, 9   # exponents: projections, normed heads, rotated q / k, v, cached v


# ------------------------------------------------------------------------------------------------------- the cases
def listed():
    base = dict(H=15, KV=5, HD=64, page=64, bits=16, window=0, norm=False, interleaved=False, rot=64)

    def c(name, kind, **kw):
        return dict(base, name=name, kind=kind, **kw)
    return [
        # one user's first short answer: nothing but latency
        c("decode_1_ctx33", "attn", B=1, ctx_lo=33, ctx_hi=33, new_lo=1, new_hi=1, page=16),
        # the framework's own decode batch: 64 sequences after prompts of up to 512 tokens, 128 tokens into the answer
        c("decode_64_ctx640", "attn", B=64, ctx_lo=128, ctx_hi=639, new_lo=1, new_hi=1),
        # long documents, 8-bit pages
        c("decode_8_ctx32k_8bit", "attn", B=8, ctx_lo=21001, ctx_hi=32767, new_lo=1, new_hi=1, bits=8),
        # a few drafted tokens a sequence checked at once, 8 query heads a group, a sliding window
        c("verify_16x5_window", "attn", B=16, ctx_lo=37, ctx_hi=4099, new_lo=1, new_hi=5, H=16, KV=2, HD=128, rot=128,
          page=32, bits=8, window=1024),
        # the framework's own prefill batch with ragged prompts
        c("prompt_64x512", "attn", B=64, ctx_lo=0, ctx_hi=0, new_lo=97, new_hi=512),
        # one long prompt
        c("prompt_1x8192", "attn", B=1, ctx_lo=0, ctx_hi=0, new_lo=8192, new_hi=8192, page=128),
        # a chunked prefill: odd chunks behind cached context, wide heads
        c("chunk_4x257_ctx8k", "attn", B=4, ctx_lo=1023, ctx_hi=8190, new_lo=255, new_hi=257, H=16, KV=4, HD=128, rot=128),
        # the rows of a whole prefill batch
        c("prep_64x512", "prep", B=64, ctx_lo=0, ctx_hi=0, new_lo=97, new_hi=512),
        # normed heads, interleaved pairs over a part of the head, 8-bit pages, ragged chunks with an empty one
        c("prep_9x1001_norm_8bit", "prep", B=9, ctx_lo=0, ctx_hi=3001, new_lo=0, new_hi=1001, H=16, KV=4, HD=128, rot=96,
          page=32, bits=8, norm=True, interleaved=True),
        # a long sequence's cached rows handed back (moved to another machine, or checked)
        c("read_3_ctx20k_8bit", "read", B=3, ctx_lo=0, ctx_hi=0, new_lo=1, new_hi=20011, bits=8),
        # the decode batch's shorter sequences handed back, small pages
        c("read_16_ctx640", "read", B=16, ctx_lo=0, ctx_hi=0, new_lo=129, new_hi=640, page=16),
        # a decode step's two calls as a layer makes them
        c("step_64_ctx640", "step", B=64, ctx_lo=128, ctx_hi=639, new_lo=1, new_hi=1),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attn", "attn", "attn", "attn", "prep", "prep", "read", "step"])
    HD = rng.choice([16, 32, 64, 64, 64, 128, 128, 256])
    KV = rng.choice([1, 2, 3, 4, 5, 8])
    G = rng.randint(1, 8)
    B = _log(rng, 1, 64)
    ctx = _log(rng, 1, 32768) - 1
    new = 1 if kind == "step" else rng.choice([1, 1, rng.randint(2, 9), _log(rng, 10, 4096)])
    window = rng.choice([0, 0, 0, _log(rng, 1, 2048)])
    top = 5.0e8  # query-head x key pairs of 64 dims, as the largest listed case has
    while True:
        pairs = B * new * (ctx + new / 2.0) * KV * G * HD / 64.0
        rows = B * new * KV * (G + 2) * HD
        held = B * (ctx + new) * KV * HD
        if pairs <= top / 2 and rows <= 4.0e7 and held <= 8.0e7:
            break
        if B > 1:
            B = max(1, B // 2)
        elif ctx > new:
            ctx //= 2
        else:
            new = max(1, new // 2)
    return dict(kind=kind, B=B, ctx_lo=ctx // 3, ctx_hi=ctx, new_lo=new if new == 1 else rng.randint(0, new), new_hi=new,
                H=KV * G, KV=KV, HD=HD, page=rng.choice([16, 32, 64, 128, 256]), bits=rng.choice([16, 8]), window=window,
                norm=rng.random() < 0.4, interleaved=rng.random() < 0.4, rot=rng.choice([HD, HD, HD // 2]))


def _lengths(case):
    """The cached tokens and the new tokens of every sequence: the case's bounds alone decide them."""
    r = random.Random("%d %d %d %d %d" % tuple(case[k] for k in ("B", "ctx_lo", "ctx_hi", "new_lo", "new_hi")))
    ctx = [r.randint(case["ctx_lo"], case["ctx_hi"]) for _ in range(case["B"])]
    new = [r.randint(case["new_lo"], case["new_hi"]) for _ in range(case["B"])]
    ctx[0], new[0] = case["ctx_hi"], case["new_hi"]
    if case["B"] > 1:
        new[-1] = case["new_lo"]
    return ctx, new


def _visible(case, ctx, n):
    """(keys that some row sees, (row, key) pairs) of one sequence."""
    w = case["window"]
    if n == 0:
        return 0, 0
    keys = ctx + n - (max(0, ctx + 1 - w) if w else 0)
    if not w:
        return keys, n * ctx + n * (n + 1) // 2
    full = [min(ctx + i + 1, w) for i in range(n)]
    return keys, sum(full)


def work(case):
    H, KV, HD = case["H"], case["KV"], case["HD"]
    ctx, new = _lengths(case)
    rows = sum(new)
    held = KV * (HD * case["bits"] // 8 + (1 if case["bits"] == 8 else 0))  # one cached row of K or of V
    seen = [_visible(case, c, n) for c, n in zip(ctx, new)]
    keys, pairs = sum(s[0] for s in seen), sum(s[1] for s in seen)
    attn = dict(bytes=4 * rows * H * HD + 2 * keys * held, flops=4 * pairs * H * HD)
    span = max(c + n for c, n in zip(ctx, new)) - min(ctx)
    prep = dict(bytes=rows * (4 * H * HD + 4 * KV * HD + 2 * held) + 4 * case["rot"] * min(rows, span),
                flops=rows * (H + KV) * HD * (10 if case["norm"] else 6) + rows * KV * HD * 2)
    read = dict(bytes=rows * (2 * held + 4 * KV * HD), flops=2 * rows * KV * HD)
    if case["kind"] == "attn":
        return attn
    if case["kind"] == "read":
        return read
    if case["kind"] == "prep":
        return dict(bytes=prep["bytes"] + read["bytes"], flops=prep["flops"] + read["flops"])
    # a step's own rows stay on the chip between its two calls, in the ideal
    return dict(bytes=prep["bytes"] + attn["bytes"] - 4 * rows * H * HD + 2 * rows * H * HD, flops=prep["flops"] + attn["flops"])


# ------------------------------------------------------------------------------------------------------- the inputs
def _scale_regs(f_s, sigma):
    """The softmax unit's scale: Cm 2^-Cs = log2(e) sigma 2^-f_s 2^12 with a 24-bit Cm."""
    c = math.log2(math.e) * sigma * 2.0 ** (F - f_s)
    cs = 23 - math.floor(math.log2(c))
    cm = int(round(c * 2.0 ** cs))
    return (cm >> 1, cs - 1) if cm >= 1 << 24 else (cm, cs)


def _entries(G, sa, sb, sc, n):
    """n 16-byte parameter entries {int32 G, int32 0, u8 sa, sb, sc}."""
    e = np.zeros((n, 16), np.uint8)
    e[:, 0:4] = np.broadcast_to(np.asarray(G, np.int64), (n,)).astype("<i4").view(np.uint8).reshape(n, 4)
    for k, v in ((8, sa), (9, sb), (10, sc)):
        e[:, k] = v
    return e


def _rot_entries(case, heads, fx):
    """The rotation's entries of every channel: products at 2^-(fx + 23) to FQ; the dims past ``rot`` from fx to FQ."""
    sc = np.full((heads, case["HD"]), fx - FQ, np.int64)
    sc[:, :case["rot"]] = fx + ROPE_BITS - FQ
    return _entries(0, 0, 0, sc.reshape(-1), heads * case["HD"])


def _bitlen(t):
    """Bits of 0 <= t < 2^15."""
    return sum((t >= (1 << k)).to(t.dtype) for k in range(15))


def _rne(x, k):
    """x / 2^k to the nearest integer, ties to even (k >= 0, tensors)."""
    q = x >> k
    r = x - (q << k)
    half = (torch.ones_like(q) << k) >> 1
    up = (k > 0) & ((r > half) | ((r == half) & ((q & 1) == 1)))
    return q + up.to(q.dtype)


def _codes(x):
    """8-bit codes and shifts of rows x [..., HD]."""
    t = torch.where(x >= 0, x, -x - 1).amax(-1, keepdim=True)
    s = (_bitlen(t) - 7).clamp(min=0)
    return _rne(x, s.expand_as(x)).clamp(-128, 127), s


def _fill(case, x, planes, shifts):
    """Whole pages from rows x [pages][KV][page][HD] (int64)."""
    if case["bits"] == 8:
        c, s = _codes(x)
        planes.copy_(c.to(torch.int8))
        shifts.copy_(s[..., 0].to(torch.uint8))
    else:
        HD = case["HD"]
        planes[..., :HD] = (x >> 8).to(torch.int8)
        planes[..., HD:] = ((x & 255) - 256 * ((x & 128) >> 7)).to(torch.int8)


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(int(seed) * 7919 + 11)
    H, KV, HD, B, page = case["H"], case["KV"], case["HD"], case["B"], case["page"]
    ctx, new = _lengths(case)
    rows = sum(new)
    blocks = [-(-(c + n) // page) for c, n in zip(ctx, new)]
    width, pages = max(blocks), sum(blocks) + 3
    ids = torch.randperm(pages, generator=g, device=dev)[:sum(blocks)].to(torch.int32)
    table = torch.full((B, width), -1, dtype=torch.int32, device=dev)
    at = 0
    for b, k in enumerate(blocks):
        table[b, :k] = ids[at:at + k]
        at += k
    cu = torch.tensor(np.concatenate([[0], np.cumsum(new)]).astype(np.int32), device=dev)
    pos = torch.tensor(ctx, dtype=torch.int32, device=dev)

    def normal(shape, std):
        return (torch.randn(shape, generator=g, device=dev) * std).round().clamp(-32768, 32767)
    std = 0.6 * (64.0 / HD) ** 0.25
    byte = (2 if case["bits"] == 16 else 1) * HD
    kc = torch.empty((pages, KV, page, byte), dtype=torch.int8, device=dev)
    vc = torch.empty_like(kc)
    ks = vs = None
    if case["bits"] == 8:
        ks = torch.empty((pages, KV, page), dtype=torch.uint8, device=dev)
        vs = torch.empty_like(ks)
    step = max(1, (1 << 24) // (KV * page * HD))
    for p in range(0, pages, step):  # in pieces: the int64 words of a long cache are large
        e = min(pages, p + step)
        _fill(case, normal((e - p, KV, page, HD), std * 2 ** FQ).to(torch.int64), kc[p:e], None if ks is None else ks[p:e])
        _fill(case, normal((e - p, KV, page, HD), 0.6 * 2 ** FV).to(torch.int64), vc[p:e], None if vs is None else vs[p:e])
    st = dict(case=case, ctx=ctx, new=new, rows=rows, kc=kc, vc=vc, ks=ks, vs=vs, table=table, cu=cu, pos=pos)
    kind = case["kind"]
    if kind in ("attn", "step"):
        f_p = 15 if max(ctx) + max(new) > 2048 else 12
        cm, cs = _scale_regs(2 * FQ - 8, 1.0 / math.sqrt(HD))
        st["smx"] = torch.tensor([[cm, cs | f_p << 8]] * H, dtype=torch.int32, device=dev)
        if kind == "attn":
            st["q"] = normal((rows, H * HD), std * 2 ** FQ).to(torch.int16)
        st["o"] = torch.empty((rows, H * HD), dtype=torch.int16, device=dev)
    if kind in ("prep", "step"):
        rot, top = case["rot"], max(c + n for c, n in zip(ctx, new))
        st["q0"], st["k0"], st["v0"] = (normal((rows, n * HD), std * 2 ** FQ0).to(torch.int16) for n in (H, KV, KV))
        ang = torch.arange(top, dtype=torch.float64, device=dev)[:, None] * \
            1e5 ** (-torch.arange(rot // 2, dtype=torch.float64, device=dev) / (rot // 2))
        st["rope"] = torch.cat([ang.cos(), ang.sin()], 1).mul(2.0 ** ROPE_BITS).round().to(torch.int32)
        fx = FN if case["norm"] else FQ0
        whole = rot == HD  # every channel alike: one broadcast entry
        for nm, n in (("pq", H), ("pk", KV)):
            e = _rot_entries(case, n, fx)
            st[nm] = torch.from_numpy(e[:1].copy() if whole else e).to(dev)
        st["pv"] = torch.from_numpy(_entries(0, 0, 0, FV0 - FV, 1)).to(dev)
        st["whole"] = whole
        if case["norm"]:
            gam = 1.0 + 0.1 * torch.randn((2, HD), generator=g, device=dev).cpu().numpy().astype(np.float64)
            G = np.rint(gam * math.sqrt(HD) * 2.0 ** 24).astype(np.int64)
            st["nq"], st["nk"] = (torch.from_numpy(_entries(G[i], 0, 0, P1_BITS + 24 - FN, HD)).to(dev) for i in (0, 1))
            st["eps"] = int(round(1e-5 * HD * 2.0 ** (2 * FQ0)))
        st["q"] = torch.empty((rows, H * HD), dtype=torch.int16, device=dev)
    if kind in ("prep", "read"):
        st["k"], st["v"] = (torch.empty((rows, KV * HD), dtype=torch.int16, device=dev) for _ in range(2))
    if own:
        from cormorant_b200 import paged
        st["cache"] = paged.PagedCache(pages=pages, page=page, KV=KV, HD=HD, bits=case["bits"],
                                       buffers=(kc, vc) if ks is None else (kc, vc, ks, vs))
        st["batch"] = paged.PagedBatch(table, cu, pos, rows=rows, max_q=max(new), max_keys=max(c + n for c, n in zip(ctx, new)))
    return st


# ------------------------------------------------------------------------------------------------------- the passes
def run(st):
    kind = st["case"]["kind"]
    if own:
        return _own(st, kind)
    if kind == "attn":
        return _attn(st, st["q"])
    if kind == "read":
        return _read(st, st["kc"], st["ks"]), _read(st, st["vc"], st["vs"])
    q, k, v = _prep(st)
    if kind == "prep":
        return q, k.to(torch.int16), v.to(torch.int16)
    _write(st, st["kc"], st["ks"], k)
    _write(st, st["vc"], st["vs"], v)
    return q, _attn(st, q)


def _own(st, kind):
    from cormorant_b200 import ops
    c, cache, batch = st["case"], st["cache"], st["batch"]
    if kind in ("prep", "step"):
        kw = dict(nq=st["nq"], nk=st["nk"], eps_q=st["eps"], eps_k=st["eps"]) if c["norm"] else {}
        ops.llm_paged_prep(cache, batch, st["q0"], st["k0"], st["v0"], st["q"], H=c["H"], rope=st["rope"], rot=c["rot"],
                           interleaved=c["interleaved"], pq=st["pq"], pk=st["pk"], pv=st["pv"], pq_bc=st["whole"],
                           pk_bc=st["whole"], pv_bc=True, **kw)
    if kind in ("attn", "step"):
        ops.llm_paged_attn(cache, batch, st["q"], st["o"], H=c["H"], smx=st["smx"], window=c["window"])
        return st["o"] if kind == "attn" else (st["q"], st["o"])
    ops.llm_paged_read(cache, batch, st["k"], st["v"])
    return (st["q"], st["k"], st["v"]) if kind == "prep" else (st["k"], st["v"])


# ------------------------------------------------------------------------------------------------------- plain forms
def _values(case, planes, shifts):
    """Cached bytes [..., byte] (and shifts [...]) as the int32 words that they stand for."""
    HD = case["HD"]
    if case["bits"] == 8:
        return planes.to(torch.int32) << shifts.to(torch.int32)[..., None]
    return planes[..., :HD].to(torch.int32) * 256 + (planes[..., HD:].to(torch.int32) & 255)


def _slots(st, b, lo, hi):
    """(page, row in the page) of the positions lo .. hi - 1 of sequence b."""
    p = torch.arange(lo, hi, device=st["table"].device)
    return st["table"][b][p // st["case"]["page"]].to(torch.int64), p % st["case"]["page"]


def _gather(st, planes, shifts, b, lo, hi):
    """Rows lo .. hi - 1 of sequence b: [rows][KV][HD]."""
    pg, r = _slots(st, b, lo, hi)
    return _values(st["case"], planes[pg, :, r], None if shifts is None else shifts[pg, :, r])


def _read(st, planes, shifts):
    out = [_gather(st, planes, shifts, b, c, c + n) for b, (c, n) in enumerate(zip(st["ctx"], st["new"]))]
    return torch.cat(out).reshape(st["rows"], -1).to(torch.int16)


def _write(st, planes, shifts, x):
    """The words x [rows][KV HD] (as the cache holds them) into the pages."""
    case = st["case"]
    at = 0
    for b, (c, n) in enumerate(zip(st["ctx"], st["new"])):
        pg, r = _slots(st, b, c, c + n)
        w = x[at:at + n].reshape(n, case["KV"], case["HD"]).to(torch.int64)
        at += n
        if case["bits"] == 8:
            code, s = _codes(w)
            planes[pg, :, r] = code.to(torch.int8)
            shifts[pg, :, r] = s[..., 0].to(torch.uint8)
        else:
            lo = w & 255
            planes[pg, :, r] = torch.cat([w >> 8, lo - 256 * (lo >> 7)], -1).to(torch.int8)


def _mulhi(a, b):
    """floor(a b / 2^32) of 0 <= a, b < 2^32 in int64."""
    return ((a >> 16) * b + (((a & 65535) * b) >> 16)) >> 16


_RSQ = {}


def _norm(x, entries, eps):
    """RMS norm of heads x [..., HD] by the row-ops unit's rsqrt."""
    if x.device not in _RSQ:
        i = torch.arange(8192, dtype=torch.float64, device=x.device)
        y = (2.0 ** RM_BITS / ((i + 0.5) * 2.0 ** 19).sqrt()).round().clamp(max=2.0 ** 32 - 1)
        _RSQ[x.device] = y.to(torch.int64)
    D = ((x * x).sum(-1, keepdim=True) + eps).clamp(min=1)
    e = sum((D >= (1 << k)).to(torch.int64) for k in range(62))
    d = e - 32
    d = d + (d & 1)
    Dm = torch.where(d >= 0, D >> d.clamp(min=0), D << (-d).clamp(min=0))
    y0 = _RSQ[x.device][Dm >> 19]
    u = _mulhi(_mulhi(Dm, y0), y0)
    y1 = (y0 + ((y0 * ((1 << 30) - u)) >> 31)).clamp(1 << 31, (1 << 32) - 1)
    P1 = (x * y1) >> (RM_BITS + (d >> 1) - P1_BITS)
    G, sc = entries[:, 0:4].contiguous().view(torch.int32)[:, 0].to(torch.int64), entries[:, 10].to(torch.int64)
    return _rne(P1 * G, sc.expand_as(P1)).clamp(-32768, 32767)


def _rotate(case, x, cos, sin, entries):
    """The rotation of heads x [rows][heads][HD] by cos / sin [rows][rot / 2]."""
    n, heads, HD = x.shape
    rot = case["rot"]
    par = entries.to(torch.int64).expand(heads * HD, 16).reshape(heads, HD, 16)
    sa, sb, sc = par[..., 8], par[..., 9], par[..., 10]
    first = torch.arange(rot // 2, device=x.device) * (2 if case["interleaved"] else 1)
    second = first + (1 if case["interleaved"] else rot // 2)
    y = x << sa
    a, b, c, s = x[..., first], x[..., second], cos[:, None, :], sin[:, None, :]
    y[..., first] = ((a * c) << sa[:, first]) - ((b * s) << sb[:, first])
    y[..., second] = ((b * c) << sa[:, second]) + ((a * s) << sb[:, second])
    return _rne(y, sc.expand_as(y)).clamp(-32768, 32767)


def _prep(st):
    """The rotated q rows (int16) and the K / V words as the cache holds them."""
    case, rows = st["case"], st["rows"]
    H, KV, HD, rot = case["H"], case["KV"], case["HD"], case["rot"]
    dev = st["q0"].device
    at = torch.cat([torch.arange(c, c + n, device=dev) for c, n in zip(st["ctx"], st["new"])])
    cos, sin = (t.to(torch.int64) for t in st["rope"][at].split(rot // 2, 1))
    q, k, v = (st[nm].to(torch.int64).reshape(rows, n, HD) for nm, n in (("q0", H), ("k0", KV), ("v0", KV)))
    if case["norm"]:
        q, k = _norm(q, st["nq"], st["eps"]), _norm(k, st["nk"], st["eps"])
    q, k = _rotate(case, q, cos, sin, st["pq"]), _rotate(case, k, cos, sin, st["pk"])
    pv = st["pv"].to(torch.int64)
    v = _rne(v << pv[:, 8], pv[:, 10].expand_as(v)).clamp(-32768, 32767)
    if case["bits"] == 8:
        k, v = (c << s for c, s in (_codes(k), _codes(v)))
    return q.reshape(rows, H * HD).to(torch.int16), k.reshape(rows, KV * HD), v.reshape(rows, KV * HD)


_TAB = {}


def _kernel_out(acc):
    """An exact sum (float64) as the kernels round it: modulo 2^32, floor / 2^8, saturated."""
    a = ((acc.to(torch.int64) + (1 << 31)) & 0xFFFFFFFF) - (1 << 31)
    return (a >> 8).clamp(-32768, 32767)


def _attn(st, q_rows):
    case = st["case"]
    H, KV, HD, w = case["H"], case["KV"], case["HD"], case["window"]
    G = H // KV
    dev = q_rows.device
    if dev not in _TAB:
        _TAB[dev] = torch.tensor([int(round(65536.0 * 2.0 ** (-k / 4096.0))) for k in range(4096)], device=dev)
    cm = st["smx"][:, 0].to(torch.int64).reshape(KV, G, 1, 1)
    cs = (st["smx"][:, 1] & 63).to(torch.int64).reshape(KV, G, 1, 1)
    fp = ((st["smx"][:, 1] >> 8) & 31).to(torch.int64).reshape(KV, G, 1, 1)
    out = torch.empty((st["rows"], H, HD), dtype=torch.int16, device=dev)
    at = 0
    for b, (c, n) in enumerate(zip(st["ctx"], st["new"])):
        some = max(1, min(n, (1 << 26) // (H * (c + n))))  # rows at a time: the scores of a long prompt do not fit at once
        for i in range(0, n, some):
            m = min(some, n - i)
            first, end = c + i, c + i + m
            lo = max(0, first + 1 - w) if w else 0
            K = _gather(st, st["kc"], st["ks"], b, lo, end).permute(1, 2, 0).to(torch.float64)
            V = _gather(st, st["vc"], st["vs"], b, lo, end).permute(1, 0, 2).to(torch.float64)
            q = q_rows[at + i:at + i + m].reshape(m, KV, G, HD).permute(1, 2, 0, 3).to(torch.float64)
            s = _kernel_out(torch.matmul(q.reshape(KV, G * m, HD), K)).reshape(KV, G, m, end - lo)
            key, row = torch.arange(lo, end, device=dev), torch.arange(first, end, device=dev)[:, None]
            seen = key <= row
            if w:
                seen = seen & (key > row - w)
            top = s.masked_fill(~seen, -32769).amax(-1, keepdim=True)
            y = ((top - s).masked_fill_(~seen, 0) * cm) >> cs
            e = (_TAB[dev][y & 4095] >> (y >> F).clamp(max=31)).masked_fill_(~seen, 0)
            R = (1 << RB) // e.sum(-1, keepdim=True)
            P = ((e * R + (torch.ones_like(fp) << (RB - 1 - fp))) >> (RB - fp)).clamp(max=32767).masked_fill_(~seen, 0)
            o = _kernel_out(torch.matmul(P.to(torch.float64).reshape(KV, G * m, end - lo), V))
            out[at + i:at + i + m] = o.reshape(KV, G, m, HD).permute(2, 0, 1, 3).reshape(m, H, HD).to(torch.int16)
        at += n
    return out.reshape(st["rows"], H * HD)


# ------------------------------------------------------------------------------------------------------- 64-bit truth
def exact(case, seed):
    """The definition row by row in numpy's 64-bit integers (and, for q.k and P.v, sums of exact products)."""
    ctx, new = _lengths(case)
    pairs = sum(_visible(case, c, n)[1] for c, n in zip(ctx, new)) * case["H"]
    if (case["kind"] in ("attn", "step") and (pairs > 1.2e7 or sum(new) * case["H"] > 1.5e5)) or sum(new) * (case["H"] + 2 * case["KV"]) * case["HD"] > 2.5e7:
        return None
    st = prepare(case, seed)
    h = {k: (v.cpu().numpy() if torch.is_tensor(v) else v) for k, v in st.items()}
    H, KV, HD, page, w = case["H"], case["KV"], case["HD"], case["page"], case["window"]
    rows = [(b, c + i) for b, (c, n) in enumerate(zip(ctx, new)) for i in range(n)]

    def sat(x):
        return np.clip(x, -32768, 32767)

    def nearest(x, k):  # ties to even, from the quotient and the remainder
        k = np.broadcast_to(np.asarray(k, np.int64), x.shape)
        two = np.left_shift(np.int64(1), k)
        q, r = np.divmod(x, two)
        return q + ((2 * r > two) | ((2 * r == two) & (q % 2 == 1)))

    def cached(planes, shifts):
        p = planes.astype(np.int64)
        return p * 2 ** shifts.astype(np.int64)[..., None] if case["bits"] == 8 else p[..., :HD] * 256 + p[..., HD:] % 256

    def held(x):  # what the cache makes of the words x [..., HD]
        if case["bits"] == 16:
            return x
        big = np.maximum(x, -1 - x).max(-1)
        s = np.maximum(np.ceil(np.log2(big + 1.0)).astype(np.int64) - 7, 0)[..., None]
        return np.clip(nearest(x, s), -128, 127) * 2 ** s

    def sequence(planes, shifts, b, n):
        pg = h["table"][b][:-(-n // page)].astype(np.int64)
        x = cached(planes[pg], None if shifts is None else shifts[pg])
        return x.transpose(0, 2, 1, 3).reshape(-1, KV, HD)[:n]
    kind = case["kind"]
    if kind in ("prep", "step"):
        at = np.array([p for _, p in rows], np.int64)
        rot = case["rot"]
        table = h["rope"].astype(np.int64)[at]
        cos, sin = table[:, None, :rot // 2], table[:, None, rot // 2:]

        def norm(x, ent):
            D = np.maximum((x * x).sum(-1) + h["eps"], 1)
            y1, sh = np.empty_like(D), np.empty_like(D)
            flat, fy, fs = D.reshape(-1), y1.reshape(-1), sh.reshape(-1)
            for i, d0 in enumerate(flat.tolist()):  # arbitrary-precision integers
                d = d0.bit_length() - 32
                d += d & 1
                dm = d0 >> d if d >= 0 else d0 << -d
                y0 = min(int(round(2.0 ** RM_BITS / math.sqrt(((dm >> 19) + 0.5) * 2.0 ** 19))), (1 << 32) - 1)
                u = (((dm * y0) >> 32) * y0) >> 32
                fy[i] = min(max(y0 + ((y0 * ((1 << 30) - u)) >> 31), 1 << 31), (1 << 32) - 1)
                fs[i] = RM_BITS + d // 2
            G = ent[:, :4].copy().view("<i4")[:, 0].astype(np.int64)
            p1 = np.right_shift(x * y1[..., None], sh[..., None] - P1_BITS)
            return sat(nearest(p1 * G, ent[:, 10].astype(np.int64)))

        def rotate(x, ent):
            n = x.shape[1]
            par = np.broadcast_to(ent.astype(np.int64), (n * HD, 16)).reshape(n, HD, 16)
            y = np.left_shift(x, par[..., 8])
            i = np.arange(rot // 2)
            a, b = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + rot // 2)
            y[..., a] = x[..., a] * cos * 2 ** par[:, a, 8] - x[..., b] * sin * 2 ** par[:, a, 9]
            y[..., b] = x[..., b] * cos * 2 ** par[:, b, 8] + x[..., a] * sin * 2 ** par[:, b, 9]
            return sat(nearest(y, par[..., 10]))
        q, k, v = (h[nm].astype(np.int64).reshape(len(rows), n, HD) for nm, n in (("q0", H), ("k0", KV), ("v0", KV)))
        if case["norm"]:
            q, k = norm(q, h["nq"]), norm(k, h["nk"])
        q, k = rotate(q, h["pq"]), held(rotate(k, h["pk"]))
        v = held(sat(nearest(v * 2 ** h["pv"][0, 8].astype(np.int64), h["pv"][0, 10])))
        if kind == "prep":
            return tuple(x.reshape(len(rows), -1).astype(np.int16) for x in (q, k, v))
    if kind == "read":
        K, V = ([sequence(h[p], h[s], b, c + n)[c:] for b, (c, n) in enumerate(zip(ctx, new))] for p, s in (("kc", "ks"), ("vc", "vs")))
        return tuple(np.concatenate(x).reshape(len(rows), -1).astype(np.int16) for x in (K, V))
    tab = np.array([math.floor(65536.0 * 2.0 ** (-k / 4096.0) + 0.5) for k in range(4096)], np.int64)

    def out(total):
        total = np.rint(total).astype(np.int64)
        return sat(((total + 2 ** 31) % 2 ** 32 - 2 ** 31) // 256)
    res = np.zeros((len(rows), H, HD), np.int16)
    r = 0
    for b, (c, n) in enumerate(zip(ctx, new)):
        if n == 0:
            continue
        K, V = sequence(h["kc"], h["ks"], b, c + n), sequence(h["vc"], h["vs"], b, c + n)
        if kind == "step":
            K, V = K.copy(), V.copy()
            K[c:], V[c:] = k[r:r + n], v[r:r + n]
            Q = q[r:r + n]
        else:
            Q = h["q"][r:r + n].astype(np.int64).reshape(n, H, HD)
        for i in range(n):
            hi, lo = c + i + 1, max(0, c + i + 1 - w) if w else 0
            for head in range(H):
                kv = head // (H // KV)
                cm, cfg = int(h["smx"][head, 0]), int(h["smx"][head, 1])
                cs, fp = cfg & 63, cfg >> 8 & 31
                s = out(K[lo:hi, kv].astype(np.float64) @ Q[i, head].astype(np.float64))
                y = ((s.max() - s) * cm) // 2 ** cs
                e = np.where(y < 17 * 4096, tab[y % 4096] // 2 ** np.minimum(y // 4096, 17), 0)
                P = np.minimum((e * (2 ** RB // int(e.sum())) + 2 ** (RB - fp - 1)) // 2 ** (RB - fp), 32767)
                res[r + i, head] = out(P.astype(np.float64) @ V[lo:hi, kv].astype(np.float64))
        r += n
    res = res.reshape(len(rows), H * HD)
    return res if kind == "attn" else (q.reshape(len(rows), H * HD).astype(np.int16), res)
