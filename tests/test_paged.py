"""The paged KV cache's operators (corm_llm_paged_prep / _attn / _read; no
counterpart in the reference): the oracle of each against the reference-pinned
restatements, the refusals and the host classes on the CPU; on the GPU every
output and every cache byte against the oracle, all exact — heads, pages,
shifts, windows and lengths where they can go wrong, rows of no sequence and
pages that are not there left alone, the kernels' own nodes, captured passes,
streams."""
import ctypes as C

import numpy as np
import pytest

from cormorant_b200 import _lib, paged
from cormorant_b200 import attention as AT
from cormorant_b200 import rowops_host as RH
from oracle import attn as OA
from oracle import paged as OP
from oracle import spec

torch = pytest.importorskip("torch")


# ------------------------------------------------------------------------------------------------ builders
def _smx(H, HD, f_s=12, f_p=12):
    cm, cs = AT.smx_scale_regs(f_s, 1.0 / np.sqrt(HD))
    return np.array([[cm, cs | f_p << 8]] * H, np.int32)


def _batch(rng, pages, page, ctx, new, *, spare=2, extra=0):
    """A block table of distinct random pages, cu and pos for sequences of ctx
    cached and new packed rows (``extra`` rows behind the last one)."""
    blocks = [-(-(c + n) // page) for c, n in zip(ctx, new)]
    ids = rng.permutation(pages)[:sum(blocks)]
    assert ids.size == sum(blocks)
    table = np.full((len(ctx), max(blocks + [1]) + spare), -1, np.int32)
    at = 0
    for b, k in enumerate(blocks):
        table[b, :k] = ids[at:at + k]
        at += k
    cu = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    return table, cu, np.asarray(ctx, np.int32), int(cu[-1]) + extra


def _random_cache(rng, pages, KV, page, HD, bits, hi=32768):
    """A cache full of random rows (a full-range or a small one), as its bytes."""
    x = rng.integers(-hi, hi, size=(2, pages, KV, page, HD))
    c = OP.Cache(*(np.zeros((pages, KV, page, HD * bits // 8), np.int8) for _ in range(2)),
                 *((np.zeros((pages, KV, page), np.uint8) for _ in range(2)) if bits == 8 else (None, None)),
                 None, None, None, HD, bits)
    for planes, shifts, v in ((c.kc, c.ks, x[0]), (c.vc, c.vs, x[1])):
        if bits == 8:
            v = v >> rng.integers(0, 15, size=(pages, KV, page, 1))  # every shift
            code, s = OP.quantise(v.reshape(-1, HD))
            planes[...] = code.reshape(v.shape)
            shifts[...] = s.reshape(shifts.shape)
        else:
            planes[..., :HD] = v >> 8
            planes[..., HD:] = (v & 255).astype(np.uint8).view(np.int8)
    return c


def _ents(rng, n, top=3, sc=(20, 27)):
    """n random entries: small up-shifts, down-shifts that keep some of the word."""
    sa, sb = rng.integers(0, top, n), rng.integers(0, top, n)
    return RH.param_block(np.zeros(n, np.int64), 0, sa, sb, rng.integers(*sc, n)).astype(np.int16)


def _rope(rows, rot, theta=1e4):
    ang = np.outer(np.arange(rows), theta ** (-np.arange(rot // 2) / max(rot // 2, 1)))
    return np.rint(np.concatenate([np.cos(ang), np.sin(ang)], 1) * 2.0 ** 23).astype(np.int32)


def _norm_entries(rng, HD, fo=12):
    w, bc, g, E = RH.rmsnorm_job(1.0 + 0.2 * rng.normal(size=HD), 1e-5, 13, np.full(HD, fo))
    return (np.tile(w, HD) if bc else w).astype(np.int16), E


# ------------------------------------------------------------------------------------------------ CPU
def test_oracle_norm_is_the_units_job():
    rng = np.random.default_rng(1)
    HD, n = 32, 5
    x = rng.integers(-3000, 3000, size=(n, HD))
    x[0] = 0
    w, E = _norm_entries(rng, HD)
    mem = np.zeros(8192, np.uint8)
    mem[:2 * n * HD] = x.astype("<i2").reshape(-1).view(np.uint8)
    mem[4096:4096 + 16 * HD] = w.view(np.uint8)
    spec.rowops_job(spec.RowOpsMem(mem), RH.opword(RH.OP_NORM), HD, n, 1, 0, 2 * HD, 0, 0, 0, 0, 2048, 2 * HD, 0, 4096,
                    E, 0, 0, 0, RH.NO_WINDOW)
    want = mem[2048:2048 + 2 * n * HD].view("<i2").astype(np.int64).reshape(n, HD)
    assert np.array_equal(OP.norm(x, w, E), want)


def test_oracle_rotation_and_attention_are_the_nodes():
    """One sequence in pages against the contiguous nodes' restatement."""
    rng = np.random.default_rng(2)
    T, H, KV, HD, page, pos = 9, 4, 2, 32, 16, 21
    G, Cn = H // KV, 48
    q0, k0, v = (rng.integers(-20000, 20000, size=(T, m * HD)) for m in (H, KV, KV))
    ang = np.outer(np.arange(Cn), 1e4 ** (-np.arange(HD // 2) / (HD // 2)))
    cos, sin = np.cos(ang).astype(np.float32), np.sin(ang).astype(np.float32)
    ck, cv = (rng.integers(-9000, 9000, size=(Cn, KV * HD)) for _ in range(2))
    f = dict(fq0=np.full(H * HD, 13), fk0=np.full(KV * HD, 13), fv=np.full(KV * HD, 13), fq=np.full(H, 10),
             fkc=np.full(KV * HD, 10), fvc=np.full(KV * HD, 9))
    smx = _smx(H, HD)
    table, cu, p, rows = _batch(rng, 5, page, [pos], [T])
    c = _random_cache(rng, 5, KV, page, HD, 16)
    c.table, c.cu, c.pos = table, cu, p
    for i in range(pos):
        c.store(c.kc, c.ks, 0, i, ck[i].reshape(KV, HD))
        c.store(c.vc, c.vs, 0, i, cv[i].reshape(KV, HD))
    ref = OA.prefill_layer(q0, k0, v, pos, T, T=T, H=H, KV=KV, HD=HD, C=Cn, cos=cos, sin=sin, ck=ck, cv=cv,
                           cm=smx[:, 0], cfg=smx[:, 1], **f)
    rope = np.rint(np.concatenate([cos, sin], 1).astype(np.float64) * 2.0 ** 23).astype(np.int64)
    pq, pk = (RH.pblock(0, 0, *RH.rope_params(np.full(n * HD, 13), n, HD, np.full(n, 10)), n * HD)[0].astype(np.int16)
              for n in (H, KV))
    sa, sc = RH.vround_params(np.full(KV * HD, 13), np.full(KV * HD, 9))
    q, o = np.zeros((T, H * HD), np.int64), np.zeros((T, H * HD), np.int64)
    OP.prep(c, q0, k0, v, q, H=H, rope=rope, rot=HD, interleaved=False, pq=pq, pk=pk,
            pv=RH.pblock(0, 0, sa, 0, sc, KV * HD)[0].astype(np.int16))
    OP.attn(c, q, o, H=H, smx=smx)
    for h in range(H):
        assert np.array_equal(q[:, h * HD:(h + 1) * HD], ref["qx"][h // G][:, (h % G) * T:(h % G + 1) * T].T)
    assert np.array_equal(o, ref["pv"])
    kk, vv = np.zeros((T, KV * HD), np.int64), np.zeros((T, KV * HD), np.int64)
    OP.read(c, kk, vv)
    assert np.array_equal(kk, ck[pos:pos + T]) and np.array_equal(vv, cv[pos:pos + T])


def test_oracle_codes():
    x = np.array([[0, 0], [127, -128], [128, 0], [-129, 0], [255, 1], [-32768, 32767], [383, -2]])
    c, s = OP.quantise(x)
    assert s.tolist() == [0, 0, 1, 1, 1, 8, 2]
    assert c.tolist() == [[0, 0], [127, -128], [64, 0], [-64, 0], [127, 0], [-128, 127], [96, 0]]


def _desc(**kw):
    """A cache descriptor that every check accepts (its addresses are never read
    on the host)."""
    d = dict(kc=4096, vc=8192, ks=0, vs=0, table=256, cu=256, pos=256, pages=4, page=16, bits=16, KV=2, HD=64, B=1,
             table_width=2, rows=1)
    d.update(kw)
    return _lib.PagedCacheDesc(*d.values())


def _prep_desc(c=None, **kw):
    d = dict(q0=16, k0=16, v0=16, q=16, rope=16, pq=16, pk=16, pv=16, nq=0, nk=0, eps_q=0, eps_k=0, ldq0=256, ldk=128,
             ldv=128, ldq=256, H=4, rot=64, interleaved=0, rope_rows=8, flags=7)
    d.update(kw)
    return _lib.PagedPrepDesc(c or _desc(), *d.values())


def _attn_desc(c=None, **kw):
    d = dict(q=16, o=16, smx=16, ldq=256, ldo=256, H=4, max_q=1, max_keys=1, window=0)
    d.update(kw)
    return _lib.PagedAttnDesc(c or _desc(), *d.values())


def _read_desc(c=None, **kw):
    d = dict(k=16, v=16, ldk=128, ldv=128)
    d.update(kw)
    return _lib.PagedReadDesc(c or _desc(), *d.values())


BAD_CACHE = [dict(kc=0), dict(vc=0), dict(table=0), dict(cu=0), dict(pos=0), dict(bits=4), dict(bits=8), dict(page=8),
             dict(page=48), dict(page=512), dict(HD=8), dict(HD=96), dict(HD=512), dict(KV=0), dict(KV=65536),
             dict(B=65536), dict(pages=1 << 31), dict(rows=1 << 31), dict(table_width=1 << 27), dict(kc=4104),
             dict(vc=8), dict(bits=8, ks=8, vs=16), dict(table=258), dict(cu=2), dict(pos=1)]


@pytest.mark.parametrize("bad", BAD_CACHE, ids=lambda b: "_".join(f"{k}{v}" for k, v in b.items()))
def test_refused_caches(bad):
    L = _lib.lib()
    for fn, d in ((L.corm_llm_paged_prep, _prep_desc(_desc(**bad))), (L.corm_llm_paged_attn, _attn_desc(_desc(**bad))),
                  (L.corm_llm_paged_read, _read_desc(_desc(**bad)))):
        assert fn(C.byref(d), None) in (_lib.CORM_EINVAL, _lib.CORM_ELIMIT)
        assert b"corm_llm_paged" in L.corm_last_error()


@pytest.mark.parametrize("bad", [dict(q0=0), dict(q=0), dict(rope=0), dict(pq=0), dict(pk=0), dict(pv=0), dict(H=0),
                                 dict(H=65536, ldq0=1 << 30, ldq=1 << 30), dict(rot=0), dict(rot=63), dict(rot=66),
                                 dict(rope_rows=0), dict(ldq0=255), dict(ldk=127), dict(ldv=127), dict(ldq=255),
                                 dict(nq=16, eps_q=1 << 62), dict(nk=16, eps_k=1 << 62), dict(nq=18), dict(q0=17),
                                 dict(k0=17), dict(v0=1), dict(q=15), dict(rope=18)],
                         ids=lambda b: "_".join(f"{k}{v}" for k, v in b.items()))
def test_refused_preps(bad):
    L = _lib.lib()
    assert L.corm_llm_paged_prep(C.byref(_prep_desc(**bad)), None) in (_lib.CORM_EINVAL, _lib.CORM_ELIMIT)


@pytest.mark.parametrize("bad", [dict(q=0), dict(o=0), dict(smx=0), dict(H=0), dict(H=3), dict(H=34, ldq=1 << 20, ldo=1 << 20),
                                 dict(ldq=255), dict(ldo=255), dict(smx=18), dict(q=17), dict(o=19)],
                         ids=lambda b: "_".join(f"{k}{v}" for k, v in b.items()))
def test_refused_attns(bad):
    L = _lib.lib()
    assert L.corm_llm_paged_attn(C.byref(_attn_desc(**bad)), None) in (_lib.CORM_EINVAL, _lib.CORM_ELIMIT)


@pytest.mark.parametrize("bad", [dict(ldk=127), dict(ldv=127), dict(k=17), dict(v=33)],
                         ids=lambda b: "_".join(f"{k}{v}" for k, v in b.items()))
def test_refused_reads(bad):
    L = _lib.lib()
    assert L.corm_llm_paged_read(C.byref(_read_desc(**bad)), None) == _lib.CORM_EINVAL


def test_host_classes_refuse():
    """The Python layer's own checks, on CPU tensors (no launch can follow)."""
    with pytest.raises(_lib.CormError):
        paged.PagedCache(4, 24, 2, 64, device="cpu")
    with pytest.raises(_lib.CormError):
        paged.PagedCache(4, 16, 2, 64, bits=4, device="cpu")
    with pytest.raises(_lib.CormError):
        paged.PagedCache(4, 16, 2, 64, buffers=(torch.zeros(4 * 2 * 16 * 128, dtype=torch.int8),))
    with pytest.raises(_lib.CormError):
        paged.PagedCache(4, 16, 2, 64, buffers=(torch.zeros(10, dtype=torch.int8),) * 2)
    i32 = dict(dtype=torch.int32)
    with pytest.raises(_lib.CormError):
        paged.PagedBatch(torch.zeros((2, 3), dtype=torch.int64), torch.zeros(3, **i32), torch.zeros(2, **i32), rows=2)
    with pytest.raises(_lib.CormError):
        paged.PagedBatch(torch.zeros((2, 3), **i32), torch.zeros(2, **i32), torch.zeros(2, **i32), rows=2)
    with pytest.raises(_lib.CormError):
        paged.PagedBatch(torch.zeros((2, 6), **i32)[:, ::2], torch.zeros(3, **i32), torch.zeros(2, **i32), rows=2)
    cache = paged.PagedCache(4, 16, 2, 64, device="cpu")
    batch = paged.PagedBatch.of([[0], [1, 2]], [1, 2], [3, 20], device="cpu")
    assert (batch.rows, batch.max_q, batch.max_keys, batch.width) == (3, 2, 22, 2)
    assert batch.table.tolist() == [[0, -1], [1, 2]] and batch.cu.tolist() == [0, 1, 3]
    from cormorant_b200 import ops
    with pytest.raises(_lib.CormError):
        ops.llm_paged_read(cache, batch, None, None)


def test_one_batch_with_two_caches():
    """A batch that two threads use with a cache each: whatever the other one does
    between two lines of a call, the descriptor is of the call's own cache."""
    import sys
    caches = [paged.PagedCache(4, 16, 2, 64, device="cpu") for _ in range(2)]
    batch = paged.PagedBatch.of([[0], [1, 2]], [1, 2], [3, 20], device="cpu")
    steps = []

    def other(frame, event, arg):  # the other thread's whole call, before every line of this one's
        if frame.f_code is paged.PagedCache.desc.__code__:
            sys.settrace(None)
            assert caches[1].desc(batch).kc == caches[1].kc.data_ptr()
            steps.append(event)
            sys.settrace(other)
            return other
    for _ in range(2):
        before = sys.gettrace()
        sys.settrace(other)
        try:
            got = caches[0].desc(batch)
        finally:
            sys.settrace(before)
        assert (got.kc, got.vc) == (caches[0].kc.data_ptr(), caches[0].vc.data_ptr())
        assert caches[0].desc(batch).kc == caches[0].kc.data_ptr()
        assert caches[1].desc(batch).kc == caches[1].kc.data_ptr()
    assert len(steps) > 6


def test_a_batch_does_not_hold_a_cache():
    """The pages go with their cache, not with the last batch used on them."""
    import gc
    import weakref
    cache = paged.PagedCache(4, 16, 2, 64, device="cpu")
    batch = paged.PagedBatch.of([[0]], [1], [3], device="cpu")
    desc, pages = cache.desc(batch), weakref.ref(cache.kc)
    assert cache.desc(batch) is desc
    del cache
    gc.collect()
    assert pages() is None
    cache = paged.PagedCache(4, 16, 2, 64, device="cpu")
    assert cache.desc(batch).kc == cache.kc.data_ptr()


def _row_views(H, HD):
    """(tensor, stride of its rows) of what a program holds 8 packed rows of H heads of
    HD in, and the tensors that do not hold them, on the CPU."""
    n, z = H * HD, lambda *s: torch.zeros(s, dtype=torch.int16)  # noqa: E731
    W = 3 * n
    good = [(z(8, n), n), (z(11, n), n), (z(8 * n), n), (z(9 * n + 5), n), (z(8, W), W), (z(8, W)[:, 5:5 + n], W),
            (z(1, 8 * n), n), (z(8, H, HD), n), (z(2, 4, n), n), (z(2, 4, H, HD), n),
            (z(8, W)[:, :n].unflatten(1, (H, HD)), W),            # a projection's heads
            (z(8, 2 * H + 1, HD)[:, 1:1 + H], (2 * H + 1) * HD),  # the same, from the heads' array
            (z(2, 4, W)[..., n:2 * n], W), (z(2, 9, n)[:, ::9], 9 * n)]
    bad = [z(7, n), z(8 * n - 1), z(16, n)[:5], z(16 * n)[:5 * n], z(16, 2 * n)[:, :n - 1], z(8, W)[:, ::2],
           z(16, H, HD)[:7], z(n, 8).t(), z(1, n).expand(8, n), z(3, 5, W)[:2, :4, :n]]
    if H > 1:
        good.append((z(8, 2 * H, HD), 2 * n))                                           # its first heads
        bad += [z(8, H, 2, HD)[:, :, 0], z(8, HD, H).transpose(1, 2), z(8, 2 * H, HD)[:, ::2]]  # heads apart
    return good, bad


@pytest.mark.parametrize("H,HD", [(4, 64), (1, 16), (3, 32)])
def test_rows_of_a_view(H, HD):
    """The stride of a packed array is its own, whatever its rank; one that does not
    hold the rows within itself is refused, though its storage might."""
    from cormorant_b200 import ops
    n = H * HD
    good, bad = _row_views(H, HD)
    for t, ld in good:
        rows = 8 if t.numel() >= 8 * n else 2
        assert ops._rows(t, "x", rows, n, None, -1) == (t.data_ptr(), ld), (t.shape, t.stride())
        assert ops._rows(t, "x", rows, n, ld, -1) == (t.data_ptr(), ld), (t.shape, t.stride())
    for t in bad:
        for ld in (None, n, 3 * n):
            with pytest.raises(_lib.CormError):
                ops._rows(t, "x", 8, n, ld, -1)
    flat = torch.zeros(7 * 3 * n + n, dtype=torch.int16)  # a stride given for a flat array
    assert ops._rows(flat, "x", 8, n, 3 * n, -1)[1] == 3 * n
    assert ops._rows(torch.zeros((24, n), dtype=torch.int16), "x", 8, n, 3 * n, -1)[1] == 3 * n
    for t, ld in ((flat, 3 * n + 1), (flat[1:], 3 * n), (flat, n - 1), (torch.zeros((8, 3 * n), dtype=torch.int16)[:, :n], n)):
        with pytest.raises(_lib.CormError):
            ops._rows(t, "x", 8, n, ld, -1)
    one = torch.zeros((5, 2 * n), dtype=torch.int16)[2:3, :n]  # one row: any stride
    assert ops._rows(one, "x", 1, n, None, -1)[0] == one.data_ptr()


def test_rotation_table_shapes():
    """A table's rows are rot wide: one of another width is refused, not read as more rows."""
    from cormorant_b200 import ops
    z = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    for t, rot, rows in ((z(8, 64), 64, 8), (z(8, 32), 32, 8), (z(256), 32, 8), (z(2, 3, 16), 16, 6)):
        assert ops._rope_rows(t, rot, -1) == rows
    for t, rot in ((z(8, 64), 32), (z(8, 32), 64), (z(4, 64), 128), (z(100), 64), (z(0, 64), 64), (z(63), 64), (z(8, 64), 0),
                   (z(8, 64), -2), (z(8, 64).long(), 64), (z(8, 128)[:, :64], 64), (z(8, 64)[::2], 64)):
        with pytest.raises(_lib.CormError, match="rope"):
            ops._rope_rows(t, rot, -1)


def test_numbers_that_do_not_fit():
    """Lengths, windows and eps that the descriptors' fields would wrap are refused (the
    hint of the keys, of which any value is right, is cut to its range)."""
    from cormorant_b200 import ops
    i32 = dict(dtype=torch.int32)
    a = torch.zeros((1, 2), **i32), torch.zeros(2, **i32), torch.zeros(1, **i32)
    for bad in (dict(rows=-1), dict(rows=1 << 31), dict(rows=1 << 32), dict(rows=4, max_q=-1), dict(rows=4, max_q=1 << 32)):
        with pytest.raises(_lib.CormError, match="PagedBatch"):
            paged.PagedBatch(*a, **bad)
    assert paged.PagedBatch(*a, rows=4, max_keys=-3).max_keys == 0
    assert paged.PagedBatch(*a, rows=4, max_keys=1 << 40).max_keys == 0x7FFFFFFF
    assert paged.PagedBatch(*a, rows=4, max_q=9).max_q == 9
    cache, batch = paged.PagedCache(4, 16, 2, 64, device="cpu"), paged.PagedBatch(*a, rows=4)
    t = torch.zeros(4, 256, dtype=torch.int16)
    for w in (-1, 1 << 32, (1 << 32) + 5):
        with pytest.raises(_lib.CormError, match="window"):
            ops.llm_paged_attn(cache, batch, t, t, H=4, smx=torch.zeros((4, 2), **i32), window=w)
    for kw in (dict(eps_q=-1), dict(eps_k=1 << 62), dict(eps_q=1 << 64), dict(eps_k=(1 << 64) + 3)):
        with pytest.raises(_lib.CormError, match="eps"):
            ops.llm_paged_prep(cache, batch, t, t, t, t, H=4, rope=torch.zeros((8, 64), **i32), pq=None, pk=None, **kw)


def test_page_pool():
    p = paged.PagePool(5, 16)
    a = p.extend("a", 17)
    assert len(a) == 2 and p.extend("a", 32) == a and len(p.extend("b", 1)) == 1
    with pytest.raises(MemoryError):
        p.extend("a", 16 * 5)
    assert p.held["a"] == a and len(p.free) == 2
    p.release("a")
    assert len(p.free) == 4 and len(p.extend("b", 80)) == 5
    p.release("nobody")


# ------------------------------------------------------------------------------------------------ GPU
gpu = pytest.mark.gpu


def _dev(a):
    return None if a is None else torch.from_numpy(np.ascontiguousarray(a)).cuda()


def _handles(c, rows, max_q=None, max_keys=None):
    cache = paged.PagedCache(c.kc.shape[0], c.page, c.kc.shape[1], c.HD, c.bits,
                             buffers=[_dev(x) for x in (c.kc, c.vc, c.ks, c.vs) if x is not None])
    return cache, paged.PagedBatch(_dev(c.table), _dev(c.cu), _dev(c.pos), rows=rows, max_q=max_q, max_keys=max_keys)


def _same_bytes(c, cache):
    for nm in ("kc", "vc", "ks", "vs"):
        if getattr(c, nm) is not None:
            assert np.array_equal(getattr(c, nm), getattr(cache, nm).cpu().numpy()), nm


PREPS = [  # HD, rot, interleaved, norm, bits, page, H, KV, broadcast
    (64, 64, False, False, 16, 16, 3, 1, True),
    (64, 64, False, True, 8, 64, 15, 5, False),
    (16, 16, False, True, 16, 32, 4, 2, False),
    (16, 8, True, True, 8, 16, 1, 1, False),
    (32, 16, False, False, 8, 128, 7, 2, False),
    (32, 32, True, True, 16, 16, 2, 2, True),
    (128, 96, True, True, 8, 32, 4, 2, False),
    (128, 128, False, False, 16, 256, 8, 1, False),
    (128, 44, False, True, 16, 64, 2, 1, False),   # rot / 2 = 22: element by element
    (64, 6, True, False, 8, 16, 5, 5, False),
    (64, 2, False, False, 16, 16, 1, 1, False),
    (256, 256, False, True, 8, 16, 3, 3, False),
    (256, 128, True, False, 16, 32, 2, 1, False),
]


def _prep_case(rng, HD, rot, interleaved, norm, bits, page, H, KV, bc, *, hi=32768, big_shifts=False):
    ctx, new = [0, page - 1, 3, 2 * page + 5, 7], [5, 4, 0, 3, 1]
    table, cu, pos, rows = _batch(rng, 16, page, ctx, new, extra=3)
    c = _random_cache(rng, 16, KV, page, HD, bits)
    c.table, c.cu, c.pos = table, cu, pos
    q0, k0, v0 = (rng.integers(-hi, hi, size=(rows, n * HD)).astype(np.int16) for n in (H, KV, KV))
    q0[0], k0[0], v0[0] = 0, 0, 0
    top = 50 if big_shifts else 3
    sc = (40, 64) if big_shifts else (20, 27)
    par = [_ents(rng, 1 if bc else n * HD, top, sc) for n in (H, KV)] + [_ents(rng, 1 if bc else KV * HD, 4, (0, 9))]
    kw = dict(rope=_rope(3 * page, rot), rot=rot, interleaved=interleaved, pq=par[0], pk=par[1], pv=par[2])
    if norm:
        (kw["nq"], kw["eps_q"]), (kw["nk"], kw["eps_k"]) = _norm_entries(rng, HD), _norm_entries(rng, HD, 13)
    return c, rows, q0, k0, v0, kw


def _run_prep(c, rows, q0, k0, v0, kw, H, bc, ld=None):
    from cormorant_b200 import ops
    cache, batch = _handles(c, rows)
    g = {k: _dev(v) if isinstance(v, np.ndarray) else v for k, v in kw.items()}
    if ld is None:
        a, qd = [_dev(x) for x in (q0, k0, v0)], torch.full((rows, H * c.HD), -7, dtype=torch.int16, device="cuda")
        ops.llm_paged_prep(cache, batch, *a, qd, H=H, pq_bc=bc, pk_bc=bc, pv_bc=bc, **g)
        got = qd.cpu().numpy()
    else:  # views of one wide array, at an odd offset and stride
        wide = torch.full((rows, ld), 99, dtype=torch.int16, device="cuda")
        at, a = 1, []
        for x in (q0, k0, v0):
            v = wide[:, at:at + x.shape[1]]
            v.copy_(_dev(x))
            a.append(v)
            at += x.shape[1]
        qd = torch.full((rows, H * c.HD + 5), -7, dtype=torch.int16, device="cuda")
        ops.llm_paged_prep(cache, batch, *a, qd[:, 3:3 + H * c.HD], H=H, pq_bc=bc, pk_bc=bc, pv_bc=bc, **g)
        assert (qd[:, :3] == -7).all() and (qd[:, 3 + H * c.HD:] == -7).all()
        got = qd[:, 3:3 + H * c.HD].cpu().numpy()
    want = np.full((rows, H * c.HD), -7, np.int64)
    OP.prep(c, q0, k0, v0, want, H=H, **kw)
    assert np.array_equal(got, want)
    _same_bytes(c, cache)
    assert ops.device_status() == 0


@gpu
@pytest.mark.parametrize("case", PREPS, ids=lambda c: "hd%d_rot%d_i%d_n%d_b%d_p%d_h%d_%d_%d" % tuple(map(int, c)))
def test_prep_vs_oracle(case):
    """Ragged rows (an empty sequence, page borders, rows of no sequence), full-range words."""
    args = _prep_case(np.random.default_rng(sum(map(int, case))), *case)
    _run_prep(*args, case[6], case[8])


@gpu
@pytest.mark.parametrize("case", [(128, 128, False, True, 16, 32, 40, 20, False), (256, 64, True, False, 8, 64, 33, 11, False),
                                  (16, 16, False, False, 16, 16, 90, 45, True)], ids=["hd128", "hd256", "hd16"])
def test_prep_and_read_of_many_heads(case):
    """More heads than a warp takes of a row, and a read-back of as many."""
    test_prep_vs_oracle(case)
    test_read_vs_oracle(case[0], case[4], case[5], case[7])


@gpu
@pytest.mark.parametrize("case", [PREPS[1], PREPS[6], PREPS[8]], ids=["hd64", "hd128", "rot44"])
def test_prep_views_and_wide_shifts(case):
    """Operands that are views of one wide row at an odd offset; entries whose shifts need 128-bit sums."""
    rng = np.random.default_rng(77)
    HD, H, KV = case[0], case[6], case[7]
    _run_prep(*_prep_case(rng, *case), H, case[8], ld=(H + 2 * KV) * HD + 9)
    _run_prep(*_prep_case(rng, *case, big_shifts=True), H, case[8])


@gpu
@pytest.mark.parametrize("bits", [16, 8])
def test_prep_missing_pages_and_late_positions(bits):
    """Table entries outside the pool, positions past the table and past the rotation's table, cu and pos out of
    range: nothing is written there, the q rows still come."""
    rng = np.random.default_rng(5)
    c, rows, q0, k0, v0, kw = _prep_case(rng, 64, 64, False, False, bits, 16, 2, 1, True)
    c.table[0, 0], c.table[1, 1], c.table[3, 2] = 16, -2, 1 << 30
    c.pos[4] = c.table.shape[1] * 16 - 1 + 40
    c.pos[2] = -9
    c.cu[-1] = rows + 11
    _run_prep(c, rows, q0, k0, v0, kw, 2, True)


@gpu
def test_prep_is_the_units_jobs():
    """The same words as the row-ops unit's NORM and ROPE jobs, v as it is."""
    from cormorant_b200 import ops
    rng = np.random.default_rng(8)
    H, KV, HD, page, n = 6, 2, 64, 16, 40
    table, cu, pos, rows = _batch(rng, 8, page, [0], [n])
    c = _random_cache(rng, 8, KV, page, HD, 16)
    c.table, c.cu, c.pos = table, cu, pos
    cache, batch = _handles(c, rows)
    q0, k0, v0 = (_dev(rng.integers(-9000, 9000, size=(n, m * HD)).astype(np.int16)) for m in (H, KV, KV))
    (wq, E), (wk, _) = _norm_entries(rng, HD), _norm_entries(rng, HD)
    ang = np.outer(np.arange(n), 1e4 ** (-np.arange(HD // 2) / (HD // 2)))
    cos, sin = np.cos(ang).astype(np.float32), np.sin(ang).astype(np.float32)
    rope = np.rint(np.concatenate([cos, sin], 1).astype(np.float64) * 2.0 ** 23).astype(np.int32)
    pe = RH.pblock(0, 0, *RH.rope_params(np.full(H * HD, 12), H, HD, np.full(H, 10)), H * HD)[0].astype(np.int16)
    q = torch.empty((n, H * HD), dtype=torch.int16, device="cuda")
    ops.llm_paged_prep(cache, batch, q0, k0, v0, q, H=H, rope=_dev(rope), pq=_dev(pe), pk=_dev(pe), pq_bc=True,
                       pk_bc=True, v_direct=True, nq=_dev(wq), nk=_dev(wk), eps_q=E, eps_k=E)
    words = _dev(RH.rope_table_words(cos, sin).astype(np.int16))
    out = []
    for x, m, w in ((q0, H, wq), (k0, KV, wk)):
        t, y = torch.empty_like(x), torch.empty_like(x)
        ops.rowops(x, None, t, _dev(w), op=RH.opword(RH.OP_NORM), n=HD, rows=n * m, a_s1=2 * HD, c_s1=2 * HD, eps=E)
        ops.rowops(t, words, y, _dev(pe), op=RH.opword(RH.OP_ROPE, RH.K_I16, RH.K_I32, RH.K_I16, b_en=True, p_bcast=True),
                   n=m * HD, rows=n, a_s1=2 * m * HD, b_s1=8 * HD, c_s1=2 * m * HD, aux=HD)
        out.append(y)
    k, v = torch.empty_like(k0), torch.empty_like(v0)
    ops.llm_paged_read(cache, batch, k, v)
    assert torch.equal(q, out[0]) and torch.equal(k, out[1]) and torch.equal(v, v0)


@gpu
@pytest.mark.parametrize("HD,bits,page,KV", [(16, 16, 16, 3), (16, 8, 256, 1), (32, 8, 32, 2), (64, 16, 64, 5),
                                             (128, 8, 16, 1), (256, 16, 32, 2)])
def test_read_vs_oracle(HD, bits, page, KV):
    from cormorant_b200 import ops
    rng = np.random.default_rng(HD + bits)
    ctx, new = [0, 3, page - 2, 0], [page + 1, 0, 5, 2]
    table, cu, pos, rows = _batch(rng, 12, page, ctx, new, extra=2)
    c = _random_cache(rng, 12, KV, page, HD, bits)
    c.table, c.cu, c.pos = table, cu, pos
    c.table[2, 1] = 99
    c.pos[3] = c.cap - 1
    cache, batch = _handles(c, rows)
    want = [np.full((rows, KV * HD), 5, np.int64) for _ in range(2)]
    OP.read(c, *want)
    for off in (0, 1):  # dense rows, then rows at an odd offset and stride
        buf = [torch.full((rows, KV * HD + 3 * off), 5, dtype=torch.int16, device="cuda") for _ in range(2)]
        view = [b[:, off:off + KV * HD] for b in buf]
        ops.llm_paged_read(cache, batch, *view)
        for g, w, b in zip(view, want, buf):
            assert np.array_equal(g.cpu().numpy(), w)
            assert off == 0 or ((b[:, :1] == 5).all() and (b[:, -2:] == 5).all())
    one = torch.full((rows, KV * HD), 5, dtype=torch.int16, device="cuda")
    ops.llm_paged_read(cache, batch, None, one)
    assert np.array_equal(one.cpu().numpy(), want[1])
    ops.llm_paged_read(cache, batch, one, None)
    assert np.array_equal(one.cpu().numpy(), want[0])


@gpu
@pytest.mark.parametrize("case", [PREPS[1], PREPS[6]], ids=["hd64", "hd128"])
@pytest.mark.parametrize("split", [True, False], ids=["columns", "heads"])
def test_head_views_in_and_out(case, split):
    """The three operators on [rows][heads][HD] views of fused arrays, cut from the
    columns of one with two dimensions or the heads of one with three: the heads
    between them are left as they were."""
    from cormorant_b200 import ops
    HD, H, KV, bc = case[0], case[6], case[7], case[8]
    c, rows, q0, k0, v0, kw = _prep_case(np.random.default_rng(sum(map(int, case))), *case)
    cache, batch = _handles(c, rows)

    def fused(*parts):  # each part's heads, a head of -7 before, between and behind them
        t = torch.full((rows, sum(parts) + len(parts) + 1, HD), -7, dtype=torch.int16, device="cuda")
        ats = [1 + sum(parts[:i]) + i for i in range(len(parts))]
        wide = t.view(rows, -1)
        return t, [wide[:, at * HD:(at + p) * HD].unflatten(1, (p, HD)) if split else t[:, at:at + p]
                   for at, p in zip(ats, parts)]

    def check(t, views, wants):
        for v, w in zip(views, wants):
            assert np.array_equal(v.reshape(rows, -1).cpu().numpy(), w)
            v.fill_(-7)
        assert (t == -7).all()
    t, ins = fused(H, KV, KV)
    for v, x in zip(ins, (q0, k0, v0)):
        v.copy_(_dev(x).view(v.shape))
    g = {k: _dev(v) if isinstance(v, np.ndarray) else v for k, v in kw.items()}
    qt, (q,) = fused(H)
    ops.llm_paged_prep(cache, batch, *ins, q, H=H, pq_bc=bc, pk_bc=bc, pv_bc=bc, **g)
    want = np.full((rows, H * HD), -7, np.int64)
    OP.prep(c, q0, k0, v0, want, H=H, **kw)
    _same_bytes(c, cache)
    smx = _smx(H, HD)
    ot, (o,) = fused(H)
    ops.llm_paged_attn(cache, batch, q, o, H=H, smx=_dev(smx))
    att = np.full((rows, H * HD), -7, np.int64)
    OP.attn(c, want, att, H=H, smx=smx)
    check(ot, [o], [att])
    check(qt, [q], [want])
    check(t, ins, [q0, k0, v0])
    kvt, kv = fused(KV, KV)
    ops.llm_paged_read(cache, batch, *kv)
    words = [np.full((rows, KV * HD), -7, np.int64) for _ in range(2)]
    OP.read(c, *words)
    check(kvt, kv, words)
    assert ops.device_status() == 0


def _run_attn(c, rows, H, smx, rng, *, window=0, max_q=None, max_keys=None, hi=32768, odd=False):
    from cormorant_b200 import ops
    cache, batch = _handles(c, rows, max_q=max_q, max_keys=max_keys)
    q = rng.integers(-hi, hi, size=(rows, H * c.HD)).astype(np.int16)
    n = H * c.HD
    if odd:
        qw = torch.zeros((rows, n + 5), dtype=torch.int16, device="cuda")
        qd = qw[:, 1:1 + n]
        qd.copy_(_dev(q))
        ow = torch.full((rows, n + 3), -7, dtype=torch.int16, device="cuda")
        o = ow[:, 1:1 + n]
    else:
        qd, ow = _dev(q), None
        o = torch.full((rows, n), -7, dtype=torch.int16, device="cuda")
    ops.llm_paged_attn(cache, batch, qd, o, H=H, smx=_dev(smx), window=window)
    want = np.full((rows, n), -7, np.int64)
    OP.attn(c, q, want, H=H, smx=smx, window=window, max_q=max_q)
    assert np.array_equal(o.cpu().numpy(), want)
    if ow is not None:
        assert (ow[:, 0] == -7).all() and (ow[:, 1 + n:] == -7).all()
    _same_bytes(c, cache)
    assert ops.device_status() == 0
    return want


ATTNS = [  # HD, bits, page, H, KV, contexts, new rows, window
    (64, 16, 64, 3, 1, [0], [1], 0),
    (64, 16, 16, 15, 5, [33, 0, 63, 64, 65, 127], [1] * 6, 0),
    (64, 8, 64, 6, 2, [200, 0, 1, 77], [1, 1, 0, 5], 0),
    (64, 16, 32, 4, 4, [0, 5], [37, 64], 0),
    (64, 16, 64, 8, 1, [3, 130], [65, 17], 40),
    (64, 8, 16, 16, 1, [0, 9], [33, 128], 1),
    (128, 16, 64, 4, 2, [100, 0], [1, 40], 0),
    (128, 8, 128, 5, 1, [10, 300], [30, 1], 100),
    (128, 16, 16, 16, 2, [0, 0, 250], [129, 1, 3], 0),
    (16, 16, 16, 2, 1, [70, 0], [1, 20], 0),
    (16, 8, 64, 14, 2, [3], [50], 7),
    (32, 16, 256, 7, 1, [300, 2], [2, 33], 0),
    (32, 8, 16, 4, 2, [100], [16], 33),
    (256, 16, 16, 3, 1, [90, 0], [1, 10], 0),
    (256, 8, 32, 2, 2, [40], [20], 16),
]


@gpu
@pytest.mark.parametrize("hi", [2000, 32768], ids=["small", "full"])
@pytest.mark.parametrize("case", ATTNS, ids=lambda c: "hd%d_b%d_p%d_h%d_%d_n%d_w%d" % (c[:5] + (max(c[6]), c[7])))
def test_attn_vs_oracle(case, hi):
    """Every head width, page size and width of the words; lengths around the
    64-key tiles and the 16- and 128-row tiles; small words (a spread softmax)
    and the full range (sums that wrap, scores that saturate)."""
    HD, bits, page, H, KV, ctx, new, w = case
    rng = np.random.default_rng(HD * 7 + bits + sum(ctx) + hi)
    pages = sum(-(-(c + n) // page) for c, n in zip(ctx, new)) + 2
    table, cu, pos, rows = _batch(rng, pages, page, ctx, new, extra=2)
    c = _random_cache(rng, pages, KV, page, HD, bits, hi)
    c.table, c.cu, c.pos = table, cu, pos
    want = _run_attn(c, rows, H, _smx(H, HD, f_s=10 if hi == 2000 else 12), rng, window=w, hi=hi, odd=hi == 2000,
                     max_q=max(new), max_keys=max(a + b for a, b in zip(ctx, new)))
    assert (want[:rows - 2] != 0).mean() > 0.3


@gpu
@pytest.mark.parametrize("HD,bits,window", [(64, 16, 0), (64, 8, 0), (128, 16, 0), (128, 8, 130), (64, 16, 1)])
def test_attn_more_tiles_than_multiprocessors(HD, bits, window):
    """Several tiles for every CTA, of unlike lengths, sequences without rows
    between them, contexts in one and in more windows."""
    rng = np.random.default_rng(HD + bits + window)
    KV, page, B = 5, 32, 44
    new = [int(rng.integers(1, 150)) if i % 5 else 0 for i in range(B)]
    ctx = [int(rng.integers(0, 200)) for i in range(B)]
    new[7], ctx[7], new[30], ctx[30] = 300, 0, 129, 800
    pages = sum(-(-(a + n) // page) for a, n in zip(ctx, new)) + 2
    table, cu, pos, rows = _batch(rng, pages, page, ctx, new, extra=2)
    c = _random_cache(rng, pages, KV, page, HD, bits, 2500)
    c.table, c.cu, c.pos = table, cu, pos
    want = _run_attn(c, rows, KV, _smx(KV, HD, f_s=10), rng, window=window, hi=2500, max_q=max(new),
                     max_keys=max(a + b for a, b in zip(ctx, new)))
    assert (want[:rows - 2] != 0).mean() > 0.3


@gpu
@pytest.mark.parametrize("HD,bits,ctx,hint", [(64, 16, 9000, 9001), (64, 8, 15001, 9), (128, 8, 7000, 7001),
                                              (256, 16, 3001, 1)])
def test_attn_long_contexts_few_rows(HD, bits, ctx, hint):
    """Many more tiles of keys than stages of copies, one row and a few."""
    rng = np.random.default_rng(ctx)
    page, new = 64, [1, 3]
    ctxs = [ctx, ctx // 3]
    pages = sum(-(-(a + n) // page) for a, n in zip(ctxs, new)) + 1
    table, cu, pos, rows = _batch(rng, pages, page, ctxs, new)
    c = _random_cache(rng, pages, 2, page, HD, bits, 2500)
    c.table, c.cu, c.pos = table, cu, pos
    _run_attn(c, rows, 6, _smx(6, HD, f_s=10), rng, hi=2500, max_q=3, max_keys=hint)


@gpu
@pytest.mark.parametrize("HD,bits,new", [(64, 16, 1), (64, 16, 70), (64, 8, 1), (128, 16, 33), (256, 16, 20)])
def test_attn_softmax_registers(HD, bits, new):
    """Registers that differ by head: shifts below 8 and from 40 up, P at 0 to
    31 bits, a scale that leaves only the maximum, one that keeps every key."""
    rng = np.random.default_rng(31)
    H, KV, page = 12, 2, 16
    smx = np.array([[0xFFFFFF, 0 | 12 << 8], [0xFFFFFF, 7 | 8 << 8], [0xFFFFFF, 8 | 15 << 8], [0x800000, 39 | 12 << 8],
                    [0x812345, 40 | 14 << 8], [0xFFFFFF, 63 | 15 << 8], [0, 20 | 12 << 8], [1, 0 | 0 << 8],
                    [0xABCDEF, 24 | 31 << 8], [0xABCDEF, 28 | 16 << 8], [0xABCDEF, 21 | 12 << 8], [0x123456, 12 | 4 << 8]],
                   np.int32)
    table, cu, pos, rows = _batch(rng, 24, page, [150, 31], [new, 1])
    c = _random_cache(rng, 24, KV, page, HD, bits, 3000)
    c.table, c.cu, c.pos = table, cu, pos
    _run_attn(c, rows, H, smx, rng, hi=3000, max_q=new, max_keys=150 + new)


@gpu
@pytest.mark.parametrize("HD,bits,H,KV,ctx,new,hint", [
    (64, 16, 3, 1, 900, 1, 1), (64, 8, 6, 2, 700, 9, 64), (128, 16, 4, 1, 500, 5, 1), (256, 16, 4, 2, 700, 3, 1),
    (64, 16, 4, 2, 1500, 40, 1), (64, 8, 4, 2, 1100, 70, 1), (128, 16, 4, 1, 1200, 40, 1), (128, 8, 4, 4, 1000, 130, 1)])
def test_attn_keys_beyond_the_hint(HD, bits, H, KV, ctx, new, hint):
    """More keys than the hint said: the scores do not fit at once and are formed
    again in windows, with the same result."""
    rng = np.random.default_rng(ctx)
    page = 32
    pages = -(-(ctx + new) // page) + 1
    table, cu, pos, rows = _batch(rng, pages, page, [ctx], [new])
    c = _random_cache(rng, pages, KV, page, HD, bits, 2500)
    c.table, c.cu, c.pos = table, cu, pos
    _run_attn(c, rows, H, _smx(H, HD, f_s=10), rng, hi=2500, max_q=new, max_keys=hint)


@gpu
@pytest.mark.parametrize("new", [1, 24])
@pytest.mark.parametrize("HD,bits", [(64, 16), (64, 8), (128, 8)])
def test_attn_missing_pages_and_late_positions(HD, bits, new):
    """Pages that are not there count as zeros; positions past the table see
    what the table covers, or nothing with a window; cu and pos out of range;
    rows past max_q left alone."""
    rng = np.random.default_rng(HD + bits)
    H, KV, page = 4, 2, 16
    ctx, n = [80, 20, 40, 0, 60], [new, new, new, new, 2 * new]
    table, cu, pos, rows = _batch(rng, 64, page, ctx, n, spare=0, extra=1)
    c = _random_cache(rng, 64, KV, page, HD, bits, 3000)
    c.table, c.cu, c.pos = table, cu, pos
    c.table[0, 1], c.table[0, 4], c.table[1, 0] = 64, -1, 1 << 30
    c.pos[2] = c.cap + 5
    c.pos[3] = -4
    c.cu[-1] = rows + 9
    for w in (0, 4, 100):
        _run_attn(c, rows, H, _smx(H, HD, f_s=10), rng, window=w, hi=3000, max_q=new, max_keys=90)


@gpu
@pytest.mark.parametrize("window", [0, 150])
@pytest.mark.parametrize("HD,bits,page", [(64, 16, 16), (64, 8, 128), (128, 16, 64), (128, 8, 256)])
def test_attn_tiles_of_missing_pages(HD, bits, page, window):
    """Rows of 128-row tiles over pages that are not there: single ones, whole tiles
    of keys (whose copies are none), one after tiles that are there; positions past
    the table, cu and pos out of range, rows past max_q."""
    rng = np.random.default_rng(HD + bits + window)
    H, KV, new = 4, 2, 70
    ctx, n = [700, 300, 0, 90], [new, new, new, new + 9]
    table, cu, pos, rows = _batch(rng, 130, page, ctx, n, spare=0, extra=1)
    c = _random_cache(rng, 130, KV, page, HD, bits, 3000)
    c.table, c.cu, c.pos = table, cu, pos
    per = max(1, 128 // page)
    c.table[0, 2 * per:4 * per] = -1                 # two tiles of keys and more
    c.table[0, 0], c.table[0, -1] = 130, 1 << 30
    c.table[1, :per] = -9                            # the first tile
    c.pos[2] = c.cap - 20                            # the last rows lie past the table
    c.pos[3] = -4
    c.cu[-1] = rows + 9
    _run_attn(c, rows, H, _smx(H, HD, f_s=10), rng, window=window, hi=3000, max_q=new, max_keys=ctx[0] + new)


@gpu
def test_attn_equal_scores_and_extremes():
    """Zero queries (every score alike: P = 1 / keys), the most negative words
    (a score of -2^15 where every sum saturates), a single key."""
    from cormorant_b200 import ops
    rng = np.random.default_rng(3)
    H, KV, HD, page = 2, 1, 64, 16
    for new in (1, 50):
        table, cu, pos, rows = _batch(rng, 12, page, [100, 0], [new, 1])
        c = _random_cache(rng, 12, KV, page, HD, 16)
        c.table, c.cu, c.pos = table, cu, pos
        for fill_q, fill_k in ((0, None), (-32768, -32768), (32767, -32768), (-32768, 32767)):
            if fill_k is not None:
                c.kc[..., :HD], c.kc[..., HD:] = fill_k >> 8, np.int64(fill_k & 255).astype(np.uint8).view(np.int8)
            cache, batch = _handles(c, rows, max_q=new, max_keys=100 + new)
            q = np.full((rows, H * HD), fill_q, np.int16)
            o = torch.zeros((rows, H * HD), dtype=torch.int16, device="cuda")
            smx = _smx(H, HD, f_p=15)
            ops.llm_paged_attn(cache, batch, _dev(q), o, H=H, smx=_dev(smx))
            want = np.zeros((rows, H * HD), np.int64)
            OP.attn(c, q, want, H=H, smx=smx)
            assert np.array_equal(o.cpu().numpy(), want), (new, fill_q, fill_k)


@gpu
def test_paged_step_captured_and_on_streams():
    """A step's two calls captured once and replayed with other positions,
    pages and rows; then the same calls on two streams at once, each with its own
    cache."""
    from cormorant_b200 import ops
    rng = np.random.default_rng(12)
    H, KV, HD, page, B = 6, 2, 64, 16, 3
    smx, pe = _smx(H, HD), RH.pblock(0, 0, 0, 0, 26, 8)[0].astype(np.int16)
    pv = RH.pblock(0, 0, 0, 0, 4, 8)[0].astype(np.int16)
    rope = _rope(400, HD)

    def fresh(seed, bits):
        r = np.random.default_rng(seed)
        ctx = [int(x) for x in r.integers(0, 300, B)]
        table, cu, pos, rows = _batch(r, 80, page, ctx, [1] * B)
        full = np.full((B, 20), -1, np.int32)
        full[:, :table.shape[1]] = table[:, :20]
        c = _random_cache(r, 80, KV, page, HD, bits, 2000)
        c.table, c.cu, c.pos = full, cu, pos
        a = [r.integers(-2000, 2000, size=(B, m * HD)).astype(np.int16) for m in (H, KV, KV)]
        return c, a

    def want(c, a):
        q, o = np.zeros((B, H * HD), np.int64), np.zeros((B, H * HD), np.int64)
        OP.prep(c, *a, q, H=H, rope=rope, rot=HD, interleaved=False, pq=pe, pk=pe, pv=pv)
        OP.attn(c, q, o, H=H, smx=smx)
        return o
    common = dict(rope=_dev(rope), pq=_dev(pe), pk=_dev(pe), pv=_dev(pv), pq_bc=True, pk_bc=True, pv_bc=True)
    sd = _dev(smx)
    for bits in (16, 8):
        c, a = fresh(1, bits)
        cache, batch = _handles(c, B, max_q=1, max_keys=320)
        ad = [_dev(x) for x in a]
        q, o = (torch.zeros((B, H * HD), dtype=torch.int16, device="cuda") for _ in range(2))

        def step():
            ops.llm_paged_prep(cache, batch, *ad, q, H=H, **common)
            ops.llm_paged_attn(cache, batch, q, o, H=H, smx=sd)
        step()
        assert np.array_equal(o.cpu().numpy(), want(c, a))
        _same_bytes(c, cache)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
        for seed in (2, 3, 4):
            c, a = fresh(seed, bits)
            for t, x in zip((cache.kc, cache.vc, cache.ks, cache.vs, batch.table, batch.cu, batch.pos, *ad),
                            (c.kc, c.vc, c.ks, c.vs, c.table, c.cu, c.pos, *a)):
                if t is not None:
                    t.copy_(_dev(x))
            o.fill_(3)
            graph.replay()
            assert np.array_equal(o.cpu().numpy(), want(c, a))
            _same_bytes(c, cache)
    # two streams at once
    cs = [fresh(20 + i, 16) for i in range(2)]
    hs = [_handles(c, B, max_q=1, max_keys=320) for c, _ in cs]
    xs = [[_dev(x) for x in a] for _, a in cs]
    outs = [[torch.zeros((B, H * HD), dtype=torch.int16, device="cuda") for _ in range(2)] for _ in cs]
    streams = [torch.cuda.Stream() for _ in cs]
    torch.cuda.synchronize()
    for _ in range(4):
        for (cache, batch), ad, (q, o), s in zip(hs, xs, outs, streams):
            with torch.cuda.stream(s):
                ops.llm_paged_prep(cache, batch, *ad, q, H=H, **common)
                ops.llm_paged_attn(cache, batch, q, o, H=H, smx=sd)
    torch.cuda.synchronize()
    for (c, a), (q, o) in zip(cs, outs):
        assert np.array_equal(o.cpu().numpy(), want(c, a))
    assert ops.device_status() == 0


@gpu
def test_prep_writes_what_attn_reads_chunk_by_chunk():
    """A prompt at once, and the same prompt in ragged chunks (each attending to
    the pages the chunks before filled), give the same rows, at 16 and 8 bits;
    the rows also come back the same."""
    from cormorant_b200 import ops
    rng = np.random.default_rng(40)
    H, KV, HD, page, n = 6, 2, 64, 16, 150
    rope = _dev(_rope(n, HD))
    pe = RH.pblock(0, 0, 0, 0, 26, 8)[0].astype(np.int16)
    par = dict(rope=rope, pq=_dev(pe), pk=_dev(pe), pq_bc=True, pk_bc=True, v_direct=True)
    x = [_dev(rng.integers(-3000, 3000, size=(n, m * HD)).astype(np.int16)) for m in (H, KV, KV)]
    smx = _dev(_smx(H, HD))
    for bits in (16, 8):
        outs, kvs = [], []
        for chunks in ([n], [1, 63, 2, 64, 20], [50] * 3):
            cache = paged.PagedCache(20, page, KV, HD, bits)
            pool, at = paged.PagePool(20, page), 0
            q, o = (torch.zeros((n, H * HD), dtype=torch.int16, device="cuda") for _ in range(2))
            for m in chunks:
                batch = paged.PagedBatch.of([pool.extend(0, at + m)], [m], [at])
                sl = slice(at, at + m)
                ops.llm_paged_prep(cache, batch, *(t[sl] for t in x), q[sl], H=H, **par)
                ops.llm_paged_attn(cache, batch, q[sl], o[sl], H=H, smx=smx)
                at += m
            k, v = (torch.zeros((n, KV * HD), dtype=torch.int16, device="cuda") for _ in range(2))
            ops.llm_paged_read(cache, paged.PagedBatch.of([pool.held[0]], [n], [0]), k, v)
            outs.append(o)
            kvs.append(torch.cat([k, v], 1))
        assert all(torch.equal(outs[0], t) for t in outs[1:]) and all(torch.equal(kvs[0], t) for t in kvs[1:])
        assert bits == 8 or torch.equal(kvs[0][:, KV * HD:], x[2])


CHUNKS = [  # HD, bits, page, H, KV, contexts, new rows, window
    (64, 16, 64, 4, 1, [900, 20, 0, 1500, 300], [40, 70, 0, 33, 64], 0),
    (64, 8, 32, 6, 2, [1100, 1100, 5], [70, 1, 65], 0),
    (128, 16, 16, 4, 1, [1700], [129], 0),
    (128, 8, 128, 8, 2, [600, 0, 1300, 64], [50, 50, 50, 50], 0),
    (64, 16, 256, 3, 1, [2500, 130], [90, 90], 700)]


@gpu
@pytest.mark.parametrize("case", CHUNKS, ids=lambda c: "hd%d_b%d_p%d_h%d_%d_w%d" % (c[:5] + (c[7],)))
def test_attn_chunks_over_contexts(case):
    """Chunks of rows behind longer and shorter contexts: the sequences taken by
    their lengths, an item's keys shared by a cluster, empty sequences between."""
    HD, bits, page, H, KV, ctx, new, w = case
    rng = np.random.default_rng(sum(ctx) + HD + bits)
    pages = sum(-(-(c + n) // page) for c, n in zip(ctx, new)) + 2
    table, cu, pos, rows = _batch(rng, pages, page, ctx, new, extra=1)
    c = _random_cache(rng, pages, KV, page, HD, bits, 2500)
    c.table, c.cu, c.pos = table, cu, pos
    _run_attn(c, rows, H, _smx(H, HD, f_s=10), rng, window=w, hi=2500, max_q=max(new),
              max_keys=max(a + b for a, b in zip(ctx, new)))


@gpu
@pytest.mark.parametrize("new,ctx", [([130, 7, 200], [0, 600, 40]), ([1, 2, 1], [2500, 30, 1300])], ids=["prompts", "decode"])
def test_attn_captured_with_other_lengths(new, ctx):
    """A captured call replayed with the rows, positions and pages of other
    batches within its max_q and rows (the hint of the keys passed, too)."""
    from cormorant_b200 import ops
    HD, KV, H, page, width = 64, 2, 6, 32, 90
    rng = np.random.default_rng(sum(new))
    smx, rows = _smx(H, HD, f_s=10), sum(new)

    def batch_of(ctx, new):
        table, cu, pos, _ = _batch(rng, 200, page, ctx, new)
        full = np.full((3, width), -1, np.int32)
        full[:, :table.shape[1]] = table
        return full, cu, pos
    c = _random_cache(rng, 200, KV, page, HD, 16, 2500)
    c.table, c.cu, c.pos = batch_of(ctx, new)
    cache, batch = _handles(c, rows, max_q=max(new), max_keys=max(a + b for a, b in zip(ctx, new)))
    qh = rng.integers(-2500, 2500, size=(rows, H * HD)).astype(np.int16)
    q, o, sd = _dev(qh), torch.zeros((rows, H * HD), dtype=torch.int16, device="cuda"), _dev(smx)
    ops.llm_paged_attn(cache, batch, q, o, H=H, smx=sd)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.llm_paged_attn(cache, batch, q, o, H=H, smx=sd)
    for perm in ([0, 1, 2], [2, 0, 1], [1, 2, 0]):
        n2 = [new[perm[0]], 0 if perm[0] == 2 else new[perm[1]], new[perm[2]]]
        c.table, c.cu, c.pos = batch_of([ctx[i] // 2 + 9 * i for i in perm], n2)
        for t, x in zip((batch.table, batch.cu, batch.pos), (c.table, c.cu, c.pos)):
            t.copy_(_dev(x))
        o.fill_(5)
        graph.replay()
        want = np.full((rows, H * HD), 5, np.int64)
        OP.attn(c, qh, want, H=H, smx=smx, max_q=max(new))
        assert np.array_equal(o.cpu().numpy(), want)
    assert ops.device_status() == 0


@gpu
def test_calls_from_two_threads():
    """Two host threads, each with its own cache, sizes and stream, at once: every
    result is the one of the call alone."""
    import threading
    from cormorant_b200 import ops
    rng = np.random.default_rng(91)
    jobs = []
    for HD, KV, ctx, new in ((64, 2, [3000, 40], [1, 2]), (64, 2, [5], [90]), (64, 2, [700, 0, 90], [1, 300, 40]),
                             (128, 1, [1500], [1])):
        page = 32
        pages = sum(-(-(a + n) // page) for a, n in zip(ctx, new)) + 1
        table, cu, pos, rows = _batch(rng, pages, page, ctx, new)
        c = _random_cache(rng, pages, KV, page, HD, 16, 2500)
        c.table, c.cu, c.pos = table, cu, pos
        cache, batch = _handles(c, rows, max_q=max(new), max_keys=max(a + b for a, b in zip(ctx, new)))
        q, smx = _dev(rng.integers(-2500, 2500, size=(rows, 2 * KV * HD)).astype(np.int16)), _dev(_smx(2 * KV, HD, f_s=10))
        want = torch.zeros((rows, 2 * KV * HD), dtype=torch.int16, device="cuda")
        ops.llm_paged_attn(cache, batch, q, want, H=2 * KV, smx=smx)
        jobs.append((cache, batch, q, smx, 2 * KV, want))
    torch.cuda.synchronize()
    bad = []

    def work(mine):
        with torch.cuda.stream(torch.cuda.Stream()):
            for i in range(60):
                cache, batch, q, smx, H, want = mine[i % len(mine)]
                o = torch.zeros_like(want)
                ops.llm_paged_attn(cache, batch, q, o, H=H, smx=smx)
                if i % 7 == 0 and not torch.equal(o, want):
                    bad.append(i)
            torch.cuda.current_stream().synchronize()
            if not torch.equal(o, want):
                bad.append(-1)
    threads = [threading.Thread(target=work, args=(m,)) for m in (jobs[:2], jobs[2:])]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad and ops.device_status() == 0


@gpu
def test_gpu_refusals():
    """Arguments of the wrong type, size, stride or device raise; nothing runs."""
    from cormorant_b200 import ops
    cache = paged.PagedCache(4, 16, 2, 64)
    batch = paged.PagedBatch.of([[0, 1]], [4], [3])
    z = lambda n, dt=torch.int16, dev="cuda": torch.zeros((4, n), dtype=dt, device=dev)  # noqa: E731
    smx = torch.zeros((4, 2), dtype=torch.int32, device="cuda")
    for q, o, kw in ((z(256, torch.int32), z(256), {}), (z(256), z(256, dev="cpu"), {}), (z(255), z(256), {}),
                     (z(256), z(256), dict(ldq=300)), (z(256), z(256), dict(ldo=200)), (z(512)[:, ::2], z(256), {})):
        with pytest.raises(_lib.CormError):
            ops.llm_paged_attn(cache, batch, q, o, H=4, smx=smx, **kw)
    with pytest.raises(_lib.CormError):
        ops.llm_paged_attn(cache, batch, z(256), z(256), H=4, smx=smx[:3])
    with pytest.raises(_lib.CormError):
        ops.llm_paged_attn(cache, batch, z(192), z(192), H=3, smx=smx)
    with pytest.raises(_lib.CormError):
        ops.llm_paged_read(cache, batch, z(64), None)
    e = torch.zeros((1, 16), dtype=torch.uint8, device="cuda")
    rope = torch.zeros((8, 64), dtype=torch.int32, device="cuda")
    ok = dict(H=4, rope=rope, pq=e, pk=e, pv=e, pq_bc=True, pk_bc=True, pv_bc=True)
    ops.llm_paged_prep(cache, batch, z(256), z(128), z(128), z(256), **ok)
    for kw in (dict(pq_bc=False), dict(pv=None), dict(rope=rope.to(torch.int64)), dict(rot=65), dict(nq=e),
               dict(rope=rope[:0])):
        with pytest.raises(_lib.CormError):
            ops.llm_paged_prep(cache, batch, z(256), z(128), z(128), z(256), **dict(ok, **kw))
    assert ops.device_status() == 0


@gpu
def test_gpu_refused_rotation_tables():
    """The preparation asks for a table of its rot's width."""
    from cormorant_b200 import ops
    cache, batch = paged.PagedCache(4, 16, 2, 64), paged.PagedBatch.of([[0, 1]], [4], [3])
    z = lambda n: torch.zeros((4, n), dtype=torch.int16, device="cuda")  # noqa: E731
    e = torch.zeros((1, 16), dtype=torch.uint8, device="cuda")
    rope = torch.zeros((8, 64), dtype=torch.int32, device="cuda")
    ok = dict(H=4, pq=e, pk=e, pv=e, pq_bc=True, pk_bc=True, pv_bc=True)
    for kw in (dict(rope=rope), dict(rope=rope.view(-1)), dict(rope=rope[:, :32].contiguous(), rot=32)):
        ops.llm_paged_prep(cache, batch, z(256), z(128), z(128), z(256), **ok, **kw)
    for kw in (dict(rope=rope, rot=32), dict(rope=rope[:, :32].contiguous()), dict(rope=rope.view(-1)[:100])):
        with pytest.raises(_lib.CormError, match="rope"):
            ops.llm_paged_prep(cache, batch, z(256), z(128), z(128), z(256), **ok, **kw)
    assert ops.device_status() == 0


@gpu
@pytest.mark.parametrize("ctx,new,codes", [([0, 0], [300, 140], range(311, 324)), ([6000], [100], range(311, 324)),
                                           ([6000], [1], [303])], ids=["tiles", "tile_cluster", "cluster"])
@pytest.mark.parametrize("HD,bits", [(64, 16), (128, 8)])
def test_attn_waits_that_run_out(HD, bits, ctx, new, codes):
    """Waits of 200 cycles, far below a copy's time, run out: the launch ends, its status
    is read once, and the next launch with the usual limit is exact."""
    from cormorant_b200 import ops
    rng = np.random.default_rng(HD + new[0])
    H, KV, page = 4, 2, 64
    pages = sum(-(-(a + n) // page) for a, n in zip(ctx, new))
    table, cu, pos, rows = _batch(rng, pages, page, ctx, new)
    c = _random_cache(rng, pages, KV, page, HD, bits, 2500)
    c.table, c.cu, c.pos = table, cu, pos
    kw = dict(max_q=max(new), max_keys=max(a + n for a, n in zip(ctx, new)))
    cache, batch = _handles(c, rows, **kw)
    smx = _smx(H, HD, f_s=10)
    q, o = (torch.zeros((rows, H * HD), dtype=torch.int16, device="cuda") for _ in range(2))
    assert ops.device_status() == 0
    L = _lib.lib()
    try:
        assert L.corm_set_wait_limit(200) == 0
        ops.llm_paged_attn(cache, batch, q, o, H=H, smx=_dev(smx))
        torch.cuda.synchronize()
    finally:
        assert L.corm_set_wait_limit(0) == 0
    assert ops.device_status() in codes
    assert ops.device_status() == 0
    _run_attn(c, rows, H, smx, rng, hi=2500, **kw)
