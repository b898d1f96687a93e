"""A Llama model served over the paged KV cache (llm_runner.PagedLlamaRunner):
prompts of unlike lengths, chunks and single tokens in one pass, sequences that
come, end and leave their pages to others, against the contiguous prefill graph
(with the same softmax unit) run over each sequence's whole tokens."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from cormorant_b200 import workloads as WL  # noqa: E402
from cormorant_b200._lib import CormError  # noqa: E402
from cormorant_b200.llm_runner import PagedLlamaRunner  # noqa: E402
from oracle import paged as OP  # noqa: E402

gpu = pytest.mark.gpu
SMALL = dict(layers=1, hidden=64, heads=4, kv_heads=2, head_dim=16, ffn=128, vocab=50)


@pytest.fixture
def paged_cpu(cpu_ops, monkeypatch):
    """The paged operators replayed on the oracle over CPU tensors, beside the
    other kernels' job models."""
    from cormorant_b200 import ops

    def host(cache, batch):
        a = [None if t is None else t.numpy() for t in (cache.kc, cache.vc, cache.ks, cache.vs, batch.table, batch.cu,
                                                        batch.pos)]
        return OP.Cache(*a, cache.HD, cache.bits)

    def rows(t, n, w):
        return t.numpy().reshape(-1)[:n * w].reshape(n, w)

    def prep(cache, batch, q0, k0, v0, q, *, H, rope, pq, pk, pv=None, rot=None, interleaved=False, pq_bc=False,
             pk_bc=False, pv_bc=False, v_direct=False, **kw):
        assert not kw
        R, nq, nk = batch.rows, H * cache.HD, cache.KV * cache.HD
        out = np.zeros((R, nq), np.int64)

        def ent(t, bc, n):
            e = t.numpy()[:8 if bc else 8 * n]
            return e.astype(np.int16)
        OP.prep(host(cache, batch), rows(q0, R, nq).astype(np.int64), rows(k0, R, nk).astype(np.int64),
                rows(v0, R, nk).astype(np.int64), out, H=H, rope=rope.numpy().reshape(-1, cache.HD).astype(np.int64),
                rot=cache.HD, interleaved=False, pq=ent(pq, pq_bc, nq), pk=ent(pk, pk_bc, nk),
                pv=None if v_direct else ent(pv, pv_bc, nk))
        rows(q, R, nq)[...] = out

    def attn(cache, batch, q, o, *, H, smx, window=0):
        R, n = batch.rows, H * cache.HD
        out = np.zeros((R, n), np.int64)
        OP.attn(host(cache, batch), rows(q, R, n).astype(np.int64), out, H=H, smx=smx.numpy(), window=window)
        rows(o, R, n)[...] = out
    monkeypatch.setattr(ops, "llm_paged_prep", prep)
    monkeypatch.setattr(ops, "llm_paged_attn", attn)


def _words(logits, n, vocab):
    return logits[:n * vocab].cpu().numpy().reshape(n, vocab)


def _contiguous(dims, seq, tokens, device):
    """The contiguous prefill's logits after the tokens, and its model."""
    from cormorant_b200.simulator import GpuSimulator
    m = WL.LlamaModel(batch=1, seq=seq, **dims)
    sim = GpuSimulator(m.prefill_graph, device=device)
    out = m.prefill_graph.output_tensors[0].onnx_name
    got = []
    for t in tokens:
        h = np.zeros((seq, m.D))
        h[:len(t)] = m.emb[np.asarray(t)]
        feeds = {"h0": h, "pos": np.array([0]), "n": np.array([len(t)])}
        raw = {x.onnx_name: (np.asarray(feeds[x.onnx_name]).astype(np.int64).reshape(-1) if x.host
                             else sim._to_raw(x, feeds[x.onnx_name])) for x in m.prefill_graph.input_tensors}
        res, _ = sim.forward_raw(raw, keep=[out], states=sim.states_to_device())
        got.append(_words(res[out], 1, m.vocab)[0])
    return np.stack(got)


def _served(dims, device, lengths, steps, seq, page, bits=16, chunk=5):
    """Two sequences from their prompts, a third joining in chunks while they
    decode, then one ended and its pages taken by a fourth; every pass's logits
    with the tokens that lead to them."""
    m = WL.LlamaModel(batch=1, seq=seq, **dims)
    rng = np.random.default_rng(1)
    prompt = {s: rng.integers(0, m.vocab, n).tolist() for s, n in zip("abcd", lengths)}
    pages = sum(-(-(lengths[i] + 3 * steps) // page) for i in range(3)) + 1
    r = PagedLlamaRunner(m, pages=pages, page=page, bits=bits, device=device)
    seen = []

    def note(tokens, logits):
        seen.extend(zip([list(t) for t in tokens], _words(logits, len(tokens), m.vocab)))
    tok = {s: list(prompt[s]) for s in "ab"}
    lg = r.append("ab", [tok["a"], tok["b"]])
    note([tok["a"], tok["b"]], lg)
    ids = torch.empty(2, dtype=torch.int32, device=r.device)
    for _ in range(steps):
        lg = r.step("ab", lg, ids)
        for s, t in zip("ab", ids.tolist()):
            tok[s].append(t)
        note([tok["a"], tok["b"]], lg)
    tok["c"] = []
    while len(tok["c"]) < lengths[2]:  # a chunk of c beside a token of a and b
        best = _words(lg, 2, m.vocab).argmax(1)
        new = prompt["c"][len(tok["c"]):len(tok["c"]) + chunk]
        for s, t in zip("ab", best.tolist()):
            tok[s].append(t)
        tok["c"] += new
        lg = r.append("acb", [tok["a"][-1:], new, tok["b"][-1:]])
        note([tok["a"], tok["c"], tok["b"]], lg)
        lg = torch.from_numpy(_words(lg, 3, m.vocab)[[0, 2]].reshape(-1).copy()).to(r.device)
    r.release("a")
    free = len(r.pool.free)
    lg = r.append("d", [prompt["d"]])
    note([prompt["d"]], lg)
    assert r.length == dict(b=len(tok["b"]), c=lengths[2], d=lengths[3]) and len(r.pool.free) < free
    return m, seen


def test_runner_host_logic_cpu(paged_cpu):
    dims = dict(SMALL, seed=4)
    _, seen = _served(dims, "cpu", (9, 3, 7, 12), 2, 32, 16)
    want = _contiguous(dims, 32, [t for t, _ in seen], "cpu")
    assert len(seen) >= 10
    for (t, got), w in zip(seen, want):
        assert np.array_equal(got, w), len(t)


def test_runner_refuses(paged_cpu):
    m = WL.LlamaModel(batch=1, seq=16, cache=32, seed=4, **SMALL)
    r = PagedLlamaRunner(m, pages=2, page=16, device="cpu")
    for seqs, ids in (("ab", [[1]]), ("aa", [[1], [2]]), ("a", [[]]), ("a", [[50]]), ("a", [[-1]]), ([], []),
                      ("a", [[1] * 33])):
        with pytest.raises(CormError):
            r.append(seqs, ids)
    with pytest.raises(MemoryError):
        r.append("abc", [[1], [2], [3]])
    assert not r.pool.held and not r.length and len(r.pool.free) == 2
    r.append("ab", [[1] * 16, [2]])
    with pytest.raises(MemoryError):
        r.append("ba", [[1], [1]])  # a has no page for its 17th token; b is as it was
    assert r.length == dict(a=16, b=1)
    r.release("b")
    r.append("a", [[1]])
    assert r.length == dict(a=17)


def test_append_takes_one_list_a_sequence(paged_cpu):
    """Tokens in an array of another shape are refused: its length is not their number."""
    m = WL.LlamaModel(batch=1, seq=16, cache=32, seed=4, **SMALL)
    r = PagedLlamaRunner(m, pages=3, page=16, device="cpu")
    for bad in (np.array([[1, 2, 3]]), [[1], [2]], torch.tensor([[4, 5]]), np.array(3)):
        with pytest.raises(CormError):
            r.append("ab", [[1], bad])
    assert not r.length and len(r.pool.free) == 3
    want = r.append("a", [[1, 2, 3]])
    for s, good in (("b", np.array([1, 2, 3], np.uint8)), ("c", torch.tensor([1, 2, 3]))):
        assert torch.equal(r.append(s, [good])[:m.vocab], want[:m.vocab])


def test_rotation_tables_of_shared_weights(paged_cpu, monkeypatch):
    """Simulators that share weights, each graph with a rotation table of its own: a
    table that is gone does not serve one that came to lie at its address."""
    import gc

    from cormorant_b200 import attention as AT
    from cormorant_b200.paged import PagedBatch, PagedCache
    from cormorant_b200.simulator import GpuSimulator
    m = WL.LlamaModel(batch=1, seq=16, cache=32, seed=4, **SMALL)
    first = GpuSimulator(m.paged_graph(4), device="cpu")
    m.rope = None
    h = torch.from_numpy(np.rint(m.emb[[3, 9, 4, 7]] * 2.0 ** m.E["fr"]).astype(np.int32).reshape(-1))

    def run(share):
        g = m.paged_graph(4)
        sim = GpuSimulator(g, device="cpu", share=share)
        sim.paged = ([PagedCache(2, 16, m.KV, m.HD, device="cpu")], PagedBatch.of([[0]], [4], [5], device="cpu"))
        out = g.output_tensors[0].onnx_name
        res, _ = sim.forward_raw({"h_step": h}, keep=[out])
        return res[out][:4 * m.D].clone()
    turned = AT.paged_rope(m.sin, m.cos)  # another rotation
    wrap = torch.from_numpy
    monkeypatch.setattr(torch, "from_numpy", lambda a: wrap(a).clone())  # as an upload to a device does
    m.rope = AT.paged_rope(m.cos, m.sin)
    at, one = id(m.rope), run(first)
    m.rope = None
    gc.collect()
    kept = []
    for _ in range(2000):
        m.rope = turned.copy()
        if id(m.rope) == at:
            break
        kept.append(m.rope)
    two = run(first)
    assert torch.equal(two, run(None)) and not torch.equal(one, two)


def test_step_refuses_before_it_writes(paged_cpu):
    """A step that cannot be made leaves ids, the sequences and the pool as they were."""
    m = WL.LlamaModel(batch=1, seq=16, cache=32, seed=4, **SMALL)
    r = PagedLlamaRunner(m, pages=3, page=16, device="cpu")
    lg = r.append("ab", [[1] * 32, [2] * 16])
    ids = torch.full((2,), -5, dtype=torch.int32)
    for seqs, err in (("aa", CormError), ("", CormError), ("ab", CormError), ("b", MemoryError)):
        with pytest.raises(err):  # twice a sequence, none, a at the model's 32 positions, no page for b's 17th token
            r.step(seqs, lg, ids)
        assert ids.tolist() == [-5, -5] and r.length == dict(a=32, b=16) and not r.pool.free
    r.release("a")
    r.step("b", lg[m.vocab:], ids)
    assert ids[0] >= 0 and ids[1] == -5 and r.length == dict(b=17)


def test_runner_on_two_threads(paged_cpu, monkeypatch):
    """Two threads on one runner, each with sequences of its own: every pass's logits are
    those of the sequence alone, wherever the other thread's passes fall."""
    import threading
    import time

    from cormorant_b200 import ops
    m = WL.LlamaModel(batch=1, seq=16, cache=32, seed=4, **SMALL)
    inner = ops.llm_paged_prep

    def slow(*a, **kw):  # the other thread has its turn in the middle of a pass
        time.sleep(0.005)
        inner(*a, **kw)
    monkeypatch.setattr(ops, "llm_paged_prep", slow)

    def serve(r, s, first):
        got = []
        for i in range(4):
            ids = torch.empty(1, dtype=torch.int32)
            lg = r.append([(s, i)], [[first + i, 7, 3]])
            got.append(_words(lg, 1, m.vocab))
            got.append(_words(r.step([(s, i)], lg, ids), 1, m.vocab))
            if i % 2:
                r.release((s, i))
        return np.stack(got)
    alone = [serve(PagedLlamaRunner(m, pages=4, page=16, device="cpu"), s, 9 * s) for s in range(2)]
    r = PagedLlamaRunner(m, pages=8, page=16, device="cpu")
    out, errors = [None, None], []

    def work(s):
        try:
            out[s] = serve(r, s, 9 * s)
        except Exception as e:  # noqa: BLE001
            errors.append(e)
    threads = [threading.Thread(target=work, args=(s,)) for s in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    assert np.array_equal(out[0], alone[0]) and np.array_equal(out[1], alone[1])
    assert sorted(r.length) == [(0, 0), (0, 2), (1, 0), (1, 2)] and len(r.pool.free) == 4


def test_runner_keeps_few_graphs(paged_cpu, monkeypatch):
    """Passes of ever other row counts: the graphs kept are bounded, the last used stay,
    one workspace serves all, and a pass over a graph built again gives the same words."""
    m = WL.LlamaModel(batch=1, seq=16, cache=32, seed=4, **SMALL)
    r = PagedLlamaRunner(m, pages=2, page=16, device="cpu")
    monkeypatch.setattr(PagedLlamaRunner, "GRAPHS", 5, raising=False)
    want = {}
    for n in list(range(1, 13)) + [1, 12, 3]:
        got = r.append("a", [list(range(1, n + 1))])[:m.vocab].clone()
        assert torch.equal(want.setdefault(n, got), got)
        r.release("a")
        assert len(r._sims) <= 5 and (n, False) in r._sims and (1, True) in r._sims
        assert all(s._ws is None for s in r._sims.values())
    assert list(r._sims)[-2:] == [(3, False), (1, True)]
    assert 1 < PagedLlamaRunner(m, pages=2, page=16, device="cpu").GRAPHS


@gpu
@pytest.mark.parametrize("dims,lengths,page", [
    (dict(layers=2, hidden=64, heads=4, kv_heads=2, head_dim=16, ffn=128, vocab=300), (9, 3, 70, 40), 16),
    (dict(layers=2, hidden=960, heads=15, kv_heads=5, head_dim=64, ffn=256, vocab=500), (33, 100, 61, 90), 64),
    (dict(layers=1, hidden=512, heads=4, kv_heads=4, head_dim=128, ffn=256, vocab=300), (5, 130, 40, 60), 32)],
    ids=["hd16", "hd64", "hd128"])
def test_gpu_runner_is_the_contiguous_model(dims, lengths, page):
    from cormorant_b200 import ops
    dims = dict(dims, seed=6)
    _, seen = _served(dims, None, lengths, 3, 160, page, chunk=33)
    want = _contiguous(dims, 160, [t for t, _ in seen], None)
    for (t, got), w in zip(seen, want):
        assert np.array_equal(got, w), len(t)
    assert ops.device_status() == 0


@gpu
def test_gpu_runner_8_bit_pages():
    """8-bit pages: a token's words do not depend on the cut into passes."""
    dims = dict(layers=2, hidden=256, heads=8, kv_heads=2, head_dim=32, ffn=256, vocab=200, seed=8)
    m = WL.LlamaModel(batch=1, seq=64, **dims)
    rng = np.random.default_rng(3)
    ids = rng.integers(0, 200, 40).tolist()
    got = []
    for cuts in ([40], [1] * 40, [7, 30, 1, 2]):
        r = PagedLlamaRunner(m, pages=6, page=16, bits=8)
        at = 0
        for i, c in enumerate(cuts):
            if i == 1:  # company
                r.append("x", [ids[:9]])
            lg = r.append("a", [ids[at:at + c]])
            at += c
        got.append(_words(lg, 1, 200))
    assert np.array_equal(got[0], got[1]) and np.array_equal(got[0], got[2])


@gpu
def test_gpu_runner_generate():
    """Greedy tokens of several prompts at once are those of each alone."""
    dims = dict(layers=2, hidden=960, heads=15, kv_heads=5, head_dim=64, ffn=256, vocab=500, seed=2)
    m = WL.LlamaModel(batch=1, seq=64, **dims)
    rng = np.random.default_rng(5)
    prompts = {s: rng.integers(0, 500, n).tolist() for s, n in (("p", 17), ("q", 1), ("r", 45))}
    r = PagedLlamaRunner(m, pages=8, page=64)
    both = r.generate(prompts, 5)
    for s, p in prompts.items():
        assert PagedLlamaRunner(m, pages=2, page=64).generate({s: p}, 5)[s] == both[s]


@gpu
def test_gpu_runner_on_streams():
    """A runner's passes on one stream after another, nothing waited for between them,
    and from two threads on two streams: the words of one stream's."""
    import threading
    dims = dict(layers=2, hidden=960, heads=15, kv_heads=5, head_dim=64, ffn=256, vocab=500, seed=2)
    m = WL.LlamaModel(batch=1, seq=64, **dims)
    prompts = {s: np.random.default_rng(s).integers(0, 500, 5 + 9 * s).tolist() for s in range(4)}
    want = {s: PagedLlamaRunner(m, pages=2, page=64).generate({s: p}, 6)[s] for s, p in prompts.items()}
    r = PagedLlamaRunner(m, pages=8, page=64)
    streams = [torch.cuda.Stream() for _ in range(3)]
    ids = torch.empty((6, 4), dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.stream(streams[0]):
        lg = r.append(list(prompts), list(prompts.values()))
    for i in range(6):
        with torch.cuda.stream(streams[(i + 1) % 3]):
            lg = r.step(list(prompts), lg, ids[i])
    torch.cuda.synchronize()
    assert ids.cpu().numpy().T.tolist() == [want[s] for s in prompts]
    for s in prompts:
        r.release(s)
    got = {}

    def work(mine):
        with torch.cuda.stream(torch.cuda.Stream()):
            for s in mine:
                got.update(r.generate({s: prompts[s]}, 6))
    threads = [threading.Thread(target=work, args=(t,)) for t in ((0, 2), (1, 3))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert got == want
