"""What ops.greedy_embed refuses before it launches anything (CPU: the checks come
before the device is looked at)."""
import pytest

torch = pytest.importorskip("torch")


def test_greedy_embed_refuses():
    """Arrays that do not hold what the launch reads or writes, on the host: too few
    logits rows, a short ids, out or table, a slice of a longer one, other types."""
    from cormorant_b200 import ops
    from cormorant_b200._lib import CormError
    B, V, D = 3, 10, 4
    i16 = lambda *s: torch.zeros(s, dtype=torch.int16)  # noqa: E731
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    ok = dict(logits=i16(B * V), table=i32(V, D), out=i32(B * D), ids=i32(B))
    for bad in (dict(logits=i16(2, V)), dict(logits=i16(6 * V)[:2 * V]), dict(logits=i16(B * V).float()),
                dict(logits=i16(B, 2 * V)[:, ::2]), dict(table=i32(V - 1, D)), dict(table=i32(V, D).long()),
                dict(out=i32(B * D - 1)), dict(out=i32(2 * B * D)[:2 * D]), dict(out=i32(B, 2 * D)[:, :D]),
                dict(ids=i32(B - 1)), dict(ids=i32(B)[:2]), dict(ids=i32(2 * B)[::2]), dict(ids=i32(B).long())):
        with pytest.raises(CormError, match=next(iter(bad))):
            a = dict(ok, **bad)
            ops.greedy_embed(a["logits"], a["table"], a["out"], a["ids"], batch=B, vocab=V, dim=D)
    with pytest.raises(CormError, match="logits"):
        ops.greedy_embed(ok["logits"], ok["table"], ok["out"], ok["ids"], batch=B, vocab=V, dim=D, ld=V + 1)
    with pytest.raises(CormError, match="CUDA"):  # all as it should be, but not on a device
        ops.greedy_embed(ok["logits"], ok["table"], ok["out"], ok["ids"], batch=B, vocab=V, dim=D)
