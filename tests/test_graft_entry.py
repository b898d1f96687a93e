"""build(): the reference's C oracle is made only where the reference has its source."""
import os
import subprocess

import pytest


@pytest.mark.parametrize("there", [False, True], ids=["without", "with"])
def test_build_makes_the_oracle_where_its_source_is(monkeypatch, there):
    import __graft_entry__ as entry
    from cormorant_b200 import build as b
    exists, made = os.path.exists, []
    monkeypatch.setattr(b, "build", lambda **kw: None)
    monkeypatch.setattr(os.path, "exists", lambda p: there if str(p).endswith("rowops_ref.h") else exists(p))
    monkeypatch.setattr(os.path, "isdir", lambda p: True)
    monkeypatch.setattr(subprocess, "run", lambda a, **kw: made.append(a))
    entry.build()
    assert bool(made) is there
