"""The build entry point compiles every source each time, also where built libraries are up to date by their times."""
import subprocess


def test_build_compiles_whatever_is_there(monkeypatch):
    import __graft_entry__
    calls = []
    monkeypatch.setattr(subprocess, "run", lambda args, **kw: calls.append((list(args), kw)))
    __graft_entry__.build()
    (args, kw), = calls
    assert args[0] == "make" and "-B" in args and kw.get("check") is True
