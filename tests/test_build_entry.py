"""The build entry point compiles what is there already as well (no GPU needed)."""
import subprocess

import __graft_entry__


def test_build_does_not_trust_what_looks_up_to_date(monkeypatch):
    calls = []
    monkeypatch.setattr(subprocess, "check_call", lambda cmd, **kw: calls.append(cmd))
    __graft_entry__.build()
    folders = [c[c.index("-C") + 1].replace("\\", "/") for c in calls]
    assert any(f.endswith("isaacgym_amd/csrc") for f in folders) and len(folders) == 3
    assert all(c[0] == "make" and "-B" in c for c in calls)
