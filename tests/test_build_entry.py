"""The build entry point compiles every source on every call."""
import glob
import os
import subprocess

from conftest import PKG


def test_build_compiles_every_source_whatever_is_built(monkeypatch):
    import __graft_entry__ as entry
    calls = []
    monkeypatch.setattr(entry.subprocess, "check_call", calls.append)
    try:
        entry.build()
    except RuntimeError:   # no library here yet
        pass
    assert len(calls) == 1
    # the same make, told to say what it would do
    said = subprocess.run(calls[0] + ["-n"], capture_output=True, text=True, check=True).stdout
    sources = [os.path.basename(f) for f in glob.glob(os.path.join(PKG, "csrc", "*.hip"))]
    assert sources and all(f" -c {f} " in said for f in sources) and "-shared" in said
