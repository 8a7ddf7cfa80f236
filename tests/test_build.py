"""The build: every source is compiled again when its flags change, and whenever build() is called."""

import subprocess
from pathlib import Path

import __graft_entry__

CSRC = Path(__graft_entry__.PKG) / "csrc"


def _compiled(*args):
    out = subprocess.run(["make", "-C", str(CSRC), "-n", *args], check=True, capture_output=True, text=True).stdout
    return {name for name in (p.name for p in CSRC.iterdir()) if f" -c {name} -o " in out}


def test_a_changed_makefile_compiles_every_source():
    """Its flags keep packed float32 instructions out of the kernels: an object of other flags must not stay."""
    sources = {p.name for p in CSRC.glob("*.hip")} | {p.name for p in CSRC.glob("*.cpp")}
    assert len(sources) > 10 and _compiled("-W", "Makefile") == sources


def test_build_compiles_what_is_there_already(monkeypatch):
    commands = []
    monkeypatch.setattr(__graft_entry__.subprocess, "run", lambda command, **kw: commands.append(command))
    __graft_entry__.build()
    (command,) = commands
    sources = {p.name for p in CSRC.glob("*.hip")} | {p.name for p in CSRC.glob("*.cpp")}
    monkeypatch.undo()
    assert command[0] == "make" and _compiled(*(a for a in command[1:] if a == "-B")) == sources
