"""CPU: the order of build()'s steps."""
import subprocess

import pytest

import __graft_entry__ as entry


def test_the_torch_side_is_built_last(monkeypatch):
    """Torch's headers and libraries are needed by the policy operators' torch side alone: where they are missing, the library of the
    C-ABI, the go_game module and the oracle are there all the same."""
    done = []

    class Compiler:
        returncode = 0

        def __init__(self, cmd, cwd):
            done.append("compile")

        def wait(self):
            return 0

    def torch_side():
        raise ImportError("torch")
    monkeypatch.setattr(subprocess, "Popen", Compiler)
    monkeypatch.setattr(entry, "_run", lambda cmd: done.append("oracle" if cmd[0] == "make" else "link"))
    monkeypatch.setattr(entry, "build_go_game", lambda: done.append("go_game"))
    monkeypatch.setattr(entry, "build_policy_ops", torch_side)
    with pytest.raises(ImportError, match="torch"):
        entry.build()
    assert done == ["compile"] * len(entry.HIP_SOURCES) + ["link", "go_game", "oracle"]
