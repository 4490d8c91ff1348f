"""The C++ binding is tied to the torch and the Python that it was built against."""
import os

import pytest
import torch

from longcat_video_b200 import _lib as L
from longcat_video_b200 import build


def test_another_torch_gets_a_binding_of_its_own(monkeypatch):
    L.binding()
    here = L.binding_path()
    assert os.path.exists(here)
    commands = []

    def run(cmd, **kw):
        commands.append(cmd)
        return type("Done", (), dict(returncode=0, stdout="", stderr=""))()
    monkeypatch.setattr(build.subprocess, "run", run)
    build._build_binding(False)
    assert commands == []  # it is there and newer than its sources
    monkeypatch.setattr(torch, "__version__", "99.0")
    monkeypatch.setattr(L, "_binding", None)
    assert L.binding_path() != here
    with pytest.raises(RuntimeError, match="build it with"):
        L.binding()
    build._build_binding(False)
    assert len(commands) == 1 and L.binding_path() in commands[0]
