"""_binding.so is rebuilt when its source, the header or the torch that it was built against is newer."""
import os

import pytest

from tokenrush_b200 import build


@pytest.mark.parametrize("newer", ["nothing", "binding.cpp", "trb_kv.h", "version.py"])
def test_out_of_date(monkeypatch, tmp_path, newer):
    sources = []
    for real in build.binding_sources():
        assert os.path.exists(real)
        p = tmp_path / os.path.basename(real)
        p.write_text("")
        os.utime(p, (3000, 3000) if p.name == newer else (1000, 1000))
        sources.append(str(p))
    so = tmp_path / "_binding.so"
    so.write_text("")
    os.utime(so, (2000, 2000))
    ran = []

    class Done:
        returncode = 0
    monkeypatch.setattr(build, "BINDING", str(so))
    monkeypatch.setattr(build, "binding_sources", lambda: sources)
    monkeypatch.setattr(build.subprocess, "run", lambda cmd, **kw: ran.append(cmd) or Done)
    assert build.build_binding() == str(so)
    assert len(ran) == (newer != "nothing")


def test_torch_is_a_source():
    import torch
    assert os.path.join(os.path.dirname(torch.__file__), "version.py") in build.binding_sources()
