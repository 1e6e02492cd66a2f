"""The autograd extension is built again when torch has been exchanged, not by file times alone."""
import types


def test_another_torch_builds_again(tmp_path, monkeypatch):
    from cafe_b200 import build
    calls = []

    def run(cmd, **kw):
        calls.append(cmd)
        so.write_bytes(b"")
        return types.SimpleNamespace(returncode=0, stdout="")
    so = tmp_path / "_dense_torch.so"
    monkeypatch.setattr(build, "TORCH_SO", so)
    monkeypatch.setattr(build, "TORCH_RECORD", tmp_path / "build" / "record")
    monkeypatch.setattr(build.subprocess, "run", run)
    build.build_torch()
    assert len(calls) == 1
    build.build_torch()
    assert len(calls) == 1                       # nothing has changed
    build.TORCH_RECORD.write_text("torch 1.0, python 2")
    build.build_torch()
    assert len(calls) == 2                       # built for another torch
    build.TORCH_RECORD.unlink()
    build.build_torch()
    build.build_torch()
    assert len(calls) == 3                       # by a build that kept no record
