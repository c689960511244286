"""What makes the extension's build compile again, with the compiler stubbed."""

import os

import pytest

from simumax_amd.kernels import build as B


@pytest.fixture
def tree(tmp_path, monkeypatch):
    """A build in its own folder; returns what each build compiled."""
    csrc = tmp_path / "csrc"
    csrc.mkdir()
    for name in B.KERNEL_SOURCES + B.HEADERS + ["wgrad.cpp", "binding.cpp"]:
        (csrc / name).write_text("")
        os.utime(csrc / name, (1000, 1000))
    for name, path in list(vars(B).items()):
        # all that the module keeps beside itself
        if isinstance(path, str) and path.startswith(B.HERE + os.sep):
            monkeypatch.setattr(B, name, str(
                tmp_path / os.path.relpath(path, B.HERE)))
    monkeypatch.setattr(B, "HERE", str(tmp_path))
    done = []

    def run(cmd, check):
        out = cmd[cmd.index("-o") + 1]
        if fail and out.endswith(fail[0]):
            raise RuntimeError("compiler")
        open(out, "w").close()
        done.append(os.path.basename(out))

    fail = []
    monkeypatch.setattr(B.subprocess, "run", run)

    def build(fails_at=None):
        done.clear()
        fail[:] = [fails_at] if fails_at else []
        try:
            B.build(verbose=False)
        except RuntimeError:
            assert fails_at
        return sorted(done)

    build.csrc = csrc
    return build


EVERYTHING = sorted([f"{s}.o" for s in B.KERNEL_SOURCES if os.path.exists(
    os.path.join(B.CSRC, s))] + ["binding.cpp.o", "wgrad.cpp.o",
                                 "simumax_hip.so"])


def test_only_what_changed_is_compiled(tree, monkeypatch):
    monkeypatch.setattr(B, "KERNEL_SOURCES", [
        s for s in B.KERNEL_SOURCES if f"{s}.o" in EVERYTHING])
    assert tree() == EVERYTHING
    assert tree() == []
    later = os.path.getmtime(B.OUT) + 100
    os.utime(tree.csrc / "rope.hip", (later, later))
    assert "rope.hip.o" in tree()


def test_other_flags_compile_everything(tree, monkeypatch):
    monkeypatch.setattr(B, "KERNEL_SOURCES", [
        s for s in B.KERNEL_SOURCES if f"{s}.o" in EVERYTHING])
    assert tree() == EVERYTHING
    first = B.ARCH
    monkeypatch.setattr(B, "ARCH", "gfx950:sramecc+")
    assert tree() == EVERYTHING
    assert tree() == []
    # a build that fails half-way leaves objects of other flags behind
    monkeypatch.setattr(B, "ARCH", first)
    assert tree(fails_at="binding.cpp.o") != EVERYTHING
    monkeypatch.setattr(B, "ARCH", "gfx950:sramecc+")
    assert tree() == EVERYTHING
