"""mgnet_amd.build: what makes an object or the library stale.  No compiler runs: a script in its place writes down its command and the output."""
import os
import stat

import pytest


@pytest.fixture
def tree(tmp_path, monkeypatch):
    from mgnet_amd import build
    src = tmp_path / "csrc"
    src.mkdir()
    (tmp_path / "include").mkdir()
    for name in ("a.hip", "a_f16.hip", "b.hip"):
        (src / name).write_text("//\n")
    (src / "h.h").write_text("//\n")
    flags = tmp_path / "build.py"
    flags.write_text("#\n")
    cc = tmp_path / "cc"
    cc.write_text('#!/bin/sh\necho "$@" >> %s\nwhile [ $# -gt 1 ]; do if [ "$1" = -o ]; then echo x > "$2"; fi; shift; done\n' % (tmp_path / "log"))
    cc.chmod(cc.stat().st_mode | stat.S_IXUSR)
    for k, v in dict(HERE=tmp_path, ROOT=tmp_path, LIB=tmp_path / "lib" / "lib.so", OBJ=tmp_path / "lib" / "obj", HIPCC=cc, SELF=flags).items():
        monkeypatch.setattr(build, k, str(v), raising=False)

    def run(**kw):
        (tmp_path / "log").write_text("")
        build.build(**kw)
        return sorted(w.split("/")[-1] for line in (tmp_path / "log").read_text().splitlines() for w in line.split() if w.endswith(".hip"))

    def touch(name):
        t = max(os.path.getmtime(p) for p in tmp_path.rglob("*")) + 10
        os.utime(tmp_path / name, (t, t))
        for p in (tmp_path / "lib").rglob("*"):      # (built earlier than that, whatever the clock)
            if p.is_file():
                os.utime(p, (t - 5, t - 5))
    return run, touch


def test_objects_follow_their_sources(tree):
    run, touch = tree
    assert run() == ["a.hip", "a_f16.hip", "b.hip"] and run() == []
    touch("csrc/b.hip")
    assert run() == ["b.hip"]
    touch("csrc/a.hip")
    assert run() == ["a.hip", "a_f16.hip"]


def test_changed_flags_make_everything_stale(tree):
    run, touch = tree
    run()
    touch("build.py")
    assert run() == ["a.hip", "a_f16.hip", "b.hip"]


def test_forced(tree):
    run, _ = tree
    run()
    assert run(force=True) == ["a.hip", "a_f16.hip", "b.hip"]


def test_the_entry_point_compiles_each_time(monkeypatch):
    import __graft_entry__ as g
    from mgnet_amd import build
    calls = []
    monkeypatch.setattr(build, "build", lambda **kw: calls.append(kw))
    g.build()
    g.build()
    assert [kw.get("force") for kw in calls] == [True, True]


def test_a_variant_is_built_with_the_librarys_flags(tmp_path):
    """tools/build_variant.sh compiles one source by itself: with the flags that every object of the library has"""
    import subprocess

    from conftest import ROOT
    from mgnet_amd import build
    (tmp_path / "tools").mkdir()
    (tmp_path / "tools" / "build_variant.sh").write_text(open(os.path.join(ROOT, "tools", "build_variant.sh")).read())
    for name in ("mgnet_amd", "include"):
        os.symlink(os.path.join(ROOT, name), tmp_path / name)
    cc = tmp_path / "cc"
    cc.write_text('#!/bin/sh\necho "$@" >> %s\n' % (tmp_path / "log"))
    cc.chmod(cc.stat().st_mode | stat.S_IXUSR)
    subprocess.run(["bash", str(tmp_path / "tools" / "build_variant.sh"), "x", "q8.hip", "-DX"], check=True, env=dict(os.environ, HIPCC=str(cc)), stdout=subprocess.DEVNULL)
    lines = [line.split() for line in open(tmp_path / "log") if " -c " in line]
    assert lines and all("-DX" in line for line in lines)
    for line in lines:
        k = line.index("-packed-fp32-ops")
        assert line[k - 3:k + 1] == ["-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]
        assert [f for f in build.CFLAGS if f.startswith("-O") or f.startswith("-std")] == [f for f in line if f.startswith("-O") or f.startswith("-std")]
