"""build.py decides what is out of date: sources, headers and the flags that a built file was made with (no compiler needed)."""
import os
import stat

import pytest


@pytest.fixture
def build(tmp_path, monkeypatch):
    from animal2vec_amd import build as B
    fake = tmp_path / "hipcc"
    fake.write_text(f'#!/bin/sh\necho "$@" >> {tmp_path}/log\nwhile [ "$1" != "-o" ]; do shift; done\n: > "$2"\n')
    fake.chmod(fake.stat().st_mode | stat.S_IXUSR)
    src = tmp_path / "csrc"
    src.mkdir()
    for f in ("one.hip", "two.hip", "common.h"):
        (src / f).write_text("")
        os.utime(src / f, (1, 1))
    monkeypatch.setenv("HIPCC", str(fake))
    for name, value in dict(HERE=str(tmp_path), CSRC=str(src), OBJ=str(src / "build"), LIB=str(tmp_path / "lib.so"), SOURCES=["one.hip", "two.hip"],
                            HEADERS=[str(src / "common.h")], FILE_FLAGS={"two.hip": ["-two"]}).items():
        monkeypatch.setattr(B, name, value, raising=False)

    def ran(go):
        log = tmp_path / "log"
        log.write_text("")
        go()
        return [os.path.basename(line.split(" -c ")[1].split(" ")[0]) if " -c " in line else "link" for line in log.read_text().splitlines()]
    return B, src, ran


def test_flags_are_part_of_what_a_file_depends_on(build, monkeypatch):
    B, src, ran = build
    go = lambda **kw: ran(lambda: B.build(verbose=False, **kw))          # noqa: E731
    assert sorted(go()) == ["link", "link", "one.hip", "one.hip", "two.hip", "two.hip"]          # both libraries
    assert go() == []
    monkeypatch.setattr(B, "FILE_FLAGS", {"two.hip": ["-other"]})
    assert sorted(go()) == ["link", "link", "two.hip", "two.hip"] and go() == []
    monkeypatch.setattr(B, "FLAGS", [*B.FLAGS, "-DX"])
    assert sorted(go()) == ["link", "link", "one.hip", "one.hip", "two.hip", "two.hip"] and go() == []
    os.utime(src / "common.h", (2e9, 2e9))
    assert len(go()) == 6
    os.utime(src / "common.h", (1, 1))
    assert go() == [] and len(go(force=True)) == 6


def test_a_file_without_a_record_of_its_flags_is_built_again(build):
    B, src, ran = build
    ran(lambda: B.build(verbose=False))
    os.remove(src / "build" / "one.o.cmd")
    assert ran(lambda: B.build(verbose=False)) == ["one.hip", "link"]
