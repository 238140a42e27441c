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


def test_no_file_is_compiled_with_packed_fp32_arithmetic(tmp_path):
    """every source of the libraries takes the flag, and what the compiler makes of the two files with hand-counted register budgets, which
    once went without, has none"""
    import re
    import shutil
    import subprocess
    from animal2vec_amd import build as B
    for s in B.SOURCES:
        assert "-packed-fp32-ops" in [*B.FLAGS, *B.FILE_FLAGS.get(s, [])], s
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not os.path.exists(hipcc):
        pytest.skip("hipcc not available")
    for src in ("a2v_gemm_p8.hip", "a2v_conv_dec.hip"):
        out = tmp_path / (src + ".s")
        subprocess.run([hipcc, *B.FLAGS, *B.FILE_FLAGS.get(src, []), "-S", "--cuda-device-only", os.path.join(B.CSRC, src), "-o", str(out)], check=True, capture_output=True)
        found = re.findall(r"\bv_pk_(?:add|mul|fma)_f32\b", out.read_text())
        assert not found, (src, len(found))
