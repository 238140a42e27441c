"""What the compiler makes of the linear attention kernels, where their correctness or their speed rests on it (no GPU needed)."""
import os
import re
import shutil
import subprocess

import pytest


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    """-> {(type, channels, heads of a workgroup, state pass): instructions}, what the compiler said"""
    from animal2vec_amd import build as B
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not os.path.exists(hipcc):
        pytest.skip("hipcc not available")
    src, out = "a2v_linattn.hip", tmp_path_factory.mktemp("isa") / "linattn.s"
    r = subprocess.run([hipcc, *B.FLAGS, *B.FILE_FLAGS.get(src, []), "-S", "--cuda-device-only", os.path.join(B.CSRC, src), "-o", str(out)], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-2000:]
    s, found = out.read_text(), {}
    for m in re.finditer(r"^_Z10lin_kernelI(DF16b|f)Li(\d+)ELi(\d+)ELb([01])EEv7LinArgs:", s, re.M):
        body = s[m.end():s.index(".amdhsa_kernel", m.end())]
        lines = [x.split(";")[0].strip() for x in body.split("\n")]
        found[m[1], int(m[2]), int(m[3]), m[4] == "1"] = [x for x in lines if x and not x.startswith(".") or x.startswith(".LBB")]
    assert len(found) == 16
    return found, r.stderr


def chunk_loop(lines):
    """the lines of the loop over chunks, wherever the compiler has put them: what a barrier can reach and come back from"""
    at = {x[:-1]: i for i, x in enumerate(lines) if x.startswith(".LBB")}
    edges = []
    for i, x in enumerate(lines):
        m = re.match(r"s_(c?)branch\w* (\.LBB\w+)", x)
        if m:
            edges.append((i, at[m[2]]))
        if (not m or m[1]) and x != "s_endpgm" and i + 1 < len(lines):
            edges.append((i, i + 1))

    def reach(start, pairs):
        to = {}
        for u, v in pairs:
            to.setdefault(u, []).append(v)
        seen, todo = set(), list(to.get(start, ()))
        while todo:
            i = todo.pop()
            if i not in seen:
                seen.add(i)
                todo += to.get(i, ())
        return seen
    for i, x in enumerate(lines):
        if x == "s_barrier":
            inside = reach(i, edges) & reach(i, [(v, u) for u, v in edges])
            if i in inside:
                return [lines[j] for j in sorted(inside)]
    raise AssertionError("no loop with a barrier")


def test_m0_is_the_loads_own(kernels):
    found, said = kernels
    assert "reserved registers" not in said
    for key, lines in found.items():
        loads = [i for i, x in enumerate(lines) if x.startswith("global_load_lds_dwordx4")]
        assert bool(loads) == (key[0] == "DF16b"), key
        for i in loads:
            assert lines[i - 2].startswith("s_mov_b32 m0, s") and lines[i - 1] == "s_nop 0", (key, lines[i - 2:i + 1])
        assert sum(bool(re.search(r"\bm0\b", x)) for x in lines) == len(loads), key


def test_no_register_is_spilled_inside_the_chunk_loop(kernels):
    for key, lines in kernels[0].items():
        loop = chunk_loop(lines)
        assert sum(x.startswith("v_mfma") for x in loop) >= 4, key
        assert not [x for x in loop if x.startswith("scratch_")], key


def test_a_chunk_waits_for_its_loads_by_a_count_that_the_next_rows_cover(kernels):
    """A chunk's loads are issued in the chunk in front of it, whose stored rows are younger: vmcnt(1) is right as long as one store is issued behind the
    last of the loads, and useful as long as nothing else in the loop waits for memory.  (vmcnt(0), the other wait written into the source, is
    for a segment's first chunk and for 32-bit rows.)"""
    for key, lines in kernels[0].items():
        if key[0] != "DF16b":
            continue
        loop = chunk_loop(lines)
        waits = [x for x in loop if re.match(r"s_waitcnt.*vmcnt", x)]
        loads = [i for i, x in enumerate(loop) if x.startswith("global_load_lds_dwordx4")]
        stores = [i for i, x in enumerate(loop) if re.match(r"global_store_dwordx4 .* nt$", x)]
        if key[3]:
            assert len(loads) == 2 and not stores and waits == ["s_waitcnt vmcnt(0)"], (key, waits)
        else:
            assert len(loads) == 3 and len(stores) == 1 and stores[0] > loads[-1], key
            assert sorted(waits) == ["s_waitcnt vmcnt(0)", "s_waitcnt vmcnt(1)"], (key, waits)
            other = [x for x in loop if re.match(r"(global|flat|buffer)_(load|store|atomic)", x) and "lds" not in x and not x.endswith(" nt")]
            assert all(x.startswith("global_store_dwordx4") for x in other) and len(other) <= 2, (key, other)          # (32-bit rows)
