"""The guard-page harness (tests/guard) without a GPU: where the allocator puts a tensor between its unmapped pages, that no GPU test reads
outside of one, and that nothing runs behind a fault."""
import ctypes
import os
import re
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


class Place(ctypes.Structure):
    _fields_ = [(n, ctypes.c_uint64) for n in ("reserved", "mapped_at", "mapped", "tensor_at")]


@pytest.fixture(scope="module")
def place():
    import __graft_entry__
    f = ctypes.CDLL(__graft_entry__.build_guard()).dpig_guard_place
    f.argtypes, f.restype = [ctypes.c_uint64, ctypes.c_uint64, ctypes.c_int, ctypes.POINTER(Place)], None

    def call(size, granularity, at_start):
        p = Place()
        f(size, granularity, at_start, ctypes.byref(p))
        return p
    return call


@pytest.mark.parametrize("granularity", [4096, 65536, 2 << 20])
@pytest.mark.parametrize("size", [0, 1, 15, 16, 17, 4095, 4096, 4097, (2 << 20) - 16, 2 << 20, (2 << 20) + 1, 3 * 10 ** 9 + 7])
def test_a_tensor_ends_or_starts_at_an_unmapped_page(place, size, granularity):
    """'hi': the 16-byte piece behind the tensor's last one is the first of the unmapped granule; 'lo': the byte before it the last of one."""
    pieces = (max(size, 1) + 15) // 16 * 16
    for at_start in (0, 1):
        p = place(size, granularity, at_start)
        end = p.mapped_at + p.mapped
        assert p.mapped_at % granularity == 0 and p.mapped % granularity == 0 and pieces <= p.mapped < pieces + granularity
        assert p.mapped_at >= granularity and p.reserved - end >= granularity                     # a granule on each side is never mapped
        assert p.mapped_at <= p.tensor_at and p.tensor_at + max(size, 1) <= end and p.tensor_at % 16 == 0
        assert p.tensor_at == p.mapped_at if at_start else p.tensor_at + pieces == end


def test_no_gpu_test_copies_from_behind_a_guarded_tensor():
    """The harness' own GPU test reads inside its 4096-byte tensor only."""
    text = open(os.path.join(ROOT, "tests", "test_guard_gpu.py")).read()
    offsets = re.findall(r'"-c", code, str\(([^)]*)\)', text)
    assert offsets and all(0 <= eval(o) <= 4096 - 16 for o in offsets), offsets


def test_a_sweep_ends_with_its_first_faulting_case(monkeypatch):
    sys.path.insert(0, os.path.join(ROOT, "tests"))
    import test_guard_gpu as G
    runs = []

    def dies(cmd, **kw):
        runs.append(cmd)
        assert len(runs) == 1, "started again behind a fault"
        return subprocess.CompletedProcess(cmd, -6, stdout="CASE 0 a\nOK 0 a\nCASE 1 b\nERR 1 b: x\nCASE 2 c\n", stderr="Memory access fault\n")
    monkeypatch.setattr(G.subprocess, "run", dies)
    faults, errs, total = G.sweep("hi")
    assert len(faults) == 1 and faults[0].startswith("2 c [rc -6] Memory access fault") and errs == ["ERR 1 b: x"] and total is None


@pytest.mark.parametrize("status,ran", [(0, 3), (5, 3), (1, 2), (134, 2), (124, 2)])
def test_the_suite_on_guard_pages_stops_at_the_first_failing_file(tmp_path, status, ran):
    """The second of three files ends with `status` (5: nothing selected); a stand-in for python counts the calls."""
    fake = tmp_path / "python"
    fake.write_text("#!/bin/sh\necho run >> %s/calls\n[ $(wc -l < %s/calls) -eq 2 ] && exit %d\nexit 0\n" % (tmp_path, tmp_path, status))
    fake.chmod(0o755)
    env = dict(os.environ, PATH="%s:%s" % (tmp_path, os.environ["PATH"]), GRAFT_REPO_ROOT=str(tmp_path))
    r = subprocess.run(["bash", os.path.join(ROOT, "scripts", "guard_suite.sh"), "hi", "a.py", "b.py", "c.py"], env=env, capture_output=True, text=True)
    assert len((tmp_path / "calls").read_text().split()) == ran, r.stdout + r.stderr
    assert r.returncode == (0 if status in (0, 5) else status)


def test_no_script_is_there_to_bring_a_fault_out():
    """Programs that load the GPU without torch's caching allocator, so that a stray access leaves mapped memory, are the guard-page tests alone."""
    held = [f for f in os.listdir(os.path.join(ROOT, "scripts")) if f.endswith((".py", ".sh"))
            and "NO_CUDA_MEMORY_CACHING" in open(os.path.join(ROOT, "scripts", f)).read()]
    assert not held
