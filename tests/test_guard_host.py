"""The guard-page harness (tests/guard) without a GPU: where the allocator puts a tensor between its unmapped pages, and that no GPU test reads
outside of one."""
import ctypes
import os
import re

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
