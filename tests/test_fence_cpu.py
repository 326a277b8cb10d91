"""The electric-fence allocator's arithmetic on the host (no GPU): the tensor's end (mode left: its start) is the mapping's, whole granules
are mapped and a granule on either side is not.  The control of tests/test_fence_gpu.py rests on this and makes no access outside."""
import ctypes
import os
import random
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "tools"))


@pytest.fixture(scope="module")
def inside():
    import guarded
    if not os.path.exists("/opt/rocm/bin/hipcc") and not os.path.exists(guarded.LIB):
        pytest.skip("hipcc not found")
    f = ctypes.CDLL(guarded.build()).ea_guard_inside
    f.argtypes = [ctypes.c_longlong, ctypes.c_longlong, ctypes.c_int, ctypes.c_longlong, ctypes.c_longlong, ctypes.c_void_p]
    return f


def test_layout_and_border(inside):
    rng = random.Random(3)
    for user in [1, 16, 4096, 4097, (1 << 20) + 64, 1 << 21] + [rng.randint(1, 1 << 30) for _ in range(100)]:
        for gran in (4096, 65536, 1 << 21):
            for right in (0, 1):
                out = (ctypes.c_longlong * 4)()
                inside(user, gran, right, 0, 1, out)
                total, start, mapped, tensor = out
                assert mapped % gran == 0 and user <= mapped < user + gran
                assert start == gran and total == start + mapped + gran                    # one granule without pages on either side
                whole = (user + 15) // 16 * 16
                assert tensor == (start + mapped - whole if right else start) and tensor % 16 == 0
                assert inside(user, gran, right, 0, user, None) == 1                       # the tensor itself
                if right:                                                                  # behind it, 16-byte pieces on: nothing
                    assert [inside(user, gran, 1, whole + d, 4, None) for d in (-4, -3, 0, 4096)] == [1, 0, 0, 0]
                else:
                    assert [inside(user, gran, 0, d, 4, None) for d in (0, -1, -4, -4096)] == [1, 0, 0, 0]


def test_the_tree_holds_no_deliberate_fault():
    """The allocator and its launcher contain no device code at all: what is outside a mapping is reported, not touched."""
    tools = os.path.join(ROOT, "tools")
    text = open(os.path.join(tools, "guard_alloc", "ea_guard_alloc.cpp")).read() + open(os.path.join(tools, "guarded.py")).read()
    assert "__global__" not in text and "hipLaunchKernel" not in text and "<<<" not in text
    assert not os.path.exists(os.path.join(tools, "fault_hunt.sh"))
