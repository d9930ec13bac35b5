"""CPU tests of the 4-bit cache's size query: arguments that the call refuses have no size,
and end nothing."""
import subprocess
import sys

ODD = [(2, 1, 2, 2, 8192, 64), (2, 1, 2, 2, 5000, 0), (2, 1, 2, 2, 4097, 1 << 20), (2, 1, 2, 2, 96, 64), (2, 1, 3, 2, 64, 64),
       (1 << 62, 1, 2, 2, 64, 64), (2, 1 << 62, 2, 2, 64, 64), (2, 1, 1 << 62, 1, 64, 64), (2, 1, 2, 1 << 62, 64, 64),
       (2, 65, 2, 2, 64, 64), (70000, 1, 2, 2, 64, 64), (2, 1, 2, 2, 64, 1 << 62), (65535, 64, 512, 2, 64, 64),
       (2, 1, 2, 2, 1 << 62, 64), (2, 1, 2, 2, -64, 64), (0, 0, 0, 0, 0, 0)]


CHILD = """
import ctypes, sys
size = ctypes.CDLL(sys.argv[1]).mom_decode_attn_int4_workspace_size
size.restype, size.argtypes = ctypes.c_size_t, [ctypes.c_int64] * 6
for args in eval(sys.argv[2]):
    print(size(*args), flush=True)
"""


def test_no_size_for_what_is_refused():
    """In a process of its own: a division by zero would end it."""
    from naylis_b200 import build
    r = subprocess.run([sys.executable, "-c", CHILD, build.build(), repr(ODD)], capture_output=True, text=True, timeout=300)
    assert r.stdout.split() == ["0"] * len(ODD) and r.returncode == 0, (r.returncode, r.stdout.split(), r.stderr[-300:])
