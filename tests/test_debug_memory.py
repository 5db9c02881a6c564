"""The debug library reads what a call names, not whole page tables: 12288 streams of 2^20 pages are 51 GB, and an exception for
want of memory would end the process at the C entry. Without a GPU the reading itself is what fails."""
import subprocess
import sys

import pytest
import torch

from whisperdrz_amd import _lib

CALL = """
import ctypes, resource, sys
sys.path.insert(0, {root!r})
lib = ctypes.CDLL({lib!r})
lib.wdrz_last_error.restype = ctypes.c_char_p
i64 = ctypes.c_int64
tables = (i64 * 10)(*[65536] * 5, 12288, 1 << 20, 16, 1 << 20, 1 << 24)
pages = (i64 * 6)(65536, 65536, 1 << 20, 4, 16, 64)
st = (i64 * 4)(256, 256, 64, 1)
used = int(open("/proc/self/statm").read().split()[0]) * 4096
resource.setrlimit(resource.RLIMIT_AS, (used + (1 << 31), used + (1 << 31)))
p = lambda x: ctypes.c_void_p(x)
rc = lib.wdrz_attn_kvpages(2, pages, tables, p(65536), st, None, None, None, None, p(65536), p(65536), p(65536), st, i64(2), i64(1), i64(4),
                           ctypes.c_float(0.125), p(65536), ctypes.c_size_t(1 << 40), None)
print(rc, lib.wdrz_last_error().decode())
"""


@pytest.mark.skipif(torch.cuda.is_available(), reason="the addresses are none")
def test_large_tables_are_not_copied_whole():
    code = CALL.format(root=str(_lib.DEBUG_LIB_PATH.parent.parent), lib=str(_lib.DEBUG_LIB_PATH))
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and "reading" in r.stdout and "failed" in r.stdout, (r.returncode, r.stdout, r.stderr[-500:])
