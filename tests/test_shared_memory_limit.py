"""A kernel's dynamic shared-memory limit under calls from two threads: it never ends up below what a call was promised.

The library runs in a process of its own whose runtime calls are stand-ins, so that the order of two first calls can be set. No GPU."""

from __future__ import annotations

import os
import shutil
import subprocess
import sys
import textwrap

import pytest

from gdn2_tilelang_b200 import build

SHIM = """
    #include <unistd.h>
    static int limit, sets;
    static volatile int slow_value, slow_entered;
    int cudaGetDevice(int* d) { *d = 0; return 0; }
    int cudaFuncSetAttribute(const void* f, int attr, int value) {
      if (attr != 8) return 0;
      if (value == slow_value) { slow_entered = 1; usleep(300000); }
      limit = value; ++sets;
      return 0;
    }
    int now(void) { return limit; }
    int count(void) { return sets; }
    int entered(void) { return slow_entered; }
    void begin(int slow) { limit = sets = 0; slow_value = slow; slow_entered = 0; }
"""
DRIVER = """
    import ctypes, sys, threading, time
    lib, shim = ctypes.CDLL(sys.argv[1]), ctypes.CDLL(sys.argv[2])
    ensure = lib._ZN4gdn219ensure_dynamic_smemEPKvm
    ensure.argtypes, ensure.restype = [ctypes.c_void_p, ctypes.c_size_t], ctypes.c_int
    for kernel, first, second in ((64, 1000, 2000), (128, 2000, 1000)):
        shim.begin(first)                        # the first call is held up inside the runtime while the second one runs
        seen = []
        def call(n):
            assert ensure(kernel, n) == 0
            seen.append((n, shim.now()))         # what this call's launch would find
        a = threading.Thread(target=call, args=(first,))
        a.start()
        while not shim.entered():
            time.sleep(0.001)
        b = threading.Thread(target=call, args=(second,))
        b.start()
        a.join(); b.join()
        assert all(limit >= n for n, limit in seen), seen
        assert shim.now() == 2000, shim.now()
        done = shim.count()
        assert ensure(kernel, 2000) == 0 and ensure(kernel, 500) == 0 and shim.now() == 2000 and shim.count() == done
"""


@pytest.mark.skipif(shutil.which("gcc") is None, reason="no C compiler")
def test_the_limit_is_only_raised(tmp_path):
    shim, driver = tmp_path / "shim.so", tmp_path / "driver.py"
    (tmp_path / "shim.c").write_text(textwrap.dedent(SHIM))
    driver.write_text(textwrap.dedent(DRIVER))
    subprocess.run(["gcc", "-shared", "-fPIC", "-o", str(shim), str(tmp_path / "shim.c")], check=True)
    lib = build.LIB if build.LIB.exists() else build.build()
    r = subprocess.run([sys.executable, str(driver), str(lib), str(shim)], env={**os.environ, "LD_PRELOAD": str(shim)},
                       capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stderr
