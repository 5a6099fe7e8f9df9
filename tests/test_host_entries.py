"""C entries of the host library under a limit on memory: lists that do not fit end as an error code, never as an exception
that leaves a C function and with it ends the process."""
import subprocess
import sys

import pytest

CAPACITY, METADATA = 4, 5

# What can be asked for in a few words: one sequence of 2^31 - 2 rows is 2^31 query blocks (60 GB) or 2^30 records (34 GB),
# one bit per slot of the largest pool 268 MB.
CALLS = {
    "attention_plan": "lib.gk_attention_plan_build(ptr(seq), 1, 16, 1, 128, -1, 148, 0, None, 0, n(), None, 0, n(), n())",
    "prefill_plan": "lib.gk_prefill_plan_build(ptr(seq), 1, 128, 1, -1, 0, None, 0, n(), None, n())",
    "prefill_plan_two_way": "lib.gk_prefill_plan_build_two_way(ptr(seq), 1, None, 128, 1, -1, 0, None, 0, n(), None, n())",
    "shared_prefix_plan": "lib.gk_shared_prefix_plan_build(ptr(seq), 1, None, None, None, 0, 16, 1, 128, -1, 148, 0, 0, 0,"
                          " C.byref(C.c_int()), None, 0, n(), None, 0, n(), n(), None, 0, n(), None, 0, n())",
    "metadata": "lib.gk_paged_metadata_validate(ptr(one), ptr(one), ptr(one), 1, ptr(one), 1, 1, 2**31 - 1, ptr(seq), n(), None)",
}


@pytest.mark.parametrize("call", CALLS)
def test_lists_that_do_not_fit(call):
    code = f"""
import ctypes as C, resource
import numpy as np
from gaudirt_b200 import abi
lib = abi.lib()
ptr = lambda a: a.ctypes.data_as(C.c_void_p)
n = lambda: C.byref(C.c_int64())
seq, one = np.array([[0, 2**31 - 2, 0, 0]], dtype=np.int32), np.zeros(4, dtype=np.int32)
mapped = int(open("/proc/self/statm").read().split()[0]) * resource.getpagesize()
resource.setrlimit(resource.RLIMIT_AS, (mapped + (200 << 20), resource.RLIM_INFINITY))
print("code", {CALLS[call]})
"""
    run = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stderr
    assert run.stdout.split()[-2:] == ["code", str(CAPACITY)]


def test_messages_outlive_the_call():
    import ctypes as C

    import numpy as np

    from gaudirt_b200 import abi
    lib = abi.lib()
    one = np.zeros(4, dtype=np.int32)
    pointer = one.ctypes.data_as(C.c_void_p)
    for slots, message in ((0, "dimensions outside"), (1, None)):
        rc = lib.gk_paged_metadata_validate(pointer, pointer, pointer, 1, pointer, 1, 1, slots, pointer, C.byref(C.c_int64()), None)
        assert rc == (METADATA if message else 0)
        assert b"dimensions outside" in lib.gk_metadata_error()      # stays until the next refusal
