"""What a kernel may take of a workgroup's LDS is an attribute of the kernel, not of a launch: two host threads that set it to
what each one's own launch needs could lower it between the other's setting and its launch.

Launches are recorded on the CPU by functions that stand in for the runtime's in a process of their own.
"""
import ctypes
import json
import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
LIBRARY = os.path.join(os.path.dirname(HERE), "vllm-v0.1.0_amd", "libpaged_attn_mi355x.so")

STAND_IN = r"""
#include <stddef.h>
#include <stdint.h>
typedef struct { uint32_t x, y, z; } dim;
typedef struct { const void* kernel; int64_t set, shared; } record;
record records[64];
int num_records;
static dim grid_, block_;
static size_t shared_;
static void* stream_;
static void add(const void* kernel, int64_t set, int64_t shared) {
  if (num_records < 64) records[num_records++] = (record){kernel, set, shared};
}
int hipFuncSetAttribute(const void* kernel, int attribute, int value) { add(kernel, value, -1); return 0; }
int __hipPushCallConfiguration(dim grid, dim block, size_t shared, void* stream) {
  grid_ = grid, block_ = block, shared_ = shared, stream_ = stream;
  return 0;
}
int __hipPopCallConfiguration(dim* grid, dim* block, size_t* shared, void** stream) {
  *grid = grid_, *block = block_, *shared = shared_, *stream = stream_;
  return 0;
}
int hipLaunchKernel(const void* kernel, dim grid, dim block, void** args, size_t shared, void* stream) {
  add(kernel, -1, (int64_t)shared);
  return 0;
}
int hipGetLastError(void) { return 0; }
"""


def calls(stand_in):
    """In the process of its own: one kernel's launches of several sizes; (kernel, set, shared) in order."""
    class Record(ctypes.Structure):
        _fields_ = [("kernel", ctypes.c_void_p), ("set", ctypes.c_int64), ("shared", ctypes.c_int64)]

    recorder = ctypes.CDLL(stand_in, mode=ctypes.RTLD_GLOBAL)
    lib = ctypes.CDLL(LIBRARY)
    p, n = ctypes.c_void_p(4096), ctypes.c_int
    lib.pa_cached_kv_attention_accumulate.argtypes = [ctypes.c_void_p] * 5 + [ctypes.c_float] + [ctypes.c_void_p] * 3 + [n] * 10 + [
        ctypes.c_int64, n, ctypes.c_void_p, ctypes.c_size_t, ctypes.c_void_p]
    for context in (4096, 4352, 4608, 4096, 2048):
        rc = lib.pa_cached_kv_attention_accumulate(p, p, p, p, p, 1.0, p, p, p, 64, 64, 32, 8, 128, 16, 512, context // 16, context, 1,
                                                   32 * 128, 1, p, 1 << 40, None)
        assert rc == 0, rc
    records = (Record * 64).in_dll(recorder, "records")
    return [(r.kernel, r.set, r.shared) for r in records[:ctypes.c_int.in_dll(recorder, "num_records").value]]


def test_launches_of_all_sizes_ask_for_the_same(tmp_path):
    assert os.path.exists(LIBRARY), "build the library first"
    source, stand_in = str(tmp_path / "stand_in.c"), str(tmp_path / "stand_in.so")
    with open(source, "w") as f:
        f.write(STAND_IN)
    subprocess.run(["gcc", "-shared", "-fPIC", "-o", stand_in, source], check=True)
    run = subprocess.run([sys.executable, os.path.abspath(__file__), stand_in], check=True, stdout=subprocess.PIPE, text=True)
    records = json.loads(run.stdout.splitlines()[-1])
    launches = [shared for _, _, shared in records if shared >= 0]
    assert len(launches) == 5 and len({kernel for kernel, _, _ in records}) == 1, records
    assert launches == [4 * 4 * (c + 4) for c in (4096, 4352, 4608, 4096)] + [4 * 4 * 16 * 132], records
    allowed = 65536  # without a word
    for _, value, shared in records:
        allowed = value if value >= 0 else allowed
        assert shared <= allowed, records
    assert len({value for _, value, _ in records if value >= 0}) == 1, f"the attribute follows the launch: {records}"


if __name__ == "__main__":
    print(json.dumps(calls(sys.argv[1])))
