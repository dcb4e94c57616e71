"""What the tree attention's launches ask for, recorded on the CPU by functions that stand in for the runtime's in a process of
their own."""
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
#include <string.h>
typedef struct { uint32_t x, y, z; } dim;
typedef struct { const void* kernel; int64_t set, shared; char arguments[192]; } record;
record records[64];
int num_records;
static dim grid_, block_;
static size_t shared_;
static void* stream_;
static void add(const void* kernel, int64_t set, int64_t shared, const void* arguments) {
  if (num_records == 64) return;
  record* r = &records[num_records++];
  r->kernel = kernel, r->set = set, r->shared = shared;
  if (arguments) memcpy(r->arguments, arguments, sizeof r->arguments);
}
int hipFuncSetAttribute(const void* kernel, int attribute, int value) { add(kernel, value, -1, 0); return 0; }
int __hipPushCallConfiguration(dim grid, dim block, size_t shared, void* stream) {
  grid_ = grid, block_ = block, shared_ = shared, stream_ = stream;
  return 0;
}
int __hipPopCallConfiguration(dim* grid, dim* block, size_t* shared, void** stream) {
  *grid = grid_, *block = block_, *shared = shared_, *stream = stream_;
  return 0;
}
int hipLaunchKernel(const void* kernel, dim grid, dim block, void** args, size_t shared, void* stream) {
  add(kernel, -1, (int64_t)shared, args[0]);
  return 0;
}
int hipGetLastError(void) { return 0; }
"""


class TreeArgs(ctypes.Structure):
    """The first argument of the kernels (pa_tree.h)."""
    _fields_ = [(n, ctypes.c_void_p) for n in ("out", "q", "kc", "vc", "tables", "ctx", "starts", "mask", "weights", "ml", "acc", "logits")] + [
        (n, ctypes.c_int64) for n in ("q_stride", "mask_stride", "logit_stride")] + [("c", ctypes.c_float)] + [
        (n, ctypes.c_int) for n in ("q_mode", "num_seqs", "num_tokens", "num_heads", "num_kv_heads", "group", "num_blocks", "block_bits",
                                    "table_width", "max_ctx", "max_query", "max_rows", "parts", "part_len", "row_tiles", "form")] + [
        ("sorted", ctypes.c_bool)]


class Record(ctypes.Structure):
    _fields_ = [("kernel", ctypes.c_void_p), ("set", ctypes.c_int64), ("shared", ctypes.c_int64), ("args", TreeArgs)]


def calls(stand_in, shapes):
    """In the process of its own: single tokens' launches of (seqs, heads, kv heads, context)."""
    assert ctypes.sizeof(TreeArgs) == 192
    recorder = ctypes.CDLL(stand_in, mode=ctypes.RTLD_GLOBAL)
    lib = ctypes.CDLL(LIBRARY)
    p, n = ctypes.c_void_p(4096), ctypes.c_int
    lib.pa_cached_kv_attention_accumulate.argtypes = [ctypes.c_void_p] * 5 + [ctypes.c_float] + [ctypes.c_void_p] * 3 + [n] * 10 + [
        ctypes.c_int64, n, ctypes.c_void_p, ctypes.c_size_t, ctypes.c_void_p]
    for seqs, heads, kv, context in shapes:
        rc = lib.pa_cached_kv_attention_accumulate(p, p, p, p, p, 1.0, p, p, p, seqs, seqs, heads, kv, 128, 16, 512, context // 16, context, 1,
                                                   heads * 128, 1, p, 1 << 40, None)
        assert rc == 0, rc
    records = (Record * 64).in_dll(recorder, "records")
    return [(r.kernel, r.set, r.shared, r.args.num_seqs, r.args.max_ctx, r.args.part_len, r.args.sorted)
            for r in records[:ctypes.c_int.in_dll(recorder, "num_records").value]]


def record(tmp_path, shapes):
    assert os.path.exists(LIBRARY), "build the library first"
    source, stand_in = str(tmp_path / "stand_in.c"), str(tmp_path / "stand_in.so")
    with open(source, "w") as f:
        f.write(STAND_IN)
    subprocess.run(["gcc", "-shared", "-fPIC", "-o", stand_in, source], check=True)
    run = subprocess.run([sys.executable, os.path.abspath(__file__), stand_in, json.dumps(shapes)], check=True, stdout=subprocess.PIPE, text=True)
    return json.loads(run.stdout.splitlines()[-1])


def test_launches_of_all_sizes_ask_for_the_same_lds(tmp_path):
    """What a kernel may take of a workgroup's LDS is an attribute of the kernel, not of a launch: two host threads that set
    it to what each one's own launch needs could lower it between the other's setting and its launch."""
    records = record(tmp_path, [(64, 32, 8, c) for c in (4096, 4352, 4608, 4096, 2048)])
    launches = [r[2] for r in records if r[2] >= 0]
    assert len(launches) == 5 and len({r[0] for r in records}) == 1, records
    assert launches == [4 * 4 * (c + 4) for c in (4096, 4352, 4608, 4096)] + [4 * 4 * 16 * 132], records
    allowed = 65536  # without a word
    for _, value, shared, *_ in records:
        allowed = value if value >= 0 else allowed
        assert shared <= allowed, records
    assert len({r[1] for r in records if r[1] >= 0}) == 1, f"the attribute follows the launch: {records}"


def test_sequences_are_ranked_where_their_length_repays_it(tmp_path):
    """Every workgroup ranks all sequences for itself: with many of them, of a few steps each, that was most of the launch."""
    short = [(118, 32, 32, 96), (256, 32, 32, 64), (256, 32, 8, 1024), (128, 32, 8, 512), (64, 32, 8, 512), (16, 32, 8, 1024)]
    long = [(96, 32, 8, 4096), (256, 32, 8, 2048), (128, 32, 8, 1536), (64, 40, 40, 2048), (32, 16, 16, 768)]
    alone = [(1, 32, 32, 8192), (8, 32, 8, 512), (257, 32, 8, 4096)]    # nothing waits for a CU, or too many to rank
    ranked = {(r[3], r[4]): r[6] for r in record(tmp_path, short + long + alone) if r[2] >= 0 and r[4] > 0 and r[5] > 0}
    for shapes, want in ((short, False), (long, True), (alone, False)):
        for seqs, _, _, context in shapes:
            assert ranked[seqs, context] == want, (seqs, context)


if __name__ == "__main__":
    print(json.dumps(calls(sys.argv[1], json.loads(sys.argv[2]))))
