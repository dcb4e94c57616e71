"""The tree attention's kernel for many rows keeps two LDS buffers of a step's keys and two of its values, for all its waves.
Between two barriers each buffer is either read or filled: a wave that is ahead would hand the others another step's keys.

A wave that reads one buffer of each kind reads a step's pieces, one load of 16 bytes for each; with more than those it
has read both buffers of a kind, and whatever it fills before the next barrier may be read by a wave that is behind.
This follows every way through the kernels of the built library and counts.
"""
import os
import re
import shutil
import subprocess

import pytest

OBJDUMP = next((p for p in (shutil.which("llvm-objdump"), "/opt/rocm/llvm/bin/llvm-objdump") if p and os.path.exists(p)), None)
LIBRARY = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "vllm-v0.1.0_amd", "libpaged_attn_mi355x.so")


def pieces(dtype, head_size):
    """Of a step's keys and values: 1 KiB each, 16 bytes to a lane."""
    x, tokens = (4, 16) if dtype == "F32" else (8, 32)
    return (head_size // x + 3) // 4 * (tokens // 16) + head_size // 16


def reads_before_a_fill(lines, limit):
    """The most 16-byte LDS reads (counted up to limit + 1) of any way from a barrier to a 16-byte LDS write without
    another barrier between, in a kernel's listing: 'op operands // address: ...' a line."""
    code, at = [], {}
    for line in lines:
        text, _, note = line.partition("//")
        parts = text.split(None, 1)
        if not parts:
            continue
        address = int(note.split(":")[0], 16)
        at[address] = len(code)
        code.append((parts[0], parts[1] if len(parts) > 1 else "", address))
    most, seen, todo = 0, {}, [(0, 0)]
    while todo:
        i, reads = todo.pop()
        if seen.get(i, -1) >= reads:
            continue
        seen[i] = reads
        op, rest, address = code[i]
        if op == "s_barrier":
            reads = 0
        elif op == "ds_read_b128":
            reads = min(reads + 1, limit + 1)
        elif op == "ds_write_b128":
            most = max(most, reads)
        if op not in ("s_endpgm", "s_branch") and i + 1 < len(code):
            todo.append((i + 1, reads))
        if op == "s_branch" or op.startswith("s_cbranch"):
            step = int(rest.split()[0], 0)
            todo.append((at[address + 4 + 4 * (step - 65536 if step > 32767 else step)], reads))
    return most


def test_the_count():
    read, fill, barrier = "ds_read_b128 v[0:3], v4 // {:X}:", "ds_write_b128 v4, v[0:3] // {:X}:", "s_barrier // {:X}:"

    def count(*ops, limit=2):
        return reads_before_a_fill([op.format(8 * i) if "{" in op else op for i, op in enumerate(ops)], limit)

    assert count(read, read, fill) == 2
    assert count(read, barrier, read, fill) == 1
    assert count(read, read, barrier, read, read, fill, barrier) == 2
    assert count(read, read, read, read, fill) == 3                       # no further than it matters
    assert count(read, read, read) == 0                                   # nothing is filled behind them
    # around a loop without a barrier, and with one
    back = "s_cbranch_scc1 {} // 10:"
    assert count(read, fill, back.format(65536 - 5)) == 3
    assert count(read, fill, barrier, "s_cbranch_scc1 65529 // 18:") == 1
    # a way round the barrier
    assert count(read, "s_cbranch_scc1 2 // 8:", barrier, "s_nop 0 // 14:", read, fill) == 2


@pytest.mark.skipif(OBJDUMP is None, reason="no llvm-objdump")
def test_built_kernels(tmp_path):
    assert os.path.exists(LIBRARY), "build the library first"
    copy = str(tmp_path / "kernels.so")
    shutil.copy(LIBRARY, copy)
    subprocess.run([OBJDUMP, "--offloading", copy], check=True, stdout=subprocess.DEVNULL)
    seen, wrong = 0, []
    for name in sorted(n for n in os.listdir(tmp_path) if "amdgcn" in n):
        text = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", str(tmp_path / name)], check=True, stdout=subprocess.PIPE, text=True).stdout
        for part in re.split(r"^[0-9a-f]+ <(?=[^>]*>:$)", text, flags=re.M)[1:]:
            kernel, _, body = part.partition(">:\n")
            form = re.search(r"pa_tree_many_kernelINS0_\d+(F16|BF16|F32)ELi(\d+)E", kernel)
            if form is None:
                continue
            seen += 1
            step = pieces(form[1], int(form[2]))
            most = reads_before_a_fill((line for line in body.splitlines() if "//" in line), step)
            if most != step:
                wrong.append((kernel, step, most))
    assert seen == 20, f"{seen} kernels found"
    assert not wrong, f"(kernel, a step's pieces, reads between barriers): {wrong}"
