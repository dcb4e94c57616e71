"""Every way through the built kernels leaves a matrix product its time before the result is touched.

The hardware does not hold an instruction back that reads a product's result too early: the compiler counts the
instructions between.  Where a short way and a long one meet it was seen to count along the long one alone.  This
reads the kernels of the built library and counts along every way.
"""
import os
import re
import shutil
import subprocess

import pytest

OBJDUMP = next((p for p in (shutil.which("llvm-objdump"), "/opt/rocm/llvm/bin/llvm-objdump") if p and os.path.exists(p)), None)
LIBRARY = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "vllm-v0.1.0_amd", "libpaged_attn_mi355x.so")

_REGS = re.compile(r"(?<![a-z0-9_])([va])(?:\[(\d+):(\d+)\]|(\d+))(?![a-z0-9_])")


def needed(op):
    """Instructions' time until a product's result can be read: 4 passes for 16 x 16 of 16 bits, 8 for the others."""
    return 10 if "x4_f32" in op else (12 if "32x32" in op else 8)


def registers(text):
    out = set()
    for kind, lo, hi, one in _REGS.findall(text):
        out.update((kind, i) for i in range(int(one or lo), int(one or hi) + 1))
    return out


def operands(text):
    return [p.strip() for p in re.split(r",\s*(?![^\[]*\])", text)]


def short_waits(lines):
    """(product, use, waits) of a kernel's listing: 'op operands // address: ...' a line."""
    code, at = [], {}
    for line in lines:
        text, _, note = line.partition("//")
        parts = text.split(None, 1)
        if not parts:
            continue
        at[int(note.split(":")[0], 16)] = len(code)
        code.append((parts[0], parts[1].strip() if len(parts) > 1 else "", int(note.split(":")[0], 16)))
    ways, touched = [], [registers(rest) for _, rest, _ in code]
    for i, (op, rest, address) in enumerate(code):
        to = []
        if op not in ("s_endpgm", "s_branch") and i + 1 < len(code):
            to.append(i + 1)
        if op == "s_branch" or op.startswith("s_cbranch"):
            step = int(rest.split()[0], 0)
            to.append(at[address + 4 + 4 * (step - 65536 if step > 32767 else step)])
        ways.append(to)
    found = []
    for i, (op, rest, _) in enumerate(code):
        if not op.startswith("v_mfma"):
            continue
        result, need, least = registers(operands(rest)[0]), needed(op), {}
        todo = [(j, 0) for j in ways[i]]
        while todo:
            j, waits = todo.pop()
            if waits >= need or least.get(j, need) <= waits:
                continue
            least[j] = waits
            other, its = code[j][:2]
            if touched[j] & result:
                # a product that adds to the result, or replaces it, follows in order; one that multiplies it does not
                if not other.startswith("v_mfma") or (registers(operands(its)[1]) | registers(operands(its)[2])) & result:
                    found.append((f"{op} {rest}", f"{other} {its}", waits))
                    continue
                if operands(its)[0] == operands(rest)[0]:
                    continue  # it is followed from there
            todo += [(k, waits + (int(its, 0) + 1 if other == "s_nop" else 1)) for k in ways[j]]
    return found


def test_the_count():
    head = ["s_mov_b32 s0, 0 // 0:", "v_mfma_f32_16x16x32_f16 v[0:3], v[8:11], v[12:15], 0 // 4:"]
    assert short_waits(head + ["s_nop 6 // C:", "v_add_f32_e32 v4, v3, v3 // 10:", "s_endpgm // 14:"])
    assert not short_waits(head + ["s_nop 7 // C:", "v_add_f32_e32 v4, v3, v3 // 10:", "s_endpgm // 14:"])
    # a way that goes round the waits
    assert short_waits(head + ["s_cbranch_scc1 1 // C:", "s_nop 7 // 10:", "v_mov_b32_e32 v4, v2 // 14:", "s_endpgm // 18:"])
    # adding up needs none, multiplying does
    assert not short_waits(head + ["v_mfma_f32_16x16x32_f16 v[0:3], v[8:11], v[12:15], v[0:3] // C:", "s_endpgm // 14:"])
    assert short_waits(head + ["v_mfma_f32_16x16x32_f16 v[4:7], v[0:3], v[12:15], 0 // C:", "s_endpgm // 14:"])
    # backwards, out of a loop
    loop = ["v_mov_b32_e32 v4, v1 // 0:", "s_nop 7 // 4:", "v_mfma_f32_16x16x32_f16 v[0:3], v[8:11], v[12:15], 0 // 8:"]
    assert short_waits(loop + ["s_cbranch_scc1 65531 // 10:", "s_endpgm // 14:"])


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
            if "v_mfma" not in part:
                continue
            kernel, _, body = part.partition(">:\n")
            seen += 1
            wrong += [(kernel,) + w for w in short_waits(line for line in body.splitlines() if "//" in line)]
    assert seen > 100, f"{seen} kernels with matrix products found"
    assert not wrong, f"{len(wrong)} results touched too early, first {wrong[0]}"
