"""Builds the native artefacts of the backend, in-tree:

  i_amd/i_kernels_gfx950.hsaco   device code object (hipcc --genco, gfx950 only): the kernels of compiled programs
  i_amd/i_attend_*_gfx950.hsaco  device code objects of the kernels of include/i_attend.h
  i_amd/libi_core.so             host runtime + compiler (C++17), linked to libamdhip64

Run as  python -m i_amd.build  (or call build()).  hipcc cross-compiles, no GPU needed.
"""
import os
import re
import subprocess
import sys
import tempfile
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

PKG = Path(__file__).resolve().parent
CSRC = PKG / "csrc"
ROCM = Path(os.environ.get("ROCM_PATH", "/opt/rocm"))
HSACO = PKG / "i_kernels_gfx950.hsaco"
LIB = PKG / "libi_core.so"
ATTEND = ("attend_forward", "attend_backward", "attend_cache")

# packed-fp32 VALU forms are disabled for all device code on purpose.
HIPCC_FLAGS = ["--offload-arch=gfx950", "-O3", "-std=c++17",
               "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]


def _run(cmd):
    print("+", " ".join(str(c) for c in cmd), flush=True)
    subprocess.run([str(c) for c in cmd], check=True)


def host_sources():
    return sorted(p for p in CSRC.rglob("*.cpp"))


def _registers(token):
    m = re.match(r"-?\|?([va])(?:\[(\d+):(\d+)\]|(\d+)\b)", token.strip())
    if not m:
        return set()
    return {(m.group(1), r) for r in range(int(m.group(2) or m.group(4)), int(m.group(3) or m.group(4)) + 1)}


def _kernels(asm_text):
    """Name, instructions (mnemonic, operands) and labels of every kernel of a listing."""
    for name, body in re.findall(r"^(\w+):[^\n]*\n(.*?)\.end_amdhsa_kernel", asm_text, re.S | re.M):
        code, labels = [], {}
        for line in body.splitlines():
            line = line.split(";")[0].strip()
            label = re.match(r"(\.LBB\w+):", line)
            if label:
                labels[label.group(1)] = len(code)
            elif line and not line.startswith((".", "//")):
                op, _, rest = line.partition(" ")
                code.append((op, [t.strip() for t in rest.split(",")]))
        yield name, code, labels


def _following(code, labels, start, limit):
    """The instructions after `start` within `limit` wait states, branches followed: (operation, operands, wait states since);
    sent a true value, what follows that instruction is left out."""
    seen, ways = {}, [(start + 1, 0)]
    while ways:
        at, waited = ways.pop()
        if at >= len(code) or waited >= limit or seen.get(at, limit) <= waited:
            continue
        seen[at] = waited
        op, args = code[at]
        if (yield op, args, waited) or op == "s_endpgm":
            continue
        if op.startswith(("s_branch", "s_cbranch")):
            ways.append((labels[args[0]], waited + 1))
            if op == "s_branch":
                continue
        ways.append((at + 1, waited + (int(args[0], 0) + 1 if op == "s_nop" else 1)))


def early_mfma_operands(asm_text):
    """Matrix instructions that may read an operand before it is there: one may read a register two wait states after an ordinary
    vector instruction wrote it at the earliest.  The compiler sees to that, but not for matrix instructions that are
    inline assembly (the four-wave GEMMs, the gradient's work on keys).  Those are written so that no such pair exists; this follows the
    compiled assembly from every vector instruction, branches included, and returns the pairs it finds all the same (a later
    compiler might place a copy there)."""
    found = []
    for name, code, labels in _kernels(asm_text):
        for start, (op, operands) in enumerate(code):
            if not op.startswith("v_") or op.startswith("v_mfma"):
                continue
            written = set().union(*map(_registers, operands[:2 if "swap" in op else 1]))
            for after, args, waited in _following(code, labels, start, 2) if written else ():
                if after.startswith("v_mfma") and set().union(*map(_registers, args[1:])) & written:
                    found.append(f"{name}: {after} {', '.join(args)} {waited} after {code[start]}")
    return found


def early_mfma_reads(asm_text):
    """Instructions that may see a matrix instruction's result before it is there.  A vector or memory instruction may
    read it no sooner than 8 wait states (bf16, 16 x 16 x 32) or 10 (f32, 16 x 16 x 4) after it was issued; the compiler fills them
    in, but not where the result is fetched from an accumulation register beyond a branch (one such kernel gave wrong
    sums).  This follows the compiled assembly from every matrix instruction, branches included, and returns what it finds."""
    found = []
    for name, code, labels in _kernels(asm_text):
        for start, (op, operands) in enumerate(code):
            need = {"v_mfma_f32_16x16x32_bf16": 8, "v_mfma_f32_16x16x4_f32": 10}.get(op)
            if need is None:
                continue
            result, way, done = _registers(operands[0]), _following(code, labels, start, need), None
            while True:
                try:
                    op, args, waited = way.send(done)
                except StopIteration:
                    break
                done = False
                if op.startswith("v_mfma"):
                    if (_registers(args[1]) | _registers(args[2])) & result:
                        found.append(f"{name}: {op} {', '.join(args)} {waited} after {code[start]}")
                    # (the next of a chain: its last one counts)
                    done = bool(set().union(*map(_registers, args)) & result)
                elif op.startswith(("v_", "ds_", "global_", "buffer_", "scratch_", "flat_")):
                    # (what a load brings arrives later than that)
                    read = args[1:] if op.startswith(("ds_read", "global_load", "buffer_load", "scratch_load", "flat_load")) else args
                    done = bool(set().union(*map(_registers, read)) & result)
                    if done:
                        found.append(f"{name}: {op} {', '.join(args)} {waited} after {code[start]}")
    return found


def check_assembly(asm_text, results=False):
    """Raises where compiled code does not wait for an operand of a matrix instruction (results: for its result)."""
    operands = early_mfma_operands(asm_text)
    if operands:
        raise RuntimeError("operands of matrix instructions read too early:\n" + "\n".join(operands))
    early = early_mfma_reads(asm_text) if results else []
    if early:
        raise RuntimeError("results of matrix instructions read too early:\n" + "\n".join(early))


def build_kernels():
    with tempfile.TemporaryDirectory() as tmp:
        # (the intermediate assembly lands in the working directory: it is read for the check below)
        print("+ cd", tmp, flush=True)
        cmd = [ROCM / "bin" / "hipcc", "--genco", *HIPCC_FLAGS, "-save-temps", CSRC / "kernels" / "kernels.hip", "-o", HSACO]
        print("+", " ".join(str(c) for c in cmd), flush=True)
        subprocess.run([str(c) for c in cmd], check=True, cwd=tmp)
        listings = list(Path(tmp).glob("*gfx950*.s"))
        if not listings:
            raise RuntimeError("hipcc left no gfx950 assembly to check")
        check_assembly(listings[0].read_text())


def build_attend(name):
    """One code object of the attention kernels with masks."""
    with tempfile.TemporaryDirectory() as tmp:
        cmd = [ROCM / "bin" / "hipcc", "--genco", *HIPCC_FLAGS, "-save-temps", CSRC / "kernels" / f"{name}.hip", "-o", PKG / f"i_{name}_gfx950.hsaco"]
        print("+", " ".join(str(c) for c in cmd), flush=True)
        subprocess.run([str(c) for c in cmd], check=True, cwd=tmp)
        check_assembly(next(Path(tmp).glob("*gfx950*.s")).read_text(), results=True)


def build_static_scratch():
    """The one host + device source: the fixed device workspace (a file-scope __device__ array) and its lookup."""
    obj = CSRC / "runtime" / "static_scratch.o"
    _run([ROCM / "bin" / "hipcc", "-c", "-fPIC", "-O2", "-std=c++17", "--offload-arch=gfx950",
          "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
          CSRC / "runtime" / "static_scratch.hip", "-o", obj])
    return obj


def build_host():
    scratch_obj = build_static_scratch()
    _run(["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-Wall", "-fvisibility=hidden", "-Wno-unused-function",
          "-D__HIP_PLATFORM_AMD__", f"-I{ROCM / 'include'}", f"-I{PKG.parent / 'include'}",
          *host_sources(), scratch_obj, "-o", LIB,
          f"-L{ROCM / 'lib'}", "-lamdhip64", f"-Wl,-rpath,{ROCM / 'lib'}", "-ldl", "-lpthread"])


def build():
    with ThreadPoolExecutor(max_workers=4) as pool:
        jobs = [pool.submit(build_kernels)] + [pool.submit(build_attend, name) for name in ATTEND]
        build_host()
        for job in jobs:
            job.result()


if __name__ == "__main__":
    build()
    sys.exit(0)
