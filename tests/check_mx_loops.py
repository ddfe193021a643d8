"""Compiles csrc/mx_gemm.hip to assembly and looks at what the hand-placed matrix instructions
of its tile kernels rely on (they are inline assembly, so the compiler's own hazard checks do not
cover them):

  * an ordinary vector instruction that writes a register has two wait states between it and a
    matrix instruction that reads it;
  * accumulators stay where they are inside the K loop (no moves between register files);
  * nothing goes through scratch memory (its loads would wait for the copies under way).

Prints one line per tile kernel and "N flagged"; exits with 1 if anything was flagged."""
import os
import re
import subprocess
import sys
import tempfile

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)


def assembly():
    import importlib.util

    spec = importlib.util.spec_from_file_location(
        "b", os.path.join(ROOT, "fastmoe_amd", "build.py"))
    build = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(build)
    with tempfile.TemporaryDirectory() as tmp:
        out = os.path.join(tmp, "mx_gemm.s")
        flags = [f for f in build.FLAGS if f != "-fPIC"]
        subprocess.run([build.HIPCC, *flags, "-S", "--cuda-device-only",
                        os.path.join(build.CSRC, "mx_gemm.hip"), "-o", out],
                       check=True, capture_output=True)
        return open(out).read()


def registers(operand):
    """The vector registers of v7, v[4:7] (a: accumulators)."""
    m = re.fullmatch(r"([va])(?:(\d+)|\[(\d+):(\d+)\])", operand.strip())
    if not m:
        return set()
    lo, hi = (m[2], m[2]) if m[2] else (m[3], m[4])
    return {(m[1], i) for i in range(int(lo), int(hi) + 1)}


def wait_states(line):
    m = re.match(r"s_nop (\d+)", line)
    return int(m[1]) + 1 if m else 1


def check(name, body):
    lines = []
    for raw in body.splitlines():
        line = raw.split(";")[0].strip()
        if re.match(r"[a-z]", line) and not line.endswith(":"):
            lines.append(line)
    bad = []
    at = [i for i, l in enumerate(lines) if l.startswith("v_mfma")]
    for i in at:
        ops = re.split(r",\s*", lines[i].split(None, 1)[1])
        reads = set().union(*(registers(o.split()[0]) for o in ops[1:6] if o))
        waited, j = 0, i - 1
        while j >= 0 and waited < 2:
            l = lines[j]
            if l.startswith("v_") and not l.startswith("v_mfma") and not l.startswith("v_cmp"):
                wrote = registers(re.split(r",\s*", l.split(None, 1)[1])[0])
                if wrote & reads:
                    bad.append(f"{l}  ->  {lines[i]}")
            waited += wait_states(l)
            j -= 1
    loop = lines[at[0]:at[-1] + 1] if at else []
    bad += [l for l in loop if "accvgpr" in l]
    bad += [l for l in lines if l.startswith("scratch_")]
    print(f"{name}: {len(at)} matrix instructions, {len(bad)} flagged")
    for b in bad[:5]:
        print("   ", b)
    return len(bad)


def main():
    text = assembly()
    total = kernels = 0
    for m in re.finditer(r"^(_ZN4fmoe14mx_tile_kernel\S*):(.*?)^\.Lfunc_end", text, re.M | re.S):
        total += check(m[1], m[2])
        kernels += 1
    print(f"{kernels} kernels, {total} flagged")
    return 1 if total or not kernels else 0


if __name__ == "__main__":
    sys.exit(main())
