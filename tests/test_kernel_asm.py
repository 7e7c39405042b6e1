"""CPU tests of the kernels' inline assembly. The compiler keeps the wait states
that instructions need between them for its own instructions and not for those
inside assembly, so what stands there must not need any."""
import glob
import os
import re
import subprocess

from flashinfer_amd import build

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "flashinfer_amd", "csrc")


def _blocks():
    """(place, the instructions' text, what follows it) of every asm statement."""
    found = []
    for path in sorted(glob.glob(os.path.join(CSRC, "*.h*"))):
        src = re.sub(r"//[^\n]*", "", open(path).read())
        for m in re.finditer(r"\basm\b(?:\s+volatile)?\s*\(", src):
            depth, end = 1, m.end()
            while depth:
                depth += {"(": 1, ")": -1}.get(src[end], 0)
                end += 1
            body = src[m.end():end - 1]
            text = re.match(r'(?:\s*"(?:[^"\\]|\\.)*")+', body)
            words = "".join(re.findall(r'"((?:[^"\\]|\\.)*)"', text[0]))
            place = f"{os.path.basename(path)}:{src[:m.start()].count(chr(10)) + 1}"
            found.append((place, words.replace("\\t", " ").split("\\n"), body[text.end():]))
    return found


def test_assembly_holds_no_vector_arithmetic():
    """A vector instruction may not write registers that a matrix instruction just issued still reads or writes."""
    blocks = _blocks()
    assert len(blocks) > 20
    allowed = re.compile(r"s_waitcnt|s_barrier|s_nop|s_mov_b32 m0|s_mov_b64|global_load_lds_dword(x4)?\b|;|$")
    bad = [(place, line) for place, lines, _ in blocks for line in lines if not allowed.match(line.strip())]
    assert not bad, bad


def test_assembly_loads_by_scalars_that_it_moves_itself():
    """A vector memory access may not read an SGPR that a vector instruction, such as the reload of a spilled scalar,
    wrote fewer than five wait states before; a scalar move in between waits for it."""
    loads = 0
    for place, lines, rest in _blocks():
        for n, line in enumerate(lines):
            m = re.match(r"\s*global_load_lds_\w+ (%\d+), (off|%\d+)", line)
            if not m:
                continue
            loads += 1
            assert m[2] == "off" or any(re.match(rf"\s*s_mov_b64 {m[2]},", before) for before in lines[:n]), (place, line)
            # M0 is written one wait state before the copy at least
            assert re.match(r"\s*s_mov_b32 m0,", lines[n - 2]), (place, lines)
    assert loads >= 5


SOURCE = """
#include "%s/lds_copy.hpp"
extern "C" __global__ void copies(const uint8_t* const* from, uint8_t* to) {
    __shared__ __attribute__((aligned(1024))) uint8_t smem[4096];
    // a base that a vector instruction leaves in SGPRs right before the copy
    const uint64_t p = (uint64_t)from[threadIdx.x];
    uint64_t base = (uint64_t)__builtin_amdgcn_readfirstlane((uint32_t)(p >> 32)) << 32;
    base |= (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)p);
    mimoe::g2l16s((const void*)base, threadIdx.x * 16, smem);
    mimoe::g2l16s_once((const void*)base, threadIdx.x * 16, smem + 1024);
    mimoe::g2l4s((const void*)base, threadIdx.x * 4, smem + 2048);
    mimoe::wait_vmem();
    __syncthreads();
    to[threadIdx.x] = smem[threadIdx.x * 8];
}
"""


def test_compiled_copies_read_no_scalar_that_a_vector_instruction_just_wrote(tmp_path):
    src, out = tmp_path / "copies.hip", tmp_path / "copies.s"
    src.write_text(SOURCE % CSRC)
    flags = [f for f in build.HIPCC_FLAGS if f != "-fPIC"]
    subprocess.run([build.hipcc(), *flags, "--cuda-device-only", "-S", str(src), "-o", str(out)], check=True,
                   capture_output=True)
    since, copies, seen = {}, 0, 0  # SGPR -> wait states since a vector instruction wrote it
    for line in out.read_text().split("copies:")[1].split("s_endpgm")[0].splitlines():
        words = line.split(";")[0].replace(",", " ").split()
        if not words or words[0].startswith(".") or words[0].endswith(":"):
            continue
        op, args = words[0], words[1:]
        states = int(args[0], 0) + 1 if op == "s_nop" else 1
        if op.startswith("global_load_lds"):
            copies += 1
            for a in args[1:]:
                low, high = (int(v) for v in re.fullmatch(r"s\[(\d+):(\d+)\]", a).groups()) if a.startswith("s[") else (1, 0)
                assert all(since.get(r, 5) >= 5 for r in range(low, high + 1)), line
        since = {r: n + states for r, n in since.items()}
        if op.startswith("v_readfirstlane"):
            seen += 1
            since[int(args[0][1:])] = 0
        elif op.startswith("s_mov") and args and args[0].startswith("s"):  # waits for what it reads, and so holds it
            for r in range(*(lambda v: (v[0], v[-1] + 1))([int(v) for v in re.findall(r"\d+", args[0])])):
                since.pop(r, None)
    assert copies == 3 and seen >= 2
