"""CPU tests of the kernels' inline assembly. The compiler keeps the wait states
that instructions need between them for its own instructions and not for those
inside assembly, so what stands there must not need any."""
import glob
import os
import re

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
