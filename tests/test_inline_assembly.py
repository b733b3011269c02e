"""Wait states behind inline assembly.  The compiler keeps two wait states between a vector instruction and a matrix instruction
that reads its result, but none behind an asm statement, into which it does not look: a statement that writes the operands of
matrix instructions ends with them itself."""
import glob
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "dl4s_amd", "csrc")


def _statements():
    """(file, instructions) of every asm statement with instructions in it."""
    for path in sorted(glob.glob(os.path.join(CSRC, "*.h")) + glob.glob(os.path.join(CSRC, "*.hip"))):
        with open(path) as f:
            text = f.read()
        for m in re.finditer(r'\basm\s*(?:volatile\s*)?\(((?:\s*"[^"]*")+)', text):
            code = "".join(re.findall(r'"([^"]*)"', m.group(1)))
            lines = [x.strip() for x in re.split(r"\\n|;", code.replace("\\t", " ")) if x.strip()]
            if lines:
                yield os.path.basename(path), lines


def test_operands_of_matrix_instructions():
    writers = [(f, lines) for f, lines in _statements() if any(x.startswith(("v_fma_mix", "v_cvt_pk")) for x in lines)]
    assert len(writers) >= 2
    for f, lines in writers:
        m = re.fullmatch(r"s_nop (\d+)", lines[-1])
        assert m and int(m.group(1)) >= 1, (f, lines[0], lines[-1])


def test_no_matrix_instruction_inside():
    """One there would need its own waits in front and behind."""
    for f, lines in _statements():
        assert not any("mfma" in x for x in lines), (f, lines)
