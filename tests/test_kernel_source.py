"""What inline assembly in the kernels has to declare and to wait for."""
import glob
import os
import re

import pytest

SRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                   "anand_mxnet_amd", "src")
FILES = [p for ext in ("h", "hip")
         for p in glob.glob(os.path.join(SRC, "**", "*." + ext),
                            recursive=True)
         if not p.endswith("_hip." + ext)]


def _asm(path):
    """The text and the clobbers of each asm statement."""
    text = open(path).read()
    for m in re.finditer(r"\basm\b[^(;]*\(", text):
        depth, i, quoted = 1, m.end(), False
        while depth:
            c = text[i]
            if c == '"' and text[i - 1] != "\\":
                quoted = not quoted
            elif not quoted:
                depth += (c == "(") - (c == ")")
            i += 1
        body = text[m.end():i - 1]
        lead = re.match(r'(\s*"(?:[^"\\]|\\.)*")+', body).group(0)
        code = "".join(re.findall(r'"((?:[^"\\]|\\.)*)"', lead))
        yield code.replace("\\t", "").split("\\n"), body[len(lead):]


@pytest.mark.parametrize("path", FILES, ids=os.path.basename)
def test_m0_is_declared_and_scalar_addresses_are_waited_for(path):
    for code, rest in _asm(path):
        if any(re.match(r"\s*s_mov_b32\s+m0\b", line) for line in code):
            assert '"m0"' in rest, code
        wait = 0  # states since the start of the statement
        for line in (x.strip() for x in code):
            op = line.split()[0] if line else ""
            # an address in scalar registers: a vector instruction before
            # the statement may have written them
            if op.startswith("global_load") and re.search(r",\s*%\d+", line):
                assert wait >= 5, code
            nop = re.match(r"s_nop\s+(\d+)", line)
            wait += int(nop.group(1)) + 1 if nop else bool(op)
