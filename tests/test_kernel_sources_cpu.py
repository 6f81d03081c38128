"""What the kernel sources have to say to the compiler: the registers that inline assembly writes."""
import glob
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "rwkv-infctx-trainer_amd", "csrc")
SOURCES = sorted(glob.glob(os.path.join(CSRC, "*.h")) + glob.glob(os.path.join(CSRC, "*.hip")))
# registers that no operand can name: a statement that writes one lists it as clobbered, or the compiler may keep a value of its own there
FIXED = ("m0", "vcc", "exec", "scc")


def statements(text):
    """The asm statements, each with its parentheses' content."""
    for m in re.finditer(r"\basm\s*(?:volatile\s*)?\(", text):
        depth, at, quoted = 1, m.end(), False
        while depth:
            c = text[at]
            if c == '"' and text[at - 1] != "\\":
                quoted = not quoted
            if not quoted:
                depth += (c == "(") - (c == ")")
            at += 1
        yield text[m.end():at - 1]


def written(statement):
    """The fixed registers that are the first operand of an instruction in the template."""
    template = "".join(re.findall(r'"((?:[^"\\]|\\.)*)"', re.split(r'"\s*:', statement)[0] + '"'))
    for line in re.split(r"\\n|\\t|;", template):
        word = line.strip().split(None, 1)
        if len(word) == 2 and word[1].split(",")[0].strip() in FIXED:
            yield word[1].split(",")[0].strip()


def test_the_search_finds_what_it_looks_for():
    text = 'asm volatile("s_mov_b32 m0, %0\\n\\ts_nop 0" ::"s"(f((int)a)), "v"(b) : "memory"); asm("v_add %0, %1" : "+v"(m0)); asm("s_mov_b32 m0, %0" ::"s"(a) : "m0");'
    found = list(statements(text))
    assert len(found) == 3 and [list(written(s)) for s in found] == [["m0"], [], ["m0"]]


@pytest.mark.parametrize("path", SOURCES, ids=os.path.basename)
def test_inline_assembly_names_the_fixed_registers_it_writes(path):
    with open(path) as f:
        text = f.read()
    for s in statements(text):
        for r in written(s):
            assert f'"{r}"' in s, f"{r} is written and not listed: {s[:90]}"
