"""Inline assembly of several instructions: what one of them writes must not share a register with an input that a later one
reads, so a vector register that is written there is an early clobber ("=&v", "+&v"). The compiler may otherwise place an input
of the same value in it."""
import glob
import os
import re

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
SOURCES = sorted(p for e in ("hip", "h") for p in glob.glob(os.path.join(HERE, "..", "flyhigh-engine_amd", "csrc", f"*.{e}")))


def blocks(text):
    """(line, instructions, outputs, inputs) of each asm statement."""
    for m in re.finditer(r"\basm\b(?:\s+volatile)?\s*\(", text):
        depth, quoted, i, parts, part = 1, False, m.end(), [], ""
        while depth:
            c = text[i]
            if c == '"' and text[i - 1] != "\\":
                quoted = not quoted
            depth += (c == "(") - (c == ")") if not quoted else 0
            if c == ":" and not quoted and depth == 1:
                parts.append(part)
                part = ""
            elif depth:
                part += c
            i += 1
        parts.append(part)
        code = "".join(re.findall(r'"((?:[^"\\]|\\.)*)"', parts[0]))
        outs, ins = (re.findall(r'"([^"]*)"\s*\(', parts[k]) if len(parts) > k else [] for k in (1, 2))
        yield text.count("\n", 0, m.start()) + 1, [c for c in code.split("\\n") if c.strip()], outs, ins


def wrong(text):
    return [(line, outs) for line, code, outs, ins in blocks(text)
            if len([c for c in code if not c.strip().startswith("s_nop")]) > 1 and any(i in ("v", "a") for i in ins) and
            any("&" not in o for o in outs)]


@pytest.mark.parametrize("path", SOURCES, ids=os.path.basename)
def test_outputs_are_early_clobbers(path):
    with open(path) as f:
        assert not wrong(f.read())


def test_the_rule_sees_a_shared_register():
    two = 'asm("v_add_f32 %0, %0, %1\\n" "v_mul_f32 %0, %0, %2" : "+v"(a) : "v"(b), "v"(c));'
    assert wrong(two) and not wrong(two.replace('"+v"', '"+&v"'))
    assert not wrong('asm("v_add_f32 %0, %0, %1" : "+v"(a) : "v"(b));') and not wrong('asm volatile("" : "+v"(a));')
