"""Inline assembly names the special registers that it writes: the compiler keeps its own values there and learns of a change in no other way."""
import glob
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "inferflow_amd", "csrc")
WRITES = {"m0": r"\bs_\w+ m0\b", "vcc": r"\b(v_cmp_\w+|s_mov_b64|s_\w+_b64) vcc\b", "exec": r"\b(s_\w+_b64|v_cmpx_\w+) exec\b", "scc": r"\bs_(cmp|add|sub|and|or|xor|lshl|lshr|bitcmp)\w*_\w+ "}


def statements(text):
    """(place, what stands in the parentheses) of each asm statement"""
    for m in re.finditer(r"\basm\s*(?:volatile)?\s*\(", text):
        depth, k, quoted = 1, m.end(), False
        while depth:
            c = text[k]
            if c == "\\":
                k += 1
            elif c == '"':
                quoted = not quoted
            elif not quoted:
                depth += (c == "(") - (c == ")")
            k += 1
        yield m.start(), text[m.end():k - 1]


def unnamed(text):
    bad = []
    for at, body in statements(text):
        strings = re.sub(r'"\s*"', "", body)
        code = re.match(r'\s*"((?:[^"\\]|\\.)*)"', strings)
        code = code.group(1).replace("\\n", "\n").replace("\\t", " ") if code else ""
        named = set(re.findall(r'"(m0|vcc|exec|scc)"', body[len(body) - len(body.split(":")[-1]):]))
        bad += [(text.count("\n", 0, at) + 1, r) for r, form in WRITES.items() if re.search(form, code) and r not in named]
    return bad


@pytest.mark.parametrize("path", sorted(glob.glob(os.path.join(CSRC, "**", "*.h"), recursive=True) + glob.glob(os.path.join(CSRC, "**", "*.hip"), recursive=True)), ids=os.path.basename)
def test_special_registers_are_named(path):
    assert unnamed(open(path).read()) == []


def test_the_reader_of_statements_finds_them():
    assert unnamed('asm volatile("s_cmp_eq_u32 %1, 0\\n\\ts_mov_b32 m0, %0" ::"s"(f(a, b)), "s"(c) : "scc");') == [(1, "m0")]
    assert unnamed('x;\nasm volatile("s_mov_b32 m0, %0" ::"s"(to) : "memory", "m0");') == []
    assert unnamed('asm volatile("v_cmp_lt_f32 vcc, %0, %1" ::"v"(a), "v"(b));') == [(1, "vcc")]
    assert unnamed('asm("" : "+v"(a)); asm volatile("s_waitcnt vmcnt(0)\\n\\ts_barrier" ::: "memory");') == []
