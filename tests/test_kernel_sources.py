"""What the kernel sources may not say: vector instructions inside asm statements."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "spokennlp_amd", "csrc")


def _asm_statements(text):
    """the template strings of every asm statement, comments taken out first"""
    text = re.sub(r"//[^\n]*|/\*.*?\*/", "", text, flags=re.S)
    for m in re.finditer(r'\basm\b(?:\s+volatile)?\s*\(\s*((?:"(?:[^"\\]|\\.)*"\s*)+)', text):
        yield "".join(re.findall(r'"((?:[^"\\]|\\.)*)"', m.group(1)))


def test_the_scanner_finds_what_it_looks_for():
    assert list(_asm_statements('asm("v_cvt %0, %1" : "=v"(r) : "v"(x));')) == ["v_cvt %0, %1"]
    assert list(_asm_statements('// asm("v_cvt")\nasm volatile("s_nop 0\\n\\t" "ds_read %0" :: "v"(x));')) == ["s_nop 0\\n\\tds_read %0"]


def test_no_vector_arithmetic_in_asm_statements():
    """the result of a transcendental or matrix instruction needs wait states before a vector instruction reads it; the compiler puts them in for its own
    instructions only, so one inside an asm statement reads the register's old value whenever the scheduler brings the two together"""
    found = []
    for f in sorted(os.listdir(CSRC)):
        if f.endswith((".hip", ".h")):
            for s in _asm_statements(open(os.path.join(CSRC, f)).read()):
                if re.search(r"\bv_\w+", s):
                    found.append((f, s))
    assert not found, found


def test_wide_buffer_stores_have_no_scalar_offset():
    """raw_buffer_store of 12 or 16 bytes: with a scalar offset in a register the compiler leaves out the two wait states that keep the data registers from being
    rewritten while the store still reads them (it puts them in where that offset is the constant 0)"""
    found, calls = [], 0
    for f in sorted(os.listdir(CSRC)):
        if f.endswith((".hip", ".h")):
            text = re.sub(r"//[^\n]*|/\*.*?\*/", "", open(os.path.join(CSRC, f)).read(), flags=re.S)
            for m in re.finditer(r"raw_(?:ptr_)?buffer_store_b(?:96|128)\((.*?)\);", text):
                calls += 1
                if not re.search(r",\s*0\s*,\s*\w+\s*$", m.group(1)):
                    found.append((f, m.group(0)))
    assert calls and not found, found
