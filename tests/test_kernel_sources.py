"""What the kernel sources may not say."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "spokennlp_amd", "csrc")


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
