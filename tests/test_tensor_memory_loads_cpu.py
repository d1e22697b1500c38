"""tcgen05.ld is asynchronous: a statement that waits for it has to name the registers that it fills, or arithmetic on them may be moved
ahead of the wait.  The sources of the int8 product, since no output shows it until a compiler does so."""
import os
import re

from tests._util import ROOT


def test_every_wait_names_the_registers_that_it_is_for():
    text = open(os.path.join(ROOT, "gemmlib_b200", "csrc", "int8_gemm.cu")).read()
    helper = re.search(r"__device__ __forceinline__ void tmem_ld_wait_for\(.*?\n}\n", text, flags=re.S)
    assert helper and '"+r"(r[' in helper.group()
    rest = text.replace(helper.group(), "")
    assert "tmem_ld_wait()" not in rest
    statements = re.findall(r"asm volatile\((.*?)\);\n", rest, flags=re.S)
    for s in statements:
        assert "wait::ld" not in s or "tcgen05.ld." in s, s
    # loads of this file either wait in their own statement or go to registers that tmem_ld_wait_for names
    for s in statements:
        assert "tcgen05.ld." not in s or "wait::ld" in s, s
    assert len(re.findall(r"tmem_ld_32x32b_x32\(.*?, next\)", rest)) == len(re.findall(r"tmem_ld_32x32b_x\d+\(", rest))
    assert "tmem_ld_wait_for(next)" in rest
