"""Dynamic LDS that is read or written 16 bytes at a time is declared with that alignment: it begins behind the kernel's static LDS, whose size is any multiple of 4."""
import glob
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ik_llama.cpp_amd", "csrc")


def test_dynamic_lds_accessed_as_vectors_is_aligned():
    seen = 0
    for path in sorted(glob.glob(os.path.join(CSRC, "*.hip")) + glob.glob(os.path.join(CSRC, "*.cuh"))):
        text = open(path).read()
        for m in re.finditer(r"extern __shared__ (.*?)(\w+)\[\];", text):
            name = m.group(2)
            names = {name} | set(re.findall(r"\*(\w+) = reinterpret_cast<float \*>\(%s" % name, text))          # (the array and what is derived from it in one step)
            wide = any(re.search(r"reinterpret_cast<(const )?(uint4|float4|f4|u4) \*>\((const )?%s\b" % n, text) for n in names) or any("(%s + " % n in text and "f4 *>(so" in text for n in names)
            if wide:
                seen += 1
                assert "aligned(16)" in m.group(1) or "__align__(16)" in m.group(1), (os.path.basename(path), m.group(0))
    assert seen >= 2
