"""Dynamic shared memory of the kernels: an array of bytes, which others are laid over, says its alignment - without one it starts wherever the static
arrays in front of it end, at any byte (no GPU)."""
import glob
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "evotrees.jl_amd", "csrc")


def test_byte_arrays_say_their_alignment():
    found = 0
    for path in sorted(glob.glob(os.path.join(CSRC, "*.h*"))):
        with open(path) as f:
            for number, line in enumerate(f, 1):
                m = re.search(r"extern __shared__ (.*?)\b(\w+)\[\]", line)
                if m is None:
                    continue
                found += 1
                if re.search(r"\b(char|uint8_t|int8_t|uint16_t|int16_t|short)\b", m.group(1)):
                    align = re.search(r"__align__\((\d+)\)", m.group(1))
                    assert align and int(align.group(1)) >= 8, "%s:%d: %s" % (os.path.basename(path), number, line.strip())
    assert found >= 10
