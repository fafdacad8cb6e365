"""What the sources of the device-memory operators have to state for the compiler, checked without a GPU."""
import glob
import os
import re

OPS = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "video-description-with-spatial-temporal-attention_amd", "csrc", "ops")


def test_byte_arrays_in_lds_state_their_alignment():
    """Bytes in LDS are read several at a time; an array of bytes promises an address of any alignment unless it says more."""
    seen = 0
    for path in sorted(glob.glob(os.path.join(OPS, "*.hip")) + glob.glob(os.path.join(OPS, "*.h"))):
        for line in open(path):
            m = re.search(r"__shared__\s+(.*?)\b(uint8_t|unsigned char|char|int8_t)\s+\w+\[", line)
            if m:
                seen += 1
                assert "aligned(" in m.group(1), "%s: %s" % (os.path.basename(path), line.strip())
    assert seen
