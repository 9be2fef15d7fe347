"""Order of the layer-side kernels' shared memory accesses, read from their sources: what lies between an access and the one that
must not overtake it.  Shuffles order no memory."""
import os
import re

CSRC = os.path.join(os.path.dirname(__file__), "..", "ttt_tk_b200", "csrc")


def source(name):
    text = open(os.path.join(CSRC, name)).read()
    return re.sub(r"//[^\n]*", "", text)


def block(text, start):
    """The text from `start` to the end of the braces that open behind it."""
    i = text.index("{", text.index(start))
    depth, j = 0, i
    while True:
        depth += {"{": 1, "}": -1}.get(text[j], 0)
        j += 1
        if not depth:
            return text[i:j]


def test_scan_backward_reads_a_token_before_a_lane_overwrites_it():
    """delta x and dy of a token are read by all lanes of its channel, and the lanes that end up with the sums put those in their place."""
    body = block(source("ttt_ssm_scan_sm100.cu"), "scan_backward_kernel(")
    walk = block(body, "for (int k = kSub - 1; k >= 0; --k)")
    stores = [m.start() for m in re.finditer(r"reinterpret_cast<float\*>\(m\.u \+", walk)]
    reads = [m.start() for m in re.finditer(r"=[^;=]*m\.u[ \[+]", walk) if "float*>(" not in m.group()]
    assert len(stores) == 2 and len(reads) == 2 and max(reads) < min(stores)
    assert "__syncwarp();" in walk[max(reads):min(stores)]
