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


def _groups_pending(commits, wait):
    """`commits`: the (ring, block) sets of the groups so far, in order; what may still be on its way behind the wait."""
    return [c for group in commits[len(commits) - wait:] for c in group] if wait else []


def test_convolution_rings_that_are_walked_together_share_their_groups():
    """Asynchronous copies are counted by groups of a thread, whichever ring they are for.  With one group for a block of all rings, a
    turn's wait leaves exactly the blocks behind the next one on their way, for one ring as for two; and what is overwritten is the block in
    front, which all lanes are through with."""
    text = source("ttt_short_conv.cu")
    start, turn = block(text, "void start("), block(text, "void turn(")
    assert text.count("cp_async_commit()") == 2 and start.count("cp_async_commit()") == turn.count("cp_async_commit()") == 1
    order = ["cp_async_wait<R::kSlots - 2>()", "__syncwarp()", "rows.advance()", "(more.advance(), ...)", "cp_async_commit()"]
    at = [turn.index(o) for o in order]
    assert at == sorted(at) and turn.count("cp_async_wait") == 1
    assert "k < R::kSlots - 1" in start and start.index("issue(k)") < start.index("cp_async_commit()")
    backward = block(text, "conv_backward_kernel(")
    advance = block(text, "void advance()")
    assert advance.index("++block") < advance.index("issue((block + kSlots - 1) % kSlots)")
    assert "start(begin, live, rows, ups);" in backward
    assert len(re.findall(r"\bturn\(rows, ups\);", backward)) == len(re.findall(r"\bturn\(", backward)) == 2
    slots = {int(v) for v in re.search(r"kSlots = sizeof\(T\) == 2 \? (\d) : (\d)", text).groups()}
    assert slots == {2, 4}
    for s in slots:
        for rings in (1, 2):
            commits = [{(r, k) for r in range(rings)} for k in range(s - 1)]
            for n in range(3 * s):
                pending = _groups_pending(commits, s - 2)
                assert all((r, n) not in pending for r in range(rings))
                assert {k for _, k in pending} == set(range(n + 1, n + s - 1))
                assert (n + s - 1) % s == (n - 1) % s      # the slot that the new block goes to
                commits.append({(r, n + s - 1) for r in range(rings)})
