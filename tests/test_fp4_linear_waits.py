"""How the 4-bit linear waits, read from its source (a wait that never ends can only be shown by reading: on a GPU it would
hang it).  Every wait is bounded, so each can give up; these are the rules that keep a warp together when one does."""
import os
import re

SOURCE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "vrhino_b200", "csrc", "vrb_fp4_linear.cu")


def _text():
    with open(SOURCE) as fh:
        return re.sub(r"//[^\n]*", "", fh.read())


def _block_heads(text, at):
    """The lines that open the blocks around position `at`, up to their brace."""
    open_at = []
    for i, c in enumerate(text[:at]):
        if c == "{":
            open_at.append(i)
        elif c == "}" and open_at:
            open_at.pop()
    return [text[text.rfind("\n", 0, i) + 1:i] for i in open_at]


def test_waits_of_a_warp_have_one_outcome():
    """A wait whose lanes may see different outcomes (the limit, another warp's abort) stands either in the vote of all lanes or
    in code of a single elected thread: a warp that went apart would not meet again at elect.sync or __syncwarp."""
    text = _text()
    calls = [m.start() for m in re.finditer(r"\bwait_barrier\(", text)]
    definition = text.index("bool wait_barrier(") + len("bool ")
    voted, elected, apart = 0, 0, []
    for at in calls:
        if at == definition:
            continue
        head = text[text.rfind("\n", 0, at):at]
        if "__all_sync(0xffffffffu, " in head:
            voted += 1
        elif any("elect_one()" in h for h in _block_heads(text, at)):
            elected += 1
        else:
            apart.append(text[at:text.index("\n", at)])
    assert not apart, apart
    assert voted == 1 and elected == 1      # wait_warp itself, and the split kernel's issuing thread
    assert len(re.findall(r"\bwait_warp\(", text)) >= 7      # its definition, and all other waits


def test_every_wait_is_bounded():
    """No loop on a barrier without the limit: the only try_wait is wait_barrier's, and that ends by time or by an abort."""
    text = _text()
    assert text.count("mbarrier.try_wait") == 1 and "mbarrier.test_wait" not in text
    body = text[text.index("bool wait_barrier("):]
    body = body[:body.index("\n}\n")]
    assert "kWaitNs" in body and "if (*abort) return false;" in body


class _Barrier:
    """An mbarrier of one arrival a phase, as the ring uses it: a wait for a parity passes once a phase of that parity is over."""

    def __init__(self):
        self.over = 0

    def arrive(self):
        self.over += 1

    def passes(self, parity):
        return self.over % 2 != parity


def _walk(ring, fills, lost=None):
    """The copying warp's walk over a ring of buffers, each emptied right after it was filled (but for fill `lost`); whether every
    wait of the last round over the ring passes."""
    empty, slot, phase = [_Barrier() for _ in range(ring)], 0, 1
    for fill in range(fills):
        assert empty[slot].passes(phase)
        if fill != lost:
            empty[slot].arrive()
        slot += 1
        if slot == ring:
            slot, phase = 0, phase ^ 1
    passed = True
    for _ in range(ring):
        passed = passed and empty[slot].passes(phase)
        slot += 1
        if slot == ring:
            slot, phase = 0, phase ^ 1
    return passed


def test_last_round_over_the_ring():
    """Once round more after the last copy: those waits pass when all buffers were emptied, used or not, and not before."""
    for ring in range(1, 7):
        for fills in range(0, 4 * ring + 2):
            assert _walk(ring, fills)
            for lost in range(max(0, fills - ring), fills):
                assert not _walk(ring, fills, lost)


def test_copying_warps_outwait_the_products():
    """Arrivals of finished products on the barriers of empty buffers come on their own time, in the pair kernel from the other
    CTA: both copying warps wait for the last of them before their CTA may end."""
    text = _text()
    loops = re.findall(r"for \(int left = (\w+(?:\.\w+)?); ok && left > 0; --left\) \{\s*ok = wait_warp\(&control\.empty\[slot\], phase, &control\.abort\);"
                       r"\s*if \(\+\+slot == (\w+(?:\.\w+)?)\) \{ slot = 0; phase \^= 1u; \}\s*\}", text)
    assert loops == [("kPairStages", "kPairStages"), ("q.ring", "q.ring")]


def test_tensor_memory_goes_back_before_a_cluster_meets():
    """An allocation of tensor memory waits until the SM has enough of it, and other libraries' kernels take it too.  A CTA of the
    split kernel that held its part while it waited for its cluster, and a pair of such a kernel's CTAs that waits for each other
    likewise, could each hold what the other needs.  So the split kernel allocates, works alone, gives back, and only then meets
    its cluster; the pair kernel, whose CTAs meet before that, leaves no shared memory for another kernel on its SMs."""
    text = _text()
    split = text[text.index("fp4_linear_split_kernel(const __grid_constant__"):]
    split = split[:split.index("\n}\n")]
    assert split.count("tcgen05.alloc") == 1 and split.count("tcgen05.dealloc") == 1
    held = split[split.index("tcgen05.alloc"):split.index("tcgen05.dealloc")]
    assert "cluster_sync" not in held and "barrier.cluster" not in held
    assert "wait_reads()" in held and "__syncthreads();" in held[held.index("wait_reads()"):]
    assert split.count("cluster_sync();") == 2
    pair = re.search(r"static_assert\(sizeof\(PairShared\) <= (\d+) \* 1024", text)
    stages, threads = (int(re.search(rf"constexpr int {name} = (\d+);", text).group(1)) for name in ("kPairStages", "kPairThreads"))
    buffers = stages * (2 * 128 * 128 + 3 * 2048) + 16 * 32 * 64 + 16 * 64 * 4
    assert pair and threads == 576 and 228 * 1024 - 1024 - buffers < 2 * 1024      # what another CTA could have beside it
