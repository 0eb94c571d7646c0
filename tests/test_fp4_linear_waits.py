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
    assert len(re.findall(r"\bwait_warp\(", text)) == 7      # its definition, and all other waits


def test_every_wait_is_bounded():
    """No loop on a barrier without the limit: the only try_wait is wait_barrier's, and that ends by time or by an abort."""
    text = _text()
    assert text.count("mbarrier.try_wait") == 1 and "mbarrier.test_wait" not in text
    body = text[text.index("bool wait_barrier("):]
    body = body[:body.index("\n}\n")]
    assert "kWaitNs" in body and "if (*abort) return false;" in body
