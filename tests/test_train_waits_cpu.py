"""The waits of the attention training kernels, read from their source: what a GPU must not be made to show."""
import re
from pathlib import Path

import rl_for_mario_b200

SOURCE = Path(rl_for_mario_b200.__file__).parent / "csrc" / "attn_train_sm100.cu"


def code():
    return re.sub(r"//[^\n]*", "", SOURCE.read_text())


def test_no_wait_without_a_limit():
    """A warp leaves its loop when a wait runs out, so whoever may wait for it has to do so with a limit: inside the
    kernels only mbarriers (mbar_wait, bounded), and barriers of the block at a kernel's entry and its end alone."""
    text = code()
    assert not re.search(r"\bnamed_bar|\bbar\.(sync|red|arrive)|\bbarrier\.|mbar_try_wait|__syncthreads_(and|or|count)", text)
    for body in re.split(r"__global__", text)[1:]:
        body = body[:body.index("\n}\n")]
        at = [m.start() for m in re.finditer(r"__syncthreads\(\)", body)]
        if "TcShared* sh" not in body:  # no wait that may fail: every thread reaches every barrier
            assert "mbar" not in body and "return;" not in body and "break;" not in body
            continue
        loops = [m.start() for m in re.finditer(r"while \(true\)", body)]
        assert len(at) == 2 and len(loops) == 1 and at[0] < loops[0] < at[1]
        assert body.index("tmem_dealloc") > at[1]


def test_scores_over_weights_wait_for_their_reader():
    """The PTX ISA orders two MMAs only when they share accumulator and shape.  In the dk, dv kernel the scores of the
    next block may lie where another product still reads its weights: before they are issued the wait for that
    product's commit has to stand, for either half of a block."""
    text = code()
    issue = text[text.index("void issue_keys("):text.index("struct ItemReader")]
    for scores, weights, barrier in (("scores_a(", "weights_a(", "p_taken"), ("scores_b(", "weights_b(", "blk_empty")):
        # Every issue of the scores is behind a wait on the barrier that the weights' commit completes ...
        wait = issue.index(f"warp_wait(&sh->{barrier}")
        assert wait < issue.index(scores) and issue.count(scores) == 1
        # ... which follows the weights directly.
        behind = issue[issue.index(weights):]
        assert behind.index(f"commit(&sh->{barrier}") < 100
    kernel = text[text.index("attn_train_dkv_tc_kernel(const"):]
    assert "OVER = 2 * kBlk + 2 * D + kBlk > (int)kCols" in kernel and "SH::STAGES, OVER>" in kernel
