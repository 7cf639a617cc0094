"""CPU: a model of how a whole warp waits on the parities of a shared-memory ring while one of its lanes works on it.

The tensor-core kernels' loading, issuing and column-summing warps all go through the ring's stages like this: every lane waits
until the stage's barrier has completed the phase of its round, then one lane sends the stage on (by loads, by MMAs' commits or by
an arrive), and the barrier's next phase may complete.  An mbarrier tells a waiting thread one bit: whether the phase of that
parity is the one under way.  The model runs every interleaving of two lanes and of the other side of the ring."""
from collections import deque


def _stuck(stages: int, blocks: int, together: bool) -> bool:
    """Whether some interleaving leaves a lane waiting for good.  together: the lanes meet after each wait."""
    # lane 0 sends, lane 1 only waits; a lane stands before block `b` with its wait still to do (seen = 0) or done (seen = 1);
    # sent: blocks that lane 0 has sent on; given: blocks the other side has made ready.  It makes block b ready once the stage's
    # last block, b - stages, has been sent on.
    start = (0, 0, 0, 0, 0)
    seen, queue = {start}, deque([start])
    while queue:
        at0, seen0, at1, seen1, given = state = queue.popleft()
        nexts = []
        if given < blocks and at0 >= given - stages + 1:
            nexts.append((at0, seen0, at1, seen1, given + 1))

        def ready(block):
            stage, turn = block % stages, block // stages
            done = (given - stage + stages - 1) // stages      # phases the stage's barrier has completed
            return done % 2 != turn % 2                        # the test that parity allows: phase `turn` is not under way

        if at0 < blocks:
            if not seen0:
                if ready(at0):
                    nexts.append((at0, 1, at1, seen1, given))
            elif not together or at1 > at0 or (at1 == at0 and seen1):
                nexts.append((at0 + 1, 0, at1, seen1, given))
        if at1 < blocks:
            if not seen1:
                if ready(at1):
                    nexts.append((at0, seen0, at1, 1, given))
            elif not together or at0 > at1 or (at0 == at1 and seen0):
                nexts.append((at0, seen0, at1 + 1, 0, given))
        if not nexts and (at0 < blocks or at1 < blocks):
            return True
        for s in nexts:
            if s not in seen:
                seen.add(s)
                queue.append(s)
    return False


def test_lanes_that_meet_after_each_wait_never_miss_a_phase():
    for stages in (2, 3, 5):
        for blocks in (1, 2 * stages, 4 * stages + 1):
            assert not _stuck(stages, blocks, together=True), (stages, blocks)


def test_lanes_that_do_not_meet_can():
    """Why they have to: the lane that sends may be two rounds of the ring ahead of one that still polls."""
    for stages in (2, 3, 5):
        assert _stuck(stages, 4 * stages + 1, together=False), stages


def test_role_loops_wait_as_a_whole_warp():
    """Every wait of those loops goes through warp_all."""
    import os
    import re

    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "kernel_optimization_b200", "nn_operators")
    for name in ("gemm/tensor_core_gemm.h", "gemm/tensor_core_gemm_pair.h", "linear/linear_epilogue.h", "layernorm/layernorm_backward.h"):
        text = open(os.path.join(root, name)).read()
        waits = [m.start() for m in re.finditer(r"\bmbar_wait(_remote)?\(", text) if not text[:m.start()].endswith("bool ")]
        assert waits, name
        for at in waits:
            assert text[:at].endswith("warp_all("), (name, text[at - 40:at + 60])


def test_tokens_hand_over_no_data():
    """A relaxed arrive at another CTA's barrier orders nothing behind it: the one there is gives a stage back to be overwritten.
    What is read after a wait was counted on that very barrier by the copies, or handed over by a releasing arrive."""
    import os
    import re

    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "kernel_optimization_b200")
    uses = []
    for folder, _, files in os.walk(root):
        for name in files:
            if name.endswith((".h", ".cu")):
                text = open(os.path.join(folder, name)).read()
                uses += re.findall(r"mbar_arrive_cluster_relaxed\((?!uint32_t)(.*?)\);", text)
    assert uses == ["map_to_cluster_rank(empty_bar(s), 1)"]
