"""CPU: the way out of the attention gradients' blocks after a wait that gave up (csrc/attention_tc_grad.cu), against a model of its barriers.

Two warps issue MMAs.  Each commits what it issued to a barrier and waits, by parity and with a limit, before the block frees its tensor memory; a commit arrives when its own warp's MMAs are
done.  With one barrier for both (a planted mistake) a warp leaves on the other's arrival, or waits for its limit."""
import os
import random
import re

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _leave(rng, barriers):
    """The two warps under one random interleaving; barriers[w]: which one warp w commits to and waits for.  Returns what went wrong."""
    done, pending, stage = [0, 0], [rng.randrange(0, 6), rng.randrange(0, 6)], ["commit", "commit"]
    arrived, polls = [False, False], [0, 0]
    while stage != ["left", "left"]:
        w = rng.randrange(4)
        if w >= 2:                                                     # the tensor cores finish one of a warp's MMAs
            w -= 2
            pending[w] = max(0, pending[w] - 1)
            if stage[w] != "commit" and not pending[w] and not arrived[w]:
                arrived[w] = True
                done[barriers[w]] += 1
        elif stage[w] == "commit":
            stage[w] = "wait"
        elif stage[w] == "wait":
            polls[w] += 1
            if done[barriers[w]] & 1:                                  # try_wait.parity of phase 0: the current phase is an odd one
                if pending[w]:
                    return "left with MMAs in flight"
                stage[w] = "left"
            elif polls[w] > 200:
                return "waited for its limit"
    return None


def _outcomes(barriers):
    return {_leave(random.Random(seed), barriers) for seed in range(500)}


def test_each_warp_waits_for_its_own():
    assert _outcomes((0, 1)) == {None}


def test_the_model_catches_one_barrier_for_both():
    assert _outcomes((0, 0)) >= {"left with MMAs in flight", "waited for its limit"}


@pytest.mark.parametrize("name", ["attention_tc.cu", "attention_tc_grad.cu"])
def test_the_kernels_commit_to_each_such_barrier_once(name):
    with open(os.path.join(ROOT, "fovi_b200", "csrc", name)) as f:
        text = f.read()
    commits, waits = (re.findall(call + r"\(smem_u32\(&hdr->(drain(?:\[\d\])?)\)", text) for call in ("tc_commit", "mbar_try_wait"))
    assert commits and commits == waits and len(set(commits)) == len(commits)
