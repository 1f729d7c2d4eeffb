"""The hand-over between the warps of the fp8 product for few tokens, as a model on the CPU.

An accumulator's "full" barrier completes a phase with two arrivals: the commit of the step's UMMAs and the warp that has written the step's
scales. Commits of several steps are on their way at once and nothing orders their arrivals. The scale warp's arrival must not complete a phase
that a late commit still belongs to: the next commit would then stand for the step after it, and the epilogue would read an accumulator early.
"""

import random
import re

import pytest

from tests.test_programmatic_launch_cpu import kernels

SLOTS, BATCH = 4, 2


def slots_waited_for() -> list[int]:
    """The steps of a batch whose barriers the scale warp waits for before it arrives on all of them, from the kernel's source."""
    body = kernels("fp8_block_mm_sm100.cu")["small_kernel"][1]
    branch = body[body.index("constexpr int kBatch = L::kBatch") :]
    before = re.search(r"const int before = ([^;]*);", branch)[1].replace(" ", "")
    steps = {"i0+kBatch-1-L::kSlots": [BATCH - 1], "i0+j-L::kSlots": list(range(BATCH))}[before]
    if len(steps) > 1:
        loop = branch[: branch.index("const int before")]
        assert re.search(r"for \(int j = 0; j < kBatch; \+\+j\) \{\s*$", loop)
    return steps


def epilogue_reads_early(waited: list[int], seed: int, steps: int = 16) -> bool:
    rng = random.Random(seed)
    arrivals, phase = [0] * SLOTS, [0] * SLOTS      # of the barriers
    issued, on_their_way, arrived = 0, set(), set()  # commits
    batch, read = 0, 0                               # batches the scale warps have done, steps the epilogue has read

    def complete(step):
        return phase[step % SLOTS] > step // SLOTS

    def arrive(step):
        slot = step % SLOTS
        arrivals[slot] += 1
        if arrivals[slot] == 2:
            arrivals[slot] = 0
            phase[slot] += 1

    while read < steps:
        moves = []
        if issued < steps and (issued < SLOTS or read > issued - SLOTS):
            moves.append("issue")
        moves += [("commit", s) for s in on_their_way]
        first = batch * BATCH
        if first < steps and all(first + j < SLOTS or complete(first + j - SLOTS) for j in waited):
            moves.append("scales")
        if complete(read):
            moves.append("read")
        assert moves, "the model is stuck"
        move = rng.choice(sorted(moves, key=str))
        if move == "issue":
            on_their_way.add(issued)
            issued += 1
        elif move == "scales":
            for j in range(BATCH):
                arrive(first + j)
            batch += 1
        elif move == "read":
            if read not in arrived:
                return True
            read += 1
        else:
            on_their_way.remove(move[1])
            arrived.add(move[1])
            arrive(move[1])
    return False


def test_the_model_sees_an_early_read():
    assert any(epilogue_reads_early([BATCH - 1], seed) for seed in range(500))


@pytest.mark.parametrize("seeds", [range(0, 500), range(500, 1000)], ids=["a", "b"])
def test_no_order_of_arrivals_lets_the_epilogue_read_early(seeds):
    waited = slots_waited_for()
    assert not any(epilogue_reads_early(waited, seed) for seed in seeds)


def test_a_cta_that_gave_up_takes_its_cluster_along():
    """With the contraction split over a cluster every CTA adds the partial sums of all: none may add those of a CTA whose wait has run out. The
    abort flag is a word of the CTA's own, so it has to reach the peers before the barrier behind which they look at theirs."""
    body = re.sub(r"\s+", " ", kernels("fp8_block_mm_sm100.cu")["small_kernel"][1])
    assert "abort_flag = tmem_slot + 1;" in body
    barrier, look = body.index("cluster_sync_all()"), body.index("column < p.width && !guard.aborted()")
    told = body.find("if (warp == 0 && lane < splits && guard.aborted()) st_shared_cluster_u32(map_to_cta(smem_u32(tmem_slot + 1), static_cast<uint32_t>(lane)), 1u);")
    assert -1 < told < barrier < look
    assert "__syncthreads(); if (splits > 1) {" in body[told - 60 : told]   # every warp of this CTA has set the flag by then, if it does


@pytest.mark.parametrize("kernel,barrier,condition", [("small_kernel", "empty", "i + L::kStages < steps"), ("pair_kernel", "load_empty", "left > kPairStages")])
def test_no_commit_that_nobody_waits_for(kernel, barrier, condition):
    """A commit arrives on its own. Where nobody waits for it, the arrival may come when the CTA (for a pair: the peer) has ended and its shared
    memory is another one's. The loader waits for a stage's release before it fills the stage again: for all of them but those of the last round."""
    body = re.sub(r"\s+", " ", kernels("fp8_block_mm_sm100.cu")[kernel][1])
    commits = [m.start() for m in re.finditer(r"umma_commit(_pair)?\([^;]*[&(]" + barrier + r"\[", body)]
    assert len(commits) == 1
    assert f"if ({condition})" in body[commits[0] - 140 : commits[0]]
    stages, steps = 4, 11
    waited = [i - stages for i in range(steps) if i >= stages]      # the fill of step i waits for the release of step i - stages
    assert [i for i in range(steps) if i + stages < steps] == [i for i in range(steps) if steps - i > stages] == waited
