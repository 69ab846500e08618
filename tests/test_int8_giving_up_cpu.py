"""The int8 kernels when a copy is late past the limit of the waits, on a model of one CTA's roles: the TMA
lane, the MMA lane and the epilogue (csrc/igemm.cuh, csrc/gemm_ckpt.cuh, csrc/gemm_ckpt_narrow.cuh). A wait
that runs out records a fault; every other wait then gives up as well. What must hold whatever is late and
whoever notices: no copy is in flight when the CTA leaves or when its ring is used for something else, and
nothing is stored from sums that are not there. The two decisions that this rests on are read from the
kernels' source: the TMA lane waits for its last copies whether or not it gave up itself, and the MMA lane
says that the sums are there only if they are."""
import itertools
import re

import pytest

from c3_b200.build import CSRC

NEVER = 10 ** 9
LIMIT = 100  # of a wait
DRAIN = 1000  # of the wait for copies in flight


def run(late, stages, blocks, always_drains, says_only_if_there):
    """One CTA over `blocks` K blocks in a ring of `stages`; late: {block: when its copy lands}."""
    lands = {}  # block -> time
    fault = NEVER  # when it was recorded

    def lands_at(b, issued):
        return late.get(b, issued + 1)

    # The two lanes depend on one another: block b is issued when b - stages has been read, and read when
    # its copy has landed. Times follow in order of b.
    read = {}
    issue_end, mma_ok, producer_ok = 0, True, True
    t_p = t_m = 0
    for b in range(blocks):
        if producer_ok:
            need = read.get(b - stages, 0) if b >= stages else 0
            if b >= stages and (b - stages) not in read:  # the MMA lane gave up: so does this one
                producer_ok = False
            else:
                t_p = max(t_p, need)
                lands[b] = lands_at(b, t_p)
        if not mma_ok or b not in lands:
            mma_ok = False
            continue
        if lands[b] > t_m + LIMIT:
            fault, mma_ok = min(fault, t_m + LIMIT), False
            t_m = t_m + LIMIT
        else:
            t_m = max(t_m, lands[b]) + 1
            read[b] = t_m
    producer_leaves = t_p
    if always_drains or not producer_ok:
        for b in lands:
            producer_leaves = max(producer_leaves, min(lands[b], t_p + DRAIN))
    says = mma_ok or not says_only_if_there
    epilogue_stores = says  # else the fault word ends its wait
    leaves = max(producer_leaves, t_m)
    in_flight = [b for b, t in lands.items() if t > t_m and epilogue_stores]  # over the ring, and at exit
    at_exit = [b for b, t in lands.items() if t > leaves]
    return epilogue_stores and len(read) < blocks, in_flight, at_exit, fault


CASES = [(s, n, late) for s, n in itertools.product((1, 2, 4, 8), (1, 2, 4, 8, 20))
         for late in [{}] + [{b: 150 + 7 * b} for b in range(n)] + [{b: 150, n - 1: 400} for b in range(n)]]


def test_nothing_is_stored_or_left_in_flight():
    late_ones = 0
    for stages, blocks, late in CASES:
        unfinished, over_ring, at_exit, fault = run(late, stages, blocks, True, True)
        assert not unfinished and not over_ring and not at_exit, (stages, blocks, late)
        late_ones += fault < NEVER
    assert late_ones > 100


def test_each_decision_is_needed():
    assert any(run(late, s, n, False, True)[2] for s, n, late in CASES)
    assert any(run(late, s, n, True, False)[0] for s, n, late in CASES)


def _kernel(file, kernel):
    text = (CSRC / file).read_text()
    start = text.index(f"    {kernel}(const __grid_constant__")
    end = text.find("__global__", start)
    return re.sub(r"//[^\n]*", "", text[start:end if end > 0 else len(text)])


def _roles(body):
    """The TMA lane's code, the MMA lane's, and what comes after all roles' loops."""
    producer = body[body.index("if (warp == 0) {"):body.index("else if (warp == 1) {")]
    mma = body[body.index("else if (warp == 1) {"):]
    return producer, mma[:mma.index("__syncwarp();")], body[body.rindex("tc_fence_before();"):]


def _drain(armed, phases):
    return rf"if \({armed} & \(1u << t\)\) gemm::drain_wait\(&full\[t\], \({phases} >> t\) & 1u\);"


@pytest.mark.parametrize("file,kernel", [("igemm.cuh", "igemm_pair_kernel"), ("gemm_ckpt.cuh", "dw_kernel")])
def test_the_pair_kernels_decide_so(file, kernel):
    """The leader's TMA lane drains behind no condition of its own; the sums are announced after a break."""
    producer, mma, _end = _roles(_kernel(file, kernel))
    assert re.search(r"\}\s*if \(leader\) \{\s*for \(int t = 0; t < STAGES; \+\+t\)\s*" + _drain("armed", "armed_par"), producer)
    assert mma.count("acc_full") == 1
    assert re.search(r"if \(!ok\) break;\s*umma_commit_pair_mc\(&acc_full", mma)


@pytest.mark.parametrize("file,kernel", [("igemm.cuh", "igemm_narrow_kernel"), ("gemm_ckpt_narrow.cuh", "dw_narrow_kernel")])
def test_the_small_tile_kernels_decide_so(file, kernel):
    """The drain is at the end, where the MMA lane gave up: otherwise that lane saw every copy land. The CTA
    meets at a barrier between the two."""
    producer, mma, end = _roles(_kernel(file, kernel))
    assert re.search(r"if \(!ok\) \*gave_up = 1u;\s*uint64_t\* done = ok \? acc_full : drain;\s*umma_commit\(done\);", mma)
    assert mma.count("acc_full") == 1
    assert re.search(r"__syncthreads\(\);\s*if \(threadIdx.x == 0 && \*gave_up != 0u\)\s*for \(int t = 0; t < \S+; \+\+t\)\s*"
                     + _drain(r"asked\[0\]", r"asked\[1\]"), end)
    assert re.search(r"asked\[0\] = armed;\s*asked\[1\] = armed_par;\s*\}\s*__syncwarp", producer)


def test_a_warp_gives_up_as_a_whole():
    """Where all lanes of a warp wait, one that gave up alone would leave the others in a shuffle or vote that
    names it: such waits are put to the vote themselves. The TMA and MMA roles are one lane each."""
    for file, roles in (("quant.cu", 0), ("igemm.cuh", 5), ("gemm_ckpt.cuh", 3), ("gemm_ckpt_narrow.cuh", 3)):
        text = re.sub(r"//[^\n]*", "", (CSRC / file).read_text())
        voted = len(re.findall(r"__all_sync\(0xffffffffu, mbar_wait\(", text))
        assert voted > 0 and len(re.findall(r"mbar_wait\(", text)) == voted + roles, file
