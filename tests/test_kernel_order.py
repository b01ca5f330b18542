"""Orders inside the kernels that no run can be relied on to show.

Shared memory of another CTA of a cluster may be touched only once that CTA is known to run, and
must not be given up while anything is still on its way into it.  A store that comes too early, or
an arrival that comes too late, is nearly always harmless by luck; so the order is read here from
the kernels' sources.
"""

import re
from pathlib import Path

CSRC = Path(__file__).resolve().parents[1] / "inferkernellab_b200" / "csrc"


def _source(name):
    """A source without its comments, white space as single blanks."""
    text = re.sub(r"//[^\n]*", "", (CSRC / name).read_text())
    return re.sub(r"\s+", " ", text)


def _in_order(text, *parts):
    at = -1
    for part in parts:
        found = text.find(part, at + 1)
        assert found >= 0, f"{part!r} is missing after position {at}"
        at = found


def test_sampler_waits_for_its_cluster_before_the_first_remote_store():
    text = _source("sample.cu")
    load = text[text.index("void load(const L* row)"):text.index("float argument(float l)")]
    assert load.index("cluster_wait()") < load.index("at(lane)->")
    kernel = text[text.index("sample_kernel(const SampleParams p)"):]
    _in_order(kernel, "cluster_arrive_relaxed()", "griddepcontrol.wait", "row.load(logits)")
    # nothing leaves, and nothing touches another CTA, between the arrival and the wait
    before = kernel[:kernel.index("row.load(logits)")]
    assert "return;" not in before and "row.at(" not in before


def test_an_abort_does_not_cut_short_the_wait_for_mmas_in_flight():
    """TMEM is freed after every MMA has ended, after an abort too: that wait must not look at the
    abort flag, as the waits inside the pipelines do."""
    for name in ("fp8_linear.cu", "prefill_tc.cu"):
        text = _source(name)
        assert "mbar_wait_bounded(mma_idle" not in text, name
        _in_order(text, "commit(mma_idle)", "mbar_drain(mma_idle, 0, p.err)", "tmem_dealloc")
    common = _source("common.cuh")
    drain = common[common.index("bool mbar_drain("):]
    assert "abort_flag" not in drain[:drain.index("return true; }")]


def test_both_ctas_of_a_pair_see_the_last_commits_before_they_leave():
    """Rank 0's commits arrive on rank 1's barriers asynchronously, and a cluster barrier does not
    wait for them: rank 1 has to, for the stages' releases and for the last commit."""
    text = _source("fp8_linear.cu")
    producer = text[text.index("int early = 0;"):text.index("sdesc_sw128(smem_u32(stages)")]
    _in_order(producer, "if (kPair && rank == 1) {", "i < it + kStages",
              "mbar_wait_bounded(&empty[i % kStages]", "mbar_drain(mma_idle, 0, p.err)",
              "drain_stages<kStages>")
    teardown = text[text.index("__syncwarp(); if (!kPair && p.splits > 1)"):]
    _in_order(teardown, "if (kPair) cluster.sync();", "tmem_dealloc_pair")
