"""Waits of the serving kernels that a run cannot show to be missing, read from their source."""

from __future__ import annotations

from pathlib import Path

CSRC = Path(__file__).resolve().parents[1] / "torque_mlx_b200" / "csrc"


def body(name: str, start: str, end: str) -> str:
    text = (CSRC / name).read_text()
    at = text.index(start)
    return text[at:text.index(end, at)]


def test_verification_waits_for_its_cluster_before_it_writes_to_it():
    """A CTA's shared memory may be written by another one only once it has started: every CTA arrives at the cluster's
    barrier on entry, and the wait comes before the first store."""
    kernel = body("tq_verify.cu", "verify_kernel(const VerifyArgs a) {", "int launch_verify(")
    arrive, wait, store = (kernel.index(x) for x in ("cluster_arrive();", "cluster_wait();", "st.shared::cluster"))
    assert arrive < kernel.index("grid_wait();") < wait < store


def test_many_row_attention_leaves_a_unit_by_one_decision():
    """Softmax and products meet at a barrier around every unit.  Whether a wait gave up is written by others at any
    time, so a thread may not leave on what it reads there by itself: the barrier at the unit's end decides for all."""
    kernel = body("tq_paged_prefill.cu", "paged_prefill_kernel(const AttendArgs a) {", "constexpr int kJoinRows")
    assert "if (failed)" not in kernel
    assert kernel.count("gave_up = meet_any<Shape::kMeeting>(!ok || failed);") == 2
    assert kernel.count("for (Unit u; !gave_up && line.next(u);)") == 2
    # every wait within the kernel has a limit
    assert kernel.count("bar_wait(") == 0 and "mbarrier.try_wait" not in kernel
