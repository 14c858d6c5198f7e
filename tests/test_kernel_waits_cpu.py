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
