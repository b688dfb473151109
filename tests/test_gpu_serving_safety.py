"""The serving operators where calls meet: waits that give up, streams, captured
graphs, buffers that overlap, requests a default could hide."""
import pytest

torch = pytest.importorskip("torch")

from akili_bench_b200 import ops  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def clean_status():
    ops.device_status()
    yield
    assert ops.device_status() == 0


@pytest.mark.parametrize("limit_us", [200, 5000])
def test_warps_that_share_a_barrier_give_up_together(limit_us):
    """One warp's limit passes before the phase completes, the other's does not: neither goes on (it would wait
    for the other at their next barrier); the status would be STATUS_SELFTEST_SHARED."""
    ops.selftest_wait_timeout(limit_us)
    assert ops.device_status() == ops.STATUS_SELFTEST
