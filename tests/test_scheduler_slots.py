"""What the scheduler leaves of its slots (host logic, no GPU)."""
import ctypes as C

import numpy as np
import pytest

from qwisp_amd import abi

from .test_scheduler import Fake, dll  # noqa: F401


@pytest.mark.parametrize("budget, rounds", [(0, 1), (0, 3), (1500, 1), (1500, 2), (1500, 4)])
def test_a_scheduler_that_is_destroyed_releases_its_slots(dll, budget, rounds):  # noqa: F811
    """Requests in all states: ended, decoding, in the middle of a prompt, let in but not begun, queued."""
    fake = Fake(slots=4)
    tok, fin = abi.TOKEN_FN(lambda user, job, t: None), abi.FINISH_FN(lambda user, job: None)
    h = C.c_void_p()
    assert dll.sl_sched_create(C.byref(fake.t), budget, tok, fin, None, C.byref(h)) == abi.SL_OK
    for n, g in [(5, 2), (700, 50), (6000, 3), (900, 8), (10, 10), (20, 20)]:
        p = np.full(n, 7, np.int32)
        assert dll.sl_sched_submit(h, p.ctypes.data_as(C.c_void_p), n, g, None, 0) >= 0
    for _ in range(rounds):
        assert dll.sl_sched_round(h) > 0
    assert any(fake.busy)
    dll.sl_sched_destroy(h)
    assert not any(fake.busy) and fake.pos == [0] * 4
