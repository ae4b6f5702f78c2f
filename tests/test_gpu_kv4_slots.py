"""Engines, lanes and schedulers on 4-bit caches: what a question, a read or a refusal leaves behind."""
import ctypes as C

import numpy as np
import pytest

from .test_gpu_kv4_engine import hybrid_model, make  # noqa: F401

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def alone(cfg, dev, jobs, **kw):
    e = make(cfg, dev, max_m=8, max_seq_len=128, **kw)
    out = []
    for p, n in jobs:
        out.append(e.greedy_generate(p, n, chain_k=4).tolist())
        assert e.lib.dll.sl_reset(e.h) == 0
    e.close()
    return out


def jobs_of(sizes, seed):
    rng = np.random.default_rng(seed)
    return [(rng.integers(0, 4096, n).tolist(), g) for n, g in sizes]


def test_asking_whether_a_request_fits_changes_nothing(hybrid_model):  # noqa: F811
    from qwisp_amd.engine import LaneScheduler
    cfg, dev = hybrid_model
    base = make(cfg, dev, page_size=16, n_pages=8, max_m=8, max_seq_len=128)
    sched = LaneScheduler(base, slots=3, chunk_rows=8, max_seq_len=128, token_budget=16, kv_budget_tokens=384)
    jobs = jobs_of([(30, 20), (10, 6), (50, 40)], 50)
    for _ in range(20):
        assert sched.table.can_admit(sched.table.ctx, 60, 100) == 1
    for p, n in jobs:
        sched.submit(p, n)
    assert sched.run(max_rounds=400) == alone(cfg, dev, jobs)
    assert base.kv4_free_pages() == 8
    sched.close()
    base.close()


@pytest.mark.parametrize("kv4", [True, False])
def test_slots_of_a_scheduler_that_is_destroyed_serve_the_next(hybrid_model, kv4):  # noqa: F811
    """The first is destroyed while one request decodes, one is in the middle of its prompt and one has not begun."""
    from qwisp_amd import abi
    from qwisp_amd.engine import LaneScheduler
    cfg, dev = hybrid_model
    base = make(cfg, dev, kv4=kv4, page_size=16, n_pages=24, max_m=8, max_seq_len=128)
    sched = LaneScheduler(base, slots=3, chunk_rows=8, max_seq_len=128, token_budget=9, kv_budget_tokens=384)
    jobs = jobs_of([(5, 60), (70, 20), (40, 30)], 51)
    for p, n in jobs:
        sched.submit(p, n)
    for _ in range(3):
        assert sched.round() == 3
    sched.lib.dll.sl_sched_destroy(sched.h)
    sched.h = C.c_void_p()
    if kv4:
        assert base.kv4_free_pages() == 24
    assert sched.lib.dll.sl_sched_create(C.byref(sched.table), 16, sched._tok, sched._fin, None, C.byref(sched.h)) == abi.SL_OK
    sched.streams.clear()
    for p, n in jobs:
        sched.submit(p, n)
    assert sched.run(max_rounds=400) == alone(cfg, dev, jobs, kv4=kv4)
    sched.close()
    base.close()


def test_a_request_that_others_pages_keep_out_for_good_ends(hybrid_model):  # noqa: F811
    """The base's own sequence holds three of eight pages: a request for seven of them would wait for ever."""
    from qwisp_amd.engine import LaneScheduler
    cfg, dev = hybrid_model
    base = make(cfg, dev, page_size=16, n_pages=8, max_m=8, max_seq_len=128)
    for i in range(5):
        assert base.step_argmax([i] * 8) is not None
    sched = LaneScheduler(base, slots=2, chunk_rows=8, max_seq_len=128, token_budget=16, kv_budget_tokens=256)
    jobs = jobs_of([(20, 10), (60, 50), (30, 40)], 52)
    for p, n in jobs:
        sched.submit(p, n)
    want = alone(cfg, dev, jobs)
    assert sched.run(max_rounds=400) == [want[0], [], want[2]]
    assert base.kv4_free_pages() == 5
    sched.close()
    base.close()


def test_large_requests_are_not_overtaken_for_ever(hybrid_model):  # noqa: F811
    """One request that needs all pages among many small ones: it begins before the small ones behind it."""
    from qwisp_amd import abi
    from qwisp_amd.engine import LaneScheduler
    cfg, dev = hybrid_model
    base = make(cfg, dev, page_size=16, n_pages=8, max_m=8, max_seq_len=128)
    sched = LaneScheduler(base, slots=3, chunk_rows=8, max_seq_len=128, token_budget=12, kv_budget_tokens=384)
    jobs = jobs_of([(20, 10), (9, 20), (70, 50)] + [(8, 6)] * 8, 53)
    ended = []
    sched._fin2 = abi.FINISH_FN(lambda user, job: ended.append(job))
    sched.lib.dll.sl_sched_destroy(sched.h)
    sched.h = C.c_void_p()
    assert sched.lib.dll.sl_sched_create(C.byref(sched.table), 12, sched._tok, sched._fin2, None, C.byref(sched.h)) == abi.SL_OK
    for p, n in jobs:
        sched.submit(p, n)
    assert sched.run(max_rounds=1000) == alone(cfg, dev, jobs)
    assert ended.index(2) == 2
    sched.close()
    base.close()


def test_reading_a_cache_changes_nothing(hybrid_model):  # noqa: F811
    """A rewound sequence still has the rows behind the rewind, and reading what is in front of it leaves them there."""
    cfg, dev = hybrid_model
    e = make(cfg, dev, page_size=16, max_m=8, max_seq_len=96)
    for i in range(5):
        assert e.step_argmax([i] * 8) is not None
    early = e.full_snapshot()
    for i in range(3):
        assert e.step_argmax([9 + i] * 8) is not None
    late, free = e.full_snapshot(), e.kv4_free_pages()
    want = int(e.step_argmax([7])[0])
    assert e.full_restore(late) and e.full_restore(early) and e.position == 40
    k, v = e.read_layer_cache(3)
    assert k.shape[1] == 40 and np.isfinite(k).all()
    assert e.full_restore(late) and e.position == 64 and e.kv4_free_pages() == free
    assert int(e.step_argmax([7])[0]) == want
    e.close()
