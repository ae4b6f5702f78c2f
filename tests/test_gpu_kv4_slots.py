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


@pytest.mark.parametrize("hybrid", [False, True])
def test_steps_and_cache_calls_take_no_memory(hybrid_model, hybrid):  # noqa: F811
    """All that they need is there once the engine and its lanes are: a device that fills up later ends no step.  (The first of two
    engines goes the same way before, so that what the runtime takes for a kernel's first launch has been taken.)"""
    from . import kv4_ref as ref
    cfg, dev = hybrid_model
    for first in (True, False):
        e = make(cfg, dev, page_size=64, n_pages=80, max_m=64, max_seq_len=2048)
        e.set_hybrid(hybrid)
        lanes = [e.new_lane(max_m=512 if i == 0 else 16, max_seq_len=2048) for i in range(3)]
        lanes[0].set_hybrid(hybrid)
        rng = np.random.default_rng(54)
        torch.cuda.synchronize()
        free = torch.cuda.mem_get_info()[0]
        kept = [(e, rng.normal(size=(2, 700, 256)).astype(np.float16)), (lanes[1], rng.normal(size=(2, 1025, 256)).astype(np.float16))]
        for x, rows in kept:
            assert x.load_layer_cache(3, rows, rows[:, ::-1])
        assert e.step_argmax([1] * 64) is not None and e.chained_step_argmax(3, 4) is not None and e.step_argmax([2] * 7) is not None
        for n in (512, 1, 300, 5):
            assert lanes[0].forward_tokens([4] * n, on_device=True)
        assert e.lane_step_argmax(lanes[::-1], [1, 2, 3]) is not None
        for x, rows in kept:
            k, v = x.read_layer_cache(3)
            n = rows.shape[1]
            for got, y in ((k, rows), (v, rows[:, ::-1])):
                assert np.array_equal(got[:, :n], ref.values(ref.quantise(y.astype(np.float64))).astype(np.float32).astype(np.float16))
        torch.cuda.synchronize()
        assert first or torch.cuda.mem_get_info()[0] == free
        for x in lanes:
            x.close()
        e.close()


def test_long_caches_are_loaded_and_read_in_pieces(hybrid_model):  # noqa: F811
    """More rows than are on their way at once (a few thousand on an engine of single rows)."""
    from . import kv4_ref as ref
    cfg, dev = hybrid_model
    e = make(cfg, dev, page_size=128, max_m=1, max_seq_len=20000)
    rng = np.random.default_rng(55)
    k, v = (rng.normal(size=(2, 19999, 256)).astype(np.float16) for _ in range(2))
    assert e.load_layer_cache(3, k, v) and e.position == 19999
    for got, x in zip(e.read_layer_cache(3), (k, v)):
        assert np.array_equal(got, ref.values(ref.quantise(x.astype(np.float64))).astype(np.float32).astype(np.float16))
    e.close()


def test_a_run_that_does_not_fit_changes_nothing(hybrid_model):  # noqa: F811
    cfg, dev = hybrid_model
    e = make(cfg, dev, page_size=16, n_pages=4, max_m=8, max_seq_len=128)
    assert e.greedy_generate([5] * 60, 6) is None and e.gpu_fault is None
    assert e.position == 0 and e.kv4_free_pages() == 4
    assert e.spec_generate([5] * 60, 6) is None and e.position == 0 and e.kv4_free_pages() == 4
    assert e.greedy_generate([5] * 60, 5) is not None and e.position == 64
    e.close()
