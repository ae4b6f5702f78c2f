"""Engines and lanes whose attention layers keep their keys and values in 4 bits (sl_set_kv4)."""
import numpy as np
import pytest

from . import kv4_ref as ref
from .gpu_util import device_and_host_model, same_bits

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def make(cfg, model, kv4=True, page_size=16, n_pages=0, **kw):
    from qwisp_amd.engine import SeedlessFusedForward
    e = SeedlessFusedForward(cfg, model, **kw)
    if kv4:
        e.set_kv4(page_size, n_pages)
    return e


@pytest.fixture(scope="module")
def hybrid_model():
    from qwisp_amd import synth
    cfg = synth.ModelConfig(n_layers=4, n_experts=16, vocab=4096)
    return cfg, device_and_host_model(cfg)[0]


@pytest.fixture(scope="module")
def attn_model():
    from qwisp_amd import synth
    cfg = synth.ModelConfig(n_layers=1, n_experts=8, vocab=0, layer_types=("attn",))
    return (cfg,) + device_and_host_model(cfg)


PROMPTS = [[3, 1415, 926, 535, 897], list(range(7, 60)), [2718], [9, 9, 9, 1, 2, 3] * 5]


def test_lanes_give_the_tokens_of_a_sequence_alone(hybrid_model):
    """Sequences of up to 128 tokens: batched steps, chains and single steps are the same bits."""
    from qwisp_amd.engine import LaneScheduler
    cfg, dev = hybrid_model
    alone = make(cfg, dev, max_m=8, max_seq_len=128)
    want = []
    for p in PROMPTS:
        want.append(alone.greedy_generate(p, 20, chain_k=4).tolist())
        assert alone.lib.dll.sl_reset(alone.h) == 0
    base = make(cfg, dev, page_size=32, n_pages=12, max_m=8, max_seq_len=128)
    sched = LaneScheduler(base, slots=3, chunk_rows=8, max_seq_len=128)
    for p in PROMPTS:
        sched.submit(p, 20)
    assert sched.run() == want
    sched.close()
    # and with the lanes of one step handed over in another order than they were made
    lanes = [base.new_lane(max_m=8, max_seq_len=128) for _ in PROMPTS]
    last = [int(l.greedy_generate(p, 1)[0]) for l, p in zip(lanes, PROMPTS)]
    got = [[t] for t in last]
    order = [2, 0, 3, 1]
    for _ in range(10):
        out = base.lane_step_argmax([lanes[i] for i in order], [got[i][-1] for i in order])
        for i, t in zip(order, out):
            got[i].append(int(t))
    assert got == [w[:11] for w in want]
    for l in lanes:
        l.close()
    base.close()
    alone.close()


def test_rollback_restore_and_reset(hybrid_model):
    cfg, dev = hybrid_model
    e = make(cfg, dev, max_m=8, max_seq_len=96)
    e.forward_tokens(PROMPTS[1][:8])
    for i in range(1, 6):
        e.forward_tokens(PROMPTS[1][8 * i:8 * i + 8])
    full, snap = e.full_snapshot(), e.snapshot()
    a = e.step_argmax([5, 6, 7])
    cache = e.read_layer_cache(3)
    assert e.rollback_one_step(snap)
    b = e.step_argmax([5, 6, 7])
    again = e.read_layer_cache(3)
    assert a.tolist() == b.tolist() and all(same_bits(x, y) for x, y in zip(cache, again))
    c = e.chained_step_argmax(int(b[-1]), 6)
    assert e.full_restore(full) and e.position == 48
    assert e.step_argmax([5, 6, 7]).tolist() == a.tolist()
    assert [int(e.step_argmax([t])[0]) for t in [int(a[-1])] + c[:-1].tolist()] == c.tolist()
    late = e.full_snapshot()                                   # 57 tokens
    assert e.full_restore(full) and e.step_argmax([1]) is not None       # pages behind 49 tokens have gone back
    assert not e.full_restore(late) and e.gpu_fault is None
    assert e.persistent_state_data() is None and e.lib.dll.sl_persist_size(e.h) == 0
    e.close()


def test_pages_run_out_and_come_back(hybrid_model):
    from qwisp_amd.lib import SeedlessError
    cfg, dev = hybrid_model
    base = make(cfg, dev, page_size=16, n_pages=4, max_m=8, max_seq_len=128)
    a, b = base.new_lane(max_m=8, max_seq_len=128), base.new_lane(max_m=8, max_seq_len=64)
    for i in range(5):
        assert a.step_argmax(list(range(8))) is not None       # 40 tokens: three pages
    assert b.step_argmax([1] * 8) is not None and b.step_argmax([2] * 8) is not None      # the fourth, full
    assert b.step_argmax([3]) is None and b.gpu_fault is None and b.position == 16
    assert base.lane_step_argmax([a, b], [1, 2]) is None and a.gpu_fault is None and a.position == 40
    assert a.chained_step_argmax(1, 9) is None and a.chained_step_argmax(1, 8) is not None
    a.close()
    assert b.step_argmax([3]) is not None and b.position == 17   # (a's pages came back)
    with pytest.raises(SeedlessError):
        base.new_lane(max_m=8, max_seq_len=129)
    with pytest.raises(SeedlessError):
        base.set_kv4(16)
    with pytest.raises(SeedlessError):
        b.set_kv4(16)
    b.close()
    base.close()
    late = make(cfg, dev, kv4=False, max_m=4, max_seq_len=64)
    with pytest.raises(SeedlessError):
        late.set_kv4(24)
    assert late.step_argmax([1]) is not None
    with pytest.raises(SeedlessError):
        late.set_kv4(16)
    late.close()


def test_loaded_rows_are_quantised_by_the_stated_rule(attn_model):
    cfg, dev, _ = attn_model
    e = make(cfg, dev, page_size=64, max_m=4, max_seq_len=200)
    rng = np.random.default_rng(0)
    k, v = (rng.normal(size=(2, 150, 256)).astype(np.float16) for _ in range(2))
    assert e.load_layer_cache(0, k, v) and e.position == 150
    for got, x in zip(e.read_layer_cache(0), (k, v)):
        assert np.array_equal(got, ref.values(ref.quantise(x.astype(np.float64))).astype(np.float32).astype(np.float16))
    assert e.lib.dll.sl_load_layer_cache(e.h, 0, k.ctypes.data, None, 150) == -1
    e.close()


@pytest.mark.parametrize("hybrid", [False, True])
def test_attention_layer_against_64_bits(attn_model, hybrid):
    """Gated attention rows from the projection rows that the engine itself formed and the cache it holds.  Tolerance: queries
    and (as they are read back) keys are rounded to fp16, 2^-11 of each product of a score, so a score is off by at
    most d = 2 * 2^-11 * sum |q k| / 16 and a weight by 4 d of itself; a value by 2^-11 for reading it back, by 2^-11 * (8 |s| + 2 |b + 8 s|)
    <= 2^-11 * 4 times the largest of its group for weights in fp16 (|s| <= largest / 7.5); the sum of n weights below fp16's
    normal numbers by n 2^-22; the result is rounded once."""
    cfg, dev, host = attn_model
    e = make(cfg, dev, page_size=32, max_m=64, max_seq_len=400)
    e.set_hybrid(hybrid)
    rng = np.random.default_rng(1)
    qw = host["layers.0.self_attn.q_norm.weight"].astype(np.float64)
    freq = np.exp(-2.0 * np.arange(32) / 64 * np.log(1e7)).astype(np.float32)
    done = 0
    for m in (64, 64, 30, 1, 7):
        assert e.attn_layer_rows(0, rng.normal(size=(m, 2048)).astype(np.float16)) is not None
        proj = e.debug_scratch(0, m * 12352).reshape(m, 12352)
        got = e.debug_scratch(1, m * 4096).reshape(m, 16, 256).astype(np.float64)
        k, v = (x.astype(np.float64) for x in e.read_layer_cache(0))
        both = proj[:, :8192].reshape(m, 16, 512)
        angle = (np.arange(done, done + m, dtype=np.float32)[:, None] * freq).astype(np.float64)
        q = ref.turn(both[:, :, :256], qw, np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32), np.arange(m), 1e-6)
        gate = 1 / (1 + np.exp(-both[:, :, 256:].astype(np.float64)))
        for i in range(m):
            n = done + i + 1
            for h in range(16):
                kk, vv = k[h // 8, :n], v[h // 8, :n]
                s = kk @ q[i, h] / 16
                w = np.exp(s - s.max())
                total = w.sum()
                w /= total
                d = 2 * 2.0 ** -11 * (np.abs(kk) @ np.abs(q[i, h])).max() / 16
                big = np.abs(vv).reshape(n, 4, 64).max(-1).max(0).repeat(64)
                want = (w @ vv) * gate[i, h]
                tol = ((2.0 ** -11 * 5 + 4 * d) * big + n * 2.0 ** -22 / total) * gate[i, h] + 2.0 ** -11 * np.abs(want) + 2.0 ** -25
                assert (np.abs(got[i, h] - want) <= tol).all(), (m, i, h)
        done += m
    e.close()


@pytest.mark.parametrize("budget", [0, 16])
def test_a_scheduler_with_fewer_pages_than_its_slots_could_use(hybrid_model, budget):
    """Ten requests of different lengths on four slots and pages for about two of them: with the gate every request gets its
    tokens; without a budget such a table is refused."""
    from qwisp_amd.engine import LaneScheduler
    from qwisp_amd.lib import SeedlessError
    cfg, dev = hybrid_model
    rng = np.random.default_rng(5)
    jobs = [(rng.integers(0, 4096, int(n)).tolist(), int(g)) for n, g in zip(rng.integers(1, 60, 10), rng.integers(1, 40, 10))]
    alone = make(cfg, dev, max_m=8, max_seq_len=128)
    want = []
    for p, n in jobs:
        want.append(alone.greedy_generate(p, n, chain_k=4).tolist())
        assert alone.lib.dll.sl_reset(alone.h) == 0
    alone.close()
    base = make(cfg, dev, page_size=16, n_pages=13, max_m=8, max_seq_len=128)
    base.step_argmax([1, 2, 3])                          # the base's own sequence holds a page
    assert base.kv4_free_pages() == 12
    if budget == 0:
        with pytest.raises(SeedlessError):
            LaneScheduler(base, slots=4, chunk_rows=8, max_seq_len=128)
        few = LaneScheduler(base, slots=1, chunk_rows=8, max_seq_len=128)
        few.submit(*jobs[0])
        assert few.run() == want[:1] and base.kv4_free_pages() == 12
        few.close()
    else:
        sched = LaneScheduler(base, slots=4, chunk_rows=8, max_seq_len=128, token_budget=budget, kv_budget_tokens=512)
        for p, n in jobs:
            sched.submit(p, n)
        sched.submit([1, 2], 0)
        sched.submit([3] * 100, 100)                     # longer than a slot
        sched.submit(*jobs[3])
        assert sched.run() == want + [[], [], want[3]]
        assert base.kv4_free_pages() == 12
        sched.close()
    base.close()


def test_pages_of_a_base_that_is_gone_are_its_lanes(hybrid_model):
    cfg, dev = hybrid_model
    base = make(cfg, dev, page_size=16, n_pages=2, max_m=8, max_seq_len=32)
    for _ in range(2):
        assert base.step_argmax(list(range(8))) is not None
    lane = base.new_lane(max_m=8, max_seq_len=32)
    assert lane.step_argmax([1]) is not None and base.kv4_free_pages() == 0
    for _ in range(2):
        assert lane.step_argmax([1] * 7) is not None
    assert lane.step_argmax([1] * 2) is None             # 15 tokens: the second page would be needed
    base.close()
    assert lane.step_argmax([1] * 2) is not None and lane.kv4_free_pages() == 0
    lane.close()
