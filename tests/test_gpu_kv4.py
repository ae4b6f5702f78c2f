"""The operators on the 4-bit cache against their plain 64-bit forms (kv4_ref), on the GPU."""
import numpy as np
import pytest

from . import kv4_ref as ref

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
HALF_STEP = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8}


def gpu(x, dtype=None):
    return torch.from_numpy(np.ascontiguousarray(x)).cuda() if dtype is None else torch.from_numpy(np.ascontiguousarray(x)).to(dtype).cuda()


def f64(t):
    return t.detach().cpu().double().numpy()


def kv4():
    from qwisp_amd import kv4 as m
    return m


# ---- plan -----------------------------------------------------------------------------------------------------------------
def plan_case(rng, n, width, page, spare, wild):
    ctx = rng.integers(0, max(1, width * page - 40), n)
    new = rng.integers(0, 40, n)
    held = np.minimum(width, -(-ctx // page) + (rng.random(n) < 0.3) * rng.integers(0, 3, n))
    if n:
        ctx[::5] = 0                                       # ended: everything goes back
        new[::5] = 0
    if wild and n > 8:
        ctx[1], new[2], held[3], held[4], ctx[6], new[7] = -3, -1, width + 2, -1, width * page, 9
    clean = np.clip(held, 0, width)
    total = int(clean.sum()) + spare
    order = rng.permutation(total).astype(np.int32)
    table = np.full((n, width), -7, np.int32)
    at = 0
    for r in range(n):
        table[r, :clean[r]] = order[at:at + clean[r]]
        at += clean[r]
    free = np.full(total, -7, np.int32)
    free[:spare] = order[at:]
    return [x.astype(np.int32) for x in (ctx, new)] + [table, held.astype(np.int32), free, np.array([spare], np.int32)]


@pytest.mark.parametrize("n, width, page, spare, wild, room", [
    (0, 0, 16, 5, False, 0), (1, 1, 16, 0, False, 100), (1, 4, 256, 2, False, 40), (32, 9, 64, 40, False, 2000), (33, 7, 16, 3, False, 2000),
    (100, 5, 32, 0, True, 4000), (700, 11, 16, 150, True, 20000), (700, 11, 16, 4000, True, 5000), (4096, 3, 16, 900, True, 100000), (64, 9, 128, 70, True, 300)])
def test_plan(n, width, page, spare, wild, room):
    case = plan_case(np.random.default_rng(n + 7 * width + spare), n, width, page, spare, wild)
    got = kv4().plan(*(gpu(x) for x in case), page, room)
    for name, g, w in zip(got._fields, got, ref.plan(*case, page, room)):
        assert np.array_equal(g.cpu().numpy(), w), name


def test_plan_takes_any_numbers():
    """Numbers that a broken program might hand over: nothing is followed out of bounds, and the counts stay in range."""
    rng = np.random.default_rng(5)
    n, width, page = 300, 6, 32
    wild = lambda k: rng.integers(-2 ** 31, 2 ** 31, k).astype(np.int32)  # noqa: E731
    for count in (-5, 2 ** 31 - 1):
        got = kv4().plan(gpu(wild(n)), gpu(wild(n)), gpu(wild((n, width))), gpu(wild(n)), gpu(wild(50)), gpu(np.array([count], np.int32)), page, 777)
        start = got.q_start.cpu().numpy()
        assert (np.diff(start) >= 0).all() and 0 <= start[0] and start[-1] <= 777
        assert 0 <= int(got.free_count) <= 50 and 0 <= int(got.unserved) <= n
        held, kv = got.held.cpu().numpy(), got.kv_len.cpu().numpy()
        assert ((held >= 0) & (held <= width)).all() and ((kv >= 0) & (kv <= width * page)).all()


# ---- append and read --------------------------------------------------------------------------------------------------------
def fresh(rng, n_pages, page, kv, dim):
    """A pool that holds anything at all."""
    m = kv4()
    return m.Pool(gpu(rng.integers(0, 256, (n_pages, m.page_bytes(page, kv, dim)), dtype=np.uint8)), page, kv, dim)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("heads, kv, page, rot, tokens, norm", [(16, 2, 64, 64, 1, True), (3, 1, 16, 16, 7, True), (8, 8, 32, 8, 33, False), (6, 3, 128, 64, 130, True), (4, 2, 256, 0, 19, True)])
def test_append(dim, dtype, heads, kv, page, rot, tokens, norm):
    m, rng, dt = kv4(), np.random.default_rng(dim + tokens), DTYPES[dtype]
    n_pages = -(-tokens // page) + 2
    pool = fresh(rng, n_pages, page, kv, dim)
    before = pool.pages.cpu().numpy().copy()
    row = gpu(rng.normal(size=(tokens, (heads + 2 * kv) * dim + 8)) * 2, dt)          # a projection's row, its parts as views
    row[:, ::29] *= 9
    row[:, 12 if dim == 64 else 70] = 0
    q, k, v = (row[:, a * dim:(a + b) * dim].unflatten(1, (b, dim)) for a, b in ((0, heads), (heads, kv), (heads + kv, kv)))
    v[0, 0] = 0.5                                                                      # a group without a range
    if tokens > 4:
        v[2, 0, 3], k[3, 0, 1], v[4, 0, 64 % dim] = float("inf"), float("nan"), float("nan")
    qw, kw = (gpu(1 + 0.2 * rng.normal(size=dim), dt) if norm else None for _ in range(2))
    pos = rng.integers(0, 90, tokens).astype(np.int32)
    slot = rng.permutation(n_pages * page)[:tokens].astype(np.int32)
    if tokens > 6:
        slot[1], slot[5], slot[6] = -1, n_pages * page, -2 ** 31
        if rot:
            pos[0], pos[2] = 90, -1
    cos, sin = m.rope_tables(90, rot) if rot else (None, None)
    out = torch.full((tokens, heads, dim + 4), 7.0, dtype=dt, device="cuda")[:, :, :dim]
    got = m.append(pool, q, k, v, gpu(slot), gpu(pos), cos, sin, qw, kw, out=out)
    assert got is out and (out._base[:, :, dim:] == 7).all()
    h = lambda t: None if t is None else f64(t)  # noqa: E731
    placed = (pos >= 0) & (pos < 90) | (rot == 0)
    where = np.where(placed, pos, 0)
    want_q = np.where(placed[:, None, None], ref.turn(f64(q), h(qw), h(cos), h(sin), where, 1e-6), 0)
    # fp32: a sum of dim squares, a root, a division and at most four products and a sum, each within 2^-24
    mag = np.abs(want_q) if not rot else np.abs(want_q) + np.abs(want_q).max(-1, keepdims=True)
    assert (np.abs(f64(got) - want_q) <= HALF_STEP[dtype] * np.abs(want_q) + (dim / 4 + 16) * 2.0 ** -24 * mag + 2.0 ** -25).all()
    # the cache: the stated codes, scales and biases at the stated places, everything else as it was
    want = ref.unpack(before, page, kv, dim)
    keep = placed & (slot >= 0) & (slot < n_pages * page)
    for name, x in (("k", ref.turn(f64(k), h(kw), h(cos), h(sin), where, 1e-6)), ("v", f64(v))):
        part = ref.quantise(x[keep])
        for key in part:
            want[name][key][slot[keep]] = part[key]
    have = ref.unpack(pool.pages.cpu().numpy(), page, kv, dim)
    for name in "kv":
        for key in ("codes", "scale", "bias"):
            assert np.array_equal(want[name][key], have[name][key], equal_nan=key != "codes"), (name, key)
    # and its rows as values
    ask = np.concatenate((slot, [0, n_pages * page - 1, n_pages * page, -1])).astype(np.int32)
    ok = (ask >= 0) & (ask < n_pages * page)
    for dt_out, np_t in ((torch.float32, np.float32), (torch.float16, np.float16)):
        for g, name in zip(m.read(pool, gpu(ask), dt_out), "kv"):
            with np.errstate(over="ignore", invalid="ignore"):
                val = ref.values(have[name])[np.where(ok, ask, 0)].astype(np.float32).astype(np_t)
            assert np.array_equal(np.where(ok[:, None, None], val, 0), g.cpu().numpy(), equal_nan=True), (name, dt_out)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_groups_of_equal_edges_and_values_between_two_codes(dtype):
    """Largest = -smallest leaves the edge 7.5 steps away, and short numbers fall halfway between two codes: the side that the
    stated arithmetic takes."""
    m, rng = kv4(), np.random.default_rng(21)
    edge = rng.integers(1, 256, (600, 1, 1)) / 2.0 ** rng.integers(0, 9, (600, 1, 1))
    x = np.rint(rng.uniform(-1, 1, (600, 1, 64)) * 16) / 16 * edge
    x[:, :, 3], x[:, :, 60] = edge[..., 0], -edge[..., 0]
    x[300:, :, 60] *= rng.choice([0.5, 0.875, 1.0, 0.25], (300, 1))
    v = gpu(x, DTYPES[dtype])
    pool = fresh(rng, 10, 64, 1, 64)
    m.append(pool, None, v, v, gpu(np.arange(600, dtype=np.int32)), None, None, None, None, None)
    have, want = ref.unpack(pool.pages.cpu().numpy(), 64, 1, 64), ref.quantise(f64(v))
    for name in "kv":
        for key in want:
            assert np.array_equal(have[name][key][:600], want[key]), (name, key)


def test_append_of_keys_and_values_alone():
    m, rng = kv4(), np.random.default_rng(3)
    pool, twin = (m.Pool(torch.zeros(4, m.page_bytes(16, 2, 128), dtype=torch.uint8, device="cuda"), 16, 2, 128) for _ in range(2))
    q, k, v = (gpu(rng.normal(size=(20, 2, 128)), torch.float16) for _ in range(3))
    slot, pos = (gpu(np.arange(20, dtype=np.int32)) for _ in range(2))
    cos, sin = m.rope_tables(20, 128)
    w = torch.ones(128, dtype=torch.float16, device="cuda")
    assert m.append(pool, None, k, v, slot, pos, cos, sin, None, w) is None
    m.append(twin, q, k, v, slot, pos, cos, sin, w, w)
    assert torch.equal(pool.pages, twin.pages)


# ---- attention ----------------------------------------------------------------------------------------------------------------
def filled(rng, lens, page, kv, dim, spare=2, dirt=True):
    """Pages of random rows for the given lengths, in mixed order; places that no request uses hold NaN scales."""
    count = [-(-n // page) for n in lens]
    n_pages = sum(count) + spare
    order = rng.permutation(n_pages).astype(np.int32)
    width = max(count + [1]) + 1
    table = np.full((len(lens), width), -1, np.int32)
    parts = [ref.quantise(rng.normal(size=(n_pages * page, kv, dim)) * rng.choice([0.3, 1.0, 2.0], size=(1, kv, dim))) for _ in range(2)]
    used, at = np.zeros(n_pages * page, bool), 0
    for r, k in enumerate(count):
        table[r, :k] = order[at:at + k]
        at += k
        j = np.arange(lens[r])
        used[table[r, j // page] * page + j % page] = True
    if dirt:
        for p in parts:
            p["scale"][~used], p["bias"][~used] = np.nan, np.inf
    m = kv4()
    pool = m.Pool(gpu(ref.pack(*parts, page, kv, dim)), page, kv, dim)
    return pool, dict(k=parts[0], v=parts[1]), table, n_pages


def check(dim, dtype, heads, kv, page, lens, rows, gate=False, spread=1.0, scale=None, seed=0, max_rows=None, max_keys=None, tail=0, edit=None):
    m, rng, dt = kv4(), np.random.default_rng(seed), DTYPES[dtype]
    pool, parts, table, n_pages = filled(rng, lens, page, kv, dim)
    if edit:
        edit(table)
    start = np.concatenate(([0], np.cumsum(rows))).astype(np.int32)
    t = int(start[-1]) + tail
    both = gpu(rng.normal(size=(t, heads, 2 * dim)) * spread, dt)                  # [query | gate] per head, as a projection leaves them
    q, g = both[:, :, :dim], both[:, :, dim:] if gate else None
    out = torch.full((t, heads, dim), 5.0, dtype=dt, device="cuda")
    most = max(rows) if max_rows is None else max_rows
    scale = dim ** -0.5 if scale is None else scale
    got = m.attention(pool, q, gpu(table), gpu(start), gpu(np.array(lens, np.int32)), max_rows=most, max_keys=max(lens + [1]) if max_keys is None else max_keys,
                      scale=scale, gate=g, out=out)
    assert got is out
    want, tol = ref.attention(f64(q), parts, table, start, lens, page, n_pages, scale, f64(g) if gate else None, most, HALF_STEP[dtype])
    have = f64(out)
    left = np.isnan(tol)
    assert (have[left] == 5).all()
    err = np.abs(have - want)[~left]
    assert (err <= tol[~left]).all(), (err.max(), (err / tol[~left]).max())
    return pool, q, table, start, out


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("heads, kv, page", [(16, 2, 64), (4, 4, 16), (6, 2, 32)])
def test_single_tokens(dim, dtype, heads, kv, page):
    check(dim, dtype, heads, kv, page, [1, 2, 15, 16, 17, 31, 32, 33, 127, 129, 400, 1, 63, 64, 65], [1] * 15, gate=kv == 2)


@pytest.mark.parametrize("dim, dtype, heads, kv, page", [(256, "f16", 16, 2, 64), (128, "bf16", 8, 8, 16), (64, "f16", 9, 3, 128), (256, "bf16", 20, 1, 32)])
@pytest.mark.parametrize("rows", [[2, 3, 1, 5], [8, 7, 6, 1]])
def test_a_few_rows(dim, dtype, heads, kv, page, rows):
    check(dim, dtype, heads, kv, page, [9, 140, 33, 300], rows, gate=True, seed=1)


@pytest.mark.parametrize("dim, dtype, heads, kv, page", [(256, "f16", 16, 2, 64), (128, "bf16", 4, 2, 16), (64, "f16", 5, 5, 32), (128, "f16", 7, 1, 256)])
def test_many_rows(dim, dtype, heads, kv, page):
    check(dim, dtype, heads, kv, page, [70, 201, 65, 130], [70, 90, 1, 37], gate=dim == 256, seed=2)


def test_rows_without_keys_and_requests_without_rows():
    check(128, "f16", 4, 2, 16, [0, 5, 3, 0, 40], [1, 0, 5, 2, 3], seed=3)       # the third's first two rows see nothing


def test_rows_behind_the_last_and_rows_over_the_limit_are_left():
    check(128, "bf16", 8, 2, 32, [50, 60], [3, 9], tail=4, max_rows=4, seed=4)


def test_pages_that_are_not_there():
    def edit(table):
        table[0, 1], table[1, 0], table[2, :] = -1, 1 << 20, -5
    check(256, "f16", 8, 1, 16, [60, 200, 33], [2, 1, 1], edit=edit, seed=5)


@pytest.mark.parametrize("spread, scale", [(30.0, None), (1.0, 0.0), (4.0, -0.3), (1e-3, None)])
def test_sharp_flat_and_turned_scores(spread, scale):
    check(128, "f16", 8, 2, 64, [700, 65], [1, 3], spread=spread, scale=scale, seed=6)


@pytest.mark.parametrize("max_keys", [1, 5000, 1 << 30])
def test_any_guess_of_the_longest_is_right(max_keys):
    check(128, "f16", 8, 2, 64, [1500, 3, 800], [1, 2, 1], max_keys=max_keys, seed=7)


@pytest.mark.parametrize("dim, dtype, page", [(256, "f16", 64), (128, "bf16", 16)])
def test_more_requests_than_a_wave(dim, dtype, page):
    rng = np.random.default_rng(30)
    lens = rng.integers(0, 300, 90).tolist()
    check(dim, dtype, 4, 2, page, lens, rng.integers(0, 3, 90).tolist(), gate=True, seed=30)


@pytest.mark.parametrize("dim, dtype, heads, kv, page, lens, rows", [
    (256, "f16", 4, 1, 32, [2600, 40, 900], [30, 25, 17]),          # 64 rows a workgroup, the long axis in parts
    (256, "bf16", 8, 1, 64, [1500, 1500], [5, 1]),                   # 40 and 8 rows: tiles of 16
    (128, "f16", 4, 2, 16, [2500, 77], [40, 20]),                    # tiles of 32
    (64, "bf16", 3, 3, 64, [3000, 1000], [33, 50])])
def test_many_rows_against_long_axes(dim, dtype, heads, kv, page, lens, rows):
    check(dim, dtype, heads, kv, page, lens, rows, gate=True, seed=31)


def test_more_than_64_requests_with_many_rows():
    rng = np.random.default_rng(32)
    check(256, "f16", 4, 1, 16, rng.integers(20, 200, 70).tolist(), [0, 20, 1] * 23 + [3], seed=32)


@pytest.mark.parametrize("dim, dtype, most, n", [(256, "bf16", 15, 70), (256, "f16", 12, 70), (128, "f16", 15, 70), (128, "bf16", 4, 130), (64, "f16", 17, 64), (64, "bf16", 4, 130)])
def test_many_rows_with_few_parts_each(dim, dtype, most, n):
    rng = np.random.default_rng(34)
    lens, rows = rng.integers(0, 90, n), rng.integers(0, 3, n)
    lens[::23], rows[::23] = 1000 + np.arange(len(lens[::23])), most
    check(dim, dtype, 8, 2, 64, lens.tolist(), rows.tolist(), gate=True, seed=34)


def test_values_at_the_edge_of_fp16():
    """Scales up to 8734: weights times scales stay within fp16 while the running maximum lags."""
    m, rng = kv4(), np.random.default_rng(33)
    n, dim, page = 700, 128, 32
    k = ref.quantise(np.sort(rng.normal(size=(n + 4, 1, dim)), axis=0))       # scores that keep growing
    v = ref.quantise(rng.choice([-65504.0, 65504.0, 1.0], size=(n + 4, 1, dim)))
    pool = m.Pool(gpu(ref.pack(k, v, page, 1, dim)), page, 1, dim)
    table = np.arange(22, dtype=np.int32)[None]
    q = gpu(np.abs(rng.normal(size=(2, 4, dim))), torch.bfloat16)
    out = m.attention(pool, q, gpu(table), gpu(np.array([0, 2], np.int32)), gpu(np.array([n], np.int32)), max_rows=2, max_keys=n)
    want, tol = ref.attention(f64(q), dict(k=k, v=v), table, [0, 2], [n], page, 22, dim ** -0.5, eps_out=HALF_STEP["bf16"])
    assert (np.abs(f64(out) - want) <= tol).all()


def test_long_context():
    check(256, "f16", 16, 2, 64, [20011, 513], [1, 1], gate=True, seed=8)


def test_keys_that_are_not_finite_show_where_they_are_seen():
    m, rng = kv4(), np.random.default_rng(9)
    pool, parts, table, _ = filled(rng, [40], 16, 1, 64)
    parts["v"]["scale"][table[0, 35 // 16] * 16 + 35 % 16] = np.nan
    pool = m.Pool(gpu(ref.pack(parts["k"], parts["v"], 16, 1, 64)), 16, 1, 64)
    q = gpu(rng.normal(size=(8, 2, 64)), torch.float16)
    out = m.attention(pool, q, gpu(table), gpu(np.array([0, 8], np.int32)), gpu(np.array([40], np.int32)), max_rows=8, max_keys=40)
    bad = torch.isnan(out).all(-1).all(-1).cpu().numpy()
    assert bad.tolist() == [i + 32 >= 35 for i in range(8)] and not torch.isnan(out[~torch.from_numpy(bad)]).any()


# ---- the operators together -------------------------------------------------------------------------------------------------
def test_a_run_of_steps():
    """Three requests from their prompts through single tokens, a cut and a new request in the place of one that ended."""
    m, rng, page, kv, heads, dim = kv4(), np.random.default_rng(10), 16, 2, 8, 128
    pool = fresh(rng, 24, page, kv, dim)
    cos, sin = m.rope_tables(200, 64)
    qw, kw = (gpu(1 + 0.1 * rng.normal(size=dim), torch.float16) for _ in range(2))
    table, held = torch.full((3, 10), -1, dtype=torch.int32, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda")
    free, count = torch.arange(24, dtype=torch.int32, device="cuda"), torch.tensor([24], dtype=torch.int32, device="cuda")
    ctx = np.zeros(3, np.int32)
    rows = [[] for _ in range(3)]                                   # the keys and values that each request should hold
    for keep, new in [((0, 0, 0), (40, 17, 1)), ((40, 17, 1), (1, 1, 1)), ((41, 18, 2), (1, 3, 0)), ((30, 0, 2), (2, 25, 50)), ((32, 25, 52), (1, 1, 1))]:
        ctx, new = np.array(keep, np.int32), np.array(new, np.int32)
        step = m.plan(gpu(ctx), gpu(new), table, held, free, count, page, 80)
        table, held, free, count = step.table, step.held, step.free, step.free_count
        t = int(new.sum())
        assert int(step.unserved) == 0 and int(count) + int(held.sum()) == 24
        qkv = gpu(rng.normal(size=(80, (heads + 2 * kv) * dim)), torch.float16)
        q, k, v = (qkv[:, a * dim:(a + b) * dim].unflatten(1, (b, dim)) for a, b in ((0, heads), (heads, kv), (heads + kv, kv)))
        qr = m.append(pool, q, k, v, step.slot, step.pos, cos, sin, qw, kw)
        out = m.attention(pool, qr, table, step.q_start, step.kv_len, max_rows=int(new.max()), max_keys=96)
        start = step.q_start.cpu().numpy()
        kk = ref.turn(f64(k), f64(kw), f64(cos), f64(sin), step.pos.cpu().numpy(), 1e-6)
        for r in range(3):
            rows[r] = rows[r][:ctx[r]] + [(kk[i], f64(v[i])) for i in range(start[r], start[r + 1])]
        # the same rows, quantised in a pool of their own, request behind request
        lens = [len(x) for x in rows]
        wide = -(-max(lens) // page)
        parts = [ref.quantise(np.concatenate([np.concatenate([np.stack([x[i] for x in rows[r]]) if rows[r] else np.zeros((0, kv, dim)),
                                                              np.zeros((wide * page - lens[r], kv, dim))]) for r in range(3)])) for i in (0, 1)]
        own_table = np.arange(3 * wide, dtype=np.int32).reshape(3, wide)
        want, tol = ref.attention(f64(qr), dict(k=parts[0], v=parts[1]), own_table, start, lens, page, 3 * wide, dim ** -0.5)
        assert (np.abs(f64(out) - want)[:t] <= tol[:t]).all()


def test_a_captured_step_replays():
    """plan, append and attention in one graph: lengths and rows change between replays, eager work runs between them."""
    m, rng, page, kv, heads, dim, n = kv4(), np.random.default_rng(11), 32, 2, 16, 256, 5
    i32 = dict(dtype=torch.int32, device="cuda")
    pool, twin = (m.Pool(torch.zeros(40, m.page_bytes(page, kv, dim), dtype=torch.uint8, device="cuda"), page, kv, dim) for _ in range(2))
    cos, sin = m.rope_tables(400, 64)
    w = gpu(1 + 0.1 * rng.normal(size=dim), torch.float16)
    ctx, new = torch.zeros(n, **i32), torch.zeros(n, **i32)
    state = [torch.full((n, 8), -1, **i32), torch.zeros(n, **i32), torch.arange(40, **i32), torch.tensor([40], **i32)]
    qkv = torch.zeros(16, (heads + 2 * kv) * dim, dtype=torch.float16, device="cuda")

    def step(p):
        q, k, v = (qkv[:, a * dim:(a + b) * dim].unflatten(1, (b, dim)) for a, b in ((0, heads), (heads, kv), (heads + kv, kv)))
        s = m.plan(ctx, new, *state, page, 16)
        qr = m.append(p, q, k, v, s.slot, s.pos, cos, sin, w, w)
        out = torch.zeros_like(qr)
        return s, m.attention(p, qr, s.table, s.q_start, s.kv_len, max_rows=4, max_keys=256, out=out)

    step(pool)
    pool.pages.zero_()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        s, out = step(pool)
    pool.pages.zero_()
    lens = np.zeros(n, np.int32)
    for i in range(6):
        more = rng.integers(0, 4, n).astype(np.int32)
        ctx.copy_(gpu(lens)), new.copy_(gpu(more))
        qkv.copy_(gpu(rng.normal(size=tuple(qkv.shape)), torch.float16))
        want_s, want = step(twin)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(s, want_s):
            assert torch.equal(a, b)
        assert torch.equal(out, want) and torch.equal(pool.pages, twin.pages)
        for to, x in zip(state, (s.table, s.held, s.free, s.free_count)):
            to.copy_(x)
        lens += more


def test_another_stream():
    m, rng = kv4(), np.random.default_rng(12)
    pool, parts, table, n_pages = filled(rng, [300, 41], 64, 2, 128)
    q, start, lens = gpu(rng.normal(size=(2, 8, 128)), torch.float16), gpu(np.array([0, 1, 2], np.int32)), gpu(np.array([300, 41], np.int32))
    tab = gpu(table)
    want = m.attention(pool, q, tab, start, lens, max_rows=1, max_keys=300)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = m.attention(pool, q, tab, start, lens, max_rows=1, max_keys=300)
    side.synchronize()
    assert torch.equal(got, want)


def test_tensors_of_the_wrong_kind_are_refused():
    m = kv4()
    from qwisp_amd.lib import SeedlessError
    pool = m.new_pool(2, 16, 1, 64)
    i32 = dict(dtype=torch.int32, device="cuda")
    q = torch.zeros(2, 1, 64, dtype=torch.float16, device="cuda")
    good = dict(table=torch.zeros(1, 1, **i32), q_start=torch.zeros(2, **i32), kv_len=torch.zeros(1, **i32), max_rows=1, max_keys=1)
    for bad in (dict(q=q.float()), dict(q=q[:, :, :32]), dict(q=q.cpu()), dict(table=good["table"].long()), dict(q_start=torch.zeros(3, **i32)), dict(kv_len=good["kv_len"].cpu()),
                dict(gate=q[:1]), dict(out=q.bfloat16()), dict(q=torch.zeros(2, 1, 128, dtype=torch.float16, device="cuda")[:, :, ::2])):
        with pytest.raises(ValueError):
            m.attention(pool, **{**dict(q=q), **good, **bad})
    with pytest.raises(SeedlessError):
        m.attention(pool, torch.zeros(2, 1, 65, dtype=torch.float16, device="cuda")[:, :, 1:], **good)       # rows that do not start on 16 bytes
    with pytest.raises(ValueError):
        m.read(m.Pool(pool.pages, 16, 2, 64), good["kv_len"])
    with pytest.raises(ValueError):
        m.new_pool(2, 24, 1, 64)
    with pytest.raises(ValueError):
        m.append(pool, q, q, q, torch.zeros(3, **i32), None, None, None, None, None)


def test_what_is_left_out_is_refused():
    m = kv4()
    from qwisp_amd.lib import SeedlessError
    pool = m.new_pool(2, 16, 1, 64)
    i32 = dict(dtype=torch.int32, device="cuda")
    q, one, few = torch.zeros(2, 1, 64, dtype=torch.float16, device="cuda"), torch.zeros(1, **i32), torch.zeros(2, **i32)
    cos, sin = m.rope_tables(4, 16)
    for bad in (dict(pos=None), dict(sin=None), dict(cos=None), dict(slot=None), dict(v=None), dict(cos=cos[0], sin=sin[0])):
        with pytest.raises(ValueError):
            m.append(pool, **{**dict(q=q, k=q, v=q, slot=few, pos=few, cos=cos, sin=sin, q_weight=None, k_weight=None), **bad})
    with pytest.raises(ValueError):
        m.attention(pool, q, torch.zeros(1, 1, **i32), few, None, max_rows=1, max_keys=1)
    # a step planned into its own inputs
    free, table, count = torch.arange(2, **i32), torch.full((1, 2), -1, **i32), torch.full((1,), 2, **i32)
    step = m.plan(one, one + 1, table, one.clone(), free, count, 16, 2)
    with pytest.raises(SeedlessError):
        m.plan(step.kv_len, one + 1, table, step.held.clone(), free, count, 16, 2, out=step)
    # numbers beyond the library's 32 bits mean what they say
    got = m.attention(pool, q, step.table, step.q_start, step.kv_len, max_rows=1 << 33, max_keys=1 << 33)
    want = m.attention(pool, q, step.table, step.q_start, step.kv_len, max_rows=2, max_keys=2)
    assert torch.equal(got[:1], want[:1])


def test_two_graphs_share_a_workspace_and_two_streams_run_side_by_side():
    m, rng = kv4(), np.random.default_rng(13)
    calls = []
    for dim, heads, kv, page, lens, rows in ((256, 8, 2, 32, [1700, 300], [40, 30]), (128, 8, 2, 64, rng.integers(1, 900, 90).tolist(), [1] * 90)):
        pool, _, table, _ = filled(rng, lens, page, kv, dim)
        start = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
        q = gpu(rng.normal(size=(int(start[-1]), heads, dim)), torch.float16)
        calls.append((pool, q, gpu(table), gpu(start), gpu(np.array(lens, np.int32)), max(rows), max(lens)))
    want = [m.attention(*c) for c in calls]
    need = [m.attention_workspace(c[0], c[1].shape[0], c[1].shape[1], c[2].shape[0], c[2].shape[1], c[5], c[6]) for c in calls]
    shared = torch.zeros(max(need), dtype=torch.uint8, device="cuda")
    graphs, outs = [], [torch.empty_like(w) for w in want]
    torch.cuda.synchronize()
    for c, o in zip(calls, outs):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            m.attention(*c, out=o, workspace=shared)
        graphs.append(g)
    for i in range(4):
        for o in outs:
            o.zero_()
        shared.fill_(255)
        for g in graphs[::1 if i % 2 else -1]:
            g.replay()
        got = m.attention(*calls[i % 2], workspace=shared)
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for o, w in zip(outs, want)) and torch.equal(got, want[i % 2])
    with pytest.raises(Exception, match="sl_kv4_attention"):
        m.attention(*calls[0], workspace=shared[:need[0] - 16])
    streams = [torch.cuda.Stream() for _ in calls]
    got = [[] for _ in calls]
    for _ in range(5):
        for s, c, o in zip(streams, calls, got):
            with torch.cuda.stream(s):
                o.append(m.attention(*c))
    torch.cuda.synchronize()
    assert all(torch.equal(x, w) for o, w in zip(got, want) for x in o)
