"""The 4-bit cache's attention where numbers are not finite, very small, very large or very unlike: against the plain 64-bit form,
with tolerances that follow the values' own size."""
import numpy as np
import pytest

from . import kv4_ref as ref
from .test_gpu_kv4 import DTYPES, HALF_STEP, f64, filled, gpu, kv4

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def call(pool, q, table, start, lens, scale=None):
    """Attention into an output that holds 5."""
    out = torch.full(tuple(q.shape), 5.0, dtype=q.dtype, device="cuda")
    rows = np.diff(start)
    return kv4().attention(pool, q, gpu(table), gpu(start), gpu(np.array(lens, np.int32)), max_rows=int(rows.max()), max_keys=max(lens), scale=scale, out=out)


def offsets(rows):
    return np.concatenate(([0], np.cumsum(rows))).astype(np.int32)


# ---- numbers that are not finite, the axis in parts ------------------------------------------------------------------------
# (dim, dtype, heads, kv, page, lengths, rows): a few rows (parts joined by a workgroup each), 32-row tiles, 64-row tiles, and parts of
# many requests (joined by a wave each)
SPLIT = [(64, "f16", 4, 2, 32, [3000, 200], [1, 1]), (128, "bf16", 6, 2, 16, [2900, 70], [3, 2]), (256, "f16", 4, 2, 64, [4000], [1]),
         (128, "f16", 4, 2, 16, [2500, 77], [40, 20]), (256, "bf16", 4, 1, 32, [2600, 40, 900], [30, 25, 17]),
         (256, "f16", 8, 2, 64, [1000, 60, 1003] + [7] * 67, [12, 1, 12] + [1] * 67), (128, "bf16", 8, 2, 64, [1000, 60, 1003] + [7] * 67, [15, 1, 12] + [1] * 67)]


@pytest.mark.parametrize("dim, dtype, heads, kv, page, lens, rows", SPLIT)
@pytest.mark.parametrize("what", ["query", "keys", "values"])
def test_what_is_not_finite_shows_however_the_axis_is_cut(dim, dtype, heads, kv, page, lens, rows, what):
    rng = np.random.default_rng(40)
    pool, parts, table, n_pages = filled(rng, lens, page, kv, dim)
    start = offsets(rows)
    q = gpu(rng.normal(size=(int(start[-1]), heads, dim)), DTYPES[dtype])
    if what == "query":                                      # NaN in one row, Inf in others, of different heads
        q[0, 0, 5], q[-1, heads - 1, dim - 1], q[rows[0] - 1, heads // 2, 0] = float("nan"), float("-inf"), float("inf")
    else:                                                    # whole parts of the first request, up to the last key that all its rows see
        first, name = lens[0] * 3 // 5 // 128 * 128, what[0]
        j = np.arange(first, lens[0] - rows[0] + 1)
        at = table[0, j // page] * page + j % page
        parts[name]["scale"][at, 0], parts[name]["bias"][at, 0] = np.nan, np.nan
        if len(lens) > 1:                                    # and the second's very last key, in its last group and head: seen by one row
            last = lens[1] - 1
            parts[name]["scale"][table[1, last // page] * page + last % page, kv - 1, -1] = np.nan
        pool = kv4().Pool(gpu(ref.pack(parts["k"], parts["v"], page, kv, dim)), page, kv, dim)
    have = f64(call(pool, q, table, start, lens))
    with np.errstate(invalid="ignore"):
        want, var, size = expected(f64(q), parts, table, start, lens, page, dim ** -0.5, HALF_STEP[dtype])
    bad = np.isnan(want)
    assert bad.any() and not bad.all() and np.array_equal(np.isnan(have), bad)
    compare(have[~bad], want[~bad], var[~bad], size[~bad])


# ---- small values, and keys that stand out ------------------------------------------------------------------------------------
H = 2.0 ** -11          # half a step of fp16, in which weights meet the matrix instructions


def expected(q, parts, table, start, lens, page, scale, eps_out):
    """Rows in 64 bits; per number the variance that the roundings on the way leave; and the sum of its terms' sizes.
    A weight p meets the values in two parts, (p s) (code - 8) and p (b + 8 s), and the normaliser: p s, p and b + 8 s are each
    rounded to fp16 (an error of at most H of itself, spread evenly: variance H^2 / 3 at most), independently of each other."""
    t, heads, dim = q.shape
    wide = lambda x: np.repeat(x, 64, -1)  # noqa: E731
    kv = parts["k"]["codes"].shape[1]
    kk, vv = ref.values(parts["k"]), ref.values(parts["v"])
    out, var, size = (np.zeros((t, heads, dim)) for _ in range(3))
    for r, length in enumerate(lens):
        rows = start[r + 1] - start[r]
        j = np.arange(length)
        at = table[r, j // page] * page + j % page
        for g in range(kv):
            k, v, s = kk[at, g], vv[at, g], wide(parts["v"]["scale"][at, g])
            mid = wide(parts["v"]["bias"][at, g]) + 8 * s
            hs = slice(g * (heads // kv), (g + 1) * (heads // kv))
            for i in range(rows):
                n = length - rows + i + 1
                x = scale * (q[start[r] + i, hs] @ k[:n].T)
                w = np.exp(x - x.max(-1, keepdims=True))
                w /= w.sum(-1, keepdims=True)
                o = w @ v[:n]
                w2 = w * w
                spread = w2 @ ((v[:n] - mid[:n]) ** 2 + 2 * mid[:n] ** 2) - 2 * o * (w2 @ mid[:n]) + o * o * w2.sum(-1, keepdims=True)
                out[start[r] + i, hs] = o
                var[start[r] + i, hs] = H * H / 3 * spread + (eps_out * o) ** 2 / 3
                size[start[r] + i, hs] = w @ (np.abs(v[:n]) + 8 * np.abs(s[:n]))
    return out, var, size


def compare(have, want, var, size, fp32=2.0 ** -15, least=2.0 ** -25):
    """The error as a whole within twice what the roundings leave at most (half a step is 0.7 of that for the average number, and the dims
    of a row share the errors of p), each number within seven times, ten times its likely size.
    fp32: a score is the difference of two sums over codes of up to 100 in units of log2, each of some rounded steps: within
    2^-24 * 100 * 4, which is 2^-15, of the weight; below fp16's normal numbers an output is within 2^-25."""
    err = np.abs(have - want)
    rms = lambda x: np.sqrt((x * x).mean())  # noqa: E731
    assert rms(err) <= 2 * np.sqrt(var.mean()) + fp32 * rms(size) + least, (rms(err), np.sqrt(var.mean()), rms(size))
    worst = err / (7 * np.sqrt(var) + 4 * fp32 * size + 2 * least)
    assert worst.max() <= 1, worst.max()


# (dim, dtype, heads, kv, page, lengths, rows)
SHAPES = [(64, "bf16", 4, 4, 32, [4096, 333], [1, 1]), (128, "f16", 8, 2, 16, [3000, 4100], [2, 3]), (256, "f16", 4, 1, 64, [5000], [1]),
          (64, "f16", 2, 2, 64, [4000], [40]), (128, "bf16", 2, 1, 32, [3500], [24]), (256, "f16", 4, 1, 64, [2048], [20])]


def case(shape, seed, values, sink=0.0, mean=1.0):
    """Keys of size one; values of the given size around a mean per dim; with a sink the first key lies along all queries
    and stands `sink` above the others, its own value near zero."""
    dim, dtype, heads, kv, page, lens, rows = shape
    rng = np.random.default_rng(seed)
    count = [-(-n // page) for n in lens]
    order = rng.permutation(sum(count) + 2).astype(np.int32)
    table = np.full((len(lens), max(count)), -1, np.int32)
    n_rows = len(order) * page
    u = rng.normal(size=dim)
    u /= np.linalg.norm(u)
    k = rng.normal(size=(n_rows, kv, dim))
    v = values * (mean * rng.normal(size=(1, kv, dim)) + 0.5 * rng.normal(size=(n_rows, kv, dim)))
    q = rng.normal(size=(sum(rows), heads, dim))
    if sink:
        k -= (k @ u)[..., None] * u
        q = 0.3 * (q - (q @ u)[..., None] * u) + 8 * u
    at = 0
    for r, c in enumerate(count):
        table[r, :c] = order[at:at + c]
        at += c
        if sink:
            first = table[r, 0] * page
            k[first] = u * (sink / 8 * dim ** 0.5)
            v[first] = 0.001 * v[first]
    parts = dict(k=ref.quantise(k), v=ref.quantise(v))
    pool = kv4().Pool(gpu(ref.pack(parts["k"], parts["v"], page, kv, dim)), page, kv, dim)
    return pool, gpu(q, DTYPES[dtype]), parts, table, offsets(rows)


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("values", [1.0, 1e-2, 1e-4, 1e-5])
@pytest.mark.parametrize("mean", [0.0, 1.0])
def test_values_of_any_size_keep_their_digits(shape, values, mean):
    dim, dtype, heads, kv, page, lens, rows = shape
    pool, q, parts, table, start = case(shape, 41, values, mean=mean)
    q = q.to(torch.bfloat16)                                 # (outputs of any size keep their digits)
    have = f64(call(pool, q, table, start, lens))
    compare(have, *expected(f64(q), parts, table, start, lens, page, dim ** -0.5, HALF_STEP["bf16"]), least=0.0)


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("values, sink", [(0.1, 10.0), (0.02, 13.0), (1.0, 16.0), (1e-3, 13.0)])
def test_one_key_far_above_the_rest(shape, values, sink):
    dim, dtype, heads, kv, page, lens, rows = shape
    pool, q, parts, table, start = case(shape, 42, values, sink)
    have = f64(call(pool, q, table, start, lens))
    compare(have, *expected(f64(q), parts, table, start, lens, page, dim ** -0.5, HALF_STEP[dtype]))


@pytest.mark.parametrize("shape", SHAPES)
def test_values_that_grow_along_the_axis(shape):
    """Values of sizes from e^-7 to e^7 within a sequence, the largest in its middle, and weights that fall as the values grow,
    so that all of them count: the unit of the weighted scales changes on the way."""
    dim, dtype, heads, kv, page, lens, rows = shape
    pool, q, parts, table, start = case(shape, 43, 1.0)
    rng = np.random.default_rng(44)
    u = rng.normal(size=dim)
    u /= np.linalg.norm(u)
    for r, n in enumerate(lens):
        at = table[r, np.arange(n) // page] * page + np.arange(n) % page
        size = 7.0 * np.sin(np.linspace(-np.pi / 2, 3 * np.pi / 2, n))[:, None, None]
        k = 0.3 * rng.normal(size=(n, kv, dim)) - size * u * (dim ** 0.5 / 8)
        for name, x in (("k", k), ("v", rng.normal(size=(n, kv, dim)) * np.exp(size))):
            for key, y in ref.quantise(x).items():
                parts[name][key][at] = y
    pool = kv4().Pool(gpu(ref.pack(parts["k"], parts["v"], page, kv, dim)), page, kv, dim)
    q = gpu(0.3 * rng.normal(size=tuple(q.shape)) + 8 * u, torch.bfloat16)
    have = f64(call(pool, q, table, start, lens))
    compare(have, *expected(f64(q), parts, table, start, lens, page, dim ** -0.5, HALF_STEP["bf16"]), least=0.0)


# ---- very large scores ------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dim, heads, kv, page, lens, rows", [(128, 4, 2, 32, [500, 33], [1, 2]), (64, 3, 3, 16, [400], [33]), (256, 4, 1, 64, [300], [20]), (256, 8, 2, 64, [3000], [1])])
@pytest.mark.parametrize("dtype, size", [("f16", 2.0 ** 15), ("bf16", 2.0 ** 20), ("bf16", 2.0 ** 60), ("bf16", 2.0 ** 105)])
def test_scores_beyond_what_fp32_tells_apart_choose_the_largest(dim, heads, kv, page, lens, rows, dtype, size):
    """Scores of 1e7 and more: one key has all the weight.  Rows whose two largest scores lie within fp32's error of them are left out."""
    rng = np.random.default_rng(45)
    pool, parts, table, _ = filled(rng, lens, page, kv, dim)
    k = ref.quantise(rng.normal(size=parts["k"]["codes"].shape) * 3000)
    bad = np.isnan(parts["k"]["scale"])
    for key in k:
        parts["k"][key] = np.where(bad if key != "codes" else False, parts["k"][key], k[key])
    pool = kv4().Pool(gpu(ref.pack(parts["k"], parts["v"], page, kv, dim)), page, kv, dim)
    start = offsets(rows)
    q = gpu(rng.normal(size=(int(start[-1]), heads, dim)).clip(-1.9, 1.9) * size, DTYPES[dtype])
    have, qq = f64(call(pool, q, table, start, lens)), f64(q)
    kk, vv = ref.values(parts["k"]), ref.values(parts["v"])
    used = 0
    for r, n in enumerate(lens):
        j = np.arange(n)
        at = table[r, j // page] * page + j % page
        for i in range(rows[r]):
            m = n - rows[r] + i + 1
            for h in range(heads):
                g = h // (heads // kv)
                terms = kk[at[:m], g] * qq[start[r] + i, h]
                s = terms.sum(-1)
                two = np.sort(s)[-2:]
                if two[1] - two[0] <= 2.0 ** -24 * (dim + 8) * 4 * np.abs(terms).sum(-1).max():
                    continue
                used += 1
                want, e = vv[at[s.argmax()], g], 2 * H * (np.abs(vv[at[s.argmax()], g]) + 8 * np.abs(np.repeat(parts["v"]["scale"][at[s.argmax()], g], 64)))
                assert (np.abs(have[start[r] + i, h] - want) <= e + HALF_STEP[dtype] * np.abs(want) + 2.0 ** -25).all()
    assert used > 0


# ---- keys whose group lies on the border of two scales ----------------------------------------------------------------------
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_normed_keys_between_two_counts_of_steps(dim, dtype):
    """A group whose largest is the opposite of its smallest lies 7.5 steps from its edge, and the last bit of the norm's factor decides
    between 7 and 8: it has to be that of x * rsqrt(mean + eps) * weight in double precision, as torch has it.  The squares and
    their sum are exact here."""
    m, rng = kv4(), np.random.default_rng(46)
    n, page = 4096, 64
    x = rng.integers(-40, 41, (n, 1, dim)) / 16.0
    edge = rng.integers(41, 64, (n, 1, dim // 64)) / 16.0
    w = 1 + 0.1 * rng.normal(size=dim)
    for g in range(dim // 64):
        x[:, :, 64 * g + 7], x[:, :, 64 * g + 50] = edge[:, :, g], -edge[:, :, g]
        w[64 * g + 7] = w[64 * g + 50] = 1.5
    k, w = gpu(x, DTYPES[dtype]), gpu(np.clip(w, 0.5, 1.5), DTYPES[dtype])
    pool = m.new_pool(n // page, page, 1, dim)
    m.append(pool, None, k, k, gpu(np.arange(n, dtype=np.int32)), None, None, None, None, w)
    y = k.double() * torch.rsqrt((k.double() * k.double()).mean(-1, keepdim=True) + 1e-6) * w.double()
    have, want = ref.unpack(pool.pages.cpu().numpy(), page, 1, dim)["k"], ref.quantise(y.cpu().numpy())
    other = (have["scale"] != want["scale"]).any(-1).sum()
    assert other == 0, f"{other} of {n} rows have another scale"
    assert np.array_equal(have["bias"], want["bias"]) and np.array_equal(have["codes"], want["codes"])


# ---- arguments --------------------------------------------------------------------------------------------------------------
def small_calls():
    """Calls that work, by keyword."""
    m = kv4()
    pool = m.new_pool(2, 16, 1, 64)
    i32 = dict(dtype=torch.int32, device="cuda")
    half = dict(dtype=torch.float16, device="cuda")
    q, one, two = torch.zeros(2, 1, 64, **half), torch.zeros(1, **i32), torch.arange(2, **i32)
    cos, sin = m.rope_tables(4, 16)
    plan = dict(ctx_len=one, new_len=one + 2, table=torch.full((1, 2), -1, **i32), held=one.clone(), free=two, free_count=one + 2, page_size=16, max_tokens=2)
    append = dict(pool=pool, q=q, k=q + 1, v=q + 2, slot=two, pos=two, cos=cos, sin=sin, q_weight=torch.ones(64, **half), k_weight=torch.ones(64, **half))
    attention = dict(pool=pool, q=q, table=torch.zeros(1, 1, **i32), q_start=one.new_tensor([0, 2]), kv_len=one + 2, max_rows=2, max_keys=2, gate=q + 1)
    return m, dict(plan=plan, append=append, attention=attention, read=dict(pool=pool, slots=two))


@pytest.mark.parametrize("name, arg", [("append", x) for x in ("q", "k", "v", "cos", "sin", "q_weight", "k_weight")] + [("attention", "q"), ("attention", "gate")])
def test_tensors_that_ask_for_gradients_are_refused(name, arg):
    m, calls = small_calls()
    args = calls[name]
    want = getattr(m, name)(**args)
    args = {**args, arg: args[arg].clone().requires_grad_()}
    with pytest.raises(ValueError, match=arg):
        getattr(m, name)(**args)
    with torch.no_grad():
        assert torch.equal(getattr(m, name)(**args), want)


def test_what_is_no_tensor_is_refused():
    m, calls = small_calls()
    for name, args in calls.items():
        for arg, t in args.items():
            if not isinstance(t, torch.Tensor):
                continue
            for bad in (None, [1, 2]):
                if bad is None and (name, arg) in (("append", "q"), ("append", "q_weight"), ("append", "k_weight"), ("attention", "gate")):
                    continue                                 # (may be left out)
                with pytest.raises(ValueError, match=arg):
                    getattr(m, name)(**{**args, arg: bad})
    with pytest.raises(ValueError, match="pages"):
        m.read(m.Pool(None, 16, 1, 64), calls["read"]["slots"])
    with pytest.raises(ValueError, match="workspace"):
        m.attention(**{**calls["attention"], "workspace": [1]})
