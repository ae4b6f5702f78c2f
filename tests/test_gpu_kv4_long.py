"""Engine steps of one and of several rows behind a long 4-bit cache, against 64 bits."""
import numpy as np
import pytest

from . import kv4_ref as ref
from .test_gpu_kv4_edges import compare, expected
from .test_gpu_kv4_engine import attn_model, make  # noqa: F401

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.mark.parametrize("hybrid", [False, True])
def test_steps_behind_a_long_cache(attn_model, hybrid):  # noqa: F811
    """Gated attention rows from the query rows that the engine formed, the loaded rows and the engine's own new ones, all as the codes
    that the stated rule gives them.  The output's rounding is half a step of fp16; the gate's factor has fp32's."""
    cfg, dev, host = attn_model
    n = 12000
    e = make(cfg, dev, page_size=64, max_m=64, max_seq_len=n + 200)
    e.set_hybrid(hybrid)
    rng = np.random.default_rng(60)
    old = [rng.normal(size=(2, n, 256)).astype(np.float16) for _ in range(2)]
    assert e.load_layer_cache(0, *old)
    kw = host["layers.0.self_attn.k_norm.weight"].astype(np.float64)
    freq = np.exp(-2.0 * np.arange(32) / 64 * np.log(1e7)).astype(np.float32)
    angle = (np.arange(n + 200, dtype=np.float32)[:, None] * freq).astype(np.float64)
    cos, sin = np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32)
    parts = [ref.quantise(np.moveaxis(x.astype(np.float64), 0, 1)) for x in old]
    done = n
    for m in (1, 8, 5, 64, 1):
        assert e.attn_layer_rows(0, rng.normal(size=(m, 2048)).astype(np.float16)) is not None
        proj = e.debug_scratch(0, m * 12352).reshape(m, 12352)
        q = e.debug_scratch(2, m * 4096).reshape(m, 16, 256).astype(np.float64)
        have = e.debug_scratch(1, m * 4096).reshape(m, 16, 256).astype(np.float64)
        gate = 1 / (1 + np.exp(-proj[:, :8192].reshape(m, 16, 512)[:, :, 256:].astype(np.float64)))
        k, v = (proj[:, at:at + 512].reshape(m, 2, 256).astype(np.float64) for at in (8192, 8704))
        new = [ref.quantise(ref.turn(k, kw, cos, sin, np.arange(done, done + m), 1e-6)), ref.quantise(v)]
        parts = [{key: np.concatenate((a[key], b[key])) for key in a} for a, b in zip(parts, new)]
        done += m
        table = np.arange(-(-done // 64), dtype=np.int32)[None]
        want, var, size = expected(q, dict(k=parts[0], v=parts[1]), table, [0, m], [done], 64, 0.0625, 2.0 ** -11)
        compare(have, want * gate, var * gate ** 2, size * gate)
    e.close()
