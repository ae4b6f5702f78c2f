"""The 4-bit cache without a GPU: its layout and quantisation rule in the plain form, and the calls that the library refuses
before it launches anything."""
import ctypes as C

import numpy as np
import pytest

from qwisp_amd import abi, lib

from . import kv4_ref as ref


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("page", [16, 64])
def test_layout_covers_every_byte_once(page, dim):
    key, ksb, value, vsb = ref.places(page, dim)
    n = page * 9 * dim // 8
    seen = np.zeros(n, int)
    for at in (key, value):
        assert np.array_equal(at[:, 0::2], at[:, 1::2])      # two dims in a byte
        np.add.at(seen, at[:, 0::2].reshape(-1), 1)
    for w in (ksb, vsb):
        for b in range(4):
            np.add.at(seen, 4 * w.reshape(-1) + b, 1)
    assert (seen == 1).all()
    assert lib.get().dll.sl_kv4_page_bytes(page, 3, dim) == 3 * n


def test_pack_is_the_inverse_of_unpack():
    rng = np.random.default_rng(0)
    parts = [ref.quantise(rng.normal(size=(32, 2, 128))) for _ in range(2)]
    back = ref.unpack(ref.pack(*parts, 16, 2, 128), 16, 2, 128)
    for p, name in zip(parts, "kv"):
        for key in p:
            assert np.array_equal(p[key], back[name][key])


def test_quantised_values_lie_within_a_step():
    rng = np.random.default_rng(1)
    x = rng.normal(size=(500, 64)) * np.exp(rng.normal(size=(500, 1)) * 3)
    p = ref.quantise(x)
    # With x = |edge| / s0 (at least 7.5, the edge being the larger of two that lie 15 s0 apart) and n = rint(x), the step
    # is s = x s0 / n, and the far end of the group lies 15 s0 - 15 s = 15 s0 (n - x) / n <= 7.5 s0 / n = 7.5 s / x <= s
    # beyond the last code; everything else lies within half a step.  Added: what fp16 leaves of the scale (15 steps of it) and of the bias.
    bound = np.abs(p["scale"]) + 15 * 2.0 ** -11 * np.abs(p["scale"]) + 2.0 ** -11 * np.abs(p["bias"]) + 16 * 2.0 ** -25
    assert (np.abs(ref.values(p) - x) <= bound).all()
    zero = ref.quantise(np.zeros((1, 64)))
    assert (ref.values(zero) == 0).all()
    assert np.isnan(ref.values(ref.quantise(np.array([[np.inf] + [1.0] * 63])))).all()
    assert (np.abs(ref.values(ref.quantise(np.full((1, 64), 1e9)))) == 65504).all()


# ---- refusals: every call below ends before a launch, so no device is needed --------------------------------------------
P = 1 << 20          # an address that is never followed


def pool(**kw):
    return abi.Kv4Pool(**{**dict(pages=P, n_pages=4, page_size=16, n_kv=2, head_dim=64), **kw})


def append(**kw):
    base = dict(n_tokens=3, n_heads=4, rot_dim=32, max_pos=100, dtype=abi.SL_F16, eps=1e-6, q=P, k=P, v=P, q_weight=P, k_weight=P, cos=P, sin=P,
                slot=P, pos=P, q_out=2 * P, q_token=256, q_head=64, k_token=128, k_head=64, v_token=128, v_head=64, out_token=256, out_head=64)
    return abi.Kv4AppendArgs(**{**base, **kw})


def attn(**kw):
    base = dict(n_req=2, n_tokens=3, n_heads=4, dtype=abi.SL_F16, table_width=4, max_rows=2, max_keys=64, scale=0.1, q=P, gate=None, out=2 * P, q_token=256,
                q_head=64, out_token=256, out_head=64, table=P, q_start=P, kv_len=P, workspace=P, workspace_bytes=1 << 40)
    return abi.Kv4AttnArgs(**{**base, **kw})


def plan(**kw):
    base = dict(n_req=2, table_width=4, n_free=8, page_size=16, max_tokens=4, ctx_len=P, new_len=P, table_in=P, held_in=P, free_in=P, free_count_in=P,
                table_out=2 * P, held_out=2 * P, free_out=2 * P, free_count_out=2 * P, q_start=2 * P, kv_len=2 * P, slot=2 * P, pos=2 * P, unserved=2 * P)
    return abi.Kv4PlanArgs(**{**base, **kw})


POOLS = [(dict(pages=None), abi.SL_ERR_ARG), (dict(pages=P + 4), abi.SL_ERR_ARG), (dict(n_pages=0), abi.SL_ERR_ARG), (dict(n_kv=0), abi.SL_ERR_ARG),
         (dict(page_size=24), abi.SL_ERR_UNSUPPORTED), (dict(page_size=8), abi.SL_ERR_UNSUPPORTED), (dict(page_size=512), abi.SL_ERR_UNSUPPORTED),
         (dict(head_dim=96), abi.SL_ERR_UNSUPPORTED), (dict(n_kv=1025), abi.SL_ERR_UNSUPPORTED), (dict(n_pages=1 << 27), abi.SL_ERR_TOO_LARGE)]


@pytest.mark.parametrize("bad, status", POOLS)
def test_bad_pools(bad, status):
    dll = lib.get().dll
    assert dll.sl_kv4_append(pool(**bad), append(), None) == status
    assert dll.sl_kv4_attention(pool(**bad), attn(), None) == status
    assert dll.sl_kv4_read(pool(**bad), P, 3, abi.SL_F32, P, P, None) == status
    assert dll.sl_kv4_append(None, append(), None) == abi.SL_ERR_ARG


@pytest.mark.parametrize("bad", [dict(dtype=2), dict(n_tokens=-1), dict(rot_dim=12), dict(rot_dim=72), dict(rot_dim=-8), dict(max_pos=0), dict(eps=-1.0),
                                 dict(eps=float("nan")), dict(k=None), dict(v=None), dict(slot=None), dict(pos=None), dict(cos=None), dict(sin=None),
                                 dict(q_out=None), dict(n_heads=0), dict(k=P + 4), dict(q=P + 2), dict(q_out=P + 2), dict(cos=P + 8), dict(k_weight=P + 2),
                                 dict(k_token=129), dict(v_head=66), dict(q_head=65), dict(out_token=2)])
def test_append_refuses(bad):
    assert lib.get().dll.sl_kv4_append(pool(), append(**bad), None) == abi.SL_ERR_ARG


@pytest.mark.parametrize("bad", [dict(dtype=2), dict(n_req=-1), dict(n_tokens=-1), dict(n_heads=0), dict(n_heads=5), dict(max_rows=-1), dict(max_keys=0), dict(q=None),
                                 dict(out=None), dict(table=None), dict(q_start=None), dict(kv_len=None), dict(q=P + 8), dict(out=P + 2), dict(gate=P + 2),
                                 dict(q_token=260), dict(out_head=12), dict(gate=P, gate_token=4), dict(table_width=-1)])
def test_attention_refuses(bad):
    assert lib.get().dll.sl_kv4_attention(pool(), attn(**bad), None) == abi.SL_ERR_ARG


@pytest.mark.parametrize("bad, status", [(dict(n_req=-1), abi.SL_ERR_ARG), (dict(max_tokens=-1), abi.SL_ERR_ARG), (dict(page_size=17), abi.SL_ERR_UNSUPPORTED),
                                         (dict(n_req=4097), abi.SL_ERR_TOO_LARGE), (dict(table_width=1 << 30), abi.SL_ERR_TOO_LARGE), (dict(ctx_len=None), abi.SL_ERR_ARG),
                                         (dict(free_count_in=None), abi.SL_ERR_ARG), (dict(slot=None), abi.SL_ERR_ARG), (dict(table_out=P), abi.SL_ERR_ARG),
                                         (dict(free_out=P), abi.SL_ERR_ARG), (dict(held_out=P), abi.SL_ERR_ARG), (dict(free_count_out=P), abi.SL_ERR_ARG)])
def test_plan_refuses(bad, status):
    assert lib.get().dll.sl_kv4_plan(plan(**bad), None) == status


@pytest.mark.parametrize("out", ["table_out", "held_out", "free_out", "free_count_out", "q_start", "kv_len", "slot", "pos", "unserved"])
@pytest.mark.parametrize("inp", ["ctx_len", "new_len", "table_in", "held_in", "free_in", "free_count_in"])
def test_plan_refuses_an_output_that_is_an_input(out, inp):
    assert lib.get().dll.sl_kv4_plan(plan(**{inp: 5 * P, out: 5 * P}), None) == abi.SL_ERR_ARG


def test_empty_calls_do_nothing():
    dll = lib.get().dll
    assert dll.sl_kv4_append(pool(), append(n_tokens=0), None) == abi.SL_OK
    assert dll.sl_kv4_attention(pool(), attn(n_req=0), None) == abi.SL_OK
    assert dll.sl_kv4_attention(pool(), attn(n_tokens=0), None) == abi.SL_OK
    assert dll.sl_kv4_attention(pool(), attn(max_rows=0), None) == abi.SL_OK
    assert dll.sl_kv4_read(pool(), None, 0, abi.SL_F32, P, P, None) == abi.SL_OK
    assert dll.sl_kv4_read(pool(), P, -1, abi.SL_F32, P, P, None) == abi.SL_ERR_ARG
    assert dll.sl_kv4_read(pool(), P, 1, abi.SL_BF16, P, P, None) == abi.SL_ERR_ARG
    assert dll.sl_kv4_read(pool(), P, 1, abi.SL_F32, P + 4, P, None) == abi.SL_ERR_ARG


def test_struct_sizes_match_the_header(tmp_path):
    import os
    import subprocess
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    src = tmp_path / "s.c"
    src.write_text('#include <stdio.h>\n#include "seedless_hip.h"\nint main(void) { printf("%zu %zu %zu %zu\\n", sizeof(sl_kv4_pool), sizeof(sl_kv4_plan_args), '
                   'sizeof(sl_kv4_append_args), sizeof(sl_kv4_attn_args)); return 0; }\n')
    subprocess.check_call(["gcc", "-I", os.path.join(root, "include"), "-o", str(tmp_path / "s"), str(src)])
    got = [int(x) for x in subprocess.check_output([str(tmp_path / "s")]).split()]
    assert got == [C.sizeof(t) for t in (abi.Kv4Pool, abi.Kv4PlanArgs, abi.Kv4AppendArgs, abi.Kv4AttnArgs)]


def test_sizes_beyond_a_launch_are_refused():
    dll = lib.get().dll
    assert dll.sl_kv4_append(pool(), append(n_tokens=0x7ffffff0), None) == abi.SL_ERR_TOO_LARGE
    assert dll.sl_kv4_read(pool(head_dim=256), P, 0x7fffffff, abi.SL_F32, P, P, None) == abi.SL_ERR_TOO_LARGE
    assert dll.sl_kv4_attention(pool(), attn(n_tokens=1 << 24, max_rows=1 << 24), None) == abi.SL_ERR_TOO_LARGE
    assert dll.sl_kv4_attention(pool(n_kv=2), attn(n_tokens=1 << 22, max_rows=1 << 22, n_heads=16, n_req=4096), None) == abi.SL_ERR_TOO_LARGE
    assert dll.sl_kv4_attention(pool(), attn(n_req=4097), None) == abi.SL_ERR_TOO_LARGE


@pytest.mark.parametrize("scale", [float("nan"), float("inf"), float("-inf")])
def test_attention_refuses_a_scale_that_is_not_finite(scale):
    assert lib.get().dll.sl_kv4_attention(pool(), attn(scale=scale), None) == abi.SL_ERR_ARG
