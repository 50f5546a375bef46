"""CPU checks of the 8-bit paged cache's oracle and of the library's refusals
(no kernel is launched here)."""

import ctypes
import struct

import numpy as np
import pytest

from oracle import kv8_oracle as kv8o
from oracle import tierkv_oracle as orc

torch = pytest.importorskip("torch")


def test_e4m3_table_and_encoder_match_torch():
    b = torch.arange(256, dtype=torch.uint8)
    ref = b.view(torch.float8_e4m3fn).double().numpy()
    np.testing.assert_array_equal(kv8o.E4M3, ref)
    rng = np.random.default_rng(0)
    x = np.concatenate([rng.normal(0, s, 4000) for s in (1e-3, 0.1, 3.0, 200.0)]).astype(np.float32)
    mid = ((kv8o.E4M3[:126] + kv8o.E4M3[1:127]) / 2).astype(np.float32)      # ties
    x = np.concatenate([x, mid, -mid, [0.0, -0.0, 448.0, 460.0, -1e9]]).astype(np.float32)
    ref = torch.from_numpy(np.clip(x, -448, 448)).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    np.testing.assert_array_equal(kv8o.encode(x, "e4m3"), ref)


def test_int8_codes_match_the_demotion_formula():
    rng = np.random.default_rng(1)
    x = rng.standard_normal((16, 128)).astype(np.float16)
    codes, scale = orc.quantize_block_s(x, 16)
    c = np.zeros((1, 1, 16, 128), np.int8)
    s = np.zeros((1, 1), np.float32)
    kv8o.write_units(x[:, None].astype(np.float32), c, s, [(0, 0, 0, 16)], "int8")
    np.testing.assert_array_equal(c[0, 0], codes)
    assert s[0, 0] == np.float32(scale)


def test_rotation_keeps_lengths_and_undoes():
    rng = np.random.default_rng(2)
    ang = rng.uniform(0, 6.28, (50, 32))
    table = np.concatenate([np.cos(ang), np.sin(ang)], 1)
    x = rng.standard_normal((9, 3, 96))
    pos = rng.integers(0, 50, (3, 9))
    for inter in (False, True):
        for pairs in (False, True):
            y = kv8o.rotate(x, pos, table, (12, 10, 10), inter, pairs)
            np.testing.assert_allclose((y ** 2).sum(-1), (x ** 2).sum(-1), rtol=1e-12)
            np.testing.assert_array_equal(y[..., 64:], x[..., 64:])
            back = np.concatenate([table[:, :32], -table[:, 32:]], 1)
            np.testing.assert_allclose(kv8o.rotate(y, pos, back, (12, 10, 10), inter, pairs), x, atol=1e-12)


def test_requantized_rows_stay_near_their_values():
    rng = np.random.default_rng(3)
    c = np.zeros((1, 1, 16, 64), np.int8)
    s = np.zeros((1, 1), np.float32)
    x = rng.standard_normal((16, 1, 64)).astype(np.float32) * np.linspace(0.5, 3, 16)[:, None, None].astype(np.float32)
    for t in range(16):
        kv8o.write_units(x, c, s, [(0, t, t, 1)], "int8")
    # each growth rounds a row again by at most half a step of the scale it gets
    assert np.abs(c[0, 0] * s[0, 0] - x[:, 0]).max() <= 0.5 * s[0, 0] * 16


def test_oracle_plan_conserves_blocks():
    rng = np.random.default_rng(4)
    for _ in range(20):
        n, bs, width = 7, 16, 6
        ctx, new = rng.integers(0, 80, n), rng.integers(0, 40, n)
        table = np.full((n, width), -1, np.int32)
        free = rng.permutation(40).astype(np.int32)
        out = kv8o.plan_step(ctx, new, table, free, 30, bs, int(new.sum()), 64, width)
        fresh = np.sort(out["table"][out["table"] >= 0])
        assert len(np.unique(fresh)) == len(fresh) == 30 - out["free_count"]
        assert out["units"][:out["num_units"], 3].sum() == sum(m for m, a in zip(new, out["admitted"]) if a)


# ---- refusals of the C entry points: host checks come before any device work

def _lib():
    from paged_tierkv_b200 import _native as N
    from paged_tierkv_b200 import build as B
    B.build()
    return N, N.load()


def _cache(N, **kw):
    f = dict(k_codes=256, v_codes=256, k_scale=256, v_scale=256, blocks=10, kv_heads=2, block_size=16,
             head_dim=128, format=0)
    f.update(kw)
    return N.TkvKv8Cache(**f)


@pytest.mark.parametrize("kw,want", [
    (dict(head_dim=96), 2), (dict(block_size=48), 2), (dict(format=2), 2), (dict(kv_heads=0), 1),
    (dict(k_codes=0), 1), (dict(v_codes=264), 1), (dict(blocks=1 << 40), 1), (dict(blocks=0), 1)])
def test_cache_refusals(kw, want):
    N, lib = _lib()
    c = _cache(N, **kw)
    a = N.TkvKv8AttentionArgs(requests=1, tokens=1, heads=2, dtype=0, table_width=1, table_stride=1, scaling=1.0)
    assert lib.tkv_kv8_attention(ctypes.addressof(c), ctypes.addressof(a), None) == want


@pytest.mark.parametrize("kw,want", [
    (dict(requests=0), 1), (dict(requests=9000), 1), (dict(heads=3), 1), (dict(heads=2 * 65), 2),
    (dict(dtype=2), 2), (dict(window=-1), 1), (dict(scaling=0.0), 1), (dict(scaling=float("inf")), 1),
    (dict(table_stride=0), 1), (dict(tokens=1 << 26), 2), (dict(tokens=-1), 1), (dict(kv_lens=0), 1)])
def test_attention_refusals(kw, want):
    N, lib = _lib()
    c = _cache(N)
    f = dict(requests=1, tokens=4, heads=2, dtype=0, table_width=1, table_stride=1, scaling=1.0, max_q_len=4,
             kv_lens=256, cu_q=256, block_table=256)
    f.update(kw)
    a = N.TkvKv8AttentionArgs(**f)
    assert lib.tkv_kv8_attention(ctypes.addressof(c), ctypes.addressof(a), None) == want


@pytest.mark.parametrize("kw,want", [
    (dict(requests=0), 1), (dict(requests=8193), 1), (dict(block_size=24), 2), (dict(context_lens=0), 1),
    (dict(units=8), 1), (dict(table_stride=2), 1), (dict(free_blocks=0), 1), (dict(tokens=-1), 1)])
def test_plan_refusals(kw, want):
    N, lib = _lib()
    f = {n: 256 for n, t in N.TkvKv8PlanArgs._fields_ if t is ctypes.c_void_p}
    f.update(requests=2, tokens=4, units_cap=4, table_width=3, table_stride=3, free_capacity=5, block_size=16)
    f.update(kw)
    a = N.TkvKv8PlanArgs(**f)
    assert lib.tkv_kv8_plan_step(ctypes.addressof(a), None) == want


def _rotary_args(N, rot=None, **kw):
    r = dict(cos_sin=256, positions=256, rows=8, axis_stride=4, positions_bytes=4, rot_dim=64, axes=1,
             sections=(ctypes.c_int32 * 4)(32))
    r.update(rot or {})
    f = dict(rotary=N.TkvRotary(**r), tokens=4, heads=2, kv_heads=0, head_dim=64, dtype=0,
             q=N.TkvTokenView(256, 128, 64), q_out=N.TkvTokenView(256, 128, 64))
    f.update(kw)
    return N.TkvRotaryArgs(**f)


@pytest.mark.parametrize("rot,kw,want", [
    (dict(rot_dim=24), {}, 2), (dict(rot_dim=128), {}, 2), (dict(axes=5), {}, 2), (dict(axes=0), {}, 2),
    (dict(positions_bytes=2), {}, 2), (dict(rows=0), {}, 1), (dict(cos_sin=0), {}, 1), (dict(positions=0), {}, 1),
    (dict(sections=(ctypes.c_int32 * 4)(31)), {}, 1), ({}, dict(head_dim=72), 2), ({}, dict(head_dim=272), 2),
    ({}, dict(dtype=2), 2), ({}, dict(heads=-1), 1)])
def test_rotary_refusals(rot, kw, want):
    N, lib = _lib()
    assert lib.tkv_rotary_embed(ctypes.addressof(_rotary_args(N, rot, **kw)), None) == want


def test_misaligned_views_are_refused():
    N, lib = _lib()
    for view in ((264, 128, 64), (256, 132, 64), (256, 128, 60), (0, 128, 64)):
        assert lib.tkv_rotary_embed(ctypes.addressof(_rotary_args(N, q=N.TkvTokenView(*view))), None) == 1


def test_append_refusals():
    N, lib = _lib()
    c = _cache(N)
    v = N.TkvTokenView(256, 256, 128)
    ok = dict(k=v, v=v, units=256, num_units=256, units_cap=1, tokens=1, heads=0, dtype=0)
    for kw, want in ((dict(heads=2), 1), (dict(dtype=2), 2), (dict(units=0), 1), (dict(num_units=0), 1),
                     (dict(k=N.TkvTokenView(8, 256, 128)), 1), (dict(tokens=-1), 1)):
        a = N.TkvKv8AppendArgs(**{**ok, **kw})
        assert lib.tkv_kv8_append(ctypes.addressof(c), ctypes.addressof(a), None) == want


def test_packed_argument_blocks_have_the_structs_sizes():
    from paged_tierkv_b200 import kv8
    N, _ = _lib()
    assert kv8._ROTARY_ARGS.size == ctypes.sizeof(N.TkvRotaryArgs)
    assert kv8._APPEND_ARGS.size == ctypes.sizeof(N.TkvKv8AppendArgs)
    assert kv8._ATTENTION_ARGS.size == ctypes.sizeof(N.TkvKv8AttentionArgs)
    assert kv8._PLAN_ARGS.size == ctypes.sizeof(N.TkvKv8PlanArgs)
    assert struct.calcsize(kv8._ROTARY) == ctypes.sizeof(N.TkvRotary)
