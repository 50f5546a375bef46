"""The 8-bit paged cache on the GPU against its oracle.

Plans, codes and scales are whole numbers or fp32 values rounded step by step:
they have to be equal.  Attention is held to a bound per element, from what the
kernels round (``mass`` is sum_j p_j |v_j|, ``size`` the largest sum_d |q_d k_d| *
scaling of the row):
  fp16 P: 2^-11 mass; logits (fp32 accumulation): 2^-18 size relative in p,
  numerator and denominator: 2^-17 size mass; exp2, fp32 sums: 2^-18 mass;
  output: half an ulp of its type, 2^-11 (fp16) or 2^-8 (bf16) of the value,
  and 2^-25 below fp16's normal range.
The LSE: 2^-18 size + 2^-19 (1 + |lse|)."""

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from oracle import kv8_oracle as kv8o  # noqa: E402

pytestmark = pytest.mark.gpu

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
CODES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    from paged_tierkv_b200 import _native, ops
    _native.load(build_if_missing=True)
    yield
    assert ops.read_device_errors() == 0


def _np(t):
    return t.detach().cpu().view(torch.uint8).numpy() if t.dtype == torch.float8_e4m3fn else t.detach().cpu().numpy()


def _i32(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")


def _codes_tensor(c, fmt):
    t = torch.from_numpy(np.ascontiguousarray(c)).cuda()
    return t if fmt == "int8" else t.view(torch.float8_e4m3fn)


def _errors():
    from paged_tierkv_b200 import ops
    return ops.read_device_errors()


# ---------------------------------------------------------------------------
# step planning
# ---------------------------------------------------------------------------

def _check_plan(ctx, new, width, bs, free, count, tokens=None, extra=0, stride=None, plan=None):
    from paged_tierkv_b200 import kv8
    n = len(ctx)
    total = int(np.maximum(new, 0).sum())
    cap = total + extra
    rng = np.random.default_rng(0)
    table = rng.integers(0, 10 ** 6, (n, stride or width)).astype(np.int32)
    dev = torch.from_numpy(table).cuda()
    plan = plan or kv8.StepPlan.allocate(n, cap, bs, "cuda")
    kv8.plan_step(plan, _i32(ctx), _i32(new), dev[:, :width], _i32(free), _i32([count]), tokens=tokens)
    tk = cap if tokens is None else tokens
    units = min(tk, tk // bs + 2 * n)
    want = kv8o.plan_step(ctx, new, table, free, count, bs, tk, units, width)
    for name in ("kv_lens", "cu_q", "admitted", "slot_map", "token_request", "positions", "units"):
        got = _np(getattr(plan, name))
        np.testing.assert_array_equal(got[:len(want[name])], want[name], err_msg=name)
    assert int(plan.num_units) == want["num_units"] and int(plan.free_count) == want["free_count"]
    np.testing.assert_array_equal(_np(dev), want["table"])
    assert bool(_errors() & 4) == want["refused"]
    return plan, want


@pytest.mark.parametrize("n,ctx_max,new_max,bs", [
    (1, 0, 1, 16), (1, 100, 1, 16), (3, 40, 0, 32), (33, 70, 1, 16), (33, 500, 90, 64), (257, 65, 33, 32),
    (1025, 300, 5, 16), (8192, 20, 2, 16)])
def test_plan_matches_the_oracle(n, ctx_max, new_max, bs):
    rng = np.random.default_rng(n + bs)
    ctx, new = rng.integers(0, ctx_max + 1, n), rng.integers(0, new_max + 1, n)
    free = rng.permutation(n * (new_max // bs + 2) + 3)
    _check_plan(ctx, new, (ctx_max + new_max) // bs + 1, bs, free, len(free), extra=n % 3)


def test_plan_one_long_prompt():
    _check_plan(np.array([5]), np.array([70001]), 4400, 16, np.random.default_rng(1).permutation(4500), 4500)


@pytest.mark.parametrize("count", [0, 1, 4, 9])
def test_plan_refuses_what_the_free_list_cannot_hold(count):
    _check_plan(np.array([3, 16, 0, 30, 15]), np.array([1, 33, 20, 1, 0]), 5, 16, np.arange(100, 110), count)


def test_plan_refuses_rows_that_do_not_fit_the_table():
    _check_plan(np.array([10, 64, 0]), np.array([60, 1, 65]), 4, 16, np.arange(50), 50, stride=7)


def test_plan_counts_negative_lengths_as_zero_and_drops_tokens_past_the_limit():
    _check_plan(np.array([-5, 7]), np.array([-3, 9]), 2, 16, np.arange(9), 9)
    _check_plan(np.array([0, 0, 0]), np.array([5, 9, 40]), 4, 16, np.arange(20), 20, tokens=11)


def test_plan_steps_in_place():
    """kv_lens and free_count feed the next step from the plan's own buffers."""
    from paged_tierkv_b200 import kv8
    plan = kv8.StepPlan.allocate(3, 40, 16, "cuda")
    table = torch.full((3, 8), -1, dtype=torch.int32, device="cuda")
    free = _i32(np.arange(30)[::-1].copy())
    ctx, count = _i32([0, 0, 0]), _i32([30])
    ref_ctx, ref_table, ref_count = np.zeros(3, int), np.full((3, 8), -1, np.int32), 30
    for new in ([20, 7, 1], [1, 1, 1], [1, 0, 16], [12, 9, 1]):
        kv8.plan_step(plan, ctx, _i32(new), table, free, count)
        want = kv8o.plan_step(ref_ctx, new, ref_table, _np(free), ref_count, 16, 40, 8, 8)
        ref_ctx, ref_table, ref_count = want["kv_lens"], want["table"], want["free_count"]
        ctx, count = plan.kv_lens, plan.free_count
        np.testing.assert_array_equal(_np(ctx), ref_ctx)
        np.testing.assert_array_equal(_np(table), ref_table)
        assert int(count) == ref_count


# ---------------------------------------------------------------------------
# rotary
# ---------------------------------------------------------------------------

def _cos_sin(rows, rot, rng):
    a = rng.uniform(0, 6.28, (rows, rot // 2))
    return np.concatenate([np.cos(a), np.sin(a)], 1).astype(np.float32)


def _check_turned(got, x, ref32, ref64, dtype):
    """One rounding of the fp32 result: bit-equal; and near the 64-bit one."""
    want = torch.from_numpy(ref32.astype(np.float32)).to(DTYPES[dtype])
    assert torch.equal(got.cpu(), want)
    eps = 2.0 ** -11 if dtype == "fp16" else 2.0 ** -8
    pair = np.abs(x).max(-1, keepdims=True) * 2
    assert np.all(np.abs(got.cpu().double().numpy() - ref64) <= eps * np.abs(ref64) + 2.0 ** -22 * pair + 2.0 ** -25)


@pytest.mark.parametrize("d,rot,sections,inter,pairs", [
    (128, 128, (64,), False, False), (128, 128, (16, 24, 24), False, False), (128, 128, (24, 20, 20), True, False),
    (64, 32, (5, 6, 5), False, False), (64, 64, (8, 8, 8, 8), True, True), (128, 64, (32,), False, True),
    (80, 16, (3, 2, 3), True, False), (256, 256, (128,), False, False), (16, 16, (0, 8), False, True)])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("tokens", [1, 37])
def test_rotary_matches_the_oracle(d, rot, sections, inter, pairs, dtype, tokens):
    from paged_tierkv_b200 import kv8
    rng = np.random.default_rng(d + rot + tokens)
    table = _cos_sin(50, rot, rng)
    qkv = torch.from_numpy(rng.standard_normal((tokens, 7, d))).to(DTYPES[dtype]).cuda()
    q, k = qkv[:, :4], qkv[:, 4:6]
    pos = rng.integers(0, 50, (len(sections), tokens))
    for p in (_i32(pos), torch.from_numpy(pos).cuda(), torch.from_numpy(pos.T.copy()).cuda().t()):
        r = kv8.Rotary(torch.from_numpy(table).cuda(), sections, inter, pairs)
        qo, ko = kv8.rotary_embed(q, k, p, r)
        for got, x in ((qo, q), (ko, k)):
            x = x.cpu().float().numpy()
            _check_turned(got, x, kv8o.rotate(x, pos, table, sections, inter, pairs, np.float32),
                          kv8o.rotate(x, pos, table, sections, inter, pairs), dtype)


def test_rotary_in_place_alone_and_unaligned():
    from paged_tierkv_b200 import kv8
    rng = np.random.default_rng(3)
    table = _cos_sin(64, 64, rng)
    r = kv8.Rotary(torch.from_numpy(table).cuda())
    pos = rng.integers(0, 64, 9)
    x = torch.from_numpy(rng.standard_normal((9, 3, 64))).half().cuda()
    want, none = kv8.rotary_embed(x, None, _i32(pos), r)
    assert none is None
    y = x.clone()
    kv8.rotary_embed(None, y, _i32(pos), r, k_out=y)
    assert torch.equal(y, want)
    odd = torch.empty(9 * 3 * 64 + 3, dtype=torch.float16, device="cuda")[3:].view(9, 3, 64)
    odd.copy_(x)                                        # 6 bytes off
    assert torch.equal(kv8.rotary_embed(odd, None, _i32(pos), r)[0], want)
    swapped = x.transpose(0, 1).contiguous().transpose(0, 1)   # heads outermost in memory
    assert torch.equal(kv8.rotary_embed(swapped, None, _i32(pos), r)[0], want)
    empty = x[:0]
    assert kv8.rotary_embed(empty, empty, _i32([]), r)[0].shape == (0, 3, 64)
    assert _errors() == 0


def test_rotary_positions_outside_the_table_are_clamped_and_reported():
    from paged_tierkv_b200 import kv8
    rng = np.random.default_rng(4)
    table = _cos_sin(10, 64, rng)
    r = kv8.Rotary(torch.from_numpy(table).cuda())
    x = torch.from_numpy(rng.standard_normal((3, 1, 64))).half().cuda()
    got, _ = kv8.rotary_embed(x, None, torch.tensor([-1, 10, 2 ** 40], device="cuda"), r)
    assert _errors() == 8
    want, _ = kv8.rotary_embed(x, None, _i32([0, 9, 9]), r)
    assert torch.equal(got, want)


# ---------------------------------------------------------------------------
# append
# ---------------------------------------------------------------------------

def _random_cache(rng, blocks, kvh, bs, d, fmt):
    x = rng.standard_normal((blocks, kvh, bs, d)).astype(np.float32) * rng.uniform(0.2, 3, (blocks, kvh, 1, 1)).astype(np.float32)
    scale = (np.abs(x).max((2, 3)) / kv8o.QMAX[fmt]).astype(np.float32)
    return kv8o.encode(x / scale[..., None, None], fmt), scale


def _units(rng, lens, bs, blocks):
    """Write units of requests (context, new) over random distinct blocks."""
    ids, u, t = iter(rng.permutation(blocks)), [], 0
    for c, n in lens:
        for j in range(c // bs, -(-(c + n) // bs)) if n else ():
            lo, hi = max(c, j * bs), min(c + n, (j + 1) * bs)
            u.append((int(next(ids)), t + lo - c, lo - j * bs, hi - lo))
        t += n
    return u, t


@pytest.mark.parametrize("d,bs,kvh", [(128, 16, 1), (128, 32, 3), (128, 64, 2), (64, 16, 5), (64, 32, 2), (64, 64, 1)])
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype,rotate", [("fp16", "none"), ("bf16", "one"), ("fp16", "three"), ("bf16", "pairs")])
def test_append_codes_and_scales_are_the_formulas(d, bs, kvh, fmt, dtype, rotate):
    from paged_tierkv_b200 import kv8
    rng = np.random.default_rng(d + bs + kvh)
    lens = [(0, 1), (5, 1), (15, 1), (16, 40), (3, bs), (2 * bs - 1, 2), (7, 0), (0, 3 * bs + 5)]
    blocks = 40
    units, tokens = _units(rng, lens, bs, blocks)
    (kc, ks), (vc, vs) = _random_cache(rng, blocks, kvh, bs, d, fmt), _random_cache(rng, blocks, kvh, bs, d, fmt)
    cache = kv8.Kv8Cache(_codes_tensor(kc, fmt), _codes_tensor(vc, fmt), torch.from_numpy(ks).cuda(),
                         torch.from_numpy(vs).cuda())
    qkv = torch.from_numpy(rng.standard_normal((tokens, 4 + 2 * kvh, d)) * 1.5).to(DTYPES[dtype]).cuda()
    q, k, v = qkv[:, :4], qkv[:, 4:4 + kvh], qkv[:, 4 + kvh:]
    plan = kv8.StepPlan(block_size=bs, units=_i32(units + [(-1,) * 4] * 3), num_units=_i32([len(units)]))
    k32, v32 = k.float().cpu().numpy(), v.float().cpu().numpy()
    if rotate == "none":
        assert kv8.append(cache, plan, k, v) is None
    else:
        half = d // 2
        sections = {"one": (half,), "three": (half - 2 * (half // 3), half // 3, half // 3), "pairs": (half // 2,)}[rotate]
        inter, pairs = rotate == "three", rotate == "pairs"
        table = _cos_sin(300, 2 * sum(sections), rng)
        pos = rng.integers(0, 300, (len(sections), tokens))
        got = kv8.append(cache, plan, k, v, q=q, positions=_i32(pos),
                         rotary=kv8.Rotary(torch.from_numpy(table).cuda(), sections, inter, pairs))
        q32 = q.float().cpu().numpy()
        _check_turned(got, q32, kv8o.rotate(q32, pos, table, sections, inter, pairs, np.float32),
                      kv8o.rotate(q32, pos, table, sections, inter, pairs), dtype)
        k32 = kv8o.rotate(k32, pos, table, sections, inter, pairs, np.float32)
    for x, codes, scale, dev_codes, dev_scale in ((k32, kc, ks, cache.k_codes, cache.k_scale),
                                                  (v32, vc, vs, cache.v_codes, cache.v_scale)):
        kv8o.write_units(x, codes, scale, units, fmt)
        np.testing.assert_array_equal(_np(dev_codes), codes)
        np.testing.assert_array_equal(_np(dev_scale), scale)
        # against the values, in 64 bits: half a step of the scale (e4m3: of the
        # value's own binade, 2^-4 of it, or of the smallest normal, 2^-10 of the scale)
        for b, t0, off, n in units:
            val = kv8o.code_values(codes[b, :, off:off + n], fmt) * scale[b].astype(np.float64)[:, None, None]
            x64 = x[t0:t0 + n].transpose(1, 0, 2).astype(np.float64)
            step = scale[b][:, None, None] * 0.5 if fmt == "int8" else np.maximum(np.abs(x64) / 16, scale[b][:, None, None] * 2.0 ** -10)
            assert np.all(np.abs(val - x64) <= step * (1 + 1e-5))


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_append_grows_a_block_token_by_token(fmt):
    from paged_tierkv_b200 import kv8
    rng = np.random.default_rng(9)
    cache = kv8.Kv8Cache.allocate(2, 2, 16, 64, "cuda", CODES[fmt])
    kc, ks = np.zeros((2, 2, 16, 64), np.int8 if fmt == "int8" else np.uint8), np.ones((2, 2), np.float32)
    vc, vs = kc.copy(), ks.copy()
    x = (rng.standard_normal((16, 2, 64)) * rng.uniform(0.1, 4, (16, 1, 1))).astype(np.float16)
    for t in range(16):
        row = torch.from_numpy(x[t:t + 1]).cuda()
        plan = kv8.StepPlan(block_size=16, units=_i32([(1, 0, t, 1)]), num_units=_i32([1]))
        kv8.append(cache, plan, row, -row)
        kv8o.write_units(x[t:t + 1].astype(np.float32), kc, ks, [(1, 0, t, 1)], fmt)
        kv8o.write_units(-x[t:t + 1].astype(np.float32), vc, vs, [(1, 0, t, 1)], fmt)
        np.testing.assert_array_equal(_np(cache.k_codes), kc)
        np.testing.assert_array_equal(_np(cache.v_codes), vc)
        np.testing.assert_array_equal(_np(cache.k_scale), ks)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_append_of_zeros_infinities_and_nan(fmt):
    from paged_tierkv_b200 import kv8
    cache = kv8.Kv8Cache.allocate(6, 1, 32, 64, "cuda", CODES[fmt])
    x = torch.ones(5 * 32, 1, 64, dtype=torch.float16, device="cuda")
    x[:32] = 0
    x[40, 0, 3], x[70, 0, 9], x[100, 0, 0] = float("nan"), float("inf"), float("-inf")
    units = [(b, 32 * b, 0, 32) for b in range(5)]
    kv8.append(cache, kv8.StepPlan(block_size=32, units=_i32(units), num_units=_i32([5])), x, x)
    s = _np(cache.k_scale)[:, 0]
    assert s[0] == 1 and np.isnan(s[1:4]).all() and s[4] == np.float32(1) / kv8o.QMAX[fmt] and s[5] == 1
    assert not _np(cache.k_codes)[:4].any()
    # a poisoned block stays poisoned when finite rows follow
    y = torch.ones(1, 1, 64, dtype=torch.float16, device="cuda")
    cache.k_scale[5] = float("nan")
    kv8.append(cache, kv8.StepPlan(block_size=32, units=_i32([(5, 0, 7, 1)]), num_units=_i32([1])), y, y)
    assert np.isnan(_np(cache.k_scale)[5, 0]) and not np.isnan(_np(cache.v_scale)[5, 0])


def test_append_skips_and_reports_units_outside():
    from paged_tierkv_b200 import kv8
    cache = kv8.Kv8Cache.allocate(4, 2, 16, 64, "cuda")
    before = [_np(t).copy() for t in (cache.k_codes, cache.v_codes, cache.k_scale, cache.v_scale)]
    x = torch.ones(8, 2, 64, dtype=torch.float16, device="cuda")
    for bad in ((4, 0, 0, 1), (-1, 0, 0, 1), (0, 0, 16, 1), (0, 0, -1, 1), (0, 0, 10, 7), (0, 7, 0, 2), (0, -1, 0, 1),
                (0, 0, 0, 0)):
        kv8.append(cache, kv8.StepPlan(block_size=16, units=_i32([bad]), num_units=_i32([1])), x, x)
        assert _errors() == 1, bad
    for was, t in zip(before, (cache.k_codes, cache.v_codes, cache.k_scale, cache.v_scale)):
        np.testing.assert_array_equal(was, _np(t))
    kv8.append(cache, kv8.StepPlan(block_size=16, units=_i32([(0, 0, 0, 8)]), num_units=_i32([0])), x, x)
    kv8.append(cache, kv8.StepPlan(block_size=16, units=_i32([(0, 0, 0, 8)]), num_units=_i32([1])), x[:0], x[:0])
    np.testing.assert_array_equal(before[0], _np(cache.k_codes))


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------

def _bounds(ref, mass, size, dtype):
    eps = 2.0 ** -11 if dtype == "fp16" else 2.0 ** -8
    s = size[..., None]
    return mass * (2.0 ** -11 + 2.0 ** -17 * s + 2.0 ** -18) * (1 + eps) + eps * np.abs(ref) + 2.0 ** -25


def _scene(rng, kv, ql, heads, kvh, d, bs, fmt, dtype, shuffle=True, size=1.0):
    """Cache, tables and queries; whatever no request owns is poisoned."""
    held = [-(-k // bs) for k in kv]
    blocks = sum(held) + 3
    (kc, ks), (vc, vs) = _random_cache(rng, blocks, kvh, bs, d, fmt), _random_cache(rng, blocks, kvh, bs, d, fmt)
    ids = rng.permutation(blocks) if shuffle else np.arange(blocks)
    width = max(max(held, default=0), 1) + 2
    table = rng.integers(-5, 10 ** 6, (len(kv), width)).astype(np.int32)     # unused cells: anything
    at = 0
    for r, (n, h) in enumerate(zip(kv, held)):
        table[r, :h] = ids[at:at + h]
        at += h
        if n % bs:                                     # rows past the end of the last block: anything
            junk = (0x7F if fmt == "e4m3" else 0x55)
            kc[table[r, h - 1], :, n % bs:] = junk
            vc[table[r, h - 1], :, n % bs:] = junk
    for b in ids[at:]:
        ks[b] = vs[b] = np.nan
    cu = np.concatenate([[0], np.cumsum(ql)])
    q = (torch.from_numpy(rng.standard_normal((int(cu[-1]), heads, d)) * size)).to(DTYPES[dtype]).cuda()
    return kc, ks, vc, vs, table, cu, q


def _attend(scene, kv, bs, fmt, scaling, window=0, **kw):
    from paged_tierkv_b200 import kv8
    kc, ks, vc, vs, table, cu, q = scene
    cache = kv8.Kv8Cache(_codes_tensor(kc, fmt), _codes_tensor(vc, fmt), torch.from_numpy(ks).cuda(),
                         torch.from_numpy(vs).cuda())
    plan = kv8.StepPlan(block_size=bs, block_table=_i32(table), kv_lens=_i32(kv), cu_q=_i32(cu))
    return kv8.attention(kw.pop("q", q), cache, plan, scaling, window=window, return_lse=True, **kw)


def _check_attention(scene, kv, bs, fmt, dtype, scaling, window=0, **kw):
    kc, ks, vc, vs, table, cu, q = scene
    out, lse = _attend(scene, kv, bs, fmt, scaling, window, **kw)
    ref, rl, mass, size = kv8o.attention(q.double().cpu().numpy(), kc, vc, ks, vs, table, kv, cu, scaling, fmt, window)
    got, gl = out.double().cpu().numpy(), lse.double().cpu().numpy()
    err, tol = np.abs(got - ref), _bounds(ref, mass, size, dtype)
    assert np.all(err <= tol), (np.nanmax(err / tol), np.argwhere(~(err <= tol))[:3])
    empty = np.isneginf(rl)
    assert np.array_equal(empty, np.isneginf(gl)) and not got[empty].any()
    el = np.abs(gl[~empty] - rl[~empty])
    assert np.all(el <= 2.0 ** -18 * size[~empty] + 2.0 ** -19 * (1 + np.abs(rl[~empty])))
    return out, lse


SHAPES = [(128, 16), (128, 32), (128, 64), (64, 16), (64, 32), (64, 64)]


@pytest.mark.parametrize("d,bs", SHAPES)
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_single_tokens(d, bs, fmt, dtype):
    """Ragged decode: lengths 0, 1, around blocks, warp tiles and steps, several steps."""
    kv = [0, 1, 2, bs - 1, bs, bs + 1, 31, 33, 127, 128, 129, 300, 777]
    rng = np.random.default_rng(d + bs)
    scene = _scene(rng, kv, [1] * len(kv), 6, 2, d, bs, fmt, dtype)
    _check_attention(scene, kv, bs, fmt, dtype, d ** -0.5, max_q_len=1)


@pytest.mark.parametrize("group,kvh", [(1, 1), (2, 3), (5, 2), (7, 1), (8, 2), (11, 1), (16, 1), (17, 1), (64, 1)])
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_groups_of_query_heads(group, kvh, fmt):
    kv = [70, 1, 0, 200]
    rng = np.random.default_rng(group)
    scene = _scene(rng, kv, [1] * 4, group * kvh, kvh, 128, 16, fmt, "fp16")
    _check_attention(scene, kv, 16, fmt, "fp16", 0.09, max_q_len=1)


@pytest.mark.parametrize("d,bs", SHAPES)
@pytest.mark.parametrize("fmt,dtype", [("int8", "bf16"), ("e4m3", "fp16")])
@pytest.mark.parametrize("window", [0, 1, 50])
def test_drafted_tokens(d, bs, fmt, dtype, window):
    """Two to four tokens a request (8 and 16 rows a tile), the first of a request among them."""
    ql, kv = [2, 3, 4, 1, 4, 0, 2], [2, 70, 129, 40, 300, 9, 161]
    rng = np.random.default_rng(d + bs + window)
    scene = _scene(rng, kv, ql, 4, 2, d, bs, fmt, dtype)
    _check_attention(scene, kv, bs, fmt, dtype, d ** -0.5, window, max_q_len=4)


@pytest.mark.parametrize("d,bs", SHAPES)
@pytest.mark.parametrize("fmt,dtype", [("int8", "fp16"), ("e4m3", "bf16")])
@pytest.mark.parametrize("window", [0, 37, 200])
def test_prompts_and_chunks(d, bs, fmt, dtype, window):
    """Long queries on the tensor cores beside single tokens: a whole prompt, a
    chunk at the end of a context, one that splits rows unevenly, empty ones."""
    ql, kv = [150, 1, 77, 0, 3, 129], [150, 260, 333, 5, 90, 129]
    rng = np.random.default_rng(d + bs + window)
    scene = _scene(rng, kv, ql, 3, 1, d, bs, fmt, dtype)
    _check_attention(scene, kv, bs, fmt, dtype, d ** -0.5, window)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("q", [1, 2, 20, 100, 300])
def test_a_lone_request(fmt, q):
    rng = np.random.default_rng(q)
    scene = _scene(rng, [700], [q], 4, 1, 128, 16, fmt, "fp16")
    _check_attention(scene, [700], 16, fmt, "fp16", 0.07)


@pytest.mark.parametrize("q,kv", [(1, 9000), (3, 5000), (40, 6000)])
def test_long_contexts_are_split_and_joined(q, kv):
    rng = np.random.default_rng(kv)
    scene = _scene(rng, [kv], [q], 8, 2, 64, 32, "int8", "fp16")
    _check_attention(scene, [kv], 32, "int8", "fp16", 0.125)


@pytest.mark.parametrize("q", [5, 90])
def test_more_queries_than_keys_see_nothing(q):
    """A request that was not admitted: query tokens before the first key."""
    kv = [3, 0, 64]
    rng = np.random.default_rng(q)
    scene = _scene(rng, kv, [q, q, q], 2, 1, 128, 16, "int8", "fp16")
    _check_attention(scene, kv, 16, "int8", "fp16", 0.1)
    _check_attention(scene, kv, 16, "int8", "fp16", 0.1, 2)


@pytest.mark.parametrize("ql", [[1] * 3, [60, 1, 45]])
def test_a_low_bound_of_the_query_lengths_costs_time_only(ql):
    kv = [100, 7, 64]
    rng = np.random.default_rng(0)
    scene = _scene(rng, kv, ql, 4, 2, 64, 16, "int8", "fp16")
    _check_attention(scene, kv, 16, "int8", "fp16", 0.125, max_q_len=1)


@pytest.mark.parametrize("ql", [[1] * 4, [30, 1, 50, 2]])
@pytest.mark.parametrize("size", [1e-4, 300.0])
def test_small_and_large_queries(ql, size):
    kv = [100, 40, 64, 200]
    rng = np.random.default_rng(5)
    scene = _scene(rng, kv, ql, 4, 2, 64, 16, "e4m3", "bf16", size=size)
    _check_attention(scene, kv, 16, "e4m3", "bf16", 0.125 / max(1.0, size / 10))


@pytest.mark.parametrize("ql", [[1, 1], [100, 33]])
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_scales_of_any_size(ql, fmt):
    """V scales from 2^-60 to 2^40 and zero in one context, K scales of zero."""
    kv = [500, 300]
    rng = np.random.default_rng(6)
    scene = _scene(rng, kv, ql, 2, 1, 64, 16, fmt, "bf16")
    kc, ks, vc, vs, table, cu, q = scene
    live = np.isfinite(vs[:, 0])
    vs[live] *= (2.0 ** rng.choice([-60, -20, 0, 3, 40], vs[live].shape)).astype(np.float32)
    vs[rng.permutation(np.flatnonzero(live))[:6]] = 0
    ks[rng.permutation(np.flatnonzero(live))[:6]] = 0
    _check_attention(scene, kv, 16, fmt, "bf16", 0.125)


@pytest.mark.parametrize("ql", [[1, 1], [80, 40]])
def test_a_rising_context_moves_the_maximum(ql):
    """Keys that grow along the context: the running maximum moves at every tile."""
    kv = [900, 600]
    rng = np.random.default_rng(7)
    scene = _scene(rng, kv, ql, 2, 1, 64, 16, "int8", "fp16", shuffle=False)
    ks = scene[1]
    ks[np.isfinite(ks[:, 0])] *= np.linspace(0.01, 6, int(np.isfinite(ks[:, 0]).sum()))[:, None].astype(np.float32)
    _check_attention(scene, kv, 16, "int8", "fp16", 0.3)


@pytest.mark.parametrize("ql", [[1, 1, 1], [70, 1, 33]])
def test_poison_reaches_only_the_rows_that_see_it(ql):
    kv = [300, 200, 100]
    rng = np.random.default_rng(8)
    for which in (1, 3):                        # K's scale, V's scale
        scene = _scene(rng, kv, ql, 2, 1, 128, 16, "int8", "fp16")
        table, cu = scene[4], scene[5]
        clean, _ = _attend(scene, kv, 16, "int8", 0.09)
        scene[which][table[0, 290 // 16], 0] = np.nan            # keys 288 .. 299 of request 0
        out, lse = _attend(scene, kv, 16, "int8", 0.09)
        sees = np.array([kv[0] - (cu[1] - t) >= 288 if t < cu[1] else False for t in range(cu[-1])])
        assert torch.isnan(out).any(-1).cpu().numpy()[sees].all()
        assert torch.equal(out[~torch.from_numpy(sees)], clean[~torch.from_numpy(sees)])


def test_non_finite_queries_stay_in_their_rows():
    rng = np.random.default_rng(10)
    for ql in ([1, 1], [50, 70]):
        scene = _scene(rng, [100, 90], ql, 2, 1, 64, 16, "int8", "bf16")
        clean, _ = _attend(scene, [100, 90], 16, "int8", 0.1)
        q = scene[6].clone()
        q[0, 1, 5], q[-1, 0, 0] = float("nan"), float("inf")
        out, _ = _attend(scene, [100, 90], 16, "int8", 0.1, q=q)
        assert torch.isnan(out[0, 1]).all() and torch.isnan(out[-1, 0]).all()
        keep = torch.ones(q.shape[:2], dtype=torch.bool, device="cuda")
        keep[0, 1] = keep[-1, 0] = False
        assert torch.equal(out[keep], clean[keep])


@pytest.mark.parametrize("ql", [[1, 1], [40, 20]])
def test_cells_outside_the_cache_read_zeros_and_are_reported(ql):
    kv = [100, 64]
    rng = np.random.default_rng(11)
    scene = _scene(rng, kv, ql, 2, 1, 128, 16, "int8", "fp16")
    scene[4][0, 2], scene[4][1, 0] = -1, scene[0].shape[0]
    _check_attention(scene, kv, 16, "int8", "fp16", 0.09)
    assert _errors() == 1


def test_shared_blocks_and_strided_inputs():
    """Two requests over one prefix; queries as a slice of a fused projection; a wide table's slice."""
    from paged_tierkv_b200 import kv8
    rng = np.random.default_rng(12)
    for ql in ([1, 1], [40, 9]):
        kv = [120, 100]
        scene = list(_scene(rng, kv, ql, 4, 2, 64, 16, "int8", "fp16"))
        scene[4][1, :6] = scene[4][0, :6]
        q = scene[6]
        fused = torch.randn(q.shape[0], 4 + 4, 64, device="cuda").half()
        fused[:, 2:6] = q
        a = _check_attention(tuple(scene), kv, 16, "int8", "fp16", 0.125)[0]
        b = _attend(tuple(scene), kv, 16, "int8", 0.125, q=fused[:, 2:6])[0]
        assert torch.equal(a, b)
        odd = torch.empty(q.numel() + 1, dtype=q.dtype, device="cuda")[1:].view(q.shape)
        odd.copy_(q)
        assert torch.equal(a, _attend(tuple(scene), kv, 16, "int8", 0.125, q=odd)[0])
        wide = torch.full((2, 40), 7, dtype=torch.int32, device="cuda")
        wide[:, 3:3 + scene[4].shape[1]] = _i32(scene[4])
        cache = kv8.Kv8Cache(*(torch.from_numpy(x).cuda() for x in (scene[0], scene[2], scene[1], scene[3])))
        plan = kv8.StepPlan(block_size=16, block_table=wide[:, 3:3 + scene[4].shape[1]], kv_lens=_i32(kv), cu_q=_i32(scene[5]))
        assert torch.equal(a, kv8.attention(q, cache, plan, 0.125))


def test_rows_of_no_request_are_left_alone():
    rng = np.random.default_rng(13)
    for ql in ([1, 1], [40, 9]):
        scene = list(_scene(rng, [50, 60], ql, 2, 1, 64, 16, "int8", "fp16"))
        n = scene[6].shape[0]
        q = torch.cat([scene[6], scene[6][:3]])
        out = torch.full(q.shape, 7.0, dtype=torch.float16, device="cuda")
        _attend(tuple(scene), [50, 60], 16, "int8", 0.125, q=q, out=out)
        assert (out[n:] == 7).all() and not (out[:n] == 7).all()


def test_repeated_calls_give_the_same_bits():
    rng = np.random.default_rng(14)
    for ql, kv in (([1] * 3, [3000, 17, 900]), ([200, 1, 31], [1500, 800, 64])):
        scene = _scene(rng, kv, ql, 4, 2, 128, 16, "int8", "fp16")
        a = _attend(scene, kv, 16, "int8", 0.09)
        for _ in range(5):
            b = _attend(scene, kv, 16, "int8", 0.09)
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("d,bs", SHAPES)
@pytest.mark.parametrize("fmt,dtype", [("int8", "bf16"), ("e4m3", "fp16")])
@pytest.mark.parametrize("window", [0, 50])
@pytest.mark.parametrize("room", [0, 700000])
def test_few_rows_under_narrow_and_wide_tables(d, bs, fmt, dtype, window, room):
    """20 to 48 rows a kv head: tables with room for long contexts take the kernel
    for many rows, narrow ones the kernel for few."""
    kv, ql = [5, 64, 300, 3, 777, 130], [5, 6, 12, 1, 2, 0]
    rng = np.random.default_rng(bs + window)
    scene = list(_scene(rng, kv, ql, 8, 2, d, bs, fmt, dtype))
    scene[4] = np.concatenate([scene[4], rng.integers(-5, 10 ** 6, (len(kv), room // bs))], 1).astype(np.int32)
    _check_attention(tuple(scene), kv, bs, fmt, dtype, d ** -0.5, window, max_q_len=12)


@pytest.mark.parametrize("kv,kvh", [
    ([5000], 1),                                          # one unit in more parts than a join takes at once
    ([1700, 1, 0, 2600], 2),                              # every CTA a part of one unit
    ([100 + 41 * r for r in range(20)], 16),              # more units than CTAs
    ([6000 + 7 * r for r in range(9)], 8),                # ranges over the boundaries of split units
])
@pytest.mark.parametrize("window", [0, 1000])
def test_how_single_tokens_are_split_over_ctas(kv, kvh, window):
    rng = np.random.default_rng(len(kv))
    scene = _scene(rng, kv, [1] * len(kv), kvh, kvh, 64, 16, "int8", "fp16")
    _check_attention(scene, kv, 16, "int8", "fp16", 0.125, window, max_q_len=1)


def test_another_stream_and_a_graph():
    from paged_tierkv_b200 import kv8
    rng = np.random.default_rng(15)
    kv, ql = [400, 90], [30, 1]
    scene = _scene(rng, kv, ql, 4, 2, 128, 16, "int8", "fp16")
    want, _ = _attend(scene, kv, 16, "int8", 0.09)
    cache = kv8.Kv8Cache(*(torch.from_numpy(x).cuda() for x in (scene[0], scene[2], scene[1], scene[3])))
    plan = kv8.StepPlan(block_size=16, block_table=_i32(scene[4]), kv_lens=_i32(kv), cu_q=_i32(scene[5]))
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    out = kv8.attention(scene[6], cache, plan, 0.09, stream=side)
    side.synchronize()
    assert torch.equal(out, want)
    with torch.cuda.stream(side):
        out = kv8.attention(scene[6], cache, plan, 0.09)
    side.synchronize()
    assert torch.equal(out, want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = kv8.attention(scene[6], cache, plan, 0.09)
    for _ in range(3):
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_demoted_blocks_can_be_attended():
    """Format S's WARM pools as a cache: one query token agrees with the tiered
    decode over the same blocks (both within the fp16 bounds of the true value)."""
    from paged_tierkv_b200 import kv8, ops
    rng = np.random.default_rng(16)
    n, kvh, bs, d, g = 9, 2, 16, 128, 4
    pools = ops.TieredPools.allocate(n, n, kvh, bs, d, "cuda", ops.FORMAT_S)
    pools.hot_k.copy_(torch.randn_like(pools.hot_k.float()))
    pools.hot_v.copy_(torch.randn_like(pools.hot_v.float()))
    ops.demote_blocks_to_warm(pools, range(n), range(n), [bs] * n)
    table = _i32(rng.permutation(n)[None])
    q = torch.randn(1, kvh * g, d, device="cuda").half()
    want, _, lse = ops.decode_attention(q, table, torch.ones_like(table), torch.full_like(table, bs), pools, n, g,
                                        0.09, return_lse=True)
    plan = kv8.StepPlan(block_size=bs, block_table=table, kv_lens=_i32([n * bs]), cu_q=_i32([0, 1]))
    out, l2 = kv8.attention(q, kv8.Kv8Cache.of_pools(pools), plan, 0.09, return_lse=True)
    assert torch.allclose(out.float(), want.float(), atol=4e-3) and torch.allclose(l2, lse, atol=1e-3)


def test_offsets_past_32_bits():
    """Caches of 4.5 GB a tensor: blocks at both ends, both kernels."""
    from paged_tierkv_b200 import kv8
    kvh, bs, d = 8, 16, 128
    blocks = (9 << 29) // (kvh * bs * d)
    cache = kv8.Kv8Cache(*(torch.empty((blocks, kvh, bs, d), dtype=torch.int8, device="cuda") for _ in range(2)),
                         *(torch.full((blocks, kvh), float("nan"), device="cuda") for _ in range(2)))
    rng = np.random.default_rng(17)
    ids = np.concatenate([np.arange(blocks - 20, blocks), np.arange(12)])
    (kc, ks), (vc, vs) = _random_cache(rng, 32, kvh, bs, d, "int8"), _random_cache(rng, 32, kvh, bs, d, "int8")
    at = torch.from_numpy(ids).cuda()
    for dev, x in ((cache.k_codes, kc), (cache.v_codes, vc), (cache.k_scale, ks), (cache.v_scale, vs)):
        dev[at] = torch.from_numpy(x).cuda()
    for q in (1, 40):
        kv = [32 * bs - 5]
        x = torch.from_numpy(rng.standard_normal((q, kvh, d))).half().cuda()
        plan = kv8.StepPlan(block_size=bs, block_table=_i32(ids[None]), kv_lens=_i32(kv), cu_q=_i32([0, q]))
        out, lse = kv8.attention(x, cache, plan, 0.09, return_lse=True)
        ref, rl, mass, size = kv8o.attention(x.double().cpu().numpy(), kc, vc, ks, vs, np.arange(32)[None], kv, [0, q], 0.09, "int8")
        assert np.all(np.abs(out.double().cpu().numpy() - ref) <= _bounds(ref, mass, size, "fp16"))
    # and a write at the far end
    row = torch.randn(1, kvh, d, device="cuda").half()
    kv8.append(cache, kv8.StepPlan(block_size=bs, units=_i32([(blocks - 1, 0, 0, 1)]), num_units=_i32([1])), row, row)
    x32 = row.float().cpu().numpy()
    c, s = np.zeros((1, kvh, bs, d), np.int8), np.ones((1, kvh), np.float32)
    kv8o.write_units(x32, c, s, [(0, 0, 0, 1)], "int8")
    np.testing.assert_array_equal(_np(cache.k_codes[-1, :, 0]), c[0, :, 0])


# ---------------------------------------------------------------------------
# refusals of the Python entry points
# ---------------------------------------------------------------------------

def test_refusals():
    from paged_tierkv_b200 import kv8
    dev = "cuda"
    cache = kv8.Kv8Cache.allocate(4, 2, 16, 64, dev)
    h = torch.zeros(3, 4, 64, dtype=torch.float16, device=dev)
    kv = h[:, :2]
    table = torch.zeros(1, 2, dtype=torch.int32, device=dev)
    plan = kv8.StepPlan(block_size=16, block_table=table, kv_lens=_i32([3]), cu_q=_i32([0, 3]), units=_i32([(0, 0, 0, 3)]),
                        num_units=_i32([1]))
    rot = kv8.Rotary(torch.zeros(8, 64, device=dev))
    pos = _i32([0, 1, 2])
    own = kv8.StepPlan.allocate(2, 8, 16, dev)
    one, two = _i32([1]), _i32([1, 1])
    bad = [
        lambda: kv8.Kv8Cache(cache.k_codes.float(), cache.v_codes, cache.k_scale, cache.v_scale),
        lambda: kv8.Kv8Cache(cache.k_codes, cache.v_codes[:2], cache.k_scale, cache.v_scale),
        lambda: kv8.Kv8Cache(cache.k_codes, cache.v_codes, cache.k_scale.half(), cache.v_scale.half()),
        lambda: kv8.Kv8Cache(cache.k_codes.cpu(), cache.v_codes.cpu(), cache.k_scale.cpu(), cache.v_scale.cpu()),
        lambda: kv8.Kv8Cache.allocate(4, 2, 16, 64, dev, torch.uint8),
        lambda: kv8.Rotary(torch.zeros(8, 64, device=dev), sections=(3, 4)),
        lambda: kv8.Rotary(torch.zeros(8, 64, device=dev).half()),
        lambda: kv8.StepPlan(block_size=16, block_table=table),
        lambda: kv8.StepPlan(block_size=16, block_table=table.long(), kv_lens=_i32([3]), cu_q=_i32([0, 3])),
        lambda: kv8.StepPlan(block_size=16, units=_i32([0, 0]), num_units=one),
        lambda: kv8.StepPlan.allocate(0, 8, 16, dev),
        lambda: kv8.StepPlan.allocate(9000, 8, 16, dev),
        lambda: kv8.plan_step(plan, one, one, table, one, one),
        lambda: kv8.plan_step(own, two.long(), two, table, one, one),
        lambda: kv8.plan_step(own, two, one, table, one, one),
        lambda: kv8.plan_step(own, two, two, table, one, one),
        lambda: kv8.plan_step(own, one, one, table, one, one, tokens=9),
        lambda: kv8.rotary_embed(None, None, pos, rot),
        lambda: kv8.rotary_embed(h.float(), None, pos, rot),
        lambda: kv8.rotary_embed(h, kv[:2], pos, rot),
        lambda: kv8.rotary_embed(h, None, pos.float(), rot),
        lambda: kv8.rotary_embed(h, None, pos[:2], rot),
        lambda: kv8.rotary_embed(h, None, pos, rot, q_out=h[:, :2]),
        lambda: kv8.rotary_embed(h[..., :32], None, pos, rot),
        lambda: kv8.append(cache, plan, h, h),
        lambda: kv8.append(cache, plan, kv, kv.bfloat16()),
        lambda: kv8.append(cache, plan, kv, kv, q=h),
        lambda: kv8.append(cache, plan, kv, kv, rotary=rot),
        lambda: kv8.append(cache, kv8.StepPlan(block_size=16), kv, kv),
        lambda: kv8.append(cache, kv8.StepPlan(block_size=32, units=plan.units, num_units=one), kv, kv),
        lambda: kv8.attention(h.float(), cache, plan, 0.1),
        lambda: kv8.attention(h[:, :3], cache, plan, 0.1),
        lambda: kv8.attention(h, cache, kv8.StepPlan(block_size=16), 0.1),
        lambda: kv8.attention(h, cache, plan, 0.0),
        lambda: kv8.attention(h, cache, plan, float("nan")),
        lambda: kv8.attention(h, cache, plan, 0.1, window=-1),
        lambda: kv8.attention(h, cache, plan, 0.1, out=h[:, :2]),
        lambda: kv8.attention(h.cpu(), cache, plan, 0.1),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            pytest.fail(f"call {i} was not refused")


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("amax", [2.0 ** -130, 2.0 ** -120, 2.0 ** -60, 1.0, 2.0 ** 100])
def test_append_of_any_magnitude(fmt, amax):
    """Scales down to subnormal ones, and quotients on rounding boundaries."""
    from paged_tierkv_b200 import kv8
    rng = np.random.default_rng(18)
    qmax = float(kv8o.QMAX[fmt])
    cache = kv8.Kv8Cache.allocate(1, 1, 64, 128, "cuda", CODES[fmt])
    x = rng.uniform(-1, 1, (64, 1, 128)) * amax
    half = np.arange(128) - 63.5 if fmt == "int8" else np.concatenate([kv8o.E4M3[:64] + kv8o.E4M3[1:65], -kv8o.E4M3[:64]]) / 2
    x[1, 0] = half * (amax / qmax)                       # on, or next to, boundaries
    x[0, 0, 0] = amax
    t = torch.from_numpy(x).to(torch.bfloat16).cuda()
    kv8.append(cache, kv8.StepPlan(block_size=64, units=_i32([(0, 0, 0, 64)]), num_units=_i32([1])), t, t)
    c = np.zeros((1, 1, 64, 128), np.int8 if fmt == "int8" else np.uint8)
    s = np.ones((1, 1), np.float32)
    kv8o.write_units(t.float().cpu().numpy(), c, s, [(0, 0, 0, 64)], fmt)
    np.testing.assert_array_equal(_np(cache.k_scale), s)
    np.testing.assert_array_equal(_np(cache.k_codes), c)
