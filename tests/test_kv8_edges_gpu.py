"""Edges of the 8-bit paged cache's operators on the GPU: scales at the ends of
fp32, blocks and positions that are not there, windows and lengths near 2^31,
workspaces that grow or are captured, and error bits across all of it.

Bounds as in test_kv8_gpu.py (``mass`` is sum_j p_j |v_j|); where V's scales are
tiny the output's floor is half of bf16's smallest number, 2^-134, and P in
fp16's subnormal range adds keys * 2^-21 of the largest |v| (V's power of two
ends at 2^127, so P of a scale of 2^-131 is normal down to 2^-10)."""

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from oracle import kv8_oracle as kv8o  # noqa: E402
from test_kv8_gpu import _attend, _check_attention, _codes_tensor, _errors, _i32, _np, _scene  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    from paged_tierkv_b200 import _native, ops
    _native.load(build_if_missing=True)
    yield
    assert ops.read_device_errors() == 0


@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 64, 2 ** 30, 2 ** 30 - 1])
@pytest.mark.parametrize("q", [5, 90])
def test_a_window_as_wide_as_an_int_is_no_window(q, window):
    """Also for a request that was not admitted: more query tokens than keys."""
    kv = [3, 0, 64]
    rng = np.random.default_rng(q)
    scene = _scene(rng, kv, [q, q, q], 2, 1, 128, 16, "int8", "fp16")
    _check_attention(scene, kv, 16, "int8", "fp16", 0.1, window)


# ---------------------------------------------------------------------------
# plans
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("tokens", [64, 2000])                   # one CTA, a cluster
def test_plans_of_lengths_near_the_end_of_an_int(tokens):
    """Lengths whose sums pass 2^31: refused, and the requests around them planned."""
    from paged_tierkv_b200 import kv8
    big = 2 ** 31 - 1
    ctx, new = [0, big, 5, 0, big - 3], [big, big, 7, 20, 30]
    plan = kv8.StepPlan.allocate(5, tokens, 16, "cuda")
    table = torch.full((5, 4), 77, dtype=torch.int32, device="cuda")
    kv8.plan_step(plan, _i32(ctx), _i32(new), table, _i32([10, 11, 12, 13]), _i32([4]))
    assert _errors() & 4
    assert _np(plan.admitted).tolist() == [0, 0, 1, 1, 0]
    assert _np(plan.kv_lens).tolist()[:3] == [0, big, 12]
    assert _np(plan.cu_q).tolist() == [0, big, big, big, big, big]
    assert int(plan.free_count) == 2 and (_np(plan.slot_map) == -1).all() and (_np(plan.token_request) == 0).all()
    np.testing.assert_array_equal(_np(plan.positions), np.arange(tokens))
    np.testing.assert_array_equal(_np(table), np.array([[77] * 4] * 3 + [[13, 12, 77, 77]] + [[77] * 4]))
    # a refused request at the end of the range, first in the batch
    kv8.plan_step(plan, _i32([big - 3, 5]), _i32([30, 7]), table, _i32([10]), _i32([1]))
    assert _errors() & 4
    assert _np(plan.cu_q)[:3].tolist() == [0, 30, 37] and _np(plan.kv_lens)[:2].tolist() == [big - 3, 12]
    want = np.full(tokens, -1)
    want[:37] = np.concatenate([np.minimum(big - 3 + np.arange(30), big), 5 + np.arange(7)])
    np.testing.assert_array_equal(_np(plan.positions), want)


@pytest.mark.parametrize("tokens", [64, 2000])
def test_plans_of_more_blocks_than_an_int_counts(tokens):
    """Forty requests that would take 2^26 - 1 blocks each: what they ask for
    never wraps into blocks that the free list holds."""
    from paged_tierkv_b200 import kv8
    n, width = 43, 2 ** 26 - 1
    new = [20] + [16 * width] * 40 + [1, 0]
    plan = kv8.StepPlan.allocate(n, tokens, 16, "cuda")
    table = torch.empty((n, width), dtype=torch.int32, device="cuda")
    kv8.plan_step(plan, _i32([0] * n), _i32(new), table, _i32(np.arange(50, 60)), _i32([10]))
    assert _errors() & 4
    assert _np(plan.admitted).tolist() == [1] + [0] * 41 + [1]
    assert _np(plan.kv_lens).tolist() == [20] + [0] * 42 and int(plan.free_count) == 8 and int(plan.num_units) == 2
    assert _np(table[0, :2]).tolist() == [59, 58]
    cu = _np(plan.cu_q)
    assert cu[:3].tolist() == [0, 20, 20 + 16 * width] and (np.diff(cu) >= 0).all() and cu[-1] == 2 ** 31 - 1
# ---------------------------------------------------------------------------
# scales
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("exponent", [-110, -124])
@pytest.mark.parametrize("mixed", [False, True])
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("kv,ql,heads", [
    ([500, 300], [1, 1], 1),            # few rows
    ([500, 300], [200, 66], 1),         # many rows, units split over CTAs
    ([60, 50, 55], [49] * 3, 100),      # many rows, whole units
])
def test_tiny_v_scales_leave_the_row_sums_alone(exponent, mixed, fmt, kv, ql, heads):
    """V scales that append writes for tiny values (2^-116 and below, subnormal
    ones too): the LSE depends on K alone, and the values stay what they are.
    Mixed: beside ordinary blocks."""
    rng = np.random.default_rng(200 + exponent)
    scene = _scene(rng, kv, ql, heads, heads, 64, 16, fmt, "bf16")
    vs = scene[3]
    live = np.isfinite(vs[:, 0])
    if mixed:
        live &= rng.integers(0, 2, len(live)).astype(bool)
    vs[live] *= np.float32(2.0 ** exponent)
    kc, ks, vc, vs, table, cu, q = scene
    out, lse = _attend(scene, kv, 16, fmt, 0.125)
    ref, rl, mass, size = kv8o.attention(q.double().cpu().numpy(), kc, vc, ks, vs, table, kv, cu, 0.125, fmt)
    got, gl = out.double().cpu().numpy(), lse.double().cpu().numpy()
    assert np.all(np.abs(gl - rl) <= 2.0 ** -18 * size + 2.0 ** -19 * (1 + np.abs(rl)))
    eps, biggest = 2.0 ** -8, np.nanmax(vs) * float(kv8o.QMAX[fmt])
    tol = (mass * (2.0 ** -11 + 2.0 ** -17 * size[..., None] + 2.0 ** -18) * (1 + eps) + eps * np.abs(ref) + 2.0 ** -134
           + max(kv) * 2.0 ** -21 * biggest)
    err = np.abs(got - ref)
    assert np.all(err <= tol), (np.nanmax(err / tol), np.argwhere(~(err <= tol))[:3])


# ---------------------------------------------------------------------------
# blocks that are not there
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("ql", [[1, 1], [40, 70]])
@pytest.mark.parametrize("d,bs", [(128, 16), (64, 32), (128, 64)])
def test_cells_outside_the_cache_read_zeros_whatever_block_0_holds(ql, d, bs):
    """Block 0 is nobody's and full of e4m3 NaN codes."""
    kv = [4 * bs + 5, 150]
    rng = np.random.default_rng(31)
    kc, ks, vc, vs, table, cu, q = _scene(rng, kv, ql, 2, 1, d, bs, "e4m3", "fp16")
    table = table + 1
    kc, vc = (np.concatenate([np.full_like(x[:1], 0x7F), x]) for x in (kc, vc))
    ks, vs = (np.concatenate([np.ones_like(x[:1]), x]) for x in (ks, vs))
    table[0, 2], table[1, 0] = -1, kc.shape[0]
    _check_attention((kc, ks, vc, vs, table, cu, q), kv, bs, "e4m3", "fp16", 0.09)
    assert _errors() == 1


# ---------------------------------------------------------------------------
# error bits
# ---------------------------------------------------------------------------

def _step(new, free, bs=16, capacity=None, width=4):
    """A plan over an empty cache of ``free`` blocks, and a batch for it."""
    from paged_tierkv_b200 import kv8
    tokens = capacity or sum(new)
    cache = kv8.Kv8Cache.allocate(max(free, 1), 1, bs, 64, "cuda")
    plan = kv8.StepPlan.allocate(len(new), tokens, bs, "cuda")
    kv8.plan_step(plan, _i32([0] * len(new)), _i32(new), torch.full((len(new), width), -1, dtype=torch.int32, device="cuda"),
                  _i32(np.arange(free)), _i32([free]))
    gen = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(tokens, 1, 64, generator=gen, device="cuda").half()
    return cache, plan, x


@pytest.mark.parametrize("axes", [1, 3])
@pytest.mark.parametrize("wide", [False, True])
def test_padding_tokens_are_no_error(axes, wide):
    """A step padded to a fixed number of tokens: positions past the last token
    are -1, which every operator takes without an error; others still count."""
    from paged_tierkv_b200 import kv8
    cache, plan, x = _step([10, 3], free=2, capacity=20)
    angle = torch.rand(16, 32, device="cuda")
    rotary = kv8.Rotary(torch.cat([angle.cos(), angle.sin()], 1), (32,) if axes == 1 else (10, 11, 11))
    pos = plan.positions.expand(axes, -1)
    pos = pos.long() if wide else pos
    q = kv8.append(cache, plan, x, x, q=x, positions=pos, rotary=rotary)
    both = kv8.rotary_embed(x, x, pos, rotary)
    assert torch.equal(both[0], q) and torch.equal(both[1], q)
    kv8.attention(q, cache, plan, 0.125)
    assert _errors() == 0
    for bad in (-2, 16):
        pos = pos.clone()
        pos[:, 12] = bad
        kv8.append(cache, plan, x, x, q=x, positions=pos, rotary=rotary)
        assert _errors() == 8
        kv8.rotary_embed(x, None, pos, rotary)
        assert _errors() == 8


def test_error_bits_survive_a_growing_workspace():
    """The first step of a fresh stream refuses a request; attention then needs a
    larger workspace, and after it a chunk a still larger one."""
    from paged_tierkv_b200 import kv8, ops
    torch.cuda.synchronize()
    ops._WORKSPACES.clear()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        cache, plan, x = _step([10, 30], free=1)
        kv8.append(cache, plan, x, x)
        kv8.attention(x, cache, plan, 0.125, max_q_len=1)
        assert ops.read_device_errors() == 4
        kv8.plan_step(plan, _i32([0, 0]), _i32([30, 1]), torch.full((2, 4), -1, dtype=torch.int32, device="cuda"),
                      _i32([0]), _i32([1]))
        big = torch.zeros(200, 1, 64, dtype=torch.float16, device="cuda")
        table = torch.zeros(1, 20, dtype=torch.int32, device="cuda")
        kv8.attention(big, cache, kv8.StepPlan(block_size=16, block_table=table, kv_lens=_i32([200]), cu_q=_i32([0, 200])), 0.125)
        assert ops.read_device_errors() == 4
        assert ops.read_device_errors() == 0


def test_one_error_is_raised_once_though_the_workspace_grows():
    """A watch that recorded the word before the growth clears the bits after it too."""
    from paged_tierkv_b200 import kv8, ops
    torch.cuda.synchronize()
    ops._WORKSPACES.clear()
    watch = ops.DeviceErrorWatch()
    cache, plan, x = _step([10, 30], free=1)
    watch.record(ops.workspace_error_word())
    kv8.attention(x, cache, plan, 0.125)
    with pytest.raises(ops.TierKVDeviceError):
        watch.check()
    watch.record(ops.workspace_error_word())
    watch.check()
    assert ops.read_device_errors() == 0


# ---------------------------------------------------------------------------
# graphs
# ---------------------------------------------------------------------------

def _decode(seed, kv=(3000, 17, 900), ql=(1, 1, 1)):
    """(call, expected output): units split over CTAs, so that the arrival
    counters of the workspace are used."""
    from paged_tierkv_b200 import kv8
    rng = np.random.default_rng(seed)
    kc, ks, vc, vs, table, cu, q = scene = _scene(rng, list(kv), list(ql), 4, 2, 128, 16, "int8", "fp16")
    want, _ = _attend(scene, list(kv), 16, "int8", 0.09)
    cache = kv8.Kv8Cache(*(torch.from_numpy(x).cuda() for x in (kc, vc, ks, vs)))
    plan = kv8.StepPlan(block_size=16, block_table=_i32(table), kv_lens=_i32(kv), cu_q=_i32(cu))
    return (lambda: kv8.attention(q, cache, plan, 0.09)), want


def _captured(call, stream=None):
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=stream):
        out = call()
    return g, out


@pytest.mark.parametrize("cold", [False, True])
def test_graphs_of_one_stream_replay_in_any_order(cold):
    from paged_tierkv_b200 import ops
    calls = [_decode(40), _decode(41, (2500, 300), (1, 30))]
    torch.cuda.synchronize()
    if cold:                                   # the captures come before any call on their stream
        ops._WORKSPACES.clear()
    graphs = [_captured(call) for call, _ in calls]
    for i in (1, 0, 0, 1, 1):
        graphs[i][1].zero_()
        graphs[i][0].replay()
        torch.cuda.synchronize()
        assert torch.equal(graphs[i][1], calls[i][1])


def test_a_graph_keeps_its_workspace_when_the_stream_needs_a_larger_one():
    from paged_tierkv_b200 import ops
    side = torch.cuda.Stream()
    (decode, want), (chunk, want_chunk) = _decode(42), _decode(43, (400, 900), (60, 200))
    torch.cuda.synchronize()
    ops._WORKSPACES.clear()
    with torch.cuda.stream(side):
        decode()
    g, out = _captured(decode, side)
    with torch.cuda.stream(side):
        assert torch.equal(chunk(), want_chunk)
        filler = [torch.full((n,), 77, dtype=torch.uint8, device="cuda") for n in [1 << 16, 1 << 20, 2 << 20, 3 << 20] * 8]
        for _ in range(3):
            out.zero_()
            g.replay()
            side.synchronize()
            assert torch.equal(out, want)
        assert all(bool((f == 77).all()) for f in filler)
        assert torch.equal(decode(), want)


def test_graphs_replay_beside_one_another():
    calls = [_decode(44), _decode(45), _decode(46, (1800, 800), (40, 1))]
    graphs = [_captured(call) for call, _ in calls]
    streams = [torch.cuda.Stream() for _ in graphs]
    torch.cuda.synchronize()
    for _ in range(50):
        for s, (g, _) in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for (_, out), (_, want) in zip(graphs, calls):
        assert torch.equal(out, want)


def test_tiered_decode_graphs_replay_in_any_order():
    from paged_tierkv_b200 import ops
    from tierkv_cases import make_case, to_device
    cases = [make_case(seed=s, batch=2, q_heads=32, kv_heads=8, head_dim=128, num_blocks=70, max_blocks=72) for s in (1, 2)]
    data = [to_device(c) for c in cases]

    def call(c, d):
        return ops.decode_attention(d["query"], d["block_table"], d["block_states"], d["block_lengths"], d["pools"],
                                    d["num_blocks"], c["groups"], c["scaling"], num_splits=6)[0]
    want = [call(c, d) for c, d in zip(cases, data)]
    torch.cuda.synchronize()
    ops._WORKSPACES.clear()
    graphs = [_captured(lambda c=c, d=d: call(c, d)) for c, d in zip(cases, data)]
    for i in (1, 0, 1):
        graphs[i][1].zero_()
        graphs[i][0].replay()
        torch.cuda.synchronize()
        assert torch.allclose(graphs[i][1].float(), want[i].float(), atol=2e-3)


def test_errors_of_replays_are_read():
    from paged_tierkv_b200 import kv8, ops
    cache = kv8.Kv8Cache.allocate(4, 1, 16, 64, "cuda")
    table = _i32([[0, 9]])
    plan = kv8.StepPlan(block_size=16, block_table=table, kv_lens=_i32([20]), cu_q=_i32([0, 1]))
    q = torch.zeros(1, 1, 64, dtype=torch.float16, device="cuda")
    assert _errors() == 0
    g, _ = _captured(lambda: kv8.attention(q, cache, plan, 0.1))
    assert _errors() == 0
    g.replay()
    g.replay()
    torch.cuda.synchronize()
    assert _errors() == 1 and _errors() == 0
    table[0, 1] = 2
    g.replay()
    torch.cuda.synchronize()
    assert _errors() == 0
    del g
    ops.release_graph_workspaces()
    assert not ops._GRAPH_WORKSPACES and _errors() == 0


@pytest.mark.parametrize("tokens,bits", [(None, 0), (23, 0), (22, 16), (0, 0)])
def test_a_step_of_more_tokens_than_its_outputs_hold_is_reported(tokens, bits):
    """The dropped tokens are counted in kv_lens but have no slot and no unit."""
    from paged_tierkv_b200 import kv8
    plan = kv8.StepPlan.allocate(2, 40, 16, "cuda")
    kv8.plan_step(plan, _i32([0, 0]), _i32([20, 3]), torch.full((2, 4), -1, dtype=torch.int32, device="cuda"),
                  _i32(np.arange(9)), _i32([9]), tokens=tokens)
    assert _errors() == bits


def test_a_window_past_an_int_is_no_window():
    rng = np.random.default_rng(50)
    scene = _scene(rng, [200], [3], 2, 1, 128, 16, "int8", "fp16")
    a, b = _attend(scene, [200], 16, "int8", 0.1), _attend(scene, [200], 16, "int8", 0.1, 2 ** 40)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_inputs_that_require_a_gradient_give_outputs_without_one():
    from paged_tierkv_b200 import kv8
    rng = np.random.default_rng(51)
    scene = _scene(rng, [40], [3], 2, 1, 64, 16, "int8", "fp16")
    out, lse = _attend(scene, [40], 16, "int8", 0.1, q=scene[6].requires_grad_())
    rotary = kv8.Rotary(torch.ones(4, 64, device="cuda"))
    turned, _ = kv8.rotary_embed(scene[6], None, _i32([0, 1, 2]), rotary)
    assert not (out.requires_grad or lse.requires_grad or turned.requires_grad)


# ---------------------------------------------------------------------------
# precision
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("group,ql", [(4, 1), (3, 1), (1, 4), (2, 2), (1, 1)])
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("d,bs", [(128, 16), (64, 32)])
def test_up_to_four_rows_keep_what_fp16_drops_of_p(group, ql, fmt, d, bs):
    """fp16 queries with up to 4 rows a kv head: P counts with two fp16 numbers,
    2^-21 of it instead of 2^-11 in the bound of the other tests."""
    kv = [700, 40, 3000]
    rng = np.random.default_rng(60 + group)
    scene = _scene(rng, kv, [ql] * 3, 2 * group, 2, d, bs, fmt, "fp16")
    kc, ks, vc, vs, table, cu, q = scene
    out, _ = _attend(scene, kv, bs, fmt, d ** -0.5, max_q_len=ql)
    ref, _, mass, size = kv8o.attention(q.double().cpu().numpy(), kc, vc, ks, vs, table, kv, cu, d ** -0.5, fmt)
    eps = 2.0 ** -11
    tol = mass * (2.0 ** -21 + 2.0 ** -17 * size[..., None] + 2.0 ** -18) * (1 + eps) + eps * np.abs(ref) + 2.0 ** -25
    err = np.abs(out.double().cpu().numpy() - ref)
    assert np.all(err <= tol), (np.nanmax(err / tol), np.argwhere(~(err <= tol))[:3])


@pytest.mark.parametrize("ql", [[1] * 3, [60, 1, 45]])
def test_a_bound_of_zero_query_tokens_costs_time_only(ql):
    kv = [100, 7, 64]
    rng = np.random.default_rng(70)
    scene = _scene(rng, kv, ql, 4, 2, 64, 16, "int8", "fp16")
    out = torch.full(scene[6].shape, 9.0, dtype=torch.float16, device="cuda")
    _check_attention(scene, kv, 16, "int8", "fp16", 0.125, max_q_len=0, out=out)
