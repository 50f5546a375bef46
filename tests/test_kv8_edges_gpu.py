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
