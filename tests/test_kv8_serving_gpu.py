"""The 8-bit cache's operators together, as the example serves with them."""

import os
import sys

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu
sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    from paged_tierkv_b200 import _native
    _native.load(build_if_missing=True)


def _dense(model, ids):
    """Logits of one sequence's last token with exact fp32 attention, no cache."""
    x = model.embed[torch.tensor(ids, device="cuda")]
    g = model.heads // model.kv_heads
    d = model.head_dim
    cs = model.rotary.cos_sin[:len(ids)]
    c, s = cs[:, None, :d // 2], cs[:, None, d // 2:]

    def turn(t):
        a, b = t.float().split(d // 2, -1)
        return torch.cat([a * c - b * s, b * c + a * s], -1)

    mask = torch.ones(len(ids), len(ids), dtype=torch.bool, device="cuda").tril()
    for qkv, proj in zip(model.qkv, model.proj):
        h = torch.nn.functional.normalize(x.float(), dim=-1).to(x.dtype) * x.shape[-1] ** 0.5
        q, k, v = (h @ qkv).view(len(ids), -1, d).split([model.heads, model.kv_heads, model.kv_heads], 1)
        q, k, v = turn(q), turn(k).repeat_interleave(g, 1), v.float().repeat_interleave(g, 1)
        z = torch.einsum("ihd,jhd->hij", q, k) * d ** -0.5
        p = torch.where(mask, z, float("-inf")).softmax(-1)
        x = x + torch.einsum("hij,jhd->ihd", p, v).to(x.dtype).flatten(1) @ proj
    return x[-1].float() @ model.embed.float().t()


@pytest.mark.parametrize("cache,limit", [(torch.int8, 0.03), (torch.float8_e4m3fn, 0.08)])
def test_chunked_serving_follows_dense_attention(cache, limit):
    """Logits after a prompt served in chunks beside others stay within the
    cache's quantization (half a step of 1/127 of a block's largest value, or
    2^-4 of a value, through two layers) of dense attention's."""
    from kv8_serving import Decoder, serve
    model = Decoder(layers=2, blocks=256, cache_dtype=cache)
    gen = torch.Generator().manual_seed(2)
    prompts = [torch.randint(0, 512, (n,), generator=gen).tolist() for n in (1, 16, 33, 200, 450)]
    for chunk in (48, 450):
        out, last = serve(model, prompts, 1, chunk)
        for p, o, logits in zip(prompts, out, last):
            want = _dense(model, p)
            assert len(o) == 1
            assert (logits - want).norm() <= limit * want.norm()


def test_decoding_runs_past_block_ends():
    from kv8_serving import Decoder, serve
    model = Decoder(layers=2, blocks=64)
    out, _ = serve(model, [[1, 2, 3], [5] * 30], 40, 16)
    assert [len(o) for o in out] == [40, 40]
    again, _ = serve(model, [[1, 2, 3], [5] * 30], 40, 16)
    assert out == again


def test_running_out_of_blocks_is_reported():
    from kv8_serving import Decoder, serve
    model = Decoder(layers=1, blocks=4)
    with pytest.raises(RuntimeError, match="free block"):
        serve(model, [[1] * 100], 2, 50)
