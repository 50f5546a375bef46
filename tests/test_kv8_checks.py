"""Checks of the 8-bit cache's front end that need no GPU: tensors are stand-ins
with a device, a type and a shape, and nothing is launched."""

import ctypes
import os
import re
import struct
import subprocess

import pytest

torch = pytest.importorskip("torch")

from paged_tierkv_b200 import _native as N  # noqa: E402
from paged_tierkv_b200 import kv8  # noqa: E402

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


class FakeTensor:
    """What the checks read of a CUDA tensor."""

    def __init__(self, *shape, dtype=torch.int32, device=0, at=0x1000, stride=None):
        self.shape, self.ndim, self.dtype, self._device, self._at = torch.Size(shape), len(shape), dtype, device, at
        self._stride = stride
        self.is_cuda, self.device, self.requires_grad = True, torch.device("cuda", device), False

    def get_device(self):
        return self._device

    def numel(self):
        return self.shape.numel()

    def is_contiguous(self):
        return True

    def stride(self):
        if self._stride is not None:
            return self._stride
        s, out = 1, []
        for n in reversed(self.shape):
            out.append(s)
            s *= n
        return tuple(reversed(out))

    def data_ptr(self):
        return self._at


def _never(*_):
    raise AssertionError("launched")


def _cache(device=0):
    codes, scale = (FakeTensor(4, 2, 16, 64, dtype=torch.int8, device=device), FakeTensor(4, 2, dtype=torch.float32, device=device))
    return kv8.Kv8Cache(codes, codes, scale, scale)


def _plan(device=0, **other):
    t = {"units": FakeTensor(3, 4), "num_units": FakeTensor(1), "block_table": FakeTensor(1, 2), "kv_lens": FakeTensor(1),
         "cu_q": FakeTensor(2)}
    for name, x in t.items():
        x._device = other.get(name, device)
    return kv8.StepPlan(block_size=16, **t)


@pytest.mark.parametrize("name", ["units", "num_units", "block_table", "kv_lens", "cu_q"])
def test_a_plan_lives_on_one_device(name):
    _plan(1)
    with pytest.raises(ValueError, match="one device"):
        _plan(0, **{name: 1})


def test_num_units_is_one_number():
    with pytest.raises(ValueError, match="num_units"):
        kv8.StepPlan(block_size=16, units=FakeTensor(3, 4), num_units=FakeTensor(2))
    with pytest.raises(ValueError, match="num_units"):
        kv8.StepPlan(block_size=16, units=FakeTensor(3, 4), num_units=FakeTensor(0))


def test_tensors_of_another_device_are_refused(monkeypatch):
    monkeypatch.setattr(kv8, "_launch", _never)
    half = {"dtype": torch.float16}
    x, kv, pos = FakeTensor(3, 4, 64, **half), FakeTensor(3, 2, 64, **half), FakeTensor(3)
    there = kv8.Rotary(FakeTensor(8, 64, dtype=torch.float32, device=1))
    pos_there = FakeTensor(3, device=1)
    for call in (lambda: kv8.append(_cache(), _plan(1), kv, kv),
                 lambda: kv8.append(_cache(), _plan(0), kv, kv, q=x, positions=pos_there, rotary=there, q_out=x),
                 lambda: kv8.append(_cache(1), _plan(1), kv, kv),
                 lambda: kv8.attention(x, _cache(), _plan(1), 0.1, out=x),
                 lambda: kv8.attention(x, _cache(1), _plan(1), 0.1, out=x),
                 lambda: kv8.rotary_embed(x, None, pos_there, there, q_out=x),
                 lambda: kv8.rotary_embed(None, kv, pos_there, there, k_out=kv),
                 lambda: kv8.rotary_embed(x, None, pos, there, q_out=x)):
        with pytest.raises(ValueError, match="device"):
            call()
    for call in (lambda: kv8.append(_cache(), _plan(0), kv, kv), lambda: kv8.attention(x, _cache(), _plan(0), 0.1, out=x)):
        with pytest.raises(AssertionError, match="launched"):
            call()


def test_tensors_whose_addresses_are_kept_cannot_be_exchanged():
    cache, plan = _cache(), _plan()
    for holder, names in ((cache, ("k_codes", "v_codes", "k_scale", "v_scale")),
                          (plan, ("kv_lens", "cu_q", "admitted", "slot_map", "token_request", "positions", "units",
                                  "num_units", "free_count", "block_table"))):
        for name in names:
            with pytest.raises(AttributeError):
                setattr(holder, name, None)
    rotary = kv8.Rotary(FakeTensor(8, 64, dtype=torch.float32))
    with pytest.raises(AttributeError):
        rotary.cos_sin = None


def test_outputs_that_name_one_element_twice_are_refused(monkeypatch):
    monkeypatch.setattr(kv8, "_launch", _never)
    half = {"dtype": torch.float16}
    x, pos, rotary = FakeTensor(3, 4, 64, **half), FakeTensor(3), kv8.Rotary(FakeTensor(8, 64, dtype=torch.float32))
    for stride in ((0, 64, 1), (256, 0, 1), (32, 64, 1), (256, 32, 1)):
        out = FakeTensor(3, 4, 64, stride=stride, **half)
        with pytest.raises(ValueError, match="one element"):
            kv8.rotary_embed(x, None, pos, rotary, q_out=out)
        with pytest.raises(ValueError, match="one element"):
            kv8.append(_cache(), _plan(), FakeTensor(3, 2, 64, **half), FakeTensor(3, 2, 64, **half), q=x, positions=pos,
                       rotary=rotary, q_out=out)
    for stride in ((256, 64, 1), (64, 192, 1), (1024, 128, 1)):      # packed, heads outermost, with room between
        with pytest.raises(AssertionError, match="launched"):
            kv8.rotary_embed(x, None, pos, rotary, q_out=FakeTensor(3, 4, 64, stride=stride, **half))
    one = FakeTensor(1, 1, 64, stride=(0, 0, 1), **half)
    with pytest.raises(AssertionError, match="launched"):
        kv8.rotary_embed(one, None, pos, rotary, q_out=one)


def _leaves(struct_type, base=0):
    """(offset, size) of every scalar of a ctypes structure, in order."""
    for name, kind in struct_type._fields_:
        at = base + getattr(struct_type, name).offset
        if hasattr(kind, "_fields_"):
            yield from _leaves(kind, at)
        elif hasattr(kind, "_length_"):
            yield from ((at + i * ctypes.sizeof(kind._type_), ctypes.sizeof(kind._type_)) for i in range(kind._length_))
        else:
            yield at, ctypes.sizeof(kind)


def _packed(fmt):
    """The same of a native struct format."""
    codes = [c for n, c in re.findall(r"(\d*)([A-Za-z])", fmt) for _ in range(int(n or 1))]
    for i, c in enumerate(codes):
        if c != "x":
            yield struct.calcsize("".join(codes[:i + 1])) - struct.calcsize(c), struct.calcsize(c)


def test_packed_argument_blocks_have_the_structs_offsets():
    for fmt, kind in ((kv8._ROTARY_ARGS, N.TkvRotaryArgs), (kv8._APPEND_ARGS, N.TkvKv8AppendArgs),
                      (kv8._ATTENTION_ARGS, N.TkvKv8AttentionArgs), (kv8._PLAN_ARGS, N.TkvKv8PlanArgs)):
        assert list(_packed(fmt.format)) == list(_leaves(kind)), kind


def test_structs_have_the_headers_offsets(tmp_path):
    pairs = (("tkv_kv8_cache", N.TkvKv8Cache), ("tkv_kv8_plan_args", N.TkvKv8PlanArgs), ("tkv_rotary", N.TkvRotary),
             ("tkv_token_view", N.TkvTokenView), ("tkv_rotary_args", N.TkvRotaryArgs),
             ("tkv_kv8_append_args", N.TkvKv8AppendArgs), ("tkv_kv8_attention_args", N.TkvKv8AttentionArgs))
    checks = "".join(f"_Static_assert(sizeof({c}) == {ctypes.sizeof(k)}, \"{c}\");\n" for c, k in pairs)
    checks += "".join(f"_Static_assert(offsetof({c}, {n}) == {getattr(k, n).offset}, \"{c}.{n}\");\n"
                      for c, k in pairs for n, _ in k._fields_)
    src = tmp_path / "offsets.c"
    src.write_text('#include <stddef.h>\n#include "tierkv_b200.h"\n' + checks)
    subprocess.run(["gcc", "-std=c11", "-fsyntax-only", "-I", os.path.join(ROOT, "include"), str(src)], check=True)
