"""Serving steps over an 8-bit paged cache.

One layer's cache (:class:`Kv8Cache`) is 8-bit throughout -- Format S int8
codes, or e4m3 -- with one fp32 scale per (block, kv head) and tensor.  A batch
of requests with any query lengths (single tokens, drafted tokens, prompt
chunks, whole prompts) takes one step in four calls:

* :func:`plan_step`     block tables, slot maps and write lists from the
  requests' lengths, on the GPU (one plan serves every layer);
* :func:`rotary_embed`  rotary positions with up to four axes, or fused into
* :func:`append`        the quantizing write of the new keys and values;
* :func:`attention`     causal attention of the new tokens over the cache.

Every computation is one call into the C-ABI library (``tkv_kv8_*`` and
``tkv_rotary_embed`` in include/tierkv_b200.h).  Errors the device finds
(out-of-cache slots, exhausted free blocks, positions outside the cos / sin
table) go to the stream's error word, ``ops.read_device_errors``.  The
reference has no counterpart: its 8-bit blocks are filled by demotion only.

These are serving operators without a backward pass: inputs that require a
gradient are taken as they are, and no output carries one.
"""

from __future__ import annotations

import ctypes
import operator
import struct
from dataclasses import dataclass

import torch

from . import _native as N
from . import ops

_FORMAT = {torch.int8: N.TKV_KV8_INT8, torch.float8_e4m3fn: N.TKV_KV8_E4M3}
_FLOATS = {torch.float16: N.TKV_DTYPE_F16, torch.bfloat16: N.TKV_DTYPE_BF16}
_POSITIONS = {torch.int32: 4, torch.int64: 8}
MAX_REQUESTS = N.TKV_KV8_MAX_REQUESTS

# The C structs of include/tierkv_b200.h, packed in one call each: filling them
# through ctypes field by field costs more host time than the small kernels take.
_VIEW = "Pqq"
_ROTARY = "PPqq9i4x"
_ROTARY_ARGS = struct.Struct(_ROTARY + 4 * _VIEW + "P5i4x")
_APPEND_ARGS = struct.Struct(4 * _VIEW + "PPP" + _ROTARY + "4i")
_ATTENTION_ARGS = struct.Struct(_VIEW + "PPPqPP7ifPQ")
_PLAN_ARGS = struct.Struct("PPPqPPPPPPPPPPPP6i")
_NO_VIEW = (0, 0, 0)
_NO_ROTARY = (0,) * 13
_INT32 = torch.int32
_CONTIGUOUS = torch.contiguous_format


# ---------------------------------------------------------------------------
# handles
# ---------------------------------------------------------------------------

def _held(name: str) -> property:
    """A tensor that calls use by its address: it can be written, not exchanged."""
    return property(operator.attrgetter("_" + name))


class Kv8Cache:
    """One layer's 8-bit cache: k_codes / v_codes [blocks, kv_heads, block_size,
    head_dim] int8 or float8_e4m3fn, k_scale / v_scale [blocks, kv_heads] fp32;
    value = code * scale.  block_size 16, 32 or 64; head_dim 64 or 128."""

    k_codes, v_codes, k_scale, v_scale = map(_held, ("k_codes", "v_codes", "k_scale", "v_scale"))

    def __init__(self, k_codes: torch.Tensor, v_codes: torch.Tensor, k_scale: torch.Tensor,
                 v_scale: torch.Tensor):
        if k_codes.ndim != 4 or k_codes.dtype not in _FORMAT:
            raise ValueError("cache codes must be int8 or float8_e4m3fn [blocks, kv_heads, block_size, head_dim].")
        if not k_codes.is_cuda:
            raise ValueError("cache tensors must be CUDA tensors.")
        for t, like in ((v_codes, k_codes), (v_scale, k_scale)):
            if t.shape != like.shape or t.dtype != like.dtype:
                raise ValueError("the value tensors must match the key tensors in shape and dtype.")
        if k_scale.dtype != torch.float32 or tuple(k_scale.shape) != tuple(k_codes.shape[:2]):
            raise ValueError("cache scales must be fp32 [blocks, kv_heads].")
        for t in (k_codes, v_codes, k_scale, v_scale):
            if not t.is_contiguous() or t.device != k_codes.device:
                raise ValueError("cache tensors must be contiguous and on one device.")
        self._k_codes, self._v_codes, self._k_scale, self._v_scale = k_codes, v_codes, k_scale, v_scale
        self.blocks, self.kv_heads, self.block_size, self.head_dim = (int(x) for x in k_codes.shape)
        self.device, self._index = k_codes.device, k_codes.get_device()
        # the tensors are held, so the addresses stay theirs
        self._struct = N.TkvKv8Cache(k_codes.data_ptr(), v_codes.data_ptr(), k_scale.data_ptr(),
                                     v_scale.data_ptr(), self.blocks, self.kv_heads, self.block_size,
                                     self.head_dim, _FORMAT[k_codes.dtype])
        self._ptr = ctypes.addressof(self._struct)

    @classmethod
    def allocate(cls, blocks: int, kv_heads: int, block_size: int, head_dim: int, device,
                 dtype: torch.dtype = torch.int8) -> "Kv8Cache":
        """A cache of zero codes with scale 1."""
        if dtype not in _FORMAT:
            raise ValueError("an 8-bit cache is int8 or float8_e4m3fn.")
        shape = (blocks, kv_heads, block_size, head_dim)
        codes = [torch.zeros(shape, dtype=torch.int8, device=device).view(dtype) for _ in range(2)]
        return cls(*codes, *(torch.ones(shape[:2], device=device) for _ in range(2)))

    @classmethod
    def of_pools(cls, pools: ops.TieredPools) -> "Kv8Cache":
        """The WARM pools of Format S, shared: blocks that demotion filled can be
        attended by any number of query tokens."""
        if pools.fmt != ops.FORMAT_S:
            raise ValueError("an 8-bit cache shares Format S pools only.")
        return cls(pools.warm_k, pools.warm_v, pools.k_scale, pools.v_scale)


class StepPlan:
    """What one step's launches share.  :func:`plan_step` fills a plan made by
    :meth:`allocate`; a program that keeps its own tables passes them here:
    ``units`` / ``num_units`` for :func:`append`, ``block_table`` / ``kv_lens``
    / ``cu_q`` for :func:`attention`.

    kv_lens [requests], cu_q [requests + 1], admitted [requests], slot_map /
    token_request / positions [tokens] (-1 past the last token), units [cap, 4]
    (block, first token, row offset, rows; -1 past the last), num_units [1],
    free_count [1]; all int32."""

    kv_lens, cu_q, admitted, slot_map, token_request, positions, units, num_units, free_count, block_table = map(
        _held, ("kv_lens", "cu_q", "admitted", "slot_map", "token_request", "positions", "units", "num_units",
                "free_count", "block_table"))

    def __init__(self, *, block_size: int, units=None, num_units=None, block_table=None, kv_lens=None,
                 cu_q=None):
        self.block_size = int(block_size)
        self._units, self._num_units = units, num_units
        self._block_table, self._kv_lens, self._cu_q = block_table, kv_lens, cu_q
        self._admitted = self._slot_map = self._token_request = self._positions = self._free_count = None
        self.requests = 0
        self._outputs = None
        for name in ("units", "num_units", "kv_lens", "cu_q"):
            t = getattr(self, name)
            if t is not None and (t.dtype != torch.int32 or not t.is_cuda or not t.is_contiguous()):
                raise ValueError(f"{name} must be a contiguous int32 CUDA tensor.")
        if units is not None and (units.ndim != 2 or units.shape[1] != 4 or num_units is None or num_units.numel() != 1):
            raise ValueError("units must be [count, 4] beside num_units [1].")
        devices = {t.get_device() for t in (units, num_units, block_table, kv_lens, cu_q) if t is not None}
        if len(devices) > 1:
            raise ValueError("a plan's tensors must be on one device.")
        self._index = devices.pop() if devices else None
        if block_table is not None:
            if kv_lens is None or cu_q is None:
                raise ValueError("a block_table needs kv_lens and cu_q.")
            self.requests = int(kv_lens.numel())
            if cu_q.numel() != self.requests + 1:
                raise ValueError("cu_q must have one entry more than kv_lens.")
            _check_table(block_table, self.requests)

    @classmethod
    def allocate(cls, max_requests: int, max_tokens: int, block_size: int, device) -> "StepPlan":
        """Buffers for steps of up to max_requests requests and max_tokens tokens."""
        if not 1 <= max_requests <= MAX_REQUESTS:
            raise ValueError(f"a step plans 1 to {MAX_REQUESTS} requests.")
        if max_tokens < 0:
            raise ValueError("max_tokens must not be negative.")
        r, t = int(max_requests), int(max_tokens)
        cap = _units_cap(r, t, block_size)
        # one buffer: [units | slot_map | token_request | positions | kv_lens | admitted | cu_q | counts]
        sizes = (4 * cap, t, t, t, r, r, r + 1, 1, 1)
        buf = torch.full((sum((n + 3) // 4 * 4 for n in sizes),), -1, dtype=torch.int32, device=device)
        at, parts = 0, []
        for n in sizes:
            parts.append(buf[at:at + n])
            at += (n + 3) // 4 * 4
        units, slot, req, pos, kv, adm, cu, num, free = parts
        plan = cls(block_size=block_size, units=units.view(cap, 4), num_units=num)
        plan._kv_lens, plan._cu_q = kv, cu
        plan._slot_map, plan._token_request, plan._positions = slot, req, pos
        plan._admitted, plan._free_count = adm, free
        plan._outputs = tuple(x.data_ptr() for x in (kv, cu, adm, slot, req, pos, units, num, free))
        plan.device, plan._index = buf.device, buf.get_device()
        plan._caps = (r, t, cap)
        return plan


@dataclass(frozen=True)
class Rotary:
    """Rotary positions: cos_sin [rows, rot_dim] fp32 (the cosines of the rot_dim
    / 2 frequencies, then their sines); ``sections`` frequencies for each of up
    to four axes (None: one axis), one run after the other or, with
    ``interleave``, axis f % axes for frequency f while that axis has any left
    (axis 0 afterwards).  ``pairs``: a pair is two adjacent elements; otherwise
    element f and f + rot_dim / 2."""

    cos_sin: torch.Tensor
    sections: tuple | None = None
    interleave: bool = False
    pairs: bool = False

    def __post_init__(self):
        t = self.cos_sin
        if t.ndim != 2 or t.dtype != torch.float32 or not t.is_cuda or not t.is_contiguous():
            raise ValueError("cos_sin must be a contiguous fp32 CUDA tensor [rows, rot_dim].")
        if t.data_ptr() % 16:
            raise ValueError("cos_sin must be 16-byte aligned.")
        half = int(t.shape[1]) // 2
        sec = (half,) if self.sections is None else tuple(int(x) for x in self.sections)
        if not 1 <= len(sec) <= 4 or any(x < 0 for x in sec) or sum(sec) != half:
            raise ValueError("sections must be 1 to 4 counts that add up to rot_dim / 2.")
        object.__setattr__(self, "axes", len(sec))
        object.__setattr__(self, "rot_dim", int(t.shape[1]))
        object.__setattr__(self, "_tail", (int(t.shape[1]), len(sec), *sec, *(0,) * (4 - len(sec)),
                                           int(bool(self.interleave)), int(bool(self.pairs))))
        object.__setattr__(self, "_head", (t.data_ptr(), int(t.shape[0]), t.get_device()))

    def _at(self, positions: torch.Tensor, tokens: int):
        """(the fields of the C struct with these positions, the tensor that backs them)."""
        ptr, rows, index = self._head
        size = _POSITIONS.get(positions.dtype)
        if size is None or positions.get_device() != index:
            raise ValueError("positions must be int32 or int64 on the table's device.")
        nd = positions.ndim
        if nd == 1 and self.axes == 1:
            n, stride, step = positions.numel(), 0, positions.stride()[0]
        elif nd == 2 and positions.shape[0] == self.axes:
            n, (stride, step) = positions.shape[1], positions.stride()
        else:
            raise ValueError("positions must have shape [axes, tokens] (or [tokens] for one axis).")
        if n < tokens:
            raise ValueError("positions must have shape [axes, tokens] (or [tokens] for one axis).")
        if step != 1 and n > 1:
            positions = positions.contiguous()
            stride = n
        return (ptr, positions.data_ptr(), rows, stride, size, *self._tail), positions


# ---------------------------------------------------------------------------
# shared checks
# ---------------------------------------------------------------------------

def _units_cap(requests: int, tokens: int, block_size: int) -> int:
    return min(tokens, tokens // block_size + 2 * requests)


def _check_table(table: torch.Tensor, requests: int):
    """(row stride, width) of a block table."""
    if table.dtype != _INT32 or not table.is_cuda or table.ndim != 2:
        raise ValueError("block_table must be an int32 CUDA tensor [requests, width].")
    rows, width = table.shape
    s0, s1 = table.stride()
    if rows < requests:
        raise ValueError("block_table must be an int32 CUDA tensor [requests, width].")
    if width > 1 and s1 != 1 or rows > 1 and s0 < width:
        raise ValueError("block_table rows must be contiguous and must not overlap.")
    return (s0 if rows > 1 else width), width


# A view is (address, token stride, head stride) of a [n, h, head_dim] tensor.
# These run on every call, and small calls cost what the host spends on them:
# device indices instead of device objects, shapes read once.

def _view(t: torch.Tensor, n: int, h: int):
    """None if it is not 16-byte aligned throughout."""
    s0, s1, s2 = t.stride()
    ptr = t.data_ptr()
    if n < 2:
        s0 = 0
    if h < 2:
        s1 = 0
    if (ptr | s0 * 2 | s1 * 2) & 15 or s2 != 1 and t.shape[2] > 1:
        return None
    return ptr, s0, s1


def _input_view(t: torch.Tensor, n: int, h: int):
    """(view, tensor that backs it): strided as it is, or through a compact copy."""
    v = _view(t, n, h)
    if v is None:
        t = t.clone(memory_format=_CONTIGUOUS)
        v = _view(t, n, h)
    return v, t


def _output_view(t: torch.Tensor | None, like: torch.Tensor, n: int, h: int, name: str):
    """(output, view): the caller's, or a new contiguous one."""
    if t is None:
        t = torch.empty_like(like, memory_format=_CONTIGUOUS)
        d = like.shape[2]
        return t, (t.data_ptr(), h * d, d)
    if t.shape != like.shape or t.dtype != like.dtype or t.device != like.device:
        raise ValueError(f"{name} must match its input in shape, dtype and device.")
    v = _view(t, n, h)
    if v is None:
        raise ValueError(f"{name} must be 16-byte aligned with head_dim contiguous.")
    d = t.shape[2]
    if n > 1 and v[1] < d or h > 1 and v[2] < d:
        raise ValueError(f"{name} must not name one element for two tokens or heads.")
    return t, v


def _heads3(t: torch.Tensor, name: str):
    """(dtype code, device index) of a tensor [tokens, heads, head_dim]."""
    code, index = _FLOATS.get(t.dtype), t.get_device()
    if code is None or t.ndim != 3:
        raise ValueError(f"{name} must be an fp16 or bf16 tensor [tokens, heads, head_dim].")
    if index < 0:
        raise ValueError(f"{name} must be a CUDA tensor.")
    return code, index


def _on_stream(stream, fn, *args, **kwargs):
    """``stream=``: the whole call -- its copies, outputs and workspace too -- runs
    on that stream, and the caching allocator learns that its inputs are used
    there.  Ordering it after the inputs' producers is the caller's part."""
    for x in (*args, *kwargs.values()):
        for t in (x,) if isinstance(x, torch.Tensor) else getattr(x, "__dict__", {}).values():
            if isinstance(t, torch.Tensor) and t.is_cuda:
                t.record_stream(stream)
    with torch.cuda.stream(stream):
        return fn(*args, **kwargs)


def _launch(index: int, fn):
    """fn(stream handle, its workspace) with device ``index`` current."""
    if index != ops._CURRENT_DEVICE():
        with torch.cuda.device(index):
            return _launch(index, fn)
    st = ops._RAW_STREAM(index) if ops._RAW_STREAM is not None else torch.cuda.current_stream().cuda_stream
    ws = None if ops._CAPTURING() else ops._WORKSPACES.get((index, st))
    return fn(st, ws if ws is not None else ops.workspace_for(torch.device("cuda", index), st, 1 << 16))


# ---------------------------------------------------------------------------
# the operators
# ---------------------------------------------------------------------------

def plan_step(plan: StepPlan, context_lens: torch.Tensor, new_lens: torch.Tensor, block_table: torch.Tensor,
              free_blocks: torch.Tensor, free_count: torch.Tensor, *, tokens: int | None = None,
              stream=None) -> StepPlan:
    """Plans one step on the GPU: request i holds context_lens[i] tokens and gets
    new_lens[i] more, packed one request after the other.

    New blocks come from the end of the free list (free_blocks [capacity],
    free_count [1]) in request order and are written into block_table
    [requests, width]; every other table cell stays.  A request whose row or
    whose share of the free list does not suffice is not admitted: its context
    stays, its tokens get slot -1 and ``TKV_DEVERR_NO_BLOCKS`` is recorded.
    Fills ``plan`` (its buffers' first entries, for fewer requests than it was
    allocated for) and returns it.  ``plan.kv_lens`` and ``plan.free_count`` may
    be passed back as the next step's context_lens and free_count.  ``tokens``:
    how many entries of the token outputs to write (default: all; 0: none are
    wanted); a step of more tokens records ``TKV_DEVERR_DROPPED``."""
    if stream is not None:
        return _on_stream(stream, plan_step, plan, context_lens, new_lens, block_table, free_blocks, free_count,
                          tokens=tokens)
    if plan._outputs is None:
        raise ValueError("plan_step fills a plan made by StepPlan.allocate.")
    n, index = context_lens.numel(), plan._index
    for t in (context_lens, new_lens, free_blocks, free_count):
        if t.dtype != _INT32 or t.get_device() != index or not t.is_contiguous():
            raise ValueError("context_lens, new_lens, free_blocks and free_count must be contiguous int32 "
                             "tensors on the plan's device.")
    max_requests, max_tokens, max_units = plan._caps
    if not 1 <= n <= max_requests or new_lens.numel() != n or free_count.numel() != 1:
        raise ValueError("context_lens and new_lens must have 1 to the plan's max_requests entries, free_count one.")
    stride, width = _check_table(block_table, n)
    if block_table.get_device() != index:
        raise ValueError("block_table must be on the plan's device.")
    tokens = max_tokens if tokens is None else int(tokens)
    if not 0 <= tokens <= max_tokens:
        raise ValueError("tokens must be between 0 and the plan's max_tokens.")
    out = plan._outputs

    def call(st, ws):
        args = _PLAN_ARGS.pack(
            context_lens.data_ptr(), new_lens.data_ptr(), block_table.data_ptr(), stride,
            free_blocks.data_ptr(), free_count.data_ptr(), *out, ws.data_ptr(), n, tokens,
            min(_units_cap(n, tokens, plan.block_size), max_units), width, free_blocks.numel(),
            plan.block_size)
        return N.load().tkv_kv8_plan_step(args, st)

    status = _launch(index, call)
    if status:
        N.check(status, "tkv_kv8_plan_step")
    plan._block_table, plan.requests = block_table, n
    return plan


def rotary_embed(q: torch.Tensor | None, k: torch.Tensor | None, positions: torch.Tensor, rotary: Rotary, *,
                 q_out: torch.Tensor | None = None, k_out: torch.Tensor | None = None, stream=None):
    """Rotates q [tokens, heads, head_dim] and k [tokens, kv_heads, head_dim]
    (fp16 / bf16, any 16-byte aligned token and head strides; either may be
    None) by their tokens' positions [axes, tokens]; returns (q_out, k_out).
    An output may be its input, but not overlap it otherwise.  Position -1 (a step's padding) counts as 0;
    others outside the table are clamped too, and recorded."""
    if stream is not None:
        return _on_stream(stream, rotary_embed, q, k, positions, rotary, q_out=q_out, k_out=k_out)
    qv = kv = qov = kov = _NO_VIEW
    heads = kv_heads = 0
    if q is not None:
        code, index = _heads3(q, "q")
        tokens, heads, d = q.shape
        if index != rotary._head[2]:
            raise ValueError("q must be on the cos / sin table's device.")
        q_out, qov = _output_view(q_out, q, tokens, heads, "q_out")
        qv, q = _input_view(q, tokens, heads)
    elif k is None:
        raise ValueError("rotary_embed needs q or k [tokens, heads, head_dim].")
    if k is not None:
        k_code, k_index = _heads3(k, "k")
        n, kv_heads, dk = k.shape
        if k_index != rotary._head[2]:
            raise ValueError("k must be on the cos / sin table's device.")
        if q is None:
            code, index, tokens, d = k_code, k_index, n, dk
        elif n != tokens or dk != d or k_code != code or k_index != index:
            raise ValueError("q and k must agree in tokens, head_dim, dtype and device.")
        k_out, kov = _output_view(k_out, k, n, kv_heads, "k_out")
        kv, k = _input_view(k, n, kv_heads)
    rot, positions = rotary._at(positions, tokens)

    def call(st, ws):
        args = _ROTARY_ARGS.pack(*rot, *qv, *kv, *qov, *kov, ws.data_ptr(), tokens, heads, kv_heads, d, code)
        return N.load().tkv_rotary_embed(args, st)

    status = _launch(index, call)
    if status:
        N.check(status, "tkv_rotary_embed")
    return (q_out if q is not None else None), (k_out if k is not None else None)


def append(cache: Kv8Cache, plan: StepPlan, k: torch.Tensor, v: torch.Tensor, *, q: torch.Tensor | None = None,
           positions: torch.Tensor | None = None, rotary: Rotary | None = None,
           q_out: torch.Tensor | None = None, stream=None) -> torch.Tensor | None:
    """Quantizes the step's new keys and values [tokens, kv_heads, head_dim] into
    the blocks of ``plan.units``; with ``rotary``, k is rotated on the way (in
    fp32) and q, when given, into q_out, which is returned.

    A block's scale is max |x| / 127 (448 for e4m3) of its rows; when a block
    that already holds rows gets larger ones, its scale grows and its codes are
    rounded again.  A block with a NaN or an infinity gets scale NaN."""
    if stream is not None:
        return _on_stream(stream, append, cache, plan, k, v, q=q, positions=positions, rotary=rotary, q_out=q_out)
    code, index = _heads3(k, "k")
    shape = k.shape
    tokens, kv_heads, d = shape
    if kv_heads != cache.kv_heads or d != cache.head_dim or v.shape != shape or v.dtype != k.dtype:
        raise ValueError("k and v must have shape [tokens, kv_heads, head_dim] of the cache and one dtype.")
    if index != cache._index or v.get_device() != index:
        raise ValueError("k and v must be on the cache's device.")
    if plan.units is None or plan.block_size != cache.block_size or plan._index != index:
        raise ValueError("append needs a plan with write units of the cache's block size, on its device.")
    rot, qv, qov, heads = _NO_ROTARY, _NO_VIEW, _NO_VIEW, 0
    if rotary is not None:
        if positions is None:
            raise ValueError("rotary needs the tokens' positions.")
        if rotary._head[2] != index:
            raise ValueError("the cos / sin table must be on the cache's device.")
        rot, positions = rotary._at(positions, tokens)
    elif q is not None:
        raise ValueError("q is rotated only: pass rotary and positions beside it.")
    if q is not None:
        q_code, q_index = _heads3(q, "q")
        n, heads, dq = q.shape
        if n != tokens or dq != d or q_code != code or q_index != index:
            raise ValueError("q must agree with k in tokens, head_dim, dtype and device.")
        q_out, qov = _output_view(q_out, q, n, heads, "q_out")
        qv, q = _input_view(q, n, heads)
    kv, k = _input_view(k, tokens, kv_heads)
    vv, v = _input_view(v, tokens, kv_heads)
    units = plan.units

    def call(st, ws):
        # no step writes more units than tokens
        args = _APPEND_ARGS.pack(*kv, *vv, *qv, *qov, units.data_ptr(), plan.num_units.data_ptr(), ws.data_ptr(), *rot,
                                 min(units.shape[0], tokens), tokens, heads, code)
        return N.load().tkv_kv8_append(cache._ptr, args, st)

    status = _launch(index, call)
    if status:
        N.check(status, "tkv_kv8_append")
    return q_out if q is not None else None


def attention(q: torch.Tensor, cache: Kv8Cache, plan: StepPlan, scaling: float, *,
              max_q_len: int | None = None, window: int = 0, out: torch.Tensor | None = None,
              return_lse: bool = False, stream=None):
    """Causal attention of the step's query tokens q [tokens, heads, head_dim]
    over the cache: request i's tokens are q[cu_q[i]:cu_q[i + 1]], the last of
    its kv_lens[i] tokens; each sees the keys up to its own position, with
    ``window`` only the last ``window`` of them.  heads: a multiple of
    kv_heads, up to 64 per kv head.  ``max_q_len``: an upper bound of the
    requests' query tokens (default: tokens).

    Returns out (q's dtype), with return_lse (out, lse [tokens, heads] fp32,
    natural log).  A token that sees nothing gets 0 and -inf; tokens that belong
    to no request are not written.  A request whose table names a block outside
    the cache reads zeros there (``TKV_DEVERR_BAD_SLOT``)."""
    if stream is not None:
        return _on_stream(stream, attention, q, cache, plan, scaling, max_q_len=max_q_len, window=window, out=out,
                          return_lse=return_lse)
    code, index = _heads3(q, "q")
    tokens, heads, d = q.shape
    if d != cache.head_dim or index != cache._index or heads % cache.kv_heads:
        raise ValueError("q must match the cache in head_dim and device, and heads be a multiple of kv_heads.")
    table = plan.block_table
    if table is None or plan.block_size != cache.block_size or plan._index != index:
        raise ValueError("attention needs a plan with block tables of the cache's block size, on its device.")
    if out is None:
        out = torch.empty_like(q, memory_format=_CONTIGUOUS)
    elif out.shape != q.shape or out.dtype != q.dtype or out.get_device() != index or not out.is_contiguous() \
            or out.data_ptr() % 16:
        raise ValueError("out must be a contiguous, 16-byte aligned tensor like q.")
    lse = q.new_empty((tokens, heads), dtype=torch.float32) if return_lse else None
    stride, width = _check_table(table, plan.requests)
    view, q = _input_view(q, tokens, heads)
    longest = tokens if max_q_len is None else min(tokens, int(max_q_len))

    def call(st, ws):
        lib = N.load()
        for attempt in range(2):
            args = _ATTENTION_ARGS.pack(
                *view, out.data_ptr(), 0 if lse is None else lse.data_ptr(), table.data_ptr(), stride,
                plan.kv_lens.data_ptr(), plan.cu_q.data_ptr(), plan.requests, tokens, heads, code,
                width, longest, min(int(window), 0x7fffffff), scaling, ws.data_ptr(), ws.numel())
            status = lib.tkv_kv8_attention(cache._ptr, args, st)
            if status != N.TKV_ERR_WORKSPACE or attempt:
                return status
            nbytes = ctypes.c_size_t()
            N.check(lib.tkv_kv8_attention_workspace(cache._ptr, args, ctypes.byref(nbytes)),
                    "tkv_kv8_attention_workspace")
            ws = ops.workspace_for(cache.device, st, nbytes.value)

    status = _launch(index, call)
    if status:
        N.check(status, "tkv_kv8_attention")
    return (out, lse) if return_lse else out
