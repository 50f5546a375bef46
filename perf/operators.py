"""Cases of the 8-bit paged cache's operators: step planning, rotary positions
with several axes, the quantizing append and attention over the cache.

``run`` computes a case either in its plain form (elementary torch operations
in 32 bits) or, with ``own`` set, through ``paged_tierkv_b200.kv8``.
"""

import random

import torch

own = False

DEVICE = "cuda"
QMAX = {"int8": 127.0, "e4m3": 448.0}
CODE = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
FLOAT = {"fp16": torch.float16, "bf16": torch.bfloat16}


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------

def listed():
    return [
        # one decode step of a small server: every request gets one token
        {"name": "plan-decode", "kind": "plan", "requests": 64, "ctx_min": 0, "ctx_max": 4096,
         "new_min": 1, "new_max": 1, "block": 16, "mix": 1},
        # a large batch that mixes prompts, chunks, single tokens and idle rows
        {"name": "plan-mixed", "kind": "plan", "requests": 1024, "ctx_min": 0, "ctx_max": 8192,
         "new_min": 0, "new_max": 255, "block": 32, "mix": 2},
        # one token of text, one axis
        {"name": "rotary-one", "kind": "rotary", "tokens": 1, "heads": 32, "kv_heads": 8, "head_dim": 128,
         "rot_dim": 128, "axes": 1, "interleave": False, "pairs": False, "dtype": "fp16", "mix": 3},
        # a video prompt: time, height and width positions
        {"name": "rotary-video", "kind": "rotary", "tokens": 16385, "heads": 32, "kv_heads": 8,
         "head_dim": 128, "rot_dim": 128, "axes": 3, "interleave": False, "pairs": False,
         "dtype": "bf16", "mix": 4},
        # one decode step's keys and values
        {"name": "append-decode", "kind": "append", "requests": 64, "ctx_min": 1, "ctx_max": 4096,
         "new_min": 1, "new_max": 1, "heads": 32, "kv_heads": 8, "head_dim": 128, "rot_dim": 128,
         "axes": 1, "interleave": False, "pairs": False, "block": 16, "dtype": "fp16",
         "cache": "int8", "mix": 5},
        # a batch of image prompts and chunks that start inside a block
        {"name": "append-prompts", "kind": "append", "requests": 13, "ctx_min": 0, "ctx_max": 777,
         "new_min": 37, "new_max": 2048, "heads": 32, "kv_heads": 8, "head_dim": 128, "rot_dim": 128,
         "axes": 3, "interleave": True, "pairs": False, "block": 32, "dtype": "bf16",
         "cache": "e4m3", "mix": 6},
        # latency: four short conversations, one token each
        {"name": "attention-decode-4", "kind": "attention", "requests": 4, "kv_min": 2048, "kv_max": 2048,
         "q_min": 1, "q_max": 1, "heads": 32, "kv_heads": 8, "head_dim": 128, "block": 16, "window": 0,
         "dtype": "fp16", "cache": "int8", "mix": 7},
        # throughput: the benchmark's batch of long sequences
        {"name": "attention-decode-32x32k", "kind": "attention", "requests": 32, "kv_min": 32768,
         "kv_max": 32768, "q_min": 1, "q_max": 1, "heads": 32, "kv_heads": 8, "head_dim": 128,
         "block": 16, "window": 0, "dtype": "fp16", "cache": "int8", "mix": 8},
        # one very long context, all of the GPU on one request
        {"name": "attention-decode-131k", "kind": "attention", "requests": 1, "kv_min": 131071,
         "kv_max": 131071, "q_min": 1, "q_max": 1, "heads": 32, "kv_heads": 8, "head_dim": 128,
         "block": 16, "window": 0, "dtype": "bf16", "cache": "e4m3", "mix": 9},
        # several drafted tokens of each request verified at once, an odd group
        {"name": "attention-verify", "kind": "attention", "requests": 23, "kv_min": 90, "kv_max": 9001,
         "q_min": 1, "q_max": 6, "heads": 28, "kv_heads": 4, "head_dim": 64, "block": 32, "window": 0,
         "dtype": "bf16", "cache": "int8", "mix": 10},
        # a whole prompt
        {"name": "attention-prompt-8k", "kind": "attention", "requests": 1, "kv_min": 8192, "kv_max": 8192,
         "q_min": 8192, "q_max": 8192, "heads": 32, "kv_heads": 8, "head_dim": 128, "block": 16,
         "window": 0, "dtype": "fp16", "cache": "int8", "mix": 11},
        # chunks of prompts beside decoding requests, a sliding window
        {"name": "attention-chunks", "kind": "attention", "requests": 7, "kv_min": 700, "kv_max": 12000,
         "q_min": 1, "q_max": 1000, "heads": 32, "kv_heads": 8, "head_dim": 128, "block": 32,
         "window": 4096, "dtype": "bf16", "cache": "e4m3", "mix": 12},
    ]


def _log(rng, lo, hi):
    """A whole number from lo to hi, spread over the logarithm."""
    return min(hi, max(lo, round(lo * (hi / lo) ** rng.random())))


def draw(rng):
    mix = rng.randrange(1 << 20)
    dtype = rng.choice(["fp16", "bf16"])
    cache = rng.choice(["int8", "e4m3"])
    head_dim = rng.choice([64, 128])
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 3, 4, 5, 7, 8])
    block = rng.choice([16, 32, 64])
    kind = rng.choice(["plan", "rotary", "append", "attention", "attention", "attention"])
    rot_dim = rng.choice([head_dim, head_dim, head_dim // 2])
    axes = rng.choice([1, 3, 4])
    style = {"rot_dim": rot_dim, "axes": axes, "interleave": rng.random() < 0.5, "pairs": rng.random() < 0.5}
    if kind == "plan":
        requests = _log(rng, 1, 1024)
        return {"kind": kind, "requests": requests, "ctx_min": 0, "ctx_max": _log(rng, 16, 8192),
                "new_min": rng.choice([0, 1]), "new_max": _log(rng, 1, 255), "block": block, "mix": mix}
    if kind == "rotary":
        return {"kind": kind, "tokens": _log(rng, 1, 16385), "heads": heads, "kv_heads": kv_heads,
                "head_dim": head_dim, **style, "dtype": dtype, "mix": mix}
    if kind == "append":
        requests = _log(rng, 1, 100)
        return {"kind": kind, "requests": requests, "ctx_min": 0, "ctx_max": _log(rng, 16, 4096),
                "new_min": 1, "new_max": _log(rng, 1, 16000 // requests), "heads": heads,
                "kv_heads": kv_heads, "head_dim": head_dim, **style, "block": block, "dtype": dtype,
                "cache": cache, "mix": mix}
    form = rng.choice(["decode", "verify", "prompt", "chunks"])
    if form == "decode":
        kv_max = _log(rng, 17, 131072) | 1
        requests, q_max = _log(rng, 1, max(1, min(200, 400000 // kv_max))), 1
    elif form == "verify":
        kv_max = _log(rng, 64, 32768) | 1
        requests, q_max = _log(rng, 1, max(1, min(64, 200000 // kv_max))), rng.randrange(2, 13)
    elif form == "prompt":
        kv_max = _log(rng, 33, 5000) | 1
        requests, q_max = rng.randrange(1, 3), kv_max
    else:
        kv_max = _log(rng, 500, 12001) | 1
        requests, q_max = rng.randrange(2, 8), _log(rng, 40, min(kv_max, 900))
    window = rng.choice([0, 0, 0, _log(rng, 8, 4096) | 1])
    kv_min = kv_max if form == "prompt" else rng.choice([kv_max, max(1, kv_max // 7)])
    q_min = 1 if form in ("verify", "chunks") else q_max
    return {"kind": kind, "requests": requests, "kv_min": kv_min, "kv_max": kv_max, "q_min": q_min,
            "q_max": q_max, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim, "block": block,
            "window": window, "dtype": dtype, "cache": cache, "mix": mix}


def _spread(rng, lo, hi):
    return lo if lo == hi else (rng.randint(lo, hi) if lo == 0 else _log(rng, lo, hi))


def _lengths(case):
    """(cached or whole length, new or query length) of every request: plain
    numbers that follow from the case alone."""
    rng = random.Random(case["mix"])
    n = case["requests"]
    if case["kind"] == "attention":
        kv = [_spread(rng, case["kv_min"], case["kv_max"]) for _ in range(n)]
        return kv, [min(k, _spread(rng, case["q_min"], case["q_max"])) for k in kv]
    ctx = [_spread(rng, case["ctx_min"], case["ctx_max"]) for _ in range(n)]
    return ctx, [_spread(rng, case["new_min"], case["new_max"]) for _ in range(n)]


def _sections(case):
    """Frequencies of each axis: a quarter for the first, the rest shared."""
    half, axes = case["rot_dim"] // 2, case["axes"]
    if axes == 1:
        return (half,)
    first = half // 4
    rest = (half - first) // (axes - 1)
    return (half - rest * (axes - 1),) + (rest,) * (axes - 1)


# ---------------------------------------------------------------------------
# work
# ---------------------------------------------------------------------------

def _pairs_seen(kv, q, window):
    """Visible (query, key) pairs of one request and the keys that any query sees."""
    first, last = kv - q + 1, kv          # keys that the first and the last query see, without a window
    if not window:
        return (first + last) * q // 2, kv
    seen = sum(min(p, window) for p in (first, last)) * q // 2 if last <= window or first >= window else \
        sum(min(p, window) for p in range(first, last + 1))
    return seen, min(kv, q + window - 1)


def work(case):
    kind = case["kind"]
    a, b = _lengths(case) if kind != "rotary" else ([], [])
    if kind == "plan":
        bs, tokens = case["block"], sum(b)
        blocks = sum(-(-(c + n) // bs) + (-c // bs) for c, n in zip(a, b))
        units = sum(-(-(c + n) // bs) - c // bs for c, n in zip(a, b) if n)
        return {"bytes": 4 * (2 + 1 + 1 + 1) * len(a) + 12 * tokens + 16 * units + 8 * blocks,
                "flops": 4 * tokens}
    heads, kvh, d = case["heads"], case["kv_heads"], case["head_dim"]
    if kind == "rotary":
        t = case["tokens"]
        return {"bytes": t * (4 * (heads + kvh) * d + 4 * case["axes"] + 4 * case["rot_dim"]),
                "flops": 3 * t * (heads + kvh) * case["rot_dim"]}
    if kind == "append":
        t, bs = sum(b), case["block"]
        units = sum(-(-(c + n) // bs) - c // bs for c, n in zip(a, b))
        move = t * (2 * (heads + 2 * kvh) * d + 2 * heads * d + 2 * kvh * d)
        return {"bytes": move + t * (4 * case["axes"] + 4 * case["rot_dim"]) + units * (16 + 8 * kvh),
                "flops": t * (3 * (heads + kvh) * case["rot_dim"] + 4 * kvh * d)}
    pairs = keys = 0
    for kv, q in zip(a, b):
        p, k = _pairs_seen(kv, q, case["window"])
        pairs, keys = pairs + p, keys + k
    scales = sum(-(-kv // case["block"]) for kv in a) * (4 + 8 * kvh)
    return {"bytes": keys * kvh * 2 * d + scales + sum(b) * heads * d * 4,
            "flops": 4 * d * heads * pairs}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def _normal(gen, *shape):
    """Activations: normal values whose channels differ in size, as keys' do."""
    x = torch.randn(shape, generator=gen, device=DEVICE)
    size = torch.randn(shape[-1], generator=gen, device=DEVICE).mul_(0.5).exp_()
    return x.mul_(size)


def _cos_sin(rows, rot_dim):
    f = torch.arange(rot_dim // 2, dtype=torch.float64, device=DEVICE)
    angle = torch.arange(rows, dtype=torch.float64, device=DEVICE)[:, None] * 10000.0 ** (-2 * f / rot_dim)
    return torch.cat([angle.cos(), angle.sin()], dim=1).float()


def _axis_positions(gen, start, axes):
    """Positions of packed tokens: text positions, or a grid's time, height and width."""
    if axes == 1:
        return start
    grid = torch.randint(0, 48, (axes, start.numel()), generator=gen, device=DEVICE, dtype=torch.int32)
    grid[0] = start
    return grid


def _filled(gen, blocks, case):
    """Codes and scales of a cache whose blocks all hold quantized activations."""
    kvh, bs, d, q = case["kv_heads"], case["block"], case["head_dim"], QMAX[case["cache"]]
    codes = torch.empty((blocks, kvh, bs, d), dtype=CODE[case["cache"]], device=DEVICE)
    scale = torch.empty((blocks, kvh), device=DEVICE)
    step = max(1, (1 << 28) // (kvh * bs * d))
    for i in range(0, blocks, step):
        x = _normal(gen, min(step, blocks - i), kvh, bs, d)
        s = x.abs().amax(dim=(2, 3)) / q
        x.div_(s[:, :, None, None])
        codes[i:i + step] = (x.round_() if case["cache"] == "int8" else x).to(codes.dtype)
        scale[i:i + step] = s
    return codes, scale


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    kind, s = case["kind"], {"case": case}
    if kind != "rotary":
        a, b = _lengths(case)
        bs = case["block"]
        total = sum(b) if kind != "attention" else 0
    if kind == "plan":
        width = -(-(case["ctx_max"] + case["new_max"]) // bs)
        held = [-(-c // bs) for c in a]
        blocks = sum(-(-(c + n) // bs) for c, n in zip(a, b)) + 5
        ids = torch.randperm(blocks, generator=gen, device=DEVICE).to(torch.int32)
        table = torch.full((len(a), width), -1, dtype=torch.int32, device=DEVICE)
        held_t = torch.tensor(held, device=DEVICE)
        cells = torch.arange(width, device=DEVICE)[None] < held_t[:, None]
        table[cells] = ids[:sum(held)]
        s.update(ctx=_i32(a), new=_i32(b), table=table, free=ids[sum(held):].contiguous(),
                 free_count=_i32([blocks - sum(held)]), tokens=total)
        return s
    dtype = FLOAT[case["dtype"]]
    heads, kvh, d = case["heads"], case["kv_heads"], case["head_dim"]
    if kind == "rotary":
        t = case["tokens"]
        qkv = _normal(gen, t, heads + 2 * kvh, d).to(dtype)
        start = torch.arange(t, device=DEVICE, dtype=torch.int32) + 11
        s.update(q=qkv[:, :heads], k=qkv[:, heads:heads + kvh], cos_sin=_cos_sin(t + 64, case["rot_dim"]),
                 positions=_axis_positions(gen, start, case["axes"]))
        return s
    if kind == "append":
        units, at, t0 = [], [], 0
        spare = 0
        for c, n in zip(a, b):
            at += range(c, c + n)
            for j in range(c // bs, -(-(c + n) // bs)):
                lo, hi = max(c, j * bs), min(c + n, (j + 1) * bs)
                units.append((spare, t0 + lo - c, lo - j * bs, hi - lo))
                spare += 1
            t0 += n
        blocks = spare + spare // 8 + 1
        ids = torch.randperm(blocks, generator=gen, device=DEVICE).to(torch.int32)
        u = _i32(units)
        u[:, 0] = ids[u[:, 0].long()]
        (kc, ks), (vc, vs) = _filled(gen, blocks, case), _filled(gen, blocks, case)
        qkv = _normal(gen, total, heads + 2 * kvh, d).to(dtype)
        s.update(q=qkv[:, :heads], k=qkv[:, heads:heads + kvh], v=qkv[:, heads + kvh:], units=u,
                 num_units=_i32([len(units)]), k_codes=kc, v_codes=vc, k_scale=ks, v_scale=vs,
                 positions=_axis_positions(gen, _i32(at), case["axes"]),
                 cos_sin=_cos_sin(max(at) + 64, case["rot_dim"]))
        return s
    width = -(-case["kv_max"] // bs)
    held = [-(-k // bs) for k in a]
    blocks = sum(held) + 3
    ids = torch.randperm(blocks, generator=gen, device=DEVICE).to(torch.int32)
    table = torch.full((len(a), width), -1, dtype=torch.int32, device=DEVICE)
    cells = torch.arange(width, device=DEVICE)[None] < torch.tensor(held, device=DEVICE)[:, None]
    table[cells] = ids[:sum(held)]
    cu = [0]
    for n in b:
        cu.append(cu[-1] + n)
    (kc, ks), (vc, vs) = _filled(gen, blocks, case), _filled(gen, blocks, case)
    s.update(q=_normal(gen, cu[-1], heads, d).to(dtype), k_codes=kc, v_codes=vc, k_scale=ks, v_scale=vs,
             table=table, kv_lens=_i32(a), cu_q=_i32(cu), max_q=max(b), max_kv=max(a), scaling=d ** -0.5)
    return s


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------

def _plan(s):
    bs, tokens = s["case"]["block"], s["tokens"]
    ctx, new, table = s["ctx"].long(), s["new"].long(), s["table"]
    n, width = table.shape
    dev = table.device
    held, want = (ctx + bs - 1) // bs, (ctx + new + bs - 1) // bs
    fits = want <= width
    need = torch.where(fits, want - held, 0)
    upto = need.cumsum(0)
    admitted = fits & ((need == 0) | (upto <= s["free_count"]))
    kv = torch.where(admitted, ctx + new, ctx)
    cu = torch.cat([torch.zeros(1, dtype=torch.long, device=dev), new.cumsum(0)])
    # table cells: cell j of a request is its (j - held)-th new block
    j = torch.arange(width, device=dev)[None]
    fresh = admitted[:, None] & (j >= held[:, None]) & (j < want[:, None])
    pick = s["free_count"] - 1 - (upto - need)[:, None] - (j - held[:, None])
    ids = s["free"][pick.clamp(0, s["free"].numel() - 1)]
    table.copy_(torch.where(fresh, ids, table))
    taken = torch.where(admitted, need, 0).sum()
    # tokens
    t = torch.arange(tokens, device=dev)
    req = torch.searchsorted(cu, t, right=True) - 1
    pos = ctx[req] + t - cu[req]
    slot = table[req, (pos // bs).clamp(max=width - 1)].long() * bs + pos % bs
    slot = torch.where(admitted[req], slot, -1)
    # write units: the blocks that the admitted requests' new tokens touch
    count = torch.where(admitted & (new > 0), want - ctx // bs, 0)
    ucu = torch.cat([torch.zeros(1, dtype=torch.long, device=dev), count.cumsum(0)])
    cap = min(tokens, tokens // bs + 2 * n)
    u = torch.arange(cap, device=dev)
    r = (torch.searchsorted(ucu, u, right=True) - 1).clamp(max=n - 1)
    block = ctx[r] // bs + u - ucu[r]
    lo = torch.maximum(block * bs, ctx[r])
    hi = torch.minimum((block + 1) * bs, ctx[r] + new[r])
    cell = table[r, block.clamp(0, width - 1)].long()
    units = torch.stack([cell, cu[r] + lo - ctx[r], lo - block * bs, hi - lo], dim=1)
    units = torch.where((u < ucu[-1])[:, None], units, -1)
    i32 = torch.int32
    return {"kv_lens": kv.to(i32), "cu_q": cu.to(i32), "admitted": admitted.to(i32),
            "slot_map": slot.to(i32), "token_request": req.to(i32), "positions": pos.to(i32),
            "units": units.to(i32), "num_units": ucu[-1:].to(i32),
            "free_count": (s["free_count"] - taken).to(i32), "table": table}


def _freq_axis(case):
    """The axis whose position turns each frequency."""
    half, axes = case["rot_dim"] // 2, case["axes"]
    sec = torch.tensor(_sections(case), device=DEVICE)
    f = torch.arange(half, device=DEVICE)
    if not case["interleave"]:
        return torch.searchsorted(sec.cumsum(0), f, right=True)
    axis = f % axes
    return torch.where(f // axes < sec[axis], axis, 0)


def _turn(x, positions, cos_sin, case):
    """x [tokens, heads, head_dim] rotated, in 32 bits."""
    half = case["rot_dim"] // 2
    p = positions.reshape(case["axes"], -1).long()[_freq_axis(case)]       # [half, tokens]
    f = torch.arange(half, device=x.device)[:, None]
    c, sn = cos_sin[p, f].t()[:, None], cos_sin[p, half + f].t()[:, None]
    y = x.float().clone()
    r = y[..., :2 * half]
    x1, x2 = (r[..., 0::2], r[..., 1::2]) if case["pairs"] else (r[..., :half], r[..., half:])
    y1, y2 = x1 * c - x2 * sn, x2 * c + x1 * sn
    y[..., :2 * half] = torch.stack([y1, y2], dim=-1).flatten(-2) if case["pairs"] else torch.cat([y1, y2], -1)
    return y


def _write(x, codes, scale, units, kind):
    """Rows of x [tokens, kv_heads, head_dim] into the blocks of the write units."""
    bs, qmax = codes.shape[2], QMAX[kind]
    block, t0, off, n = units.long().unbind(1)
    row = torch.arange(bs, device=x.device)[None]
    new = (row >= off[:, None]) & (row < (off + n)[:, None])               # [units, bs]
    old = row < off[:, None]
    rows = x[(t0[:, None] + row - off[:, None]).clamp(0, x.shape[0] - 1)].transpose(1, 2)
    most = torch.where(new[:, None, :, None], rows.abs(), 0).amax(dim=(2, 3))
    s_new = most / torch.full_like(most, qmax)
    s_old = scale[block]
    s = torch.where((off > 0)[:, None], torch.maximum(s_old, s_new), s_new)
    s = torch.where(s == 0, 1.0, s)
    was = codes[block].float()
    again = was * (s_old / s)[:, :, None, None]
    fresh = rows / s[:, :, None, None]
    if kind == "int8":
        again, fresh = again.round(), fresh.round()
    again = torch.where((s > s_old)[:, :, None, None], again, was).clamp(-qmax, qmax)
    y = torch.where(new[:, None, :, None], fresh.clamp(-qmax, qmax),
                    torch.where(old[:, None, :, None], again, was))
    codes[block] = y.to(codes.dtype)
    scale[block] = s


def _attend(s):
    case = s["case"]
    kvh, d, bs, window = case["kv_heads"], case["head_dim"], case["block"], case["window"]
    group = case["heads"] // kvh
    n, width = s["table"].shape
    length, most = s["max_kv"], s["max_q"]
    wide = -(-length // bs)
    cells = s["table"][:, :wide].long().clamp(min=0)

    def cached(codes, scale):
        x = codes[cells].float() * scale[cells][..., None, None]           # [n, wide, kvh, bs, d]
        return x.transpose(1, 2).reshape(n, kvh, wide * bs, d)[:, :, :length]

    cu, kv = s["cu_q"].long(), s["kv_lens"].long()
    q_len = cu[1:] - cu[:-1]
    i = torch.arange(most, device=cu.device)[None]
    token = (cu[:-1, None] + i).clamp(max=s["q"].shape[0] - 1)             # [n, most]
    q = s["q"].float()[token].reshape(n, most, kvh, group, d).permute(0, 2, 3, 1, 4)
    q = q.reshape(n, kvh, group * most, d)
    logits = (q @ cached(s["k_codes"], s["k_scale"]).transpose(2, 3)).mul_(s["scaling"])
    logits = logits.view(n, kvh, group, most, length)
    key = torch.arange(length, device=cu.device)
    pos = (kv - q_len)[:, None] + i                                        # [n, most]
    hidden = (key > pos[..., None]) | (key >= kv[:, None, None])
    if window:
        hidden |= key <= pos[..., None] - window
    logits.masked_fill_(hidden[:, None, None], float("-inf"))
    top = logits.amax(-1, keepdim=True)
    top = torch.where(top == float("-inf"), 0.0, top)
    p = logits.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    o = p.view(n, kvh, group * most, length) @ cached(s["v_codes"], s["v_scale"])
    o = o.view(n, kvh, group, most, d) / torch.where(total == 0, 1.0, total)
    lse = (total.log() + top).squeeze(-1)
    o = o.permute(0, 3, 1, 2, 4).reshape(n, most, kvh * group, d)
    lse = lse.permute(0, 3, 1, 2).reshape(n, most, kvh * group)
    live = i < q_len[:, None]
    return {"out": o[live].to(s["q"].dtype), "lse": lse[live]}


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def _own(s):
    from paged_tierkv_b200 import kv8
    case, kind = s["case"], s["case"]["kind"]
    if kind == "plan":
        if "plan" not in s:
            s["plan"] = kv8.StepPlan.allocate(case["requests"], s["tokens"], case["block"], DEVICE)
        p = kv8.plan_step(s["plan"], s["ctx"], s["new"], s["table"], s["free"], s["free_count"])
        return {"kv_lens": p.kv_lens, "cu_q": p.cu_q, "admitted": p.admitted, "slot_map": p.slot_map,
                "token_request": p.token_request, "positions": p.positions, "units": p.units,
                "num_units": p.num_units, "free_count": p.free_count, "table": s["table"]}
    if kind != "attention" and "rotary" not in s:
        s["rotary"] = kv8.Rotary(s["cos_sin"], sections=_sections(case), interleave=case["interleave"],
                                 pairs=case["pairs"])
    if kind == "rotary":
        return kv8.rotary_embed(s["q"], s["k"], s["positions"], s["rotary"])
    if "cache" not in s:
        s["cache"] = kv8.Kv8Cache(s["k_codes"], s["v_codes"], s["k_scale"], s["v_scale"])
    if kind == "append":
        if "plan" not in s:
            s["plan"] = kv8.StepPlan(units=s["units"], num_units=s["num_units"], block_size=case["block"])
        q = kv8.append(s["cache"], s["plan"], s["k"], s["v"], q=s["q"], positions=s["positions"],
                       rotary=s["rotary"])
        return {"q": q, "k_codes": s["k_codes"], "v_codes": s["v_codes"], "k_scale": s["k_scale"],
                "v_scale": s["v_scale"]}
    if "plan" not in s:
        s["plan"] = kv8.StepPlan(block_table=s["table"], kv_lens=s["kv_lens"], cu_q=s["cu_q"],
                                 block_size=case["block"])
    out, lse = kv8.attention(s["q"], s["cache"], s["plan"], s["scaling"], max_q_len=s["max_q"],
                             window=case["window"], return_lse=True)
    return {"out": out, "lse": lse}


def run(s):
    if own:
        return _own(s)
    case, kind = s["case"], s["case"]["kind"]
    if kind == "plan":
        return _plan(s)
    if kind == "rotary":
        return tuple(_turn(s[x], s["positions"], s["cos_sin"], case).to(s[x].dtype) for x in ("q", "k"))
    if kind == "append":
        q = _turn(s["q"], s["positions"], s["cos_sin"], case).to(s["q"].dtype)
        k = _turn(s["k"], s["positions"], s["cos_sin"], case)
        _write(k, s["k_codes"], s["k_scale"], s["units"], case["cache"])
        _write(s["v"].float(), s["v_codes"], s["v_scale"], s["units"], case["cache"])
        return {"q": q, "k_codes": s["k_codes"], "v_codes": s["v_codes"], "k_scale": s["k_scale"],
                "v_scale": s["v_scale"]}
    return _attend(s)


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------

def _turn64(x, positions, cos_sin, case):
    y = x.double().clone()
    half, axes, sec = case["rot_dim"] // 2, case["axes"], _sections(case)
    pos = positions.view(axes, -1).long()
    for f in range(half):
        if case["interleave"]:
            axis = f % axes if f // axes < sec[f % axes] else 0
        else:
            axis = next(a for a in range(axes) if f < sum(sec[:a + 1]))
        c, s = (cos_sin[pos[axis], col].double()[:, None] for col in (f, half + f))
        i, j = (2 * f, 2 * f + 1) if case["pairs"] else (f, f + half)
        x1, x2 = x[..., i].double(), x[..., j].double()
        y[..., i], y[..., j] = x1 * c - x2 * s, x1 * s + x2 * c
    return y


def _write64(x, codes, scale, units, case):
    """(values of the codes that stand after the write, or None for whole codes; scales)."""
    qmax = QMAX[case["cache"]]
    codes, scale = codes.clone(), scale.double()
    for block, t0, off, n in units.tolist():
        rows = x[t0:t0 + n].transpose(0, 1)
        s = rows.abs().amax(dim=(1, 2)) / qmax
        if off:
            grown = torch.maximum(s, scale[block])
            back = codes[block, :, :off].double() * (scale[block] / grown)[:, None, None]
            codes[block, :, :off] = (back if case["cache"] == "e4m3" else back.round()).to(codes.dtype)
            s = grown
        y = (rows / s[:, None, None]).clamp(-qmax, qmax)
        codes[block, :, off:off + n] = (y if case["cache"] == "e4m3" else y.round()).to(codes.dtype)
        scale[block] = s
    return (codes.double() if case["cache"] == "e4m3" else None), scale


def _attend64(s, r, out, lse):
    """Request r's rows of out and lse, query heads and runs of queries one by one."""
    case = s["case"]
    kvh, d, window = case["kv_heads"], case["head_dim"], case["window"]
    group, bs = case["heads"] // kvh, case["block"]
    t0, t1, kv = int(s["cu_q"][r]), int(s["cu_q"][r + 1]), int(s["kv_lens"][r])
    cells = s["table"][r, :-(-kv // bs)].long()
    for h in range(kvh):
        k, v = ((codes[cells, h].double() * scale[cells, h].double()[:, None, None]).view(-1, d)[:kv]
                for codes, scale in ((s["k_codes"], s["k_scale"]), (s["v_codes"], s["v_scale"])))
        for a in range(t0, t1, 2048):
            b = min(t1, a + 2048)
            at = torch.arange(a, b, device=DEVICE)[:, None] - t1 + kv
            j = torch.arange(kv, device=DEVICE)[None]
            seen = (j <= at) & ((j > at - window) if window else (j >= 0))
            for g in range(h * group, (h + 1) * group):
                z = s["q"][a:b, g].double() @ k.t() * s["scaling"]
                z = torch.where(seen, z, float("-inf"))
                lse[a:b, g] = torch.logsumexp(z, dim=1)
                out[a:b, g] = torch.softmax(z, dim=1) @ v


def exact(case, seed):
    if case["kind"] == "plan":
        return None                        # whole numbers only
    s = prepare(case, seed)
    if case["kind"] == "rotary":
        return tuple(_turn64(s[x], s["positions"], s["cos_sin"], case) for x in ("q", "k"))
    if case["kind"] == "append":
        q, k = (_turn64(s[x], s["positions"], s["cos_sin"], case) for x in ("q", "k"))
        kc, ks = _write64(k, s["k_codes"], s["k_scale"], s["units"], case)
        vc, vs = _write64(s["v"].double(), s["v_codes"], s["v_scale"], s["units"], case)
        return {"q": q, "k_codes": kc, "v_codes": vc, "k_scale": ks, "v_scale": vs}
    out = torch.empty(s["q"].shape, dtype=torch.float64, device=DEVICE)
    lse = torch.empty(s["q"].shape[:2], dtype=torch.float64, device=DEVICE)
    for r in range(case["requests"]):
        _attend64(s, r, out, lse)
    return {"out": out, "lse": lse}
