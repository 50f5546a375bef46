"""Numpy restatement of the 8-bit paged cache's operators (test infrastructure).

Planning and codes are exact (whole numbers, fp32 arithmetic rounded step by
step); rotation and attention are evaluated in float64.
"""

from __future__ import annotations

import numpy as np

QMAX = {"int8": np.float32(127), "e4m3": np.float32(448)}


def _e4m3_table() -> np.ndarray:
    """Value of each e4m3 byte (4 exponent bits, bias 7; 3 mantissa bits; no infinities)."""
    b = np.arange(256)
    sign = np.where(b >= 128, -1.0, 1.0)
    e, m = (b >> 3) & 15, b & 7
    v = np.where(e == 0, m * 2.0 ** -9, (8 + m) * 2.0 ** (e - 10.0))
    v = sign * v
    v[(b & 127) == 127] = np.nan
    return v


E4M3 = _e4m3_table()
_E4M3_POS = E4M3[:127]            # 0 .. 448, increasing


def code_values(codes: np.ndarray, fmt: str) -> np.ndarray:
    """float64 values of int8 codes or of e4m3 bytes (uint8)."""
    return codes.astype(np.float64) if fmt == "int8" else E4M3[codes.view(np.uint8)]


def encode(x: np.ndarray, fmt: str) -> np.ndarray:
    """fp32 values to codes: to the nearest, ties to even, clamped."""
    if fmt == "int8":
        return np.clip(np.rint(x), -127, 127).astype(np.int8)
    a = np.minimum(np.abs(x.astype(np.float64)), 448.0)
    hi = np.searchsorted(_E4M3_POS, a)               # first value >= a
    lo = np.maximum(hi - 1, 0)
    dl, dh = a - _E4M3_POS[lo], _E4M3_POS[hi] - a
    pick = np.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)
    return (pick + np.where(np.signbit(x), 128, 0)).astype(np.uint8)


def plan_step(context, new, table, free, free_count, block_size, tokens, units_cap, width):
    """One step, request by request; returns the outputs and the updated table."""
    n, bs = len(context), block_size
    table = table.copy()
    out = {"kv_lens": [], "admitted": [], "cu_q": [0]}
    slot, req, pos, units = [], [], [], []
    left, asked, taken, refused = max(0, min(free_count, len(free))), 0, 0, False
    for i in range(n):
        c, m = max(0, int(context[i])), max(0, int(new[i]))
        held, want = -(-c // bs), -(-(c + m) // bs)
        need = want - held if want <= width else 0
        ok = want <= width and (need == 0 or asked + need <= left)
        if ok:
            for j in range(need):
                table[i, held + j] = free[left - 1 - (asked + j)]
            taken += need
        asked += need
        out["kv_lens"].append(c + m if ok else c)
        out["admitted"].append(int(ok))
        refused |= not ok and m > 0
        for t in range(c, c + m):
            slot.append(int(table[i, t // bs]) * bs + t % bs if ok else -1)
            req.append(i)
            pos.append(t)
        for j in range(c // bs, want) if ok and m else ():
            lo, hi = max(c, j * bs), min(c + m, (j + 1) * bs)
            units.append((int(table[i, j]), out["cu_q"][-1] + lo - c, lo - j * bs, hi - lo))
        out["cu_q"].append(out["cu_q"][-1] + m)

    def fill(x, size):
        return np.array((x + [-1] * size)[:size], np.int32)

    out = {k: np.array(v, np.int32) for k, v in out.items()}
    out.update(slot_map=fill(slot, tokens), token_request=fill(req, tokens), positions=fill(pos, tokens),
               units=np.array((units + [(-1,) * 4] * units_cap)[:units_cap], np.int32).reshape(units_cap, 4),
               num_units=min(len(units), units_cap), free_count=left - taken, table=table, refused=refused)
    return out


def freq_axis(half: int, sections, interleave: bool) -> np.ndarray:
    f = np.arange(half)
    if not interleave:
        return np.searchsorted(np.cumsum(sections), f, side="right")
    a = f % len(sections)
    return np.where(f // len(sections) < np.asarray(sections)[a], a, 0)


def rotate(x, positions, cos_sin, sections, interleave=False, pairs=False, step=np.float64):
    """x [tokens, heads, head_dim] rotated; ``step`` is the type every product
    and sum is rounded to (float64, or float32 as the kernels do)."""
    half = cos_sin.shape[1] // 2
    p = np.asarray(positions).reshape(len(sections), -1)[freq_axis(half, sections, interleave)]   # [half, tokens]
    p = np.clip(p, 0, cos_sin.shape[0] - 1)
    c = cos_sin[p, np.arange(half)[:, None]].T[:, None].astype(step)
    s = cos_sin[p, half + np.arange(half)[:, None]].T[:, None].astype(step)
    y = x.astype(step)
    r = y[..., :2 * half]
    x1, x2 = (r[..., 0::2], r[..., 1::2]) if pairs else (r[..., :half], r[..., half:])
    y1, y2 = x1 * c - x2 * s, x2 * c + x1 * s
    out = y.copy()
    if pairs:
        out[..., 0:2 * half:2], out[..., 1:2 * half:2] = y1, y2
    else:
        out[..., :half], out[..., half:2 * half] = y1, y2
    return out


def write_units(x, codes, scale, units, fmt):
    """Quantizes rows of x [tokens, kv_heads, head_dim] (fp32) into codes
    [blocks, kv_heads, block_size, head_dim] and scale [blocks, kv_heads], in place."""
    with np.errstate(all="ignore"):
        for block, t0, off, n in units:
            for h in range(x.shape[1]):
                rows = x[t0:t0 + n, h].astype(np.float32)
                amax = np.max(np.abs(rows)) if np.all(np.isfinite(rows)) else np.float32(np.inf)
                old = scale[block, h] if off else np.float32(0)
                if not np.isfinite(amax) or not np.isfinite(old):
                    scale[block, h] = np.nan
                    codes[block, h, off:off + n] = 0
                    continue
                s = max(np.float32(amax / QMAX[fmt]), old)
                s = np.float32(1) if s == 0 else s
                if off and s > old:
                    was = code_values(codes[block, h, :off], fmt).astype(np.float32)
                    codes[block, h, :off] = encode(was * np.float32(old / s), fmt)
                codes[block, h, off:off + n] = encode(rows / s, fmt)
                scale[block, h] = s


def attention(q, k_codes, v_codes, k_scale, v_scale, table, kv_lens, cu_q, scaling, fmt, window=0):
    """(out, lse, sum of p |v|, largest sum of |q k| scaling) in float64; tokens of
    no request stay NaN.  Table cells outside the cache read as zeros."""
    blocks, kvh, bs, d = k_codes.shape
    t, heads, _ = q.shape
    group = heads // kvh
    out = np.full((t, heads, d), np.nan)
    lse = np.full((t, heads), np.nan)
    mass, size = np.zeros((t, heads, d)), np.zeros((t, heads))
    for r in range(len(kv_lens)):
        a, b, kv = int(cu_q[r]), int(cu_q[r + 1]), int(kv_lens[r])
        lo = max(0, kv - (b - a) - window + 1) if window else 0
        cells = table[r, lo // bs:-(-kv // bs)].astype(np.int64)
        good = (cells >= 0) & (cells < blocks)
        safe = np.where(good, cells, 0)
        for h in range(kvh):
            def values(codes, scale):
                with np.errstate(invalid="ignore"):
                    x = code_values(codes[safe, h], fmt) * scale[safe, h].astype(np.float64)[:, None, None]
                x[~good] = 0
                return x.reshape(-1, d)
            k, v = values(k_codes, k_scale), values(v_codes, v_scale)
            at = np.arange(lo // bs * bs, lo // bs * bs + k.shape[0])
            for i in range(a, b):
                pos = kv - (b - i)
                see = (at <= pos) & (at < kv) & ((at > pos - window) if window else True)
                for g in range(h * group, (h + 1) * group):
                    if not see.any():
                        out[i, g], lse[i, g] = 0, -np.inf
                        continue
                    qq = q[i, g].astype(np.float64)
                    z = k[see] @ qq * scaling
                    m = z.max()
                    p = np.exp(z - m)
                    w = p / p.sum()
                    out[i, g], lse[i, g] = w @ v[see], np.log(p.sum()) + m
                    mass[i, g] = w @ np.abs(v[see])
                    size[i, g] = (np.abs(k[see]) @ np.abs(qq)).max() * scaling
    return out, lse, mass, size
