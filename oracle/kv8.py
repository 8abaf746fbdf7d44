"""ORACLE (test infrastructure only): the 8-bit paged KV cache in 64 bits.

No counterpart in the reference.  Codes are OCP e4m3 bytes, a value is code *
scale with one power of two for K and one for V of every 16 slots and head:

  decode / encode  the 256 codes' values, and the nearest code (ties to the
                   even one) by search over them
  append           the append functions' rule for one cache, block by block
  load             values at slots
  attention        softmax(q K^T / sqrt(128)) V over float64 values, with the
                   sums that bound the kernel's rounding errors

Pinned by tests/test_oracle_kv8.py: the format's published corner values, ties
and the overflow border, torch's float8_e4m3fn conversions, a hand-computed
append with a growing scale, and oracle/brute.py's attention.
"""

from __future__ import annotations

import math

import torch

BLOCK = 16
TOP = 448.0
MIN_SCALE = 2.0 ** -118
CAP = {torch.bfloat16: 1.875 * 2.0 ** 127, torch.float16: 61440.0}


def _table():
    c = torch.arange(256)
    e, m = ((c >> 3) & 15).double(), (c & 7).double()
    v = torch.where(e > 0, (8 + m) * torch.exp2(e - 10), m * 2.0 ** -9)
    v[c & 127 == 127] = math.nan
    return torch.where(c >= 128, -v, v)


VALUES = _table()


def decode(codes):
    return VALUES[codes.view(torch.uint8).long()]


def encode(x):
    """Nearest code of float64 x; NaN codes for what is not finite or rounds
    past 448."""
    x = x.double()
    grid = VALUES[:127]
    a = x.abs().clamp_max(1e300)
    hi = torch.searchsorted(grid, a).clamp_max(126)
    lo = (hi - 1).clamp_min(0)
    dl, dh = a - grid[lo], grid[hi] - a
    code = torch.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)
    code[~torch.isfinite(x) | (a > 464)] = 127
    return (code + 128 * torch.signbit(x).long()).to(torch.uint8)


def need(amax: float) -> float:
    s = MIN_SCALE
    while amax > TOP * s:
        s *= 2
    return s


def append(codes, scales, side, x, slots, dtype):
    """One cache (codes uint8 [slots][hkv][128], scales [blocks][hkv][2], side
    0 K / 1 V) after appending x (float64 [rows][hkv][128]) of a call."""
    codes, scales = codes.clone(), scales.clone()
    cap = CAP[dtype]
    x = torch.where(torch.isfinite(x), x.clamp(-cap, cap), x)
    rows = [(r, s) for r, s in enumerate(slots.tolist()) if 0 <= s < codes.shape[0]]
    for b in sorted({s // BLOCK for _, s in rows}):
        mine = [(r, s) for r, s in rows if s // BLOCK == b]
        for h in range(codes.shape[1]):
            vals = torch.stack([x[r, h] for r, _ in mine])
            amax = torch.where(torch.isfinite(vals), vals.abs(), torch.zeros_like(vals)).max().item()
            new, old = need(amax), float(scales[b, h, side])
            if all(s % BLOCK for _, s in mine):
                if old > new:
                    new = old
                elif new > old:
                    held = codes[b * BLOCK:(b + 1) * BLOCK, h]
                    codes[b * BLOCK:(b + 1) * BLOCK, h] = encode(decode(held) * (old / new))
            for (r, s), v in zip(mine, vals):
                codes[s, h] = encode(v / new)
            scales[b, h, side] = new
    return codes, scales


def load(codes, scales, side, slots):
    return decode(codes[slots]) * scales[slots // BLOCK][:, :, side, None].double()


def norm_rope(x, w, eps, pos, table, max_pos):
    """float64 [rows][heads][128]: RMSNorm (w None: none), then NeoX rotation
    by fp32 table rows; and |a| + |b| of each pair, which bounds rounding."""
    x = x.double()
    if w is not None:
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()
    a, b = x[..., :64], x[..., 64:]
    ok = (pos >= 0) & (pos < max_pos)
    t = table[torch.where(ok, pos, 0)].double()[:, None]
    c, s = t[..., :64], t[..., 64:]
    y = torch.cat([a * c - b * s, b * c + a * s], -1)
    size = a.abs() + b.abs()
    return torch.where(ok[:, None, None], y, x), torch.cat([size, size], -1)


def attention(b, q, k, v, causal):
    """(out, lse, size, score, total) for a feattn.workloads.Batch; k, v float64 values
    [slots][hkv][128].  size = sum p |v|; score = the largest sum |q||k| /
    sqrt(128) over a row's keys; total = sum |v| over the sequence."""
    out = torch.zeros(b.rows, b.hq, 128, dtype=torch.float64)
    size, total = torch.zeros_like(out), torch.zeros_like(out)
    lse = torch.full((b.rows, b.hq), -math.inf, dtype=torch.float64)
    score = torch.zeros(b.rows, b.hq, dtype=torch.float64)
    for i in range(b.batch):
        n, rows = b.lens[i], b.qlens[i]
        if rows == 0:
            continue
        t = torch.arange(n)
        pages = torch.tensor(b.pages[b.kv[i]:b.kv[i + 1]])
        at = pages[t // b.page] * b.page + t % b.page
        r = slice(b.qo[i], b.qo[i + 1])
        kk = k[at].repeat_interleave(b.group, 1).permute(1, 2, 0).contiguous()
        vv = v[at].repeat_interleave(b.group, 1).permute(1, 0, 2).contiguous()
        x = q[r].double().permute(1, 0, 2).contiguous()
        s = torch.matmul(x, kk) / math.sqrt(128)
        mags = torch.matmul(x.abs(), kk.abs()) / math.sqrt(128)
        if causal:
            hide = t[None] > (n - rows + torch.arange(rows))[:, None]
            s.masked_fill_(hide, -math.inf)
            mags.masked_fill_(hide, 0)
        l = torch.logsumexp(s, -1)
        p = torch.exp(s - l[..., None])
        out[r] = torch.matmul(p, vv).permute(1, 0, 2)
        size[r] = torch.matmul(p, vv.abs()).permute(1, 0, 2)
        total[r] = vv.abs().sum(1)[None]
        lse[r] = l.permute(1, 0)
        score[r] = mags.amax(-1).permute(1, 0)
    return out, lse, size, score, total
