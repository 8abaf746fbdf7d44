"""GPU tests of the 8-bit paged KV cache (append, load, attention) against
oracle/kv8.py's 64-bit results.

Tolerances.  u = finfo.eps / 2 of the 16-bit type (2^-8 bf16, 2^-11 fp16).
* Values appended from 16-bit inputs without arithmetic (store, V): the codes
  are the oracle's.  Rotated keys carry two fp32 roundings of products of
  |a| + |b| and one of their sum, 3 * 2^-24 of |a| + |b| together; normalized
  ones up to 32 roundings of 2^-24 before that (a sum of 128 squares in 16
  steps and 3, its mean, root, reciprocal within an ulp, and two products).  So
  a code or query is the nearest to some value within 2^-22 (2^-18) of
  |a| + |b| of the 64-bit one: its distance to that is half a step more.
* Attention: every probability is rounded to 16 bits once (u each, so u times
  A = sum p |v| in the result) and the output once (u |o|); a row split over
  several work units has its parts rounded too (u A).  fp16 probabilities below
  2^-14 of a sum that is at least 1 are off by 2^-25 instead.  fp32: scores are sums of
  128 products, off by at most 128 * 2^-24 of sum |q||k| / sqrt(128) = score, plus
  2^-22 score for the scaling and the exponent's argument, and the exponential, sums
  and quotients by 2^-20 relative: e = 2^-16 score + 2^-19 in the logarithm,
  twice that times A in the result."""

import math

import pytest
import torch

import feattn
from feattn import workloads as W
from oracle import kv8

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f16": torch.float16}
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def filled(blocks, hkv, seed, dtype, spread=0.5):
    """Random codes (uint8 [blocks * 16][hkv][128]) and scales; values of order
    one, blocks of different size."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(blocks, 16, hkv, 128, generator=g)
    x *= torch.exp2((torch.randn(blocks, 1, hkv, 1, generator=g) * 2 * spread).round())
    s = torch.exp2(torch.ceil(torch.log2(x.abs().amax((1, 3)) / kv8.TOP)))
    codes = kv8.encode(x / s[:, None, :, None]).view(blocks * 16, hkv, 128)
    return codes, s


def cache(blocks, hkv, seed, dtype=torch.bfloat16, spread=0.5):
    kc, ks = filled(blocks, hkv, 2 * seed, dtype, spread)
    vc, vs = filled(blocks, hkv, 2 * seed + 1, dtype, spread)
    return kc, vc, torch.stack([ks, vs], -1).contiguous()


def half_step16(x, dtype):
    """Half a step of the 16-bit type at |x|, as float64."""
    bits, low = (8, -126) if dtype == torch.bfloat16 else (11, -14)
    e = torch.floor(torch.log2(x.abs().clamp_min(2.0 ** low)))
    return torch.exp2(e - bits)


def half_step8(x, scale):
    e = torch.floor(torch.log2((x / scale).abs().clamp_min(2.0 ** -6)))
    return torch.exp2(e - 4) * scale


# ---------------------------------------------------------------------------
# Append
# ---------------------------------------------------------------------------

def rows_of(starts, qlens, blocks, seed):
    """Slots and positions of sequences with `starts` cached and `qlens` new
    tokens over randomly ordered blocks."""
    g = torch.Generator().manual_seed(seed)
    perm = torch.randperm(blocks, generator=g).tolist()
    slots, pos = [], []
    for s, n in zip(starts, qlens):
        table = [perm.pop() for _ in range(-(-(s + n) // 16))]
        for p in range(s, s + n):
            pos.append(p)
            slots.append(table[p // 16] * 16 + p % 16)
    return torch.tensor(slots), torch.tensor(pos)


BATCHES = [
    ([0], [1]),
    ([5], [1]),
    ([0], [16]),
    ([3], [40]),
    ([15, 16, 17, 0, 31], [1, 1, 1, 1, 1]),
    ([7, 30, 2, 100, 64], [5, 5, 5, 5, 5]),
    ([0, 9, 33], [77, 130, 16]),
    ([k % 16 for k in range(70)], [1] * 70),
]


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("batch", range(len(BATCHES)))
@pytest.mark.parametrize("hkv", [1, 3, 8])
def test_store(dev, dtype, batch, hkv):
    """Codes and scales of the touched blocks are the oracle's, everything else
    is as it was; a padding row and one past the cache between the sequences."""
    dt = DT[dtype]
    starts, qlens = BATCHES[batch]
    blocks = sum(-(-(s + n) // 16) for s, n in zip(starts, qlens)) + 2
    slots, _ = rows_of(starts, qlens, blocks, batch)
    ends = torch.tensor(qlens).cumsum(0)
    at = int(ends[0])
    slots = torch.cat([slots[:at], torch.tensor([-1, blocks * 16]), slots[at:]])
    g = torch.Generator().manual_seed(100 + batch)
    k, v = (torch.randn(len(slots), hkv, 128, generator=g) * torch.exp(torch.randn(len(slots), 1, 1, generator=g))
            for _ in range(2))
    k, v = k.to(dt), v.to(dt)
    kc, vc, scales = cache(blocks, hkv, batch, dt)
    want_k, s1 = kv8.append(kc, scales, 0, k.double(), slots, dt)
    want_v, s2 = kv8.append(vc, s1, 1, v.double(), slots, dt)
    kd, vd, sd = kc.to(dev), vc.to(dev), scales.to(dev)
    feattn.store_kv8(k.to(dev), v.to(dev), kd, vd, sd, slots.to(dev), len(slots), hkv, 128, dtype == "bf16",
                     blocks * 16)
    torch.cuda.synchronize()
    assert torch.equal(sd.cpu(), s2)
    # (what a started block's later slots held is lost)
    keep = torch.ones(blocks * 16, dtype=torch.bool)
    used = [s for s in slots.tolist() if 0 <= s < blocks * 16]
    for b in {s // 16 for s in used if s % 16 == 0}:
        keep[[s for s in range(16 * b, 16 * b + 16) if s not in used]] = False
    assert torch.equal(kd.cpu()[keep], want_k[keep])
    assert torch.equal(vd.cpu()[keep], want_v[keep])


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("hq,hkv,batch,extra", [(32, 8, 6, 0), (16, 8, 7, 0), (40, 8, 5, 64), (6, 3, 3, 8), (5, 1, 4, 0),
                                                (0, 8, 6, 0)])
def test_rope_append(dev, dtype, norm, hq, hkv, batch, extra):
    """Queries, codes and scales of both append forms; one row without a
    position, one with one past the table, one not stored.  hq = 0: keys and
    values only.  The queries of the form without a norm are fe_rope's bits."""
    dt, bf16, max_pos, eps = DT[dtype], dtype == "bf16", 300, 1e-6
    starts, qlens = BATCHES[batch]
    blocks = sum(-(-(s + n) // 16) for s, n in zip(starts, qlens)) + 1
    slots, pos = rows_of(starts, qlens, blocks, batch)
    rows = len(slots)
    pos[0], pos[-1] = -1, max_pos
    if rows > 3:
        slots[0] = -5
    g = torch.Generator().manual_seed(7 * batch + hq)
    stride = (hq + 2 * hkv) * 128 + extra
    qkv = (torch.randn(rows, stride, generator=g) * 2).to(dt)
    heads = qkv[:, :(hq + 2 * hkv) * 128].reshape(rows, -1, 128)
    q, k, v = (t.contiguous() for t in heads.split([hq, hkv, hkv], 1))
    qw, kw = ((1 + 0.1 * torch.randn(128, generator=g)).to(dt) for _ in range(2))
    table = W.rope_table(max_pos, 1e6)
    kc, vc, scales = cache(blocks, hkv, batch, dt)
    kd, vd, sd = kc.to(dev), vc.to(dev), scales.to(dev)
    qd = q.to(dev)
    if norm:
        feattn.norm_rope_append_kv8(qkv.to(dev), stride, qw.to(dev) if hq else None, kw.to(dev), eps,
                                    qd if hq else None, kd, vd, sd, pos.to(dev), slots.to(dev), table.to(dev), rows,
                                    hq, hkv, bf16, max_pos, blocks * 16)
    else:
        feattn.rope_append_kv8(qd if hq else None, k.to(dev), v.to(dev), kd, vd, sd, pos.to(dev), slots.to(dev),
                               table.to(dev), rows, hq, hkv, 128, bf16, max_pos, blocks * 16)
    torch.cuda.synchronize()
    rel = 2.0 ** -18 if norm else 2.0 ** -22
    want_q, size_q = kv8.norm_rope(q, qw if norm else None, eps, pos, table, max_pos)
    want_k, size_k = kv8.norm_rope(k, kw if norm else None, eps, pos, table, max_pos)
    if hq:
        err = (qd.cpu().double() - want_q).abs()
        assert (err <= half_step16(want_q.abs() + rel * size_q, dt) + rel * size_q).all()
    if hq and not norm:
        plain, other = q.to(dev), k.to(dev)
        feattn.rope(plain, other, pos.to(dev), table.to(dev), rows, hq, hkv, 128, bf16, max_pos)
        assert torch.equal(plain.view(torch.int16), qd.view(torch.int16))
    _, s1 = kv8.append(kc, scales, 0, want_k, slots, dt)
    want_vc, s2 = kv8.append(vc, s1, 1, v.double(), slots, dt)
    assert torch.equal(sd.cpu(), s2)
    ok = (slots >= 0) & (slots < blocks * 16)
    at = slots[ok]
    got = kv8.load(kd.cpu(), s2, 0, at)
    scale = s2[at // 16][:, :, 0, None].double()
    slack = rel * size_k[ok]
    assert ((got - want_k[ok]).abs() <= half_step8(want_k[ok].abs() + slack, scale) + slack).all()
    assert torch.equal(vd.cpu()[at], want_vc[at])
    rest = torch.ones(blocks * 16, dtype=torch.bool)
    rest[(at[:, None] // 16 * 16 + torch.arange(16)).reshape(-1)] = False
    assert torch.equal(kd.cpu()[rest], kc[rest]) and torch.equal(vd.cpu()[rest], vc[rest])


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_token_by_token(dev, dtype):
    """40 single-token appends whose size wanders over 2^32 (fp16: 2^20), V
    falling where K rises: after each call codes and scales are the oracle's."""
    dt = DT[dtype]
    hkv, blocks = 2, 4
    g = torch.Generator().manual_seed(5)
    kc, vc, scales = cache(blocks, hkv, 3, dt)
    kd, vd, sd = kc.to(dev), vc.to(dev), scales.to(dev)
    for t in range(40):
        e = (8 if dtype == "bf16" else 5) * math.sin(0.9 * t) * 2
        k = (torch.randn(1, hkv, 128, generator=g) * 2.0 ** e).to(dt)
        v = (torch.randn(1, hkv, 128, generator=g) * 2.0 ** -e).to(dt)
        slots = torch.tensor([16 + t])
        kc, scales = kv8.append(kc, scales, 0, k.double(), slots, dt)
        vc, scales = kv8.append(vc, scales, 1, v.double(), slots, dt)
        feattn.store_kv8(k.to(dev), v.to(dev), kd, vd, sd, slots.to(dev), 1, hkv, 128, dtype == "bf16", blocks * 16)
        live = slice(16, 17 + t)
        assert torch.equal(sd.cpu(), scales), t
        assert torch.equal(kd.cpu()[live], kc[live]) and torch.equal(vd.cpu()[live], vc[live]), t


def test_rejected_drafts(dev):
    """Runs of five written at positions that step back by what was rejected,
    over block borders, the rejected rows large: live codes and all scales are
    the oracle's."""
    hkv, blocks, dt = 3, 4, torch.bfloat16
    g = torch.Generator().manual_seed(15)
    kc, vc, scales = cache(blocks, hkv, 3, dt)
    kd, vd, sd = kc.to(dev), vc.to(dev), scales.to(dev)
    at = 0
    for accepted in (5, 2, 3, 1, 5, 1, 2, 4, 1, 1, 5, 3, 2):
        k, v = (torch.randn(5, hkv, 128, generator=g) for _ in range(2))
        k[accepted:] *= 64
        k, v = k.to(dt), v.to(dt)
        slots = torch.arange(at, at + 5)
        kc, scales = kv8.append(kc, scales, 0, k.double(), slots, dt)
        vc, scales = kv8.append(vc, scales, 1, v.double(), slots, dt)
        feattn.store_kv8(k.to(dev), v.to(dev), kd, vd, sd, slots.to(dev), 5, hkv, 128, True, blocks * 16)
        live = slice(0, at + 5)
        assert torch.equal(sd.cpu(), scales), at
        assert torch.equal(kd.cpu()[live], kc[live]) and torch.equal(vd.cpu()[live], vc[live]), at
        at += accepted


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_special_values(dev, dtype):
    """NaN, infinities, the largest finite values, zeros and subnormals: the
    rest of their block keeps its precision, and a cached value is finite in the
    type or NaN."""
    dt = DT[dtype]
    hkv, blocks = 2, 5
    g = torch.Generator().manual_seed(9)
    x = torch.randn(64, hkv, 128, generator=g).to(dt)
    x[3, 0, 5], x[4, 1, 7], x[5, 0, 9] = math.nan, math.inf, -math.inf
    x[16, 0, :8] = torch.finfo(dt).max
    x[17, 1, :8] = -torch.finfo(dt).max
    x[32:48] = 0
    x[33, 0, 0] = -0.0
    x[48:64] = (torch.randn(16, hkv, 128, generator=g) * torch.finfo(dt).smallest_normal / 8).to(dt)
    slots = torch.arange(64)
    kc, vc, scales = cache(blocks, hkv, 4, dt)
    want, s1 = kv8.append(kc, scales, 0, x.double(), slots, dt)
    want_v, s2 = kv8.append(vc, s1, 1, x.double(), slots, dt)
    kd, vd, sd = kc.to(dev), vc.to(dev), scales.to(dev)
    feattn.store_kv8(x.to(dev), x.to(dev), kd, vd, sd, slots.to(dev), 64, hkv, 128, dtype == "bf16", blocks * 16)
    out = torch.zeros(2, 64, hkv, 128, dtype=dt, device=dev)
    feattn.load_kv8(kd, vd, sd, slots.to(dev), out[0], out[1], 64, hkv, 128, dtype == "bf16", blocks * 16)
    torch.cuda.synchronize()
    assert torch.equal(sd.cpu(), s2)
    nan = torch.isnan(kv8.decode(want))  # (NaN codes of either sign)
    assert int(nan[:64].sum()) == 3
    for got, w in ((kd, want), (vd, want_v)):
        assert torch.equal(torch.isnan(kv8.decode(got.cpu())), nan)
        assert torch.equal(got.cpu()[~nan], w[~nan])
    back = out[0].cpu().double()
    assert torch.equal(torch.isnan(back), nan[:64]) and not torch.isinf(back).any()


@pytest.mark.parametrize("eps", [1e-6, 0.0])
def test_norm_of_extreme_rows(dev, eps):
    """Keys whose root mean square is near the ends of bf16's range, and one with
    an infinity, whose norm leaves zeros and NaNs."""
    hkv, rows, max_pos = 2, 48, 64
    g = torch.Generator().manual_seed(8)
    x = torch.randn(rows, 3 * hkv, 128, generator=g)
    x[:16] *= 2.0 ** 125
    x[16:32] *= 2.0 ** -126
    x = x.to(torch.bfloat16)
    x[40, 0, 3] = math.inf
    x[41, 1, 70] = math.nan
    assert torch.isfinite(x[:32]).all()
    kw = (1 + 0.1 * torch.randn(128, generator=g)).to(torch.bfloat16)
    kc, vc, scales = cache(4, hkv, 5)
    kd, vd, sd = kc.to(dev), vc.to(dev), scales.to(dev)
    pos, slots, table = torch.arange(rows), torch.arange(rows), W.rope_table(max_pos, 1e6)
    qkv = x[:, hkv:].contiguous()
    qkv[:, :hkv] = x[:, :hkv]
    feattn.norm_rope_append_kv8(qkv.to(dev), 2 * hkv * 128, None, kw.to(dev), eps, None, kd, vd, sd, pos.to(dev),
                                slots.to(dev), table.to(dev), rows, 0, hkv, True, max_pos, 64)
    torch.cuda.synchronize()
    want, size = kv8.norm_rope(qkv[:, :hkv], kw, eps, pos, table, max_pos)
    nan = torch.isnan(want)
    assert int(nan.sum()) == 2 + 128
    _, s1 = kv8.append(kc, scales, 0, want, slots, torch.bfloat16)
    assert torch.equal(sd.cpu()[:3, :, 0], s1[:3, :, 0])
    got = kv8.load(kd.cpu(), s1, 0, slots)
    assert torch.equal(torch.isnan(got), nan)
    slack = 2.0 ** -18 * size
    bound = half_step8(want.abs() + slack, s1[slots // 16][:, :, 0, None].double()) + slack
    assert ((got - want).abs() <= bound)[~nan].all()


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("rows,hkv", [(1, 1), (33, 3), (700, 8)])
def test_load(dev, dtype, rows, hkv):
    """Every code at scales across the type's range; rows outside the cache and
    the elements behind the last row stay as they were."""
    dt = DT[dtype]
    blocks = 24
    g = torch.Generator().manual_seed(rows)
    codes = torch.randint(0, 256, (2, blocks * 16, hkv, 128), dtype=torch.uint8, generator=g)
    lo, hi = (-118, 117) if dtype == "bf16" else (-15, 6)
    scales = torch.exp2(torch.randint(lo, hi + 1, (blocks, hkv, 2), generator=g).double()).float()
    slots = torch.randint(0, blocks * 16, (rows,), generator=g)
    if rows > 5:
        slots[1], slots[3] = -1, blocks * 16
    out = torch.full((2, rows + 1, hkv, 128), 7.0, dtype=dt, device=dev)
    feattn.load_kv8(codes[0].to(dev), codes[1].to(dev), scales.to(dev), slots.to(dev), out[0], out[1], rows, hkv, 128,
                    dtype == "bf16", blocks * 16)
    torch.cuda.synchronize()
    ok = (slots >= 0) & (slots < blocks * 16)
    for side in range(2):
        got = out[side].cpu()
        want = kv8.load(codes[side], scales, side, slots[ok])
        assert torch.equal(got[:rows][ok].double().nan_to_num(-3), want.to(dt).double().nan_to_num(-3))
        assert (got[:rows][~ok] == 7.0).all() and (got[rows:] == 7.0).all()


def test_append_is_capturable_and_repeatable(dev):
    """A captured append and load, replayed with eager work between, gives the
    eager calls' bits every time."""
    hq, hkv, max_pos = 32, 8, 400
    starts, qlens = BATCHES[6]
    blocks = sum(-(-(s + n) // 16) for s, n in zip(starts, qlens)) + 1
    slots, pos = rows_of(starts, qlens, blocks, 1)
    rows = len(slots)
    g = torch.Generator().manual_seed(1)
    stride = (hq + 2 * hkv) * 128
    kc, vc, scales = (t.to(dev) for t in cache(blocks, hkv, 8))
    table = W.rope_table(max_pos, 1e6).to(dev)
    w = torch.ones(128, dtype=torch.bfloat16, device=dev)
    buf = {n: t.clone() for n, t in (("k", kc), ("v", vc), ("s", scales))}
    qkv = torch.zeros(rows, stride, dtype=torch.bfloat16, device=dev)
    q = torch.zeros(rows, hq, 128, dtype=torch.bfloat16, device=dev)
    out = torch.zeros(2, rows, hkv, 128, dtype=torch.bfloat16, device=dev)
    slots, pos = slots.to(dev), pos.to(dev)

    def step():
        feattn.norm_rope_append_kv8(qkv, stride, w, w, 1e-6, q, buf["k"], buf["v"], buf["s"], pos, slots, table, rows,
                                    hq, hkv, True, max_pos, blocks * 16)
        feattn.load_kv8(buf["k"], buf["v"], buf["s"], slots, out[0], out[1], rows, hkv, 128, True, blocks * 16)

    def reset():
        buf["k"].copy_(kc)
        buf["v"].copy_(vc)
        buf["s"].copy_(scales)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(4):
        qkv.copy_((torch.randn(rows, stride, generator=g) * 2.0 ** i).to(torch.bfloat16))
        reset()
        step()
        want = [t.clone() for t in (q, out, buf["k"], buf["v"], buf["s"])]
        reset()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(want, (q, out, buf["k"], buf["v"], buf["s"])):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8)), i


# ---------------------------------------------------------------------------
# Attention
# ---------------------------------------------------------------------------

def check_attention(b, q, kc, vc, scales, out, lse, causal):
    at = torch.arange(kc.shape[0])
    want, want_lse, size, score, total = kv8.attention(b, q, kv8.load(kc, scales, 0, at), kv8.load(vc, scales, 1, at),
                                                       causal)
    u = U[q.dtype]
    e = score * 2.0 ** -16 + 2.0 ** -19
    bound = u * (2 * size + want.abs()) + 2 * e[..., None] * size + torch.finfo(q.dtype).smallest_normal
    if q.dtype == torch.float16:
        bound += 2.0 ** -25 * total
    err = (out.double() - want).abs()
    assert (err <= bound).all(), (err / bound).max().item()
    assert ((lse.double() - want_lse).abs() <= e + 2.0 ** -21 * want_lse.abs()).all()


def attend(dev, b, q, kc, vc, scales, causal, plan=None, graph=False, max_pages=None):
    own = plan is None
    if own:
        plan = feattn.Plan(b.hq, b.hkv, 128, b.page, max(1, b.batch), max_pages or b.max_pages(),
                           q.dtype == torch.bfloat16, b.blocks)
    plan.prepare(b.qo, b.kv, b.pages, b.last, b.batch, b.rows, graph=graph)
    out = torch.full((b.rows + 1, b.hq, 128), 7.0, dtype=q.dtype, device=dev)
    lse = torch.full((b.rows + 1, b.hq), 7.0, device=dev)
    plan.run_kv8(q.to(dev), kc.to(dev), vc.to(dev), scales.to(dev), out, causal=causal, lse=lse)
    torch.cuda.synchronize()
    assert (out[b.rows:] == 7.0).all() and (lse[b.rows:] == 7.0).all()
    lists = plan.lists(causal)
    if own:
        plan.close()
    return out[:b.rows].cpu(), lse[:b.rows].cpu(), lists


def case(hq, hkv, starts, qlens, seed, dtype="bf16", page=16, spread=0.5):
    b = W.make_batch(hq, hkv, starts=starts, qlens=qlens, seed=seed, page=page, extra_pages=2)
    q, _, _ = W.make_tensors(W.make_batch(hq, hkv, starts=[0], qlens=[1], seed=1), seed=1)
    g = torch.Generator().manual_seed(seed)
    q = torch.randn(b.rows, hq, 128, generator=g).to(DT[dtype])
    kc, vc, scales = cache((b.blocks + 1) * page // 16, hkv, seed, DT[dtype], spread)
    return b, q, kc, vc, scales


SHAPES = [
    # decode: lengths of one, block and page borders, whole and split
    (32, 8, [0, 15, 16, 17, 30, 31, 32, 47, 48], [1] * 9),
    (16, 8, [511] * 4, [1] * 4),
    (32, 8, [2999, 100, 1700, 0], [1] * 4),
    (8, 8, [1000, 33], [1, 1]),
    (40, 8, [300, 5, 1200], [5, 5, 5]),
    (32, 8, [900, 20], [8, 3]),
    # many sequences: decode shares of several items
    (32, 8, [37 * k % 700 + 3 for k in range(90)], [1] * 90),
    (16, 4, [53 * k % 900 for k in range(130)], [1] * 130),
    # kv head counts with fewer wavefronts a workgroup
    (6, 3, [400, 31, 64], [1, 1, 1]),
    (12, 2, [777, 40], [1, 2]),
    (4, 1, [1500, 3, 16], [1, 1, 1]),
    # tiles: prompts, chunks over a prefix, draft blocks, odd sizes
    (32, 8, [0], [64]),
    (16, 8, [0, 3, 65], [77, 130, 33]),
    (32, 4, [500, 17], [40, 300]),
    (32, 8, [700, 20, 333], [16, 16, 16]),
    (40, 8, [100], [129]),
    (24, 3, [2000, 100, 900, 17], [8, 5, 1, 7]),
    (64, 1, [400, 33, 150], [1, 1, 1]),
    # tiles and decode pieces in one batch
    (32, 8, [1300, 5, 260, 0], [1, 70, 1, 20]),
]


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
@pytest.mark.parametrize("causal", [True, False])
def test_attention(dev, dtype, shape, causal):
    hq, hkv, starts, qlens = SHAPES[shape]
    b, q, kc, vc, scales = case(hq, hkv, starts, qlens, 20 + shape, dtype)
    out, lse, _ = attend(dev, b, q, kc, vc, scales, causal)
    check_attention(b, q, kc, vc, scales, out, lse, causal)


@pytest.mark.parametrize("page", [32, 64, 256])
@pytest.mark.parametrize("causal", [True, False])
def test_page_sizes(dev, page, causal):
    b, q, kc, vc, scales = case(32, 8, [page - 1, page, 3 * page + 5, 0, 2 * page - 3, 700], [1, 1, 40, page + 3, 4, 1],
                                page, page=page)
    out, lse, _ = attend(dev, b, q, kc, vc, scales, causal)
    check_attention(b, q, kc, vc, scales, out, lse, causal)


@pytest.mark.parametrize("qlens", [[1, 3, 1, 1, 2], [1, 3, 50, 20, 16]])
@pytest.mark.parametrize("causal", [True, False])
def test_stale_slots(dev, qlens, causal):
    """Slots no sequence holds have NaN codes, blocks no sequence holds NaN and
    infinite scales: nothing of it reaches the results."""
    b, q, kc, vc, scales = case(32, 8, [700, 5, 33, 0, 2000], qlens, 9)
    live = torch.zeros(kc.shape[0], dtype=torch.bool)
    for s in range(b.batch):
        t = torch.arange(b.lens[s])
        live[torch.tensor(b.tables[s])[t // 16] * 16 + t % 16] = True
    kz, vz = kc.clone(), vc.clone()
    kz[~live], vz[~live] = 0, 0
    kc[~live], vc[~live] = 0x7f, 0xff
    bad = scales.clone()
    dead = ~live.view(-1, 16).any(1)
    assert dead.any()
    bad[dead] = torch.tensor([math.nan, math.inf])
    out, lse, _ = attend(dev, b, q, kc, vc, bad, causal)
    assert torch.isfinite(out).all() and torch.isfinite(lse).all()
    check_attention(b, q, kz, vz, scales, out, lse, causal)


@pytest.mark.parametrize("rows", [1, 20])
def test_large_scores(dev, rows):
    """Scales that differ by 2^12 from block to block: scores of thousands,
    probabilities that are one token's."""
    b, q, kc, vc, scales = case(32, 8, [1000, 90, 300], [rows] * 3, 31, spread=3.0)
    out, lse, _ = attend(dev, b, q, kc, vc, scales, True)
    check_attention(b, q, kc, vc, scales, out, lse, True)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_graph_replays(dev, dtype):
    """A graph plan's launch captured once, replayed on batches that are planned
    as shares, as short-context items and with merges."""
    hq, hkv, n = 32, 8, 12
    batches = [[100 * (k + 1) for k in range(n)], [20 + k for k in range(n)], [2500 - 200 * k for k in range(n)],
               [0] * n, [300] * 5]
    dt = DT[dtype]
    pool = 1200
    plan = feattn.Plan(hq, hkv, 128, 16, n, 200, dtype == "bf16", pool)
    g = torch.Generator().manual_seed(2)
    kc, vc, scales = cache(pool + 1, hkv, 2, dt)
    kd, vd, sd = kc.to(dev), vc.to(dev), scales.to(dev)
    q = torch.zeros(n, hq, 128, dtype=dt, device=dev)
    out, lse = torch.zeros_like(q), torch.zeros(n, hq, device=dev)
    graph = None
    for i, starts in enumerate(batches):
        b = W.make_batch(hq, hkv, starts=starts, qlens=[1] * len(starts), seed=i, pool=pool)
        plan.prepare(b.qo, b.kv, b.pages, b.last, b.batch, b.rows, graph=True)
        qc = torch.randn(b.rows, hq, 128, generator=g).to(dt)
        q[:b.rows] = qc.to(dev)
        if graph is None:
            plan.run_kv8(q, kd, vd, sd, out, lse=lse)
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                plan.run_kv8(q, kd, vd, sd, out, lse=lse)
        out.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        assert (out[b.rows:] == 7.0).all()
        check_attention(b, qc, kc, vc, scales, out[:b.rows].cpu(), lse[:b.rows].cpu(), True)
    plan.close()


def test_graph_replays_with_tiles(dev):
    hq, hkv = 32, 8
    pool = 600
    plan = feattn.Plan(hq, hkv, 128, 16, 8, 200, True, pool)
    kc, vc, scales = cache(pool + 1, hkv, 6)
    kd, vd, sd = kc.to(dev), vc.to(dev), scales.to(dev)
    g = torch.Generator().manual_seed(3)
    q = torch.zeros(400, hq, 128, dtype=torch.bfloat16, device=dev)
    out, lse = torch.zeros_like(q), torch.zeros(400, hq, device=dev)
    graph = None
    for i, (starts, qlens) in enumerate([([300, 40], [16, 16]), ([0, 1000, 64], [200, 1, 33]), ([900] * 4, [16] * 4)]):
        b = W.make_batch(hq, hkv, starts=starts, qlens=qlens, seed=i, pool=pool)
        plan.prepare(b.qo, b.kv, b.pages, b.last, b.batch, b.rows, graph=True)
        qc = torch.randn(b.rows, hq, 128, generator=g).to(torch.bfloat16)
        q[:b.rows] = qc.to(dev)
        if graph is None:
            plan.run_kv8(q, kd, vd, sd, out, lse=lse, causal=False)
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                plan.run_kv8(q, kd, vd, sd, out, lse=lse, causal=False)
        graph.replay()
        torch.cuda.synchronize()
        check_attention(b, qc, kc, vc, scales, out[:b.rows].cpu(), lse[:b.rows].cpu(), False)
    plan.close()


def test_one_plan_serves_both_caches(dev):
    """The 16-bit call of the same plan, on a cache that holds the same values,
    before and after: same results within the roundings, its own bits kept."""
    b, q, kc, vc, scales = case(32, 8, [1000, 30, 5], [1, 40, 1], 12)
    at = torch.arange(kc.shape[0])
    k16 = kv8.load(kc, scales, 0, at).to(torch.bfloat16).view(b.blocks + 1, 16, 8, 128).to(dev)
    v16 = kv8.load(vc, scales, 1, at).to(torch.bfloat16).view(b.blocks + 1, 16, 8, 128).to(dev)
    plan = feattn.Plan(32, 8, 128, 16, 3, b.max_pages(), True, b.blocks)
    plan.prepare(b.qo, b.kv, b.pages, b.last, b.batch, b.rows)
    qd = q.to(dev)
    outs = [torch.zeros_like(qd) for _ in range(3)]
    lses = [torch.zeros(b.rows, 32, device=dev) for _ in range(3)]
    plan.run(qd, k16, v16, outs[0], lse=lses[0])
    plan.run_kv8(qd, kc.to(dev), vc.to(dev), scales.to(dev), outs[1], lse=lses[1])
    plan.run(qd, k16, v16, outs[2], lse=lses[2])
    torch.cuda.synchronize()
    plan.close()
    assert torch.equal(outs[0], outs[2]) and torch.equal(lses[0], lses[2])
    for o, l in zip(outs, lses):
        check_attention(b, q, kc, vc, scales, o.cpu(), l.cpu(), True)


def test_refusals_on_a_plan(dev):
    b, q, kc, vc, scales = case(32, 8, [10], [1], 1)
    plan = feattn.Plan(32, 8, 128, 16, 1, b.max_pages(), True, b.blocks)
    qd, kd, vd, sd = q.to(dev), kc.to(dev), vc.to(dev), scales.to(dev)
    out = torch.zeros_like(qd)
    with pytest.raises(RuntimeError, match="before prepare"):
        plan.run_kv8(qd, kd, vd, sd, out)
    plan.prepare(b.qo, b.kv, b.pages, b.last, b.batch, b.rows)
    with pytest.raises(RuntimeError, match="null"):
        plan.run_kv8(qd, kd, vd, None, out)
    with pytest.raises(RuntimeError, match="8-byte"):
        plan.run_kv8(qd, kd, vd, sd.view(-1)[1:], out)
    with pytest.raises(RuntimeError, match="16-byte"):
        plan.run_kv8(qd, kd.view(-1)[8:], vd, sd, out)
    plan.close()


def test_steps_together(dev):
    """A prompt in two chunks, then decode steps, each an append and attention on
    a side stream: what attention sees is what the oracle's cache holds."""
    hq, hkv, max_pos, eps = 16, 8, 400, 1e-6
    pool = 40
    g = torch.Generator().manual_seed(11)
    perm = torch.randperm(pool, generator=g).tolist()
    tables = [perm[:16], perm[16:24], perm[24:]]
    kc = torch.zeros((pool + 1) * 16, hkv, 128, dtype=torch.uint8)
    scales = torch.zeros(pool + 1, hkv, 2)
    kd, vd, sd = kc.to(dev), kc.to(dev), scales.to(dev)
    table = W.rope_table(max_pos, 1e6)
    kw = (1 + 0.1 * torch.randn(128, generator=g)).to(torch.bfloat16)
    plan = feattn.Plan(hq, hkv, 128, 16, 3, 20, True, pool)
    stream = torch.cuda.Stream()
    done = [0, 0, 0]
    stride = (hq + 2 * hkv) * 128
    vc = kc.clone()
    for qlens in ([70, 3, 100], [41, 50, 17], [1, 1, 1], [1, 1, 1], [5, 5, 5], [1, 1, 1]):
        b = W.Batch(hq=hq, hkv=hkv, page=16, blocks=pool, starts=list(done), qlens=qlens, tables=tables)
        W.build_metadata(b)
        qkv = (torch.randn(b.rows, stride, generator=g) * torch.exp(torch.randn(b.rows, 1, generator=g)))
        qkv = qkv.to(torch.bfloat16)
        pos, slots = torch.from_numpy(b.positions), torch.from_numpy(b.slots)
        args = [t.to(dev) for t in (qkv, kw, pos, slots, table)]
        q = torch.zeros(b.rows, hq, 128, dtype=torch.bfloat16, device=dev)
        out, lse = torch.zeros_like(q), torch.zeros(b.rows, hq, device=dev)
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            feattn.norm_rope_append_kv8(args[0], stride, args[1], args[1], eps, q, kd, vd, sd, args[2], args[3],
                                        args[4], b.rows, hq, hkv, True, max_pos, b.cache_slots)
            plan.prepare(b.qo, b.kv, b.pages, b.last, b.batch, b.rows)
            plan.run_kv8(q, kd, vd, sd, out, lse=lse)
        torch.cuda.synchronize()
        heads = qkv.view(b.rows, -1, 128)
        want_k, size = kv8.norm_rope(heads[:, hq:hq + hkv], kw, eps, pos, table, max_pos)
        _, s1 = kv8.append(kc, scales, 0, want_k, slots, torch.bfloat16)
        vc, s2 = kv8.append(vc, s1, 1, heads[:, hq + hkv:].double(), slots, torch.bfloat16)
        assert torch.equal(sd.cpu(), s2)
        # (keys within the norm's roundings, values exactly; the next step goes on from the device's keys)
        kc, scales = kd.cpu(), s2
        got, slack = kv8.load(kc, scales, 0, slots), 2.0 ** -18 * size
        half = half_step8(want_k.abs() + slack, scales[slots // 16][:, :, 0, None].double())
        assert ((got - want_k).abs() <= half + slack).all()
        done = [d + n for d, n in zip(done, qlens)]
        for i, n in enumerate(done):
            t = torch.arange(n)
            at = torch.tensor(tables[i])[t // 16] * 16 + t % 16
            assert torch.equal(vd.cpu()[at], vc[at])
        check_attention(b, q.cpu(), kc, vc, scales, out.cpu(), lse.cpu(), True)
    plan.close()


def test_cache_past_4_gib(dev):
    """Codes behind 4 GiB: an append there, attention over it, and a load."""
    hq, hkv = 8, 8
    blocks = (5 << 30) // (16 * hkv * 128) - 1
    kd = torch.zeros((blocks + 1) * 16, hkv, 128, dtype=torch.uint8, device=dev)
    vd = torch.zeros_like(kd)
    sd = torch.zeros(blocks + 1, hkv, 2, device=dev)
    n = 100
    g = torch.Generator().manual_seed(3)
    tables = [[blocks - 1 - 3 * i for i in range(7)]]
    b = W.Batch(hq=hq, hkv=hkv, page=16, blocks=blocks, starts=[0], qlens=[n], tables=tables)
    W.build_metadata(b)
    slots = torch.from_numpy(b.slots)
    k, v = (torch.randn(n, hkv, 128, generator=g).to(torch.bfloat16) for _ in range(2))
    feattn.store_kv8(k.to(dev), v.to(dev), kd, vd, sd, slots.to(dev), n, hkv, 128, True, b.cache_slots)
    got = torch.zeros(2, n, hkv, 128, dtype=torch.bfloat16, device=dev)
    feattn.load_kv8(kd, vd, sd, slots.to(dev), got[0], got[1], n, hkv, 128, True, b.cache_slots)
    small = torch.zeros(112, hkv, 128, dtype=torch.uint8)
    at = torch.arange(n)
    wk, s = kv8.append(small, torch.zeros(7, hkv, 2), 0, k.double(), at, torch.bfloat16)
    wv, s = kv8.append(small, s, 1, v.double(), at, torch.bfloat16)
    torch.cuda.synchronize()
    assert torch.equal(got[0].cpu().double(), kv8.load(wk, s, 0, at))
    assert torch.equal(got[1].cpu().double(), kv8.load(wv, s, 1, at))
    for rows in (1, n):
        bb = W.Batch(hq=hq, hkv=hkv, page=16, blocks=blocks, starts=[n - rows], qlens=[rows], tables=tables)
        W.build_metadata(bb)
        q = torch.randn(rows, hq, 128, generator=g).to(torch.bfloat16)
        plan = feattn.Plan(hq, hkv, 128, 16, 1, 10, True, blocks)
        plan.prepare(bb.qo, bb.kv, bb.pages, bb.last, 1, rows)
        out, lse = torch.zeros_like(q, device=dev), torch.zeros(rows, hq, device=dev)
        plan.run_kv8(q.to(dev), kd, vd, sd, out, lse=lse)
        torch.cuda.synchronize()
        plan.close()
        sb = W.Batch(hq=hq, hkv=hkv, page=16, blocks=6, starts=[n - rows], qlens=[rows], tables=[list(range(7))])
        W.build_metadata(sb)
        check_attention(sb, q, wk, wv, s, out.cpu(), lse.cpu(), True)


# Batches whose lists take the paths that small ones do not: more than one
# workgroup a compute unit, several items a workgroup, shares evened out.
LISTS = [
    # longest first, wide items, 512 shares of one to three items
    (32, 8, [9, 100, 0, 31, 250, 77] * 2, [300, 201, 77, 128, 250, 33] * 2),
    (16, 8, [7 * k % 90 for k in range(30)], [200 - 3 * k for k in range(30)]),
    (64, 2, [11 * k % 400 for k in range(20)], [1 + 7 * k % 90 for k in range(20)]),
    (6, 3, [7 * k % 50 for k in range(14)], [450 - 10 * k for k in range(14)]),
    # narrow items, longest first (one kv head a workgroup)
    (32, 8, [7 * k % 480 for k in range(70)], [16] * 70),
    (24, 3, [13 * k % 470 for k in range(200)], [8] * 200),
    # narrow items, equal cuts: pairs of kv heads, an odd count
    (32, 8, [37 * k % 1500 + 300 for k in range(30)], [16] * 30),
    (16, 2, [997, 3000, 40, 1800, 0, 512], [8, 5, 7, 8, 8, 8]),
    (16, 4, [900] * 9, [9, 16, 12] * 3),
    (24, 3, [2000, 900, 1711, 30], [8] * 4),
    # equal cuts of wide items
    (32, 8, [3000, 700, 12], [60, 33, 140]),
]


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("shape", range(len(LISTS)))
@pytest.mark.parametrize("causal", [True, False])
def test_lists(dev, dtype, shape, causal):
    hq, hkv, starts, qlens = LISTS[shape]
    b, q, kc, vc, scales = case(hq, hkv, starts, qlens, 60 + shape, dtype)
    out, lse, lists = attend(dev, b, q, kc, vc, scales, causal)
    assert lists.tile_items > 0
    if shape < 6:
        assert lists.tile_items > 256 and lists.merge_rows == 0
    check_attention(b, q, kc, vc, scales, out, lse, causal)
    again, lse2, _ = attend(dev, b, q, kc, vc, scales, causal)
    assert torch.equal(out, again) and torch.equal(lse, lse2)


@pytest.mark.parametrize("starts,qlens", [([3000, 5000, 1200, 4000], [16] * 4), ([9000, 4000], [60, 70]),
                                          ([4000, 7000, 9000, 2500], [1, 1, 5, 1])])
def test_split_rows_in_fp16(dev, starts, qlens):
    """fp16 rows split over several work units carry two roundings of their size,
    as unsplit ones do: 2^0.5 times the output's alone in the mean square (three
    would be 1.73), over 10^5 values and more to within a few per cent."""
    b, q, kc, vc, scales = case(32, 8, starts, qlens, 91, "f16")
    out, lse, lists = attend(dev, b, q, kc, vc, scales, False)
    assert lists.merge_rows == b.rows
    check_attention(b, q, kc, vc, scales, out, lse, False)
    at = torch.arange(kc.shape[0])
    want = kv8.attention(b, q, kv8.load(kc, scales, 0, at), kv8.load(vc, scales, 1, at), False)[0]
    err = (out.double() - want).square().mean().sqrt()
    rounding = (want.half().double() - want).square().mean().sqrt()
    assert err <= 1.55 * rounding, (err / rounding).item()


GROUPS = [
    # head counts at the borders of the work units' columns
    (33, 1, [70, 1000], [1, 2]),
    (48, 1, [300, 40, 2000], [1, 1, 1]),
    (96, 2, [1500, 20], [1, 3]),
    (128, 1, [200, 900], [1, 2]),
    (130, 2, [100, 700], [1, 1]),
    (64, 2, [30, 800], [2, 4]),
    (7, 7, [500, 20, 90], [1, 3, 40]),
    (10, 5, [600, 33], [16, 70]),
    (16, 16, [260, 1100], [1, 33]),
]


@pytest.mark.parametrize("graph", [False, True])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("shape", range(len(GROUPS)))
def test_group_sizes(dev, shape, causal, graph):
    hq, hkv, starts, qlens = GROUPS[shape]
    b, q, kc, vc, scales = case(hq, hkv, starts, qlens, 80 + shape, "bf16")
    out, lse, _ = attend(dev, b, q, kc, vc, scales, causal, graph=graph)
    check_attention(b, q, kc, vc, scales, out, lse, causal)


def test_shares_of_many_items(dev):
    """More items a share than a wavefront has lanes: 34000 sequences of two
    rows over the same three pages.  The first is right, the others are its bits."""
    hq, hkv, n = 64, 1, 34000
    one = W.Batch(hq=hq, hkv=hkv, page=16, blocks=4, starts=[38], qlens=[2], tables=[[2, 0, 3]])
    W.build_metadata(one)
    kc, vc, scales = cache(5, hkv, 3)
    g = torch.Generator().manual_seed(4)
    q = torch.randn(2, hq, 128, generator=g).to(torch.bfloat16)
    b = W.Batch(hq=hq, hkv=hkv, page=16, blocks=4, starts=[38] * n, qlens=[2] * n, tables=[[2, 0, 3]] * n)
    W.build_metadata(b)
    plan = feattn.Plan(hq, hkv, 128, 16, n, one.max_pages(), True, 4)
    plan.prepare(b.qo, b.kv, b.pages, b.last, b.batch, b.rows)
    assert plan.lists(True).tile_items == n
    qd = q.to(dev).repeat(n, 1, 1)
    out, lse = torch.zeros_like(qd), torch.zeros(2 * n, hq, device=dev)
    plan.run_kv8(qd, kc.to(dev), vc.to(dev), scales.to(dev), out, lse=lse)
    torch.cuda.synchronize()
    plan.close()
    check_attention(one, q, kc, vc, scales, out[:2].cpu(), lse[:2].cpu(), True)
    assert (out.view(n, 2, hq, 128) == out[:2]).all() and (lse.view(n, 2, hq) == lse[:2]).all()


@pytest.mark.parametrize("qlens", [[1, 1, 1], [16, 16, 16], [70, 1, 20]])
def test_without_lse(dev, qlens):
    """No lse asked for: the same rows.  A batch without sequences writes nothing."""
    b, q, kc, vc, scales = case(32, 8, [900, 30, 1500], qlens, 5)
    want, _, _ = attend(dev, b, q, kc, vc, scales, True)
    plan = feattn.Plan(32, 8, 128, 16, 3, b.max_pages(), True, b.blocks)
    qd, kd, vd, sd = q.to(dev), kc.to(dev), vc.to(dev), scales.to(dev)
    out = torch.full_like(qd, 7.0)
    plan.prepare([0], [0], [], [], 0, 0)
    plan.run_kv8(qd, kd, vd, sd, out)
    torch.cuda.synchronize()
    assert (out == 7.0).all()
    plan.prepare(b.qo, b.kv, b.pages, b.last, b.batch, b.rows)
    plan.run_kv8(qd, kd, vd, sd, out)
    torch.cuda.synchronize()
    plan.close()
    assert torch.equal(out.cpu(), want)


def test_two_plans_on_two_streams(dev):
    """Two plans' calls in flight at once, eager and as graphs, over caches of
    their own: each has its own results."""
    cases = [case(32, 8, [1500, 30, 700], [1, 1, 1], 5), case(32, 8, [1200, 64, 9], [40, 16, 130], 6)]
    plans, tensors, graphs = [], [], []
    for b, q, kc, vc, scales in cases:
        plan = feattn.Plan(32, 8, 128, 16, 3, b.max_pages(), True, b.blocks)
        plan.prepare(b.qo, b.kv, b.pages, b.last, b.batch, b.rows, graph=True)
        t = [x.to(dev) for x in (q, kc, vc, scales)] + [torch.zeros_like(q, device=dev)]
        lse = torch.zeros(b.rows, 32, device=dev)
        plan.run_kv8(*t, lse=lse)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            plan.run_kv8(*t, lse=lse)
        plans.append(plan)
        tensors.append((t, lse))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in cases]
    for replay in (False, True):
        for t, lse in tensors:
            t[-1].zero_()
            lse.zero_()
        torch.cuda.synchronize()
        for _ in range(5):
            for plan, (t, lse), graph, st in zip(plans, tensors, graphs, streams):
                with torch.cuda.stream(st):
                    graph.replay() if replay else plan.run_kv8(*t, lse=lse)
        torch.cuda.synchronize()
        for (b, q, kc, vc, scales), (t, lse) in zip(cases, tensors):
            check_attention(b, q, kc, vc, scales, t[-1].cpu(), lse.cpu(), True)
    for plan in plans:
        plan.close()


def test_nothing_to_do(dev):
    """No rows, or no kv heads and no queries: the calls return and write nothing."""
    kc, vc, scales = (t.to(dev) for t in cache(2, 8, 1))
    before = [t.clone() for t in (kc, vc, scales)]
    x = torch.zeros(4, 8, 128, dtype=torch.bfloat16, device=dev)
    slots = torch.zeros(4, dtype=torch.int64, device=dev)
    table = W.rope_table(8, 1e4).to(dev)
    for rows, hkv in ((0, 8), (4, 0)):
        feattn.store_kv8(x, x, kc, vc, scales, slots, rows, hkv, 128, True, 32)
        feattn.load_kv8(kc, vc, scales, slots, x, x, rows, hkv, 128, True, 32)
    feattn.rope_append_kv8(x, x, x, kc, vc, scales, slots, slots, table, 0, 8, 8, 128, True, 8, 32)
    torch.cuda.synchronize()
    for t, w in zip((kc, vc, scales), before):
        assert torch.equal(t, w)
    assert not x.any()
