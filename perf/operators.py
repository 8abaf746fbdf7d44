"""The 8-bit paged KV cache's operators, case by case: how they are called,
their plain forms, the work they cannot do without and their 64-bit results.

The caches hold e4m3 codes [blocks + 1][page][kv heads][128]; `scales`
[(blocks + 1) * page / 16][kv heads][2] holds a power of two for K and one for
V of every 16-token block and head; a value is code * scale.

* append: (norm,) RoPE and append of a step's new tokens, whose blocks may
  hold earlier tokens; the touched blocks are read back as 16-bit rows, so that
  the pass returns the queries and the values the cache holds afterwards.
* load: cached tokens as 16-bit rows (a prefix handed to another cache).
* attention: a prepared batch over the cached codes.
* step: a layer's append and attention of one decode step.
"""

import math
import os
import sys

import torch

own = False

DIM = 128
PAGE = 16
EPS = 1e-6
THETA = 1e6
MAX_POS = 40000
TOP = 448.0  # the largest e4m3 value
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
CODE = torch.float8_e4m3fn


def _case(name, kind, hq, hkv, seqs=0, rows=1, ctx=(0, 0), chunks=0, tokens=0, prefix=(0, 0), causal=True, norm=True,
          dtype="bf16", lens_seed=1):
    """`seqs` sequences with `rows` new tokens each over ctx[0]..ctx[1] cached
    ones, and `chunks` prompt chunks of `tokens` new tokens together, each over
    prefix[0]..prefix[1] cached ones."""
    return {"name": name, "kind": kind, "hq": hq, "hkv": hkv, "seqs": seqs, "rows": rows, "ctx_lo": ctx[0],
            "ctx_hi": ctx[1], "chunks": chunks, "tokens": tokens, "prefix_lo": prefix[0], "prefix_hi": prefix[1],
            "causal": causal, "norm": norm, "dtype": dtype, "lens_seed": lens_seed}


def listed():
    return [
        # The append of a full decode batch: one token for each sequence, most
        # of them into blocks that hold earlier tokens.
        _case("append_decode", "append", 32, 8, seqs=64, ctx=(511, 4095), lens_seed=2),
        # The append of a prefill budget filled by chunks of eight prompts.
        _case("append_prefill", "append", 32, 8, chunks=8, tokens=8192, prefix=(0, 2048), lens_seed=3),
        # Draft tokens under verification, float16, keys rotated but not
        # normalised: runs of five that start anywhere in a block.
        _case("append_verify_f16", "append", 40, 8, seqs=24, rows=5, ctx=(200, 6000), norm=False, dtype="f16",
              lens_seed=7),
        # A long cached prefix handed on as 16-bit rows.
        _case("load_prefix", "load", 32, 4, seqs=1, ctx=(30000, 30000)),
        # The same of a few short conversations, float16.
        _case("load_short_f16", "load", 16, 8, seqs=3, ctx=(20, 200), dtype="f16", lens_seed=9),
        # One layer of a decode step of a few short conversations on a small
        # model: append, then attention; bound by launches and latency.
        _case("step_small", "step", 16, 8, seqs=4, ctx=(511, 511)),
        # Attention of a full decode batch of an 8B-class model.
        _case("decode_8b", "attention", 32, 8, seqs=64, ctx=(511, 4095), lens_seed=2),
        # Long contexts, which a cache is held in 8 bits for.
        _case("decode_long", "attention", 32, 8, seqs=16, ctx=(32767, 32767)),
        # Verification of 4 draft tokens + 1 for each sequence, float16.
        _case("verify_f16", "attention", 40, 8, seqs=24, rows=5, ctx=(200, 6000), dtype="f16", lens_seed=7),
        # Draft blocks: 16 rows that see each other and a long context.
        _case("dflash_blocks", "attention", 32, 8, seqs=32, rows=16, ctx=(2048, 16384), causal=False, lens_seed=5),
        # The prefill budget of an 8B-class model: chunks of eight prompts,
        # some over a cached prefix.
        _case("prefill_8b", "attention", 32, 8, chunks=8, tokens=8192, prefix=(0, 2048), lens_seed=3),
        # One chunk of a long document: 2048 new tokens over 30000 cached.
        _case("prefill_long", "attention", 32, 4, chunks=1, tokens=2048, prefix=(30000, 30000)),
    ]


_HEADS = [(16, 8), (32, 8), (32, 4), (40, 8)]


def _log_int(rng, lo, hi):
    """An integer of [lo, hi], spread evenly over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    kind = rng.choice(["append", "append", "load", "step", "attention", "attention", "attention", "attention"])
    form = {"load": "decode", "step": "decode", "append": rng.choice(["decode", "verify", "prefill"]),
            "attention": rng.choice(["decode", "decode", "verify", "block", "prefill", "prefill"])}[kind]
    hq, hkv = rng.choice(_HEADS)
    dtype = rng.choice(["bf16", "bf16", "f16"])
    ls = rng.randrange(1, 1 << 20)
    norm = rng.random() < 0.7
    if form == "prefill":
        tokens = _log_int(rng, 64, 8192)
        chunks = min(rng.randint(1, 8), max(1, tokens // 64))
        most = 2048 * 30000 * 32 // hq - tokens * tokens // 2  # (row, cached token) pairs
        prefix = min(rng.choice([0, _log_int(rng, 16, 30000)]), most // tokens)
        c = _case("", kind, hq, hkv, chunks=chunks, tokens=tokens, prefix=(rng.randint(0, prefix), prefix), norm=norm,
                  dtype=dtype, lens_seed=ls)
    else:
        most = {"decode": 500000, "verify": 250000, "block": 300000}[form]  # cached tokens of the batch
        most = 30000 if kind == "load" else most
        hi = _log_int(rng, 16, 30000 if kind == "load" else 32767)
        seqs = min(_log_int(rng, 1, 256 if form == "decode" else 64), max(1, most // hi))
        rows = {"decode": 1, "verify": rng.randint(2, 8), "block": rng.choice([8, 16, 16])}[form]
        c = _case("", kind, hq, hkv, seqs=seqs, rows=rows, ctx=(rng.randint(1, hi), hi), causal=form != "block",
                  norm=norm, dtype=dtype, lens_seed=ls)
    del c["name"]
    return c


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------

def _lens(case):
    """(cached tokens, new tokens) of every sequence: from the case alone."""
    g = torch.Generator().manual_seed(case["lens_seed"])
    ints = lambda lo, hi, n: torch.randint(lo, hi + 1, (n,), generator=g).tolist()  # noqa: E731
    starts, rows = ints(case["ctx_lo"], case["ctx_hi"], case["seqs"]), [case["rows"]] * case["seqs"]
    n = case["chunks"]
    if n:
        starts += ints(case["prefix_lo"], case["prefix_hi"], n)
        least = min(64, case["tokens"] // n)
        share = torch.rand(n, generator=g, dtype=torch.float64) + 0.5
        ends = [0] + ((case["tokens"] - least * n) * share.cumsum(0) / share.sum()).round().long().tolist()
        rows += [least + b - a for a, b in zip(ends, ends[1:])]
    return starts, rows


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _randn(shape, gen, dtype, scale=1.0):
    x = torch.randn(shape, generator=gen, device="cuda", dtype=dtype)
    return x.mul_(scale) if scale != 1.0 else x


def _weight(n, gen, dtype):
    return (1 + 0.1 * torch.randn(n, generator=gen, device="cuda")).to(dtype)


def _need(amax):
    """The smallest power of two with amax <= TOP * it (2^-118 at least)."""
    m, x = torch.frexp(amax)
    e = torch.where(amax > 0, x - 9 + (m > 0.875).to(x.dtype), -118).clamp_min(-118)
    return (e.int() + 127 << 23).view(torch.float32)


def _filled(blocks, hkv, gen):
    """A cache of `blocks` 16-token blocks whose values are normal, with
    channels (K) and tokens (V) of different size, as codes, and its scales."""
    codes, scales = [], torch.empty(blocks, hkv, 2, device="cuda")
    for side in range(2):
        x = _randn((blocks, PAGE, hkv, DIM), gen, torch.float32)
        size = torch.randn((1, 1, hkv, DIM) if side == 0 else (blocks, PAGE, 1, 1), generator=gen, device="cuda")
        x *= size.mul_(0.5).exp_()
        scales[..., side] = _need(x.abs().amax((1, 3)))
        codes.append((x / scales[:, None, :, side, None]).to(CODE))
    return codes[0], codes[1], scales


def _angles(dtype=torch.float32):
    inv = 1.0 / torch.pow(torch.tensor(THETA, dtype=dtype, device="cuda"),
                          torch.arange(0, DIM, 2, dtype=dtype, device="cuda") / DIM)
    f = torch.arange(MAX_POS, dtype=dtype, device="cuda")[:, None] * inv
    return torch.cat([f.cos(), f.sin()], 1)


def _ints(v, dtype=torch.int64):
    return torch.tensor(v, dtype=dtype, device="cuda")


def prepare(case, seed):
    """Random activations and a filled cache, pages in random order."""
    dt, kind = DTYPES[case["dtype"]], case["kind"]
    hq, hkv = case["hq"], case["hkv"]
    starts, rows = _lens(case)
    lens = [s + n for s, n in zip(starts, rows)]
    npages = [-(-n // PAGE) for n in lens]
    blocks = sum(npages)  # page `blocks` is the padding page
    gen = _gen(seed)
    perm = torch.randperm(blocks, generator=gen, device="cuda")
    kv = [0]
    for n in npages:
        kv.append(kv[-1] + n)
    qo = [0]
    for n in rows:
        qo.append(qo[-1] + n)
    n_rows = qo[-1]
    kc, vc, scales = _filled(blocks + 1, hkv, gen)
    seq = torch.repeat_interleave(torch.arange(len(rows), device="cuda"), _ints(rows))
    local = torch.arange(n_rows, device="cuda") - _ints(qo)[seq]
    pos = _ints(starts)[seq] + local
    slots = perm[_ints(kv)[seq] + pos // PAGE] * PAGE + pos % PAGE
    st = {"case": dict(case), "kind": kind, "bf16": dt == torch.bfloat16, "dtype": dt, "kc": kc, "vc": vc,
          "scales": scales, "rows": n_rows, "lens": lens, "qlens": rows, "kv": kv, "qo": qo, "perm": perm,
          "blocks": blocks, "cache_slots": (blocks + 1) * PAGE, "pos": pos, "slots": slots}
    if kind in ("append", "step"):
        st["table"] = _angles()
        heads = hq + 2 * hkv
        if case["norm"]:
            st.update(qkv=_randn((n_rows, heads * DIM), gen, dt, 2.0), qw=_weight(DIM, gen, dt),
                      kw=_weight(DIM, gen, dt), q=torch.empty((n_rows, hq, DIM), device="cuda", dtype=dt))
        else:
            st.update(q=_randn((n_rows, hq, DIM), gen, dt), k=_randn((n_rows, hkv, DIM), gen, dt),
                      v=_randn((n_rows, hkv, DIM), gen, dt))
        # The touched blocks, and which of their tokens hold something after the call.
        touched, index = torch.unique(slots // PAGE, return_inverse=True)
        last = torch.zeros_like(touched).scatter_reduce(0, index, slots % PAGE, "amax")
        at = torch.arange(PAGE, device="cuda")[None]
        fresh = torch.zeros(len(touched), dtype=torch.bool, device="cuda")
        fresh[index[slots % PAGE == 0]] = True
        st.update(touched=touched, index=index, fresh=fresh,
                  read=(touched[:, None] * PAGE + at)[at <= last[:, None]])
    elif kind == "load":
        seq = torch.repeat_interleave(torch.arange(len(rows), device="cuda"), _ints(lens))
        p = torch.arange(sum(lens), device="cuda") - _ints([0] + lens).cumsum(0)[seq]
        st["read"] = perm[_ints(kv)[seq] + p // PAGE] * PAGE + p % PAGE
    else:
        st["q"] = _randn((n_rows, hq, DIM), gen, dt)
    if kind in ("append", "load"):
        shape = (len(st["read"]), hkv, DIM)
        st.update(k_out=torch.empty(shape, device="cuda", dtype=dt), v_out=torch.empty(shape, device="cuda", dtype=dt))
    if kind in ("attention", "step"):
        st["out"] = torch.empty((n_rows, hq, DIM), device="cuda", dtype=dt)
        st["lse"] = torch.empty((n_rows, hq), device="cuda")
        # Every sequence's tokens and rows, padded to the longest one's.
        t = torch.arange(max(lens), device="cuda")[None]
        page = torch.clamp(_ints(kv)[:-1, None] + t // PAGE, max=blocks - 1)
        st["at"] = perm[page] * PAGE + t % PAGE
        r = torch.arange(max(rows), device="cuda")[None]
        have = r < _ints(rows)[:, None]
        sees = _ints(starts)[:, None] + r if case["causal"] else (_ints(lens) - 1)[:, None].expand(-1, max(rows))
        st.update(row_at=torch.clamp(_ints(qo)[:-1, None] + r, max=n_rows - 1), have=have,
                  sees=torch.minimum(sees, _ints(lens)[:, None] - 1))
        if own:
            feattn = _feattn()
            pages = perm.tolist()
            last = [(n - 1) % PAGE + 1 for n in lens]
            st["plan"] = feattn.Plan(hq, hkv, DIM, PAGE, len(rows), max(npages) + 1, st["bf16"], blocks)
            st["plan"].prepare(qo, kv, pages, last, len(rows), n_rows)
    return st


def _feattn():
    pkg = os.path.join(os.getcwd(), "flashengine.cpp_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import feattn

    return feattn


# ---------------------------------------------------------------------------
# The plain forms
# ---------------------------------------------------------------------------

def _rope(x, cs):
    c, s = cs[:, None, :DIM // 2], cs[:, None, DIM // 2:]
    a, b = x[..., :DIM // 2], x[..., DIM // 2:]
    return torch.cat([a * c - b * s, b * c + a * s], -1)


def _rms(x, w):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w


def _values(codes, scales, side, blocks):
    """The values of whole blocks."""
    return codes.view(torch.uint8)[blocks].view(CODE).float() * scales[blocks][:, None, :, side, None]


def _put(st, codes, side, x):
    """Appends the rows x (fp32) to one cache: new scales, the touched blocks'
    earlier tokens on them, the new tokens' codes."""
    touched, index, scales = st["touched"], st["index"], st["scales"]
    amax = torch.zeros(len(touched), x.shape[1], device=x.device)
    amax.scatter_reduce_(0, index[:, None].expand(-1, x.shape[1]), x.abs().amax(-1), "amax")
    old = scales[touched][..., side]
    new = torch.where(st["fresh"][:, None], _need(amax), torch.maximum(old, _need(amax)))
    held = _values(codes, scales, side, touched)
    held.view(-1, *x.shape[1:])[index * PAGE + st["slots"] % PAGE] = x
    codes.view(torch.uint8)[touched] = (held / new[:, None, :, None]).clamp(-TOP, TOP).to(CODE).view(torch.uint8)
    scales[..., side][touched] = new


def _append(st):
    c, cs = st["case"], st["table"][st["pos"]]
    hq, hkv = c["hq"], c["hkv"]
    if c["norm"]:
        h = st["qkv"].float().view(-1, hq + 2 * hkv, DIM)
        q, k, v = _rms(h[:, :hq], st["qw"].float()), _rms(h[:, hq:hq + hkv], st["kw"].float()), h[:, hq + hkv:]
    else:
        q, k, v = st["q"].float(), st["k"].float(), st["v"].float()
    st["q"].copy_(_rope(q, cs))
    _put(st, st["kc"], 0, _rope(k, cs))
    _put(st, st["vc"], 1, v)


def _rows(st, codes, side, slots):
    x = codes.view(torch.uint8).view(-1, st["case"]["hkv"], DIM)[slots].view(CODE).float()
    return x * st["scales"][slots // PAGE][..., side, None]


def _load(st):
    st["k_out"].copy_(_rows(st, st["kc"], 0, st["read"]))
    st["v_out"].copy_(_rows(st, st["vc"], 1, st["read"]))


def _attention(st):
    c, at = st["case"], st["at"]
    hq, hkv = c["hq"], c["hkv"]
    b, t = at.shape
    n = st["row_at"].shape[1]
    k = _rows(st, st["kc"], 0, at.reshape(-1)).view(b, t, hkv, DIM).permute(0, 2, 3, 1).contiguous()
    v = _rows(st, st["vc"], 1, at.reshape(-1)).view(b, t, hkv, DIM).permute(0, 2, 1, 3).contiguous()
    q = st["q"][st["row_at"]].float().view(b, n, hkv, -1, DIM).permute(0, 2, 1, 3, 4).reshape(b, hkv, -1, DIM)
    s = torch.matmul(q, k).div_(math.sqrt(DIM)).view(b, hkv, n, -1, t)
    s.masked_fill_((torch.arange(t, device=s.device) > st["sees"][..., None])[:, None, :, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    p = s.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(b, hkv, -1, t), v).view(b, hkv, n, -1, DIM) / total
    lse = (top + total.log())[..., 0]
    st["out"].copy_(o.permute(0, 2, 1, 3, 4).reshape(b, n, hq, DIM)[st["have"]])
    st["lse"].copy_(lse.permute(0, 2, 1, 3).reshape(b, n, hq)[st["have"]])


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------

def _own_append(st, feattn):
    c = st["case"]
    if c["norm"]:
        feattn.norm_rope_append_kv8(st["qkv"], st["qkv"].shape[1], st["qw"], st["kw"], EPS, st["q"], st["kc"],
                                    st["vc"], st["scales"], st["pos"], st["slots"], st["table"], st["rows"], c["hq"],
                                    c["hkv"], st["bf16"], MAX_POS, st["cache_slots"])
    else:
        feattn.rope_append_kv8(st["q"], st["k"], st["v"], st["kc"], st["vc"], st["scales"], st["pos"], st["slots"],
                               st["table"], st["rows"], c["hq"], c["hkv"], DIM, st["bf16"], MAX_POS,
                               st["cache_slots"])


def run(st):
    kind = st["kind"]
    if own:
        feattn = _feattn()
        if kind in ("append", "step"):
            _own_append(st, feattn)
        if kind in ("append", "load"):
            feattn.load_kv8(st["kc"], st["vc"], st["scales"], st["read"], st["k_out"], st["v_out"], len(st["read"]),
                            st["case"]["hkv"], DIM, st["bf16"], st["cache_slots"])
        else:
            st["plan"].run_kv8(st["q"], st["kc"], st["vc"], st["scales"], st["out"], causal=st["case"]["causal"],
                               lse=st["lse"])
    else:
        if kind in ("append", "step"):
            _append(st)
        if kind in ("append", "load"):
            _load(st)
        else:
            _attention(st)
    return _outputs(st, st)


def _outputs(st, v):
    keys = {"append": ("q", "k_out", "v_out"), "load": ("k_out", "v_out"), "attention": ("out", "lse"),
            "step": ("q", "out", "lse")}[st["kind"]]
    return {k: v[k] for k in keys}


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------

def work(case):
    starts, rows = _lens(case)
    hq, hkv, kind = case["hq"], case["hkv"], case["kind"]
    new, token = sum(rows), hkv * 2 * DIM  # bytes of a token's codes
    nbytes = flops = 0
    if kind in ("append", "step"):
        # projections in, queries out, codes out, position, slot and angles;
        # the scale and, where a block holds earlier tokens, nothing else
        nbytes += new * ((2 * hq + 2 * hkv) * DIM * 2 + token + 16 + 4 * DIM)
        nbytes += sum(-(-(s % PAGE + n) // PAGE) for s, n in zip(starts, rows)) * hkv * 8
        flops += 10 * new * (hq + hkv) * DIM
    if kind in ("append", "load"):
        held = sum(s % PAGE + n for s, n in zip(starts, rows)) if kind == "append" else sum(starts) + new
        nbytes += held * (3 * token + 8)
        flops += held * token
    if kind in ("attention", "step"):
        cached = sum(s + n for s, n in zip(starts, rows))
        pages = sum(-(-(s + n) // PAGE) for s, n in zip(starts, rows))
        nbytes += cached * token + pages * (8 * hkv + 4) + new * hq * (2 * DIM * 2 + 4)
        pairs = sum(n * s + (n * (n + 1) // 2 if case["causal"] else n * n) for s, n in zip(starts, rows))
        flops += 4 * hq * DIM * pairs
    return {"bytes": nbytes, "flops": flops}


# ---------------------------------------------------------------------------
# The same results in 64 bits
# ---------------------------------------------------------------------------

def _turn64(x, pos, hold):
    """Rotation by the table's angles; `hold`: the table as it was given."""
    half = DIM // 2
    z = torch.complex(x[..., :half], x[..., half:])
    w = torch.complex(hold[pos][:, :half].double(), hold[pos][:, half:].double())
    y = z * w[:, None]
    return torch.cat([y.real, y.imag], -1)


def _exp2_64(e):
    return (e.long() + 1023 << 52).view(torch.float64)


def _power64(top):
    e = torch.frexp(top.clamp_min(2.0 ** -200) / TOP)[1].long()  # top / TOP in [2^(e - 1), 2^e)
    e = e - (top <= TOP * _exp2_64(e - 1)).long()
    return _exp2_64(e.clamp_min(-118))


def _e4m3_64(x):
    """x rounded to the nearest e4m3 value, ties to even."""
    step = _exp2_64(torch.frexp(x.abs().clamp_min(2.0 ** -6))[1] - 4)
    return torch.round(x / step) * step


def _append64(st):
    """The queries, and the values of the whole cache after the append."""
    c = st["case"]
    hq, hkv = c["hq"], c["hkv"]
    if c["norm"]:
        h = st["qkv"].double().view(-1, hq + 2 * hkv, DIM)
        unit = h / (h.pow(2).sum(-1, keepdim=True) / DIM + EPS).sqrt()
        q, k, v = unit[:, :hq] * st["qw"].double(), unit[:, hq:hq + hkv] * st["kw"].double(), h[:, hq + hkv:]
    else:
        q, k, v = st["q"].double(), st["k"].double(), st["v"].double()
    q, k = _turn64(q, st["pos"], st["table"]), _turn64(k, st["pos"], st["table"])
    blk, off = st["slots"] // PAGE, st["slots"] % PAGE
    caches = []
    for side, (codes, x) in enumerate(((st["kc"], k), (st["vc"], v))):
        scale = st["scales"][..., side].double()
        value = codes.double() * scale[:, None, :, None]
        top = torch.zeros_like(scale).scatter_reduce(0, blk[:, None].expand(-1, hkv), x.abs().amax(-1), "amax")
        grown = _power64(top)
        first = torch.zeros(len(scale), dtype=torch.bool, device=x.device)
        first[blk[off == 0]] = True
        hit = torch.zeros_like(first)
        hit[blk] = True
        grown = torch.where(first[:, None], grown, torch.maximum(grown, scale))
        value[blk, off] = x
        at = torch.nonzero(hit)[:, 0]
        value[at] = _e4m3_64(value[at] / grown[at][:, None, :, None]) * grown[at][:, None, :, None]
        caches.append(value.view(-1, hkv, DIM))
    return q, caches[0], caches[1]


def _attention64(st, q, k, v):
    c = st["case"]
    group = c["hq"] // c["hkv"]
    out = torch.empty(q.shape, dtype=torch.float64, device=q.device)
    lse = torch.empty(q.shape[:2], dtype=torch.float64, device=q.device)
    for i, (n, rows) in enumerate(zip(st["lens"], st["qlens"])):
        pages = st["perm"][st["kv"][i]:st["kv"][i + 1]]
        at = (pages[:, None] * PAGE + torch.arange(PAGE, device=q.device)).reshape(-1)[:n]
        for h in range(c["hkv"]):
            kh, vh = k(at, h), v(at, h)
            x = q[st["qo"][i]:st["qo"][i + 1], h * group:(h + 1) * group].double().reshape(-1, DIM)
            s = x @ kh.t() / DIM ** 0.5
            if c["causal"]:
                row = torch.arange(rows, device=q.device).repeat_interleave(group)[:, None]
                s = s.masked_fill(torch.arange(n, device=q.device) > n - rows + row, -math.inf)
            l = torch.logsumexp(s, -1, keepdim=True)
            o = torch.exp(s - l) @ vh
            out[st["qo"][i]:st["qo"][i + 1], h * group:(h + 1) * group] = o.view(rows, group, DIM)
            lse[st["qo"][i]:st["qo"][i + 1], h * group:(h + 1) * group] = l.view(rows, group)
    return out, lse


def exact(case, seed):
    st = prepare(case, seed)
    kind = case["kind"]
    res = {}
    if kind in ("append", "step"):
        res["q"], kc, vc = _append64(st)
    else:
        wide = lambda codes, side: lambda at, h: (codes.view(-1, case["hkv"], DIM)[:, h].double()[at]  # noqa: E731
                                                  * st["scales"][at // PAGE][:, h, side, None].double())
        k, v = wide(st["kc"], 0), wide(st["vc"], 1)
    if kind == "append":
        res["k_out"], res["v_out"] = kc[st["read"]], vc[st["read"]]
    elif kind == "load":
        heads = range(case["hkv"])
        res["k_out"] = torch.stack([k(st["read"], h) for h in heads], 1)
        res["v_out"] = torch.stack([v(st["read"], h) for h in heads], 1)
    else:
        if kind == "step":
            k, v = (lambda at, h: kc[at, h]), (lambda at, h: vc[at, h])
        # (queries as the layer holds them, in their 16-bit type)
        res["out"], res["lse"] = _attention64(st, res["q"].to(st["dtype"]) if kind == "step" else st["q"], k, v)
    return _outputs(st, res)
