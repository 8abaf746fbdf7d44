"""Pins oracle/kv8.py: e4m3 corner values, rounding, the append's scale rule by
hand, and its attention against the scalar-loop one."""

import math

import numpy as np
import pytest
import torch

from feattn import workloads as W
from oracle import brute, kv8


def test_corner_values():
    v = kv8.VALUES
    assert v[0] == 0 and v[1] == 2.0 ** -9 and v[8] == 2.0 ** -6 and v[0x38] == 1.0 and v[0x7e] == 448.0
    assert math.isnan(v[0x7f]) and math.isnan(v[0xff]) and v[0xfe] == -448.0
    want = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    assert torch.equal(v.nan_to_num(-1), want.nan_to_num(-1))


def test_rounding():
    x = torch.tensor([0.0, -0.0, 1.0625, 1.1875, 2.0 ** -10, 2.0 ** -10 * 1.001, 448.0, 464.0, 465.0, -300.0])
    assert kv8.encode(x).tolist() == [0, 0x80, 0x38, 0x3a, 0, 1, 0x7e, 0x7e, 0x7f, 0xf9]
    assert kv8.encode(torch.tensor([math.inf, -math.inf, math.nan])).tolist()[0] == 0x7f
    g = torch.Generator().manual_seed(1)
    x = torch.randn(20000, generator=g) * torch.exp2(torch.randint(-12, 8, (20000,), generator=g).float())
    x = x.clamp(-440, 440)
    assert torch.equal(kv8.encode(x), x.to(torch.float8_e4m3fn).view(torch.uint8))
    # every code comes back
    c = torch.arange(256, dtype=torch.uint8)
    keep = c % 128 != 127
    assert torch.equal(kv8.encode(kv8.decode(c))[keep], c[keep])


@pytest.mark.parametrize("amax,want", [(448.0, 1.0), (448.1, 2.0), (224.0, 0.5), (1.75, 2.0 ** -8), (1.8, 2.0 ** -7),
                                       (0.0, 2.0 ** -118), (2.0 ** -130, 2.0 ** -118)])
def test_need(amax, want):
    assert kv8.need(amax) == want


def test_append_by_hand():
    """Slots 16, 17 open block 1 with 1.75 (scale 2^-8: codes 448 and 256);
    slot 18 brings 7.0 (scale 2^-6), slot 19 a small value that keeps it."""
    codes = torch.full((48, 1, 128), 0x55, dtype=torch.uint8)
    scales = torch.full((3, 1, 2), 7.0)
    row = lambda v: torch.full((1, 1, 128), v, dtype=torch.float64)  # noqa: E731
    codes, scales = kv8.append(codes, scales, 0, torch.cat([row(1.75), row(1.0)]), torch.tensor([16, 17]),
                               torch.bfloat16)
    assert scales[1, 0, 0] == 2.0 ** -8 and scales[1, 0, 1] == 7.0 and scales[0, 0, 0] == 7.0
    assert (codes[16] == 0x7e).all() and kv8.decode(codes[17, 0, :1]) == 256
    codes, scales = kv8.append(codes, scales, 0, row(7.0), torch.tensor([18]), torch.bfloat16)
    assert scales[1, 0, 0] == 2.0 ** -6 and kv8.decode(codes[16, 0, :1]) == 112
    codes, scales = kv8.append(codes, scales, 0, torch.cat([row(0.01), row(9.0)]), torch.tensor([19, -1]),
                               torch.bfloat16)
    assert scales[1, 0, 0] == 2.0 ** -6
    got = kv8.load(codes, scales, 0, torch.tensor([16, 17, 18, 19]))[:, 0, 0]
    assert got[:3].tolist() == [1.75, 1.0, 7.0] and abs(got[3] - 0.01) <= 0.01 / 16
    assert (codes[:16] == 0x55).all() and (codes[32:] == 0x55).all()


def test_attention_against_scalar_loops():
    b = W.make_batch(4, 2, starts=[3, 0, 17], qlens=[2, 5, 1], seed=4)
    q, kc, vc = W.make_tensors(b, seed=4)
    for causal in (True, False):
        out, lse, size, score, total = kv8.attention(b, q, kc.double().view(-1, 2, 128), vc.double().view(-1, 2, 128), causal)
        want, want_lse = brute.attention(b.qo, b.kv, b.pages, b.last, b.batch, b.page, q.double().numpy(),
                                          kc.double().numpy(), vc.double().numpy(), 4, 2, causal)
        assert np.allclose(out.numpy(), want, atol=1e-12) and np.allclose(lse.numpy(), want_lse, atol=1e-12)
        assert (size >= out.abs() - 1e-12).all() and (score > 0).all() and (total >= size - 1e-12).all()
