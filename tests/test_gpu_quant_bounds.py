"""Attention over quantised rows within bounds that are close enough to show a lost tile, a wrong scale or a lost partial (the
CPU tests show what falls outside them), and at the ends of the numbers' range."""

from __future__ import annotations

import math

import pytest
import torch

from sparse_kv_reads_b200 import QuantAttentionGraph, QuantKVCache
from sparse_kv_reads_b200._lib import lib
from _caches import pack, quantise
from _helpers import DEV
from _quant_bounds import attention_bound

pytestmark = pytest.mark.gpu
SCALE = 1.0 / math.sqrt(128)


def normal_rows(B, H, L, seed, mean=0.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(B, H, L, 128, generator=g) + mean) * torch.randn(128, generator=g).abs()


def device_cache(codes, bits, lens=None):
    """``codes``: key codes, key scales, value codes, value scales; rows behind a sequence's length get NaN scales."""
    kc, ks, vc, vs = codes
    scale = torch.stack((ks, vs), -2).contiguous()
    for b, n in enumerate(lens or []):
        scale[b, :, n:] = float("nan")
    return QuantKVCache.from_tensors([pack(kc, bits).to(DEV)], [pack(vc, bits).to(DEV)], [scale.to(DEV)], bits)


def outside(got, q, codes, lens, bits, scale=SCALE):
    """Sequences and heads with a component outside the bound."""
    B, H = codes[0].shape[:2]
    q, got, bad = q.view(B, H, -1, 128), got.cpu().double().view(B, H, -1, 128), []
    for b, n in enumerate(lens):
        for h in range(H):
            out, bound = attention_bound(q[b, h], *(c[b, h, :n] for c in codes), bits, scale)
            if not bool(((got[b, h] - out).abs() <= bound).all()):
                bad.append((b, h, float(((got[b, h] - out).abs() / bound).max())))
    return bad


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("H,G,lens", [(3, 1, [1]), (3, 2, [16]), (3, 4, [33]), (3, 8, [300]), (2, 3, [1000]), (8, 2, [700]),
                                      (2, 4, [0, 1, 500, 333, 64, 0, 499]), (1, 8, [0] * 5 + [1] * 5 + [900]),
                                      (8, 2, [37 * b % 301 for b in range(40)])])
@pytest.mark.parametrize("ctas", [None, 1, 7, 64])
def test_attention_within_close_bounds(bits, H, G, lens, ctas):
    B, L = len(lens), max(lens)
    codes = (*quantise(normal_rows(B, H, L, L, 0.7), bits), *quantise(normal_rows(B, H, L, L + 1), bits))
    cache = device_cache(codes, bits, lens)
    q = (torch.randn(B * H * G, 128, generator=torch.Generator().manual_seed(4)) * 2).to(torch.bfloat16)
    attn = QuantAttentionGraph(H=B * H * G, H_kv=B * H, d=128, dtype=torch.bfloat16, device=DEV)
    attn.n_group = H
    if ctas is not None:
        attn.ctas = ctas
        attn.ws = torch.zeros(lib().skv_quant_workspace_bytes(B * H, G, 128, ctas), dtype=torch.uint8, device=DEV)
    n_dev = torch.tensor(lens, dtype=torch.int32, device=DEV)
    out = attn(q.to(DEV), cache, 0, n_dev).clone()
    assert torch.equal(attn(q.to(DEV), cache, 0, n_dev), out)
    assert outside(out, q, codes, lens, bits) == []


def random_codes(H, n, bits, seed, most=None):
    top = most or (127 if bits == 8 else 7)
    return torch.randint(-top, top + 1, (1, H, n, 128), generator=torch.Generator().manual_seed(seed))


def scales(H, n, bits, value):
    return torch.full((1, H, n, 1 if bits == 8 else 4), value, dtype=torch.float32).to(torch.bfloat16)


def run_alone(q, codes, bits, dtype=torch.bfloat16):
    """All rows of a cache of one sequence."""
    H, n = codes[0].shape[1:3]
    attn = QuantAttentionGraph(H=q.shape[0], H_kv=H, d=128, dtype=dtype, device=DEV)
    return attn(q.to(DEV).to(dtype), device_cache(codes, bits), 0, torch.tensor([n], dtype=torch.int32, device=DEV)).clone()


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("n", [40, 300])
def test_queries_up_to_the_largest_number(bits, n):
    """A few components in [2^127, 2^128), keys so small that the scores are ordinary."""
    H, G = 2, 3
    codes = (random_codes(H, n, bits, 1, 5), scales(H, n, bits, 2.0 ** -126), *quantise(normal_rows(1, H, n, 2), bits))
    g = torch.Generator().manual_seed(n)
    q = torch.randn(H * G, 128, generator=g) * 2.0 ** 110
    q[:, 5::31] = (1 + 0.99 * torch.rand(H * G, 4, generator=g)) * 2.0 ** 127
    assert outside(run_alone(q.to(torch.bfloat16), codes, bits), q.to(torch.bfloat16), codes, [n], bits) == []


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("size", [2.0 ** e for e in (-126, -122, -110, -60, -30, -20, 0, 60, 100, 116, 120, 122)])
def test_scores_of_queries_and_keys_at_opposite_ends(bits, size):
    """Ordinary scores from queries of one end of the numbers and keys of the other."""
    H, G, n = 2, 3, 300
    key = 2.0 ** (-4 if bits == 8 else -2) / size
    codes = (random_codes(H, n, bits, 3), scales(H, n, bits, key), *quantise(normal_rows(1, H, n, 4), bits))
    q = (torch.randn(H * G, 128, generator=torch.Generator().manual_seed(5)) * size).to(torch.bfloat16)
    assert outside(run_alone(q, codes, bits), q, codes, [n], bits) == []


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("size", [2.0 ** 60, 2.0 ** 116, 2.0 ** 120, 2.0 ** 127])
def test_scores_far_beyond_ordinary_ones(bits, dtype, sign, size):
    """Finite scores of up to 2^126, all positive or all negative: the largest one takes all."""
    H, G, n = 2, 2, 200
    kc = torch.zeros(1, H, n, 128, dtype=torch.int64)
    top = 120 if bits == 8 else 6
    kc[..., 7] = torch.tensor([top if sign > 0 else -top] * n)
    best = [3, 177]
    for h, j in enumerate(best):                           # one step above the others
        kc[0, h, j, 7] += 1
    key = 2.0 ** 50 if size < 2.0 ** 100 else 2.0 ** -7 if bits == 8 else 2.0 ** -3
    codes = (kc, scales(H, n, bits, key), *quantise(normal_rows(1, H, n, 6), bits))
    q = torch.zeros(H * G, 128)
    q[:, 7] = size
    got = run_alone(q, codes, bits, dtype).cpu().double().view(H, G, 128)
    value = codes[2].double() * codes[3].double().repeat_interleave(128 if bits == 8 else 32, -1)
    for h, j in enumerate(best):
        assert torch.equal(got[h], value[0, h, j].to(dtype).double().expand(G, -1)), h


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n", [20, 300, 3000])
def test_a_key_without_a_number_leaves_no_number_and_a_value_its_own_group(bits, dtype, n):
    """NaN scales among the rows: of a key, and the head has no answer; of a value, and its components have none."""
    H, G, size = 4, 2, 128 if bits == 8 else 32
    kc, ks, vc, vs = (*quantise(normal_rows(1, H, n, 7, 0.7), bits), *quantise(normal_rows(1, H, n, 8), bits))
    ks[0, 1, n // 2, -1] = vs[0, 3, n - 1, 0] = float("nan")
    q = (torch.randn(H * G, 128, generator=torch.Generator().manual_seed(1)) * 2).to(torch.bfloat16)
    got = run_alone(q, (kc, ks, vc, vs), bits, dtype).view(H, G, 128).isnan()
    assert bool(got[1].all()) and not bool(got[0].any()) and not bool(got[2].any())
    assert bool(got[3, :, :size].all()) and not bool(got[3, :, size:].any())


@pytest.mark.parametrize("apart", [0, 6, 12, 16, 20, 24, 40, 100])
@pytest.mark.parametrize("n", [16, 300, 1000])
def test_value_groups_of_very_different_sizes(apart, n):
    """The four value scales of a 4-bit row lie far apart, and not in the same order in every row or head."""
    H, G = 3, 3
    kc, ks, vc, vs = (*quantise(normal_rows(1, H, n, 7, 0.7), 4), *quantise(normal_rows(1, H, n, 8), 4))
    down = torch.zeros(1, H, n, 4)
    down[:, 0, :, 1:] = torch.tensor([apart / 3, apart * 2 / 3, apart])                 # the same order everywhere
    down[:, 1, :, 2] = apart                                                            # one small group
    g = torch.Generator().manual_seed(n)
    down[:, 2] = torch.randint(0, 2, (n, 4), generator=g) * apart                       # by row
    vs = (vs.float() * torch.exp2(-down.round())).to(torch.bfloat16)
    codes = (kc, ks, vc, vs)
    q = (torch.randn(H * G, 128, generator=g) * 2).to(torch.bfloat16)
    assert outside(run_alone(q, codes, 4), q, codes, [n], 4) == []


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("size", [2.0 ** -128, 2.0 ** -130])
def test_queries_below_the_normal_numbers(bits, size):
    """Every bf16 number down to 2^-133 counts, with keys so large that the scores are ordinary."""
    H, G, n = 2, 3, 300
    codes = (random_codes(H, n, bits, 3), scales(H, n, bits, 2.0 ** (122 if bits == 8 else 127)), *quantise(normal_rows(1, H, n, 4), bits))
    q = (torch.randn(H * G, 128, generator=torch.Generator().manual_seed(5)) * size).to(torch.bfloat16)
    assert outside(run_alone(q, codes, bits), q, codes, [n], bits) == []


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("H,G,lens,ctas", [(8, 2, [300], None), (8, 2, [20000], None), (4, 4, [3000, 17, 0, 9000, 128], None),
                                           (2, 8, [37 * b % 301 + 1 for b in range(80)], None), (1, 1, [6000, 1, 500], 7)])
def test_every_tile_and_partial_counts(bits, H, G, lens, ctas):
    """Values that are one in a component of their own for each 1/128 of the rows, weights all alike: an output component is
    the share of its rows, so that one that is lost or counted twice shows."""
    B, L = len(lens), max(lens)
    g = torch.Generator().manual_seed(L)
    v = torch.zeros(B, H, L, 128)
    for b, n in enumerate(lens):
        v[b, :, :n] = torch.eye(128)[torch.arange(n) * 128 // max(n, 1)]
    codes = (*quantise(torch.randn(B, H, L, 128, generator=g), bits), *quantise(v, bits))
    q = (torch.randn(B * H * G, 128, generator=g) * 0.05).to(torch.bfloat16)
    attn = QuantAttentionGraph(H=B * H * G, H_kv=B * H, d=128, dtype=torch.bfloat16, device=DEV)
    attn.n_group = H
    if ctas is not None:
        attn.ctas = ctas
        attn.ws = torch.zeros(lib().skv_quant_workspace_bytes(B * H, G, 128, ctas), dtype=torch.uint8, device=DEV)
    out = attn(q.to(DEV), device_cache(codes, bits, lens), 0, torch.tensor(lens, dtype=torch.int32, device=DEV))
    assert outside(out, q, codes, lens, bits) == []
