"""The quantised KV cache on the GPU against its definition in 64 bits: rows as they are written and read back, the
attention over them, and the decode step that uses both."""

from __future__ import annotations

import math

import pytest
import torch

from sparse_kv_reads_b200 import GraphDecoder, QuantAttentionGraph, QuantKVCache, Qwen3Config, Qwen3Model
from sparse_kv_reads_b200._lib import SkvError, check, lib
from _caches import attention, output_bound, pack, quantise, restore
from _helpers import DEV

pytestmark = pytest.mark.gpu
SCALE = 1.0 / math.sqrt(128)


def rows_of(B, H, T, dtype, seed, spread=True):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(B, H, T, 128, generator=g)
    if spread:                                             # channels of very different sizes, rows too
        x = x * torch.randn(128, generator=g).exp() * (torch.randn(B, H, T, 1, generator=g) * 3).exp()
    return x.to(dtype)


def same(a, b):
    return torch.equal(a.cpu().float().nan_to_num(nan=12345.0), b.cpu().float().nan_to_num(nan=12345.0))


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("B,H,T,at", [(1, 1, 1, 0), (2, 3, 17, 5), (3, 8, 1, 62), (1, 2, 63, 1), (1, 5, 300, 0)])
def test_rows_are_stored_and_read_back_by_their_definition(bits, dtype, B, H, T, at):
    k, v = rows_of(B, H, T, dtype, 1), rows_of(B, H, T, dtype, 2)
    k[0, 0, 0] = 0.0                                       # a row of zeros
    v[-1, -1, -1, 40] = 1e-3 if T > 1 else v[-1, -1, -1, 40]
    cache = QuantKVCache(2, B, H, 320, 128, bits, DEV)
    untouched = [t.clone() for t in (cache.k[0], cache.v[0], cache.scale[0])]
    # as a projection leaves them: [B, T, H, 128] seen per head
    kd = k.to(DEV).transpose(1, 2).contiguous().transpose(1, 2)
    cache.write(1, kd, v.to(DEV), at)
    for x, codes, which in ((k, cache.k[1], 0), (v, cache.v[1], 1)):
        code, scale = quantise(x, bits)
        assert torch.equal(codes[:, :, at:at + T].cpu(), pack(code, bits))
        assert torch.equal(cache.scale[1][:, :, at:at + T, which].cpu(), scale)
        # the nearest code: within half a scale, but for the quotient's own rounding (2^-24 of at most 127.5)
        value = restore(code, scale, bits)
        step = scale.to(torch.float64).repeat_interleave(128 if bits == 8 else 32, -1)
        assert bool(((x.double() - value).abs() <= step * (0.5 + 127.5 * 2.0 ** -24)).all())
        got = cache.read(1, at, T, dtype=dtype)[which]
        assert torch.equal(got.cpu(), value.to(dtype))     # 15 significant bits: float32 holds them all
    # nothing else was written
    assert int(cache.k[1][:, :, :at].sum()) == 0 and int(cache.k[1][:, :, at + T:].sum()) == 0
    assert int(cache.scale[1][:, :, at + T:].float().abs().sum()) == 0
    assert all(torch.equal(a, b) for a, b in zip(untouched, (cache.k[0], cache.v[0], cache.scale[0])))
    assert cache.check_status() == 0


@pytest.mark.parametrize("bits", [8, 4])
def test_extreme_rows(bits):
    """Inf and NaN spoil their scale group alone; the largest and the smallest numbers keep the definition."""
    x = rows_of(1, 1, 9, torch.bfloat16, 5, spread=False)
    x[0, 0, 0, 3] = float("nan")
    x[0, 0, 1, 77] = float("-inf")
    x[0, 0, 2] = torch.finfo(torch.bfloat16).max
    x[0, 0, 3] = -torch.finfo(torch.bfloat16).max
    x[0, 0, 4] *= 1e-37                                    # 3e-37 / 127 lies below the normal numbers (1.2e-38), / 7 not
    x[0, 0, 5] *= 1e-30
    x[0, 0, 6, :] = 0.0
    x[0, 0, 6, 5] = 2.0 ** -120
    x[0, 0, 7] = torch.arange(128) * 0.5                   # half-way quotients
    cache = QuantKVCache(1, 1, 1, 16, 128, bits, DEV)
    cache.write(0, x.to(DEV), x.to(DEV), 0)
    code, scale = quantise(x, bits)
    assert same(cache.scale[0][:, :, :9, 0], scale) and same(cache.scale[0][:, :, :9, 1], scale)
    finite = torch.isfinite(scale.float()).repeat_interleave(128 if bits == 8 else 32, -1)
    got = cache.read(0, 0, 9, dtype=torch.float32)[0].cpu()
    assert torch.equal(torch.isfinite(got), finite)
    assert torch.equal(got[finite], restore(code, scale, bits).float()[finite])
    assert bool((got[0, 0, 4] == 0).all()) == (bits == 8) and not bool((got[0, 0, 5] == 0).all())


@pytest.mark.parametrize("bits", [8, 4])
def test_positions_in_device_memory_one_per_sequence_and_outside_the_cache(bits):
    B, H, T, L = 4, 2, 6, 40
    k, v = rows_of(B, H, T, torch.bfloat16, 7), rows_of(B, H, T, torch.bfloat16, 8)
    cache = QuantKVCache(1, B, H, L, 128, bits, DEV)
    at = [0, 37, -2, 21]                                   # 37: three rows do not fit; -2: none is written
    pos = torch.tensor(at, device=DEV)
    cache.write(0, k.to(DEV), v.to(DEV), pos)
    rk, rv = cache.read(0, pos, T)
    ck, sk = quantise(k, bits)
    want = restore(ck, sk, bits).to(torch.bfloat16)
    want[1, :, 3:] = 0
    want[2] = 0
    assert torch.equal(rk.cpu(), want)
    assert cache.status.cpu().view(B, H)[:, 0].tolist() == [0, 4, 4, 0] and cache.check_status() == 4
    assert int(cache.k[0][2].sum()) == 0
    # the same position for all, from a one-element tensor; the first two sequences only
    cache.status.zero_()
    cache.write(0, k[:2].to(DEV), v[:2].to(DEV), torch.tensor([10], device=DEV))
    assert torch.equal(cache.read(0, 10, T, batch=2)[0].cpu(), restore(ck, sk, bits).to(torch.bfloat16)[:2])
    assert int(cache.k[0][3, :, 10:16].sum()) == 0 and cache.check_status() == 0


def test_a_sequence_of_the_cache_and_foreign_strides():
    cache = QuantKVCache(1, 3, 2, 32, 128, 4, DEV)
    wide = rows_of(1, 2, 8, torch.bfloat16, 3).to(DEV).repeat(1, 1, 1, 3)[..., 64:192]        # rows 768 bytes apart
    odd = torch.zeros(1, 2, 8, 132, dtype=torch.bfloat16, device=DEV)[..., 1:129].copy_(wide)  # not 16-byte aligned
    cache.sequence(1).write(0, wide, odd, 4)
    k, v = cache.read(0, 4, 8)
    code, scale = quantise(wide.cpu(), 4)
    want = restore(code, scale, 4).to(torch.bfloat16)[0]
    assert torch.equal(k[1].cpu(), want) and torch.equal(v[1].cpu(), want) and int(cache.k[0][0].sum()) == 0


def random_cache(B, H, L, bits, seed, lens=None):
    """A cache of quantised normal rows (host codes kept); rows behind a sequence's length hold NaN scales."""
    g = torch.Generator().manual_seed(seed)
    k = (torch.randn(B, H, L, 128, generator=g) + 0.7) * torch.randn(128, generator=g).abs()
    v = torch.randn(B, H, L, 128, generator=g)
    (ck, sk), (cv, sv) = quantise(k, bits), quantise(v, bits)
    scale = torch.stack((sk, sv), -2)
    for b, n in enumerate(lens or []):
        scale[b, :, max(0, n):] = float("nan")
    cache = QuantKVCache.from_tensors([pack(ck, bits).to(DEV)], [pack(cv, bits).to(DEV)], [scale.contiguous().to(DEV)], bits)
    return cache, restore(ck, sk, bits), restore(cv, sv, bits)


def score_error(q, k, bits):
    """Error of a base-e score of the tensor-core path: codes enter the products with an offset (1,024 to 1,152 for half
    floats) that the accumulators start without; a partial sum is at most that times the sum of the queries' magnitudes
    and is rounded (or cut) 16 times to 2^-22 of its size.  The key's scale and the softmax scale apply to all of it."""
    top = 7 if bits == 4 else 127
    step = k.abs().amax(-1) / top                          # at least the key's scale
    return float((step.max() * q.double().abs().sum(-1).max()) * 1152 * 16 * 2.0 ** -22 * SCALE)


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("G", [1, 2, 3, 4, 7, 8])
@pytest.mark.parametrize("n", [0, 1, 15, 16, 17, 31, 33, 63, 64, 65, 300, 1000])
def test_attention_over_quantised_rows(bits, G, n):
    H, L = 3, max(n, 1) + 5
    cache, k, v = random_cache(1, H, L, bits, 11 + n, [n])
    q = (torch.randn(H * G, 128, generator=torch.Generator().manual_seed(n)) * 2).to(torch.bfloat16)
    for dtype in (torch.bfloat16, torch.float32):
        attn = QuantAttentionGraph(H=H * G, H_kv=H, d=128, dtype=dtype, device=DEV)
        got = attn(q.to(DEV).to(dtype), cache, 0, torch.tensor([n], dtype=torch.int32, device=DEV)).cpu().double()
        for h in range(H):
            ref, mag = attention(q[h * G:(h + 1) * G], k[0, h, :n], v[0, h, :n], SCALE)
            e = score_error(q[h * G:(h + 1) * G], k[0, h, :n], bits) if n and dtype == torch.bfloat16 else 2.0 ** -16
            assert bool(((got[h * G:(h + 1) * G] - ref).abs() <= output_bound(ref, mag, dtype, e)).all()), (dtype, h)


@pytest.mark.parametrize("bits", [8, 4])
def test_a_ragged_batch_with_empty_sequences_and_lengths_beyond_the_cache(bits):
    B, H, G, L = 7, 2, 4, 700
    lens = [0, 1, 700, 333, 64, 0, 699]
    cache, k, v = random_cache(B, H, L, bits, 3, lens)
    q = (torch.randn(B * H * G, 128, generator=torch.Generator().manual_seed(4)) * 2).to(torch.bfloat16)
    attn = QuantAttentionGraph(H=B * H * G, H_kv=B * H, d=128, dtype=torch.bfloat16, device=DEV)
    attn.n_group = H
    said = list(lens)
    said[2], said[5] = 90000, -3                           # counts as the capacity, and as nothing
    n_dev = torch.tensor(said, dtype=torch.int32, device=DEV)
    out = attn(q.to(DEV), cache, 0, n_dev).clone()
    got = out.cpu().double().view(B, H, G, 128)
    for b, n in enumerate(lens):
        for h in range(H):
            qh = q.view(B, H, G, 128)[b, h]
            ref, mag = attention(qh, k[b, h, :n], v[b, h, :n], SCALE)
            e = score_error(qh, k[b, h, :n], bits) if n else 0.0
            assert bool(((got[b, h] - ref).abs() <= output_bound(ref, mag, torch.bfloat16, e)).all()), (b, h)
    assert bool((got[0] == 0).all()) and bool((got[5] == 0).all())
    assert torch.equal(attn(q.to(DEV), cache, 0, n_dev), out)                    # the same bits every time


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("H,G,lens", [(8, 2, [37 * b % 301 for b in range(90)]),           # more heads than CTAs, several a CTA
                                      (1, 8, [0] * 20 + [1] * 20 + [2000]), (1, 3, [6000, 1, 500]), (5, 1, [3000] * 4)])
@pytest.mark.parametrize("ctas", [None, 1, 7, 64])
def test_every_way_of_sharing_rows_out(bits, H, G, lens, ctas):
    """Many short heads, one long among them, few CTAs: runs that meet several heads and heads that meet several runs."""
    B = len(lens)
    cache, k, v = random_cache(B, H, max(lens), bits, B + H, lens)
    q = (torch.randn(B * H * G, 128, generator=torch.Generator().manual_seed(B)) * 2).to(torch.bfloat16)
    attn = QuantAttentionGraph(H=B * H * G, H_kv=B * H, d=128, dtype=torch.bfloat16, device=DEV)
    attn.n_group = H
    if ctas is not None:
        attn.ctas = ctas
        attn.ws = torch.zeros(lib().skv_quant_workspace_bytes(B * H, G, 128, ctas), dtype=torch.uint8, device=DEV)
    n_dev = torch.tensor(lens, dtype=torch.int32, device=DEV)
    out = attn(q.to(DEV), cache, 0, n_dev).clone()
    assert torch.equal(attn(q.to(DEV), cache, 0, n_dev), out)
    got = out.cpu().double().view(B, H, G, 128)
    for b, n in enumerate(lens):
        for h in range(H):
            qh = q.view(B, H, G, 128)[b, h]
            ref, mag = attention(qh, k[b, h, :n], v[b, h, :n], SCALE)
            e = score_error(qh, k[b, h, :n], bits) if n else 0.0
            assert bool(((got[b, h] - ref).abs() <= output_bound(ref, mag, torch.bfloat16, e)).all()), (b, h)


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("per_head", [False, True])
@pytest.mark.parametrize("ctas", [None, 5, 33])
def test_more_lengths_than_a_warp_has_lanes(bits, per_head, ctas):
    """A length per sequence or per head, more of them than 32, empty ones at both ends and in rows among them."""
    H, G = 2, 3
    lens = [0, 0] + [(37 * i) % 211 for i in range(40)] + [900, 0, 0, 0, 1, 640, 0]
    B = len(lens)
    cache, k, v = random_cache(B, H, max(lens), bits, 71, lens)
    q = (torch.randn(B * H * G, 128, generator=torch.Generator().manual_seed(6)) * 2).to(torch.bfloat16)
    attn = QuantAttentionGraph(H=B * H * G, H_kv=B * H, d=128, dtype=torch.bfloat16, device=DEV)
    attn.n_group = 1 if per_head else H
    if ctas is not None:
        attn.ctas = ctas
        attn.ws = torch.zeros(lib().skv_quant_workspace_bytes(B * H, G, 128, ctas), dtype=torch.uint8, device=DEV)
    each = [[max(n - 3 * h, 0) if per_head else n for h in range(H)] for n in lens]
    n_dev = torch.tensor([n for row in each for n in row] if per_head else lens, dtype=torch.int32, device=DEV)
    out = attn(q.to(DEV), cache, 0, n_dev).clone()
    assert torch.equal(attn(q.to(DEV), cache, 0, n_dev), out)
    got = out.cpu().double().view(B, H, G, 128)
    for b in range(B):
        for h in range(H):
            n, qh = each[b][h], q.view(B, H, G, 128)[b, h]
            ref, mag = attention(qh, k[b, h, :n], v[b, h, :n], SCALE)
            e = score_error(qh, k[b, h, :n], bits) if n else 0.0
            assert bool(((got[b, h] - ref).abs() <= output_bound(ref, mag, torch.bfloat16, e)).all()), (b, h)


def test_queries_that_alias_the_output_and_a_negative_softmax_scale():
    H, G, n = 2, 4, 300
    cache, k, v = random_cache(1, H, n, 8, 41)
    attn = QuantAttentionGraph(H=H * G, H_kv=H, d=128, dtype=torch.bfloat16, device=DEV)
    n_dev = torch.tensor([n], dtype=torch.int32, device=DEV)
    q = torch.randn(H * G, 128, generator=torch.Generator().manual_seed(5)).to(torch.bfloat16).to(DEV)
    want = attn(q, cache, 0, n_dev).clone()
    attn.out.copy_(q)
    assert torch.equal(attn(attn.out, cache, 0, n_dev), want)
    wide = torch.zeros(H * G, 129, dtype=torch.bfloat16, device=DEV)[:, 1:].copy_(q)         # strided and off the boundary
    assert torch.equal(attn(wide, cache, 0, n_dev), want)
    attn._scale = -attn._scale
    assert torch.equal(attn(-q, cache, 0, n_dev), want)


@pytest.mark.parametrize("bits", [8, 4])
def test_large_and_small_queries_keep_their_scores(bits):
    """Queries and keys far from 1: the queries' own scale must not matter."""
    H, G, n = 2, 2, 200
    cache, k, v = random_cache(1, H, n, bits, 21)
    attn = QuantAttentionGraph(H=H * G, H_kv=H, d=128, dtype=torch.bfloat16, device=DEV)
    n_dev = torch.tensor([n], dtype=torch.int32, device=DEV)
    base = torch.randn(H * G, 128, generator=torch.Generator().manual_seed(5))
    for size in (2.0 ** 40, 2.0 ** -40):
        q = (base * size).to(torch.bfloat16)
        small = QuantKVCache.from_tensors(cache.k, cache.v, [cache.scale[0].clone()], bits)
        small.scale[0][..., 0, :] *= 2.0 ** -40 if size > 1 else 2.0 ** 40
        got = attn(q.to(DEV), small, 0, n_dev).cpu().double()
        for h in range(H):
            qh = q[h * G:(h + 1) * G].double() / size
            ref, mag = attention(qh, k[0, h], v[0, h], SCALE)
            e = score_error(qh, k[0, h], bits)
            assert bool(((got[h * G:(h + 1) * G] - ref).abs() <= output_bound(ref, mag, torch.bfloat16, e)).all())
    zero = torch.zeros(H * G, 128, dtype=torch.bfloat16, device=DEV)             # every row alike: the values' mean
    got = attn(zero, cache, 0, n_dev).cpu().double()
    for h in range(H):
        ref, mag = attention(zero[:G].cpu(), k[0, h], v[0, h], SCALE)
        assert bool(((got[h * G:(h + 1) * G] - ref).abs() <= output_bound(ref, mag, torch.bfloat16)).all())


@pytest.mark.parametrize("bits", [8, 4])
def test_one_value_scale_far_above_the_others(bits):
    """Values of very different sizes: the largest may come first, last or in between."""
    H, G, n = 1, 2, 400
    cache, k, v = random_cache(1, H, n, bits, 31)
    q = torch.randn(G, 128, generator=torch.Generator().manual_seed(6)).to(torch.bfloat16)
    attn = QuantAttentionGraph(H=G, H_kv=H, d=128, dtype=torch.bfloat16, device=DEV)
    n_dev = torch.tensor([n], dtype=torch.int32, device=DEV)
    for at in (0, 137, n - 1):
        c = QuantKVCache.from_tensors(cache.k, cache.v, [cache.scale[0].clone()], bits)
        c.scale[0][:, :, at, 1] *= 2.0 ** 20
        vv = v.clone()
        vv[:, :, at] *= 2.0 ** 20
        ref, mag = attention(q, k[0, 0], vv[0, 0], SCALE)
        got = attn(q.to(DEV), c, 0, n_dev).cpu().double()
        e = score_error(q, k[0, 0], bits)
        assert bool(((got - ref).abs() <= output_bound(ref, mag, torch.bfloat16, e)).all())
    c = QuantKVCache.from_tensors(cache.k, cache.v, [cache.scale[0].clone()], bits)
    c.scale[0][:, :, :, 1] = 0                             # all values zero
    assert bool((attn(q.to(DEV), c, 0, n_dev) == 0).all())


def test_offsets_beyond_31_bits():
    """A head whose rows begin more than 2^31 bytes into the codes, and a row more than 2^31 bytes into its head."""
    L = 2_400_000
    cache = QuantKVCache(1, 1, 8, L, 128, 8, DEV)
    assert 7 * L * 128 > 2 ** 31 - 1
    k, v = rows_of(1, 8, 5, torch.bfloat16, 1, False), rows_of(1, 8, 5, torch.bfloat16, 2, False)
    cache.write(0, k.to(DEV), v.to(DEV), 2)
    code, scale = quantise(k, 8)
    assert torch.equal(cache.read(0, 2, 5)[0].cpu(), restore(code, scale, 8).to(torch.bfloat16))
    cache.write(0, k.to(DEV), v.to(DEV), 0)
    q = (torch.randn(16, 128, generator=torch.Generator().manual_seed(3)) * 2).to(torch.bfloat16)
    attn = QuantAttentionGraph(H=16, H_kv=8, d=128, dtype=torch.bfloat16, device=DEV)
    got = attn(q.to(DEV), cache, 0, torch.tensor([5], dtype=torch.int32, device=DEV)).cpu().double()
    vc, vs = quantise(v, 8)
    kk, vv = restore(code, scale, 8), restore(vc, vs, 8)
    for h in range(8):
        ref, mag = attention(q[2 * h:2 * h + 2], kk[0, h], vv[0, h], SCALE)
        e = score_error(q[2 * h:2 * h + 2], kk[0, h], 8)
        assert bool(((got[2 * h:2 * h + 2] - ref).abs() <= output_bound(ref, mag, torch.bfloat16, e)).all())
    del cache, attn
    torch.cuda.empty_cache()
    n = 17_000_000
    long = QuantKVCache(1, 1, 1, n, 128, 8, DEV)           # unwritten rows: keys and values of zero
    assert (n - 4) * 128 > 2 ** 31
    big = torch.full((1, 1, 4, 128), 2.0, dtype=torch.bfloat16, device=DEV)
    val = torch.full((1, 1, 4, 128), 8.0, dtype=torch.bfloat16, device=DEV)
    long.write(0, big, val, n - 4)
    attn = QuantAttentionGraph(H=1, H_kv=1, d=128, dtype=torch.bfloat16, device=DEV)
    qq = torch.full((1, 128), 0.75, dtype=torch.bfloat16, device=DEV)
    got = attn(qq, long, 0, torch.tensor([n], dtype=torch.int32, device=DEV)).cpu().double()
    kq, ks = quantise(big.cpu(), 8)
    vq, vs = quantise(val.cpu(), 8)
    weight = 4 * math.exp(float((restore(kq, ks, 8)[0, 0, 0] * 0.75).sum()) * SCALE)     # the others: exp(0) each
    ref = restore(vq, vs, 8)[0, 0, :1] * weight / (weight + n - 4)
    e = score_error(qq.cpu(), restore(kq, ks, 8)[0, 0], 8)
    # (17 million weights of one are summed by thousands of partial sums: 2^-16 of them at most is lost)
    assert bool(((got - ref).abs() <= output_bound(ref, ref.abs(), torch.bfloat16, e + 2.0 ** -16)).all())


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("per_seq", [False, True])
def test_the_decode_steps_write_equals_the_rotary_launch_and_a_write(bits, per_seq):
    B, H, Hk, L = 3, 8, 4, 64
    g = torch.Generator().manual_seed(9)
    qkv = torch.randn(B, (H + 2 * Hk) * 128, generator=g).to(torch.bfloat16).to(DEV)
    qw, kw = (torch.randn(128, generator=g).to(torch.bfloat16).to(DEV) for _ in range(2))
    ang = torch.rand(L, 128, generator=g) * 6
    cos, sin = ang.cos().to(torch.bfloat16).to(DEV), ang.sin().to(torch.bfloat16).to(DEV)
    pos = torch.tensor([5, 63, 31] if per_seq else [63], device=DEV)
    st = torch.cuda.current_stream().cuda_stream
    kc, vc = (torch.zeros(B, Hk, L, 128, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    q1, q2 = (torch.zeros(B * H, 128, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    check(lib().skv_qk_rope_cache(qkv.data_ptr(), qw.data_ptr(), kw.data_ptr(), cos.data_ptr(), sin.data_ptr(),
                                  pos.data_ptr(), int(per_seq), q1.data_ptr(), kc.data_ptr(), vc.data_ptr(), B, H, Hk, 128,
                                  kc.stride(0), kc.stride(1), kc.stride(2), 1e-6, st), "skv_qk_rope_cache")
    one, two = QuantKVCache(1, B, Hk, L, 128, bits, DEV), QuantKVCache(1, B, Hk, L, 128, bits, DEV)
    check(lib().skv_qk_rope_quant(one._st[0], qkv.data_ptr(), qw.data_ptr(), kw.data_ptr(), cos.data_ptr(), sin.data_ptr(),
                                  pos.data_ptr(), int(per_seq), q2.data_ptr(), B, H, 1e-6, st), "skv_qk_rope_quant")
    at = pos.tolist() if per_seq else pos.tolist() * B
    new = [torch.stack([c[b, :, p:p + 1] for b, p in enumerate(at)]) for c in (kc, vc)]
    two.write(0, new[0], new[1], pos)
    assert torch.equal(q1, q2)
    assert torch.equal(one.k[0], two.k[0]) and torch.equal(one.v[0], two.v[0]) and torch.equal(one.scale[0], two.scale[0])
    # a position outside the cache: recorded, nothing written for that sequence
    bad = torch.tensor([5, 64, 31], device=DEV)
    before = one.k[0].clone()
    check(lib().skv_qk_rope_quant(one._st[0], qkv.data_ptr(), qw.data_ptr(), kw.data_ptr(), cos.data_ptr(), sin.data_ptr(),
                                  bad.data_ptr(), 1, q2.data_ptr(), B, H, 1e-6, st), "skv_qk_rope_quant")
    assert torch.equal(one.k[0][1], before[1]) and one.status.view(B, Hk).cpu()[:, 0].tolist() == [0, 4, 0]


def test_a_captured_call_replays_with_new_lengths_on_another_stream():
    B, H, G, L = 2, 2, 2, 500
    cache, k, v = random_cache(B, H, L, 4, 17)
    attn = QuantAttentionGraph(H=B * H * G, H_kv=B * H, d=128, dtype=torch.bfloat16, device=DEV)
    attn.n_group = H
    new = rows_of(B, H, 1, torch.bfloat16, 6, False).to(DEV)
    q = (torch.randn(B * H * G, 128, generator=torch.Generator().manual_seed(8)) * 2).to(torch.bfloat16).to(DEV)
    pos = torch.tensor([10, 20], device=DEV)
    n_dev = torch.tensor([11, 21], dtype=torch.int32, device=DEV)

    def both():
        cache.write(0, new, new, pos)
        return attn(q, cache, 0, n_dev), cache.read(0, pos, 1)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, back = both()
    for at in ([30, 40], [499, 0]):
        pos.copy_(torch.tensor(at))
        n_dev.copy_(torch.tensor([a + 1 for a in at], dtype=torch.int32))
        new.mul_(-1.5)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            graph.replay()
        side.synchronize()
        got, rows = out.clone(), back.clone()
        want, want_rows = both()
        assert torch.equal(got, want) and torch.equal(rows, want_rows)
    assert cache.check_status() == 0


TINY = dict(hidden_size=256, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2, head_dim=128,
            intermediate_size=512, vocab_size=1000, max_position_embeddings=2048)


def tiny_model(dtype=torch.bfloat16, seed=3):
    with torch.device(DEV):
        m = Qwen3Model(Qwen3Config(**TINY))
    return m.to(dtype).eval().init_random(seed=seed, std=0.05)


def decode(model, ids, cache, P, T, capture, **kw):
    out = []
    with torch.no_grad():
        model.prefill(ids[:, :P], cache, chunk=128)
        dec = GraphDecoder(model, cache, mode="dense", **kw)
        dec.prepare(P)
        if capture:
            dec.capture()
        for t in range(P, P + T):
            out.append(dec.step(ids[:, t:t + 1], t)[:, -1].float().clone())
    return torch.stack(out, 1)


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("batch", [1, 3, 9])
def test_decoding_with_a_quantised_cache(bits, batch):
    """Prefill in chunks, decode through the graph: the graph equals the eager step bit for bit, and the model's own
    forward over the same quantised cache (rows read back, library attention) to the tolerance of its bf16 layers."""
    model, P, T = tiny_model(), 200, 12
    ids = torch.randint(0, 1000, (batch, P + T), generator=torch.Generator().manual_seed(1)).to(DEV)
    graph = decode(model, ids, model.alloc_cache(P + T, batch, bits=bits), P, T, True)
    eager = decode(model, ids, model.alloc_cache(P + T, batch, bits=bits), P, T, False)
    assert torch.equal(graph, eager)
    with torch.no_grad():
        cache = model.alloc_cache(P + T, batch, bits=bits)
        model.prefill(ids[:, :P], cache, chunk=77)
        own = torch.stack([model(ids[:, t:t + 1], cache, start_pos=t)[:, -1].float() for t in range(P, P + T)], 1)
    assert cache.check_status() == 0
    # the fused step rounds between its launches like the modules do; 4-bit codes of a key that differs in its last bf16
    # bit can differ by one step, 1/14 of the group's largest value, in a few rows of 200
    torch.testing.assert_close(own, graph, rtol=5e-2, atol=5e-2 if bits == 8 else 2e-1)


def test_a_ragged_quantised_batch_equals_separate_sequences():
    model, T = tiny_model(), 6
    lens = [130, 77, 9]
    g = torch.Generator().manual_seed(2)
    prompts = [torch.randint(0, 1000, (n,), generator=g).to(DEV) for n in lens]
    tail = torch.randint(0, 1000, (3, T), generator=g).to(DEV)
    cache = model.alloc_cache(140, 3, bits=8)
    with torch.no_grad():
        model.prefill_ragged(prompts, cache, chunk=64)
        dec = GraphDecoder(model, cache, mode="dense")
        dec.prepare(lens)
        dec.capture()
        got = torch.stack([dec.step(tail[:, t:t + 1], [n + t for n in lens])[:, -1].float().clone() for t in range(T)], 1)
        for b, n in enumerate(lens):
            ids = torch.cat((prompts[b], tail[b])).view(1, -1)
            c = model.alloc_cache(140, 1, bits=8)
            model.prefill(ids[:, :n], c, chunk=64)
            d = GraphDecoder(model, c, mode="dense")
            d.prepare(n)
            one = torch.stack([d.step(ids[:, t:t + 1], t)[:, -1].float().clone() for t in range(n, n + T)], 1)
            torch.testing.assert_close(got[b:b + 1], one, rtol=5e-2, atol=5e-2)
    assert cache.check_status() == 0
    with pytest.raises(ValueError, match="outside the cache"):
        dec.step(tail[:, :1], [140, 90, 20])


def test_a_float32_model_decodes_with_a_quantised_cache():
    model, P, T = tiny_model(torch.float32), 100, 5
    ids = torch.randint(0, 1000, (2, P + T), generator=torch.Generator().manual_seed(1)).to(DEV)
    got = decode(model, ids, model.alloc_cache(P + T, 2, bits=8), P, T, True)
    with torch.no_grad():
        cache = model.alloc_cache(P + T, 2, bits=8)
        model.prefill(ids[:, :P], cache, chunk=100)
        own = torch.stack([model(ids[:, t:t + 1], cache, start_pos=t)[:, -1] for t in range(P, P + T)], 1)
    # float32 throughout: what is left is a code that falls on the other side of a border, one step of 1/254 of a row
    torch.testing.assert_close(got, own, rtol=1e-2, atol=1e-2)


def test_refused_on_the_gpu_too():
    model = tiny_model()
    with pytest.raises(ValueError, match="plain cache"):
        GraphDecoder(model, model.alloc_cache(64, bits=8), mode="cluster")
    with pytest.raises(SkvError):
        QuantAttentionGraph(H=18, H_kv=2, d=128, dtype=torch.bfloat16, device=DEV)
    cache = QuantKVCache(1, 1, 2, 8, 128, 8, DEV)
    x = torch.zeros(1, 2, 1, 128, dtype=torch.bfloat16, device=DEV, requires_grad=True)
    with pytest.raises(ValueError, match="no gradient"):
        cache.write(0, x, x, 0)


@pytest.mark.parametrize("bits", [16, 8])
def test_a_second_ragged_batch_runs_through_the_captured_step(bits):
    """New prompts in the same cache, prepare() with their lengths, no new capture: as a fresh decoder has it."""
    model, T = tiny_model(), 4
    g = torch.Generator().manual_seed(12)
    batches = [[torch.randint(0, 1000, (n,), generator=g).to(DEV) for n in lens] for lens in ([40, 3, 77], [8, 90, 21])]
    tail = torch.randint(0, 1000, (3, T), generator=g).to(DEV)

    def run(dec, cache, prompts, capture):
        lens = [len(p) for p in prompts]
        with torch.no_grad():
            model.prefill_ragged(prompts, cache, chunk=32)
        dec.prepare(lens)
        if capture:
            dec.capture()
        return torch.stack([dec.step(tail[:, t:t + 1], [n + t for n in lens])[:, -1].float().clone() for t in range(T)], 1)

    cache = model.alloc_cache(128, 3, bits=bits)
    dec = GraphDecoder(model, cache, mode="dense")
    run(dec, cache, batches[0], True)
    graph = dec.graph
    got = run(dec, cache, batches[1], False)
    assert dec.graph is graph
    other = model.alloc_cache(128, 3, bits=bits)
    assert torch.equal(got, run(GraphDecoder(model, other, mode="dense"), other, batches[1], True))


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("H,L", [(1, 33), (3, 27), (1, 34)])
def test_a_sequence_whose_scales_begin_off_the_boundary(bits, H, L):
    """One KV head and an odd length: written, read and attended over as the same rows of the whole cache."""
    B, G, n = 4, 2, 20
    whole, parts = (QuantKVCache(1, B, H, L, 128, bits, DEV) for _ in range(2))
    k, v = rows_of(B, H, n, torch.bfloat16, 1, False).to(DEV), rows_of(B, H, n, torch.bfloat16, 2, False).to(DEV)
    whole.write(0, k, v, 5)
    q = torch.randn(B, H * G, 128, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16).to(DEV)
    n_dev = torch.tensor([5 + n], dtype=torch.int32, device=DEV)
    for b in range(B):
        parts.sequence(b).write(0, k[b:b + 1], v[b:b + 1], 5)
        assert torch.equal(parts.sequence(b).read(0, 5, n)[0], whole.read(0, 5, n)[0][b:b + 1])
    parts.sequence(3).write(0, k[:1], v[:1], torch.tensor([L - 3], device=DEV))              # recorded in its own words
    assert parts.status.view(B, H).cpu().tolist() == [[0] * H] * 3 + [[4] * H]
    assert all(torch.equal(a[:3], b[:3]) for a, b in zip((whole.k[0], whole.v[0], whole.scale[0]),
                                                         (parts.k[0], parts.v[0], parts.scale[0])))
    attn = QuantAttentionGraph(H=H * G, H_kv=H, d=128, dtype=torch.bfloat16, device=DEV)
    whole_attn = QuantAttentionGraph(H=B * H * G, H_kv=B * H, d=128, dtype=torch.bfloat16, device=DEV)
    want = whole_attn(q.view(B * H * G, 128), whole, 0, n_dev).view(B, H * G, 128)
    for b in range(3):
        assert torch.equal(attn(q[b], parts.sequence(b), 0, n_dev), want[b])
