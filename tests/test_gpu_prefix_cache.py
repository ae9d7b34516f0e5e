"""Attention of a batch over a prefix that its sequences share, on the GPU against its definition in 64 bits, and the
decode step over a shared-prefix cache against separate decodes over whole caches."""

from __future__ import annotations

import math

import pytest
import torch

from sparse_kv_reads_b200 import GraphDecoder, PrefixAttentionGraph, PrefixKVCache, Qwen3Config, Qwen3Model
from _caches import attention, output_bound
from _helpers import DEV

pytestmark = pytest.mark.gpu
SCALE = 1.0 / math.sqrt(128)


def inputs(B, Hk, G, P, L, lens, seed, dtype=torch.bfloat16):
    g = torch.Generator().manual_seed(seed)
    q = (torch.randn(B * Hk * G, 128, generator=g) * 2).to(dtype)
    kp, vp = (torch.randn(Hk, P, 128, generator=g) + 0.3).to(dtype), torch.randn(Hk, P, 128, generator=g).to(dtype)
    k, v = (torch.randn(B * Hk, L, 128, generator=g) + 0.3).to(dtype), torch.randn(B * Hk, L, 128, generator=g).to(dtype)
    for b, n in enumerate(lens):
        k[b * Hk:(b + 1) * Hk, max(0, n):] = float("nan")
        v[b * Hk:(b + 1) * Hk, max(0, n):] = float("nan")
    return q, kp, vp, k, v


def score_error(q, k, dtype):
    """A score is a sum of 128 exact products in float32, each partial sum cut to 2^-22 of its size at the worst."""
    if k.shape[0] == 0:
        return 0.0
    return float((q.double().abs() @ k.double().abs().T).max()) * 2.0 ** -22 * SCALE


def check_against_definition(out, q, kp, vp, k, v, lens, G, dtype):
    B, Hk = len(lens), kp.shape[0]
    got = out.cpu().double().view(B, Hk, G, 128)
    q = q.view(B, Hk, G, 128)
    for b, n in enumerate(lens):
        for h in range(Hk):
            kk, vv = torch.cat((kp[h], k[b * Hk + h, :max(0, n)])), torch.cat((vp[h], v[b * Hk + h, :max(0, n)]))
            ref, mag = attention(q[b, h], kk, vv, SCALE)
            bound = output_bound(ref, mag, dtype, score_error(q[b, h], kk, dtype))
            assert bool(((got[b, h] - ref).abs() <= bound).all()), (b, h, float((got[b, h] - ref).abs().max()))


def run(q, kp, vp, k, v, lens, B, Hk, G, ragged=True, dtype=torch.bfloat16):
    attn = PrefixAttentionGraph(B=B, H=Hk * G, H_kv=Hk, d=128, dtype=dtype, device=DEV)
    attn.n_group = Hk if ragged else 0
    n_dev = torch.tensor(lens if ragged else lens[:1], dtype=torch.int32, device=DEV)
    args = [t.to(DEV) for t in (q, kp, vp, k, v)]
    first = attn(*args, n_dev).clone()
    assert torch.equal(attn(*args, n_dev), first)          # the same bits, and the workspace is ready again
    return first, attn


@pytest.mark.parametrize("P", [0, 1, 15, 16, 63, 64, 65, 127, 128, 129, 255, 257, 1000])
@pytest.mark.parametrize("G", [1, 2, 5, 8])
def test_prefix_lengths_and_group_sizes(P, G):
    B, Hk = 3, 2
    lens = [0, 19, 1]
    x = inputs(B, Hk, G, P, 24, lens, P + G)
    out, attn = run(*x, lens, B, Hk, G)
    check_against_definition(out, *x, lens, G, torch.bfloat16)
    if P == 0:
        assert bool((out.view(B, Hk, G, 128)[0] == 0).all())           # no key at all
    assert int(attn.status.abs().sum()) == 0


@pytest.mark.parametrize("B,Hk,G", [(1, 1, 1), (2, 8, 2), (7, 3, 4), (16, 1, 8), (17, 2, 8), (33, 1, 4), (64, 2, 4), (130, 1, 2)])
@pytest.mark.parametrize("P", [70, 700])
def test_batch_sizes(B, Hk, G, P):
    lens = [(37 * b) % 90 for b in range(B)]
    x = inputs(B, Hk, G, P, 96, lens, B)
    out, _ = run(*x, lens, B, Hk, G)
    check_against_definition(out, *x, lens, G, torch.bfloat16)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_long_own_rows_equal_lengths_and_both_types(dtype):
    B, Hk, G, P, L = 4, 2, 4, 300, 1500
    lens = [1234] * B
    x = inputs(B, Hk, G, P, L, lens, 5, dtype)
    out, _ = run(*x, lens, B, Hk, G, ragged=False, dtype=dtype)
    check_against_definition(out, *x, lens, G, dtype)


def test_views_of_larger_caches_and_rows_that_hold_nan():
    """The prefix as a slice of a cache whose later rows hold NaN, own rows in a wider layout, lengths out of range."""
    B, Hk, G, P, L = 5, 2, 2, 333, 40
    lens = [40, 3, 0, 40, 17]
    q, kp, vp, k, v = inputs(B, Hk, G, P, L, lens, 9)
    big = torch.full((2, Hk, 512, 128), float("nan"), dtype=torch.bfloat16, device=DEV)
    big[0, :, :P], big[1, :, :P] = kp.to(DEV), vp.to(DEV)
    wide = torch.full((B * Hk, L, 3, 128), float("nan"), dtype=torch.bfloat16, device=DEV)
    wide[:, :, 0], wide[:, :, 2] = k.to(DEV), v.to(DEV)
    attn = PrefixAttentionGraph(B=B, H=Hk * G, H_kv=Hk, d=128, dtype=torch.bfloat16, device=DEV)
    attn.n_group = Hk
    said = [90000, 3, -7, 40, 17]
    out = attn(q.to(DEV), big[0, :, :P], big[1, :, :P], wide[:, :, 0], wide[:, :, 2],
               torch.tensor(said, dtype=torch.int32, device=DEV))
    check_against_definition(out, q, kp, vp, k, v, lens, G, torch.bfloat16)
    assert attn.status.view(B, Hk).cpu()[:, 0].tolist() == [4, 0, 0, 0, 0]


def test_scores_far_apart_and_rescaled_sums():
    """The largest score first, last, in the prefix or in the own rows: running maxima that jump by hundreds."""
    B, Hk, G, P, L = 9, 1, 8, 520, 30
    lens = [30] * B
    q, kp, vp, k, v = inputs(B, Hk, G, P, L, lens, 13)
    for where, at in (("p", 0), ("p", 300), ("p", P - 1), ("k", 0), ("k", 29)):
        kp2, k2 = kp.clone(), k.clone()
        if where == "p":
            kp2[0, at] = q[3] * 4
        else:
            k2[2, at] = q[2 * 8 + 1] * 4
        out, _ = run(q, kp2, vp, k2, v, lens, B, Hk, G)
        check_against_definition(out, q, kp2, vp, k2, v, lens, G, torch.bfloat16)


@pytest.mark.parametrize("B,Hk,G,P,n", [(2, 2, 2, 300, 9), (40, 2, 4, 2000, 9), (9, 1, 8, 9000, 70)])
def test_queries_that_alias_the_output_a_negative_scale_and_no_own_rows(B, Hk, G, P, n):
    """By the list and by the tiles: queries in the output buffer, the softmax scale's sign, a cache without own rows."""
    lens = [n] * B
    q, kp, vp, k, v = (t.to(DEV) for t in inputs(B, Hk, G, P, n, lens, B))
    attn = PrefixAttentionGraph(B=B, H=Hk * G, H_kv=Hk, d=128, dtype=torch.bfloat16, device=DEV)
    n_dev = torch.tensor([n], dtype=torch.int32, device=DEV)
    want = attn(q, kp, vp, k, v, n_dev).clone()
    check_against_definition(want, *(t.cpu() for t in (q, kp, vp, k, v)), lens, G, torch.bfloat16)
    attn.out.copy_(q)
    assert torch.equal(attn(attn.out, kp, vp, k, v, n_dev), want)
    attn._scale = -attn._scale
    assert torch.equal(attn(-q, kp, vp, k, v, n_dev), want)
    attn._scale = -attn._scale
    got = attn(q, kp, vp, k[:, :0], v[:, :0], torch.zeros_like(n_dev))
    check_against_definition(got, *(t.cpu() for t in (q, kp, vp, k, v)), [0] * B, G, torch.bfloat16)


@pytest.mark.parametrize("B,Hk,G", [(1, 1, 1), (30, 2, 4), (100, 1, 3), (70, 4, 8)])
def test_long_prefixes_through_the_tiles(B, Hk, G):
    """Enough rows that the prefix goes through the tensor-core tiles: ragged last tiles, one and more groups of 256 rows."""
    P = 128 * 40 + 77 if B > 1 else 70000
    lens = [(11 * b) % 40 for b in range(B)]
    x = inputs(B, Hk, G, P, 40, lens, B)
    out, attn = run(*x, lens, B, Hk, G)
    check_against_definition(out, *x, lens, G, torch.bfloat16)
    assert int(attn.status.abs().sum()) == 0


@pytest.mark.parametrize("B,P", [(2100, 64), (2100, 65), (1100, 127), (1100, 128), (1100, 129), (700, 257)])
def test_short_prefixes_through_the_tiles(B, P):
    """Batches so large that even a short prefix goes through the tiles: one tile, a tile with one row, masked halves."""
    G = 2
    lens = [b % 3 for b in range(B)]
    q, kp, vp, k, v = inputs(B, 1, G, P, 4, lens, P)
    out, _ = run(q, kp, vp, k, v, lens, B, 1, G)
    got = out.cpu().double().view(B, G, 128)
    for n in (0, 1, 2):                                    # all sequences of a length at once
        at = torch.tensor([b for b in range(B) if lens[b] == n])
        kk = torch.cat((kp.expand(len(at), -1, -1), k[at, :n]), 1).double()
        vv = torch.cat((vp.expand(len(at), -1, -1), v[at, :n]), 1).double()
        qq = q.view(B, G, 128)[at].double()
        w = torch.softmax(qq @ kk.transpose(1, 2) * SCALE, -1)
        ref, mag = w @ vv, w @ vv.abs()
        e = float((qq.abs() @ kk.abs().transpose(1, 2)).max()) * 2.0 ** -22 * SCALE
        assert bool(((got[at] - ref).abs() <= output_bound(ref, mag, torch.bfloat16, e)).all())


def test_a_prefix_that_no_tensor_map_can_describe():
    """One KV head's rows for all heads (a stride of zero): served by the list."""
    B, Hk, G, P = 40, 2, 2, 3000
    lens = [5] * B
    q, kp, vp, k, v = inputs(B, Hk, G, P, 8, lens, 2)
    one_k, one_v = kp[:1].to(DEV).expand(Hk, -1, -1), vp[:1].to(DEV).expand(Hk, -1, -1)
    attn = PrefixAttentionGraph(B=B, H=Hk * G, H_kv=Hk, d=128, dtype=torch.bfloat16, device=DEV)
    out = attn(q.to(DEV), one_k, one_v, k.to(DEV), v.to(DEV), torch.tensor([5], dtype=torch.int32, device=DEV))
    check_against_definition(out, q, kp[:1].expand(Hk, -1, -1), vp[:1].expand(Hk, -1, -1), k, v, lens, G, torch.bfloat16)


def test_offsets_beyond_31_bits():
    """A prefix head that begins more than 2^31 bytes into its tensor."""
    Hk, P, L = 3, 40, 16
    rows = 4_300_000
    big = torch.zeros(Hk, rows, 128, dtype=torch.bfloat16, device=DEV)
    assert 2 * rows * 256 > 2 ** 31
    lens = [5, 9]
    q, kp, vp, k, v = inputs(2, Hk, 2, P, L, lens, 3)
    big[:, :P] = kp.to(DEV)
    attn = PrefixAttentionGraph(B=2, H=Hk * 2, H_kv=Hk, d=128, dtype=torch.bfloat16, device=DEV)
    attn.n_group = Hk
    n_dev = torch.tensor(lens, dtype=torch.int32, device=DEV)
    out = attn(q.to(DEV), big[:, :P], vp.to(DEV), k.to(DEV), v.to(DEV), n_dev)
    check_against_definition(out, q, kp, vp, k, v, lens, 2, torch.bfloat16)


def test_two_objects_on_two_streams_and_a_captured_call():
    sets = []
    for seed, (B, Hk, G, P) in enumerate([(20, 2, 4, 900), (3, 4, 2, 400)]):
        lens = [(13 * b) % 30 for b in range(B)]
        x = [t.to(DEV) for t in inputs(B, Hk, G, P, 32, lens, seed)]
        attn = PrefixAttentionGraph(B=B, H=Hk * G, H_kv=Hk, d=128, dtype=torch.bfloat16, device=DEV)
        attn.n_group = Hk
        sets.append((attn, x, torch.tensor(lens, dtype=torch.int32, device=DEV)))
    want = [a(*x, n).clone() for a, x, n in sets]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(20):
        for s, (a, x, n) in zip(streams, sets):
            with torch.cuda.stream(s):
                a(*x, n)
    torch.cuda.synchronize()
    assert all(torch.equal(a.out, w) for (a, _, _), w in zip(sets, want))
    attn, x, n = sets[0]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = attn(*x, n)
    n.add_(1)
    x[3][:], x[4][:] = x[3].nan_to_num(0.5), x[4].nan_to_num(0.25)
    graph.replay()
    got = out.clone()
    assert torch.equal(attn(*x, n), got) and not torch.equal(got, want[0])


TINY = dict(hidden_size=256, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2, head_dim=128,
            intermediate_size=512, vocab_size=1000, max_position_embeddings=2048)


def tiny_model(dtype=torch.bfloat16):
    with torch.device(DEV):
        m = Qwen3Model(Qwen3Config(**TINY))
    return m.to(dtype).eval().init_random(seed=3, std=0.05)


@pytest.mark.parametrize("batch,dtype", [(2, torch.bfloat16), (9, torch.bfloat16), (3, torch.float32)])
def test_decoding_behind_a_shared_prefix_equals_whole_caches(batch, dtype):
    """One prompt, ``batch`` continuations: the graph equals the eager step bit for bit, and separate decodes over whole
    caches to the tolerance of the model's bf16 layers."""
    model, P, T = tiny_model(dtype), 150, 10
    g = torch.Generator().manual_seed(1)
    prompt, tail = torch.randint(0, 1000, (1, P), generator=g).to(DEV), torch.randint(0, 1000, (batch, T), generator=g).to(DEV)

    def shared(capture):
        cache = model.alloc_prefix_cache(P + 30, T, batch)
        with torch.no_grad():
            model.prefill(prompt, cache.prefix, chunk=64)
            dec = GraphDecoder(model, cache, mode="dense")
            dec.prepare(P)
            cache.cur_len = P
            if capture:
                dec.capture()
            out = torch.stack([dec.step(tail[:, t:t + 1], P + t)[:, -1].float().clone() for t in range(T)], 1)
        assert cache.cur_len == P + T
        return out, dec

    graph, dec = shared(True)
    eager, _ = shared(False)
    assert torch.equal(graph, eager)
    with pytest.raises(ValueError, match="outside the cache"):
        dec.step(tail[:, :1], P + T)
    with torch.no_grad():
        whole = model.alloc_cache(P + T, batch)
        model.prefill(prompt.expand(batch, -1), whole, chunk=64)
        d = GraphDecoder(model, whole, mode="dense")
        d.prepare(P)
        want = torch.stack([d.step(tail[:, t:t + 1], P + t)[:, -1].float().clone() for t in range(T)], 1)
    tol = 5e-2 if dtype == torch.bfloat16 else 1e-3
    torch.testing.assert_close(graph, want, rtol=tol, atol=tol)


def test_questions_of_different_lengths_about_one_document():
    """Each sequence's own prompt is prefilled behind the shared one, then a ragged batch decodes."""
    model, P, T = tiny_model(), 120, 5
    g = torch.Generator().manual_seed(4)
    doc = torch.randint(0, 1000, (1, P), generator=g).to(DEV)
    lens = [7, 31, 1]
    asks = [torch.randint(0, 1000, (n,), generator=g).to(DEV) for n in lens]
    tail = torch.randint(0, 1000, (3, T), generator=g).to(DEV)
    cache = model.alloc_prefix_cache(P, 40, 3)
    with torch.no_grad():
        model.prefill(doc, cache.prefix)
        last = model.prefill_ragged(asks, cache, chunk=16)
        assert cache.cur_len == [P + n for n in lens]
        dec = GraphDecoder(model, cache, mode="dense")
        dec.prepare(cache.cur_len)
        dec.capture()
        got = torch.stack([dec.step(tail[:, t:t + 1], [P + n + t for n in lens])[:, -1].float().clone()
                           for t in range(T)], 1)
        for b, n in enumerate(lens):
            ids = torch.cat((doc[0], asks[b], tail[b])).view(1, -1)
            c = model.alloc_cache(P + n + T)
            first = model.prefill(ids[:, :P + n], c, chunk=64)
            torch.testing.assert_close(last[b].float(), first.float(), rtol=5e-2, atol=5e-2)
            d = GraphDecoder(model, c, mode="dense")
            d.prepare(P + n)
            one = torch.stack([d.step(ids[:, t:t + 1], t)[:, -1].float().clone() for t in range(P + n, P + n + T)], 1)
            torch.testing.assert_close(got[b:b + 1], one, rtol=5e-2, atol=5e-2)
        model.prefill(doc[:, :50], cache.prefix)           # another, shorter document
        with pytest.raises(ValueError, match="prefix has changed"):
            dec.step(tail[:, :1], [P + 1] * 3)


def test_a_prefix_cache_is_refused_by_the_clustered_mode():
    model = tiny_model()
    with pytest.raises(ValueError, match="plain cache"):
        GraphDecoder(model, model.alloc_prefix_cache(16, 16, 2), mode="cluster")
    assert isinstance(model.alloc_prefix_cache(16, 16, 2), PrefixKVCache)


def test_a_captured_step_does_not_outlive_its_prefix():
    """Another document after the capture: prepare() alone, then a new capture, both as a fresh decoder has it."""
    model, T, B = tiny_model(), 4, 3
    g = torch.Generator().manual_seed(6)
    docs = [torch.randint(0, 1000, (1, n), generator=g).to(DEV) for n in (150, 60)]
    tail = torch.randint(0, 1000, (B, T), generator=g).to(DEV)

    def steps(dec, P):
        return torch.stack([dec.step(tail[:, t:t + 1], P + t)[:, -1].float().clone() for t in range(T)], 1)

    with torch.no_grad():
        cache = model.alloc_prefix_cache(160, T, B)
        model.prefill(docs[0], cache.prefix)
        dec = GraphDecoder(model, cache, mode="dense")
        dec.prepare(150)
        cache.cur_len = 150
        dec.capture()
        first = steps(dec, 150)
        model.prefill(docs[1], cache.prefix)
        dec.prepare(60)
        second = steps(dec, 60)
        cache.cur_len = 60
        dec.capture()
        assert torch.equal(steps(dec, 60), second)
        fresh = model.alloc_prefix_cache(160, T, B)
        model.prefill(docs[1], fresh.prefix)
        other = GraphDecoder(model, fresh, mode="dense")
        other.prepare(60)
        assert torch.equal(steps(other, 60), second) and not torch.equal(first, second)


def run_plain(q, kp, vp, k, v, B, Hk, G, dtype=torch.bfloat16):
    attn = PrefixAttentionGraph(B=B, H=Hk * G, H_kv=Hk, d=128, dtype=dtype, device=DEV)
    n = torch.tensor([k.shape[1]], dtype=torch.int32, device=DEV)
    return attn(*(t.to(DEV) for t in (q, kp, vp, k, v)), n).clone()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("B,P,n", [(2, 100, 20), (60, 5000, 20), (130, 5000, 7)])
@pytest.mark.parametrize("size", [2.0 ** 105, -2.0 ** 105])
def test_scores_far_beyond_ordinary_ones(dtype, B, P, n, size):
    """Finite scores of 2^118, all positive or all negative: the largest one takes all, be it the prefix's or an own one."""
    Hk, G = 1, 2
    q, kp, vp, k, v = inputs(B, Hk, G, P, n, [n] * B, 3, dtype)
    q[:], kp[:], k[:] = 0, 0, 0
    q[:, 9], kp[..., 9], k[..., 9] = size, (65536.0 if size > 0 else 66048.0), (65536.0 if size > 0 else 66048.0)
    best = 66048.0 if size > 0 else 65536.0
    kp[0, 77, 9] = best                                    # even sequences: the prefix's row; odd ones: an own row beyond it
    k[1::2, n // 2, 9] = best * (2 if size > 0 else 0.5)
    got = run_plain(q, kp, vp, k, v, B, Hk, G, dtype).cpu().view(B, G, 128)
    for b in range(B):
        assert torch.equal(got[b], (v[b, n // 2] if b % 2 else vp[0, 77]).expand(G, -1)), b


@pytest.mark.parametrize("B,G,P", [(3, 2, 100), (60, 4, 5000), (130, 4, 1000), (130, 4, 1024)])
def test_a_softmax_scale_of_zero_gives_the_mean(B, G, P):
    """By the list and in the range of the tiles, whole and ragged: every row counts alike."""
    Hk, n = 1, 9
    q, kp, vp, k, v = inputs(B, Hk, G, P, n, [n] * B, 4)
    attn = PrefixAttentionGraph(B=B, H=G, H_kv=Hk, d=128, dtype=torch.bfloat16, device=DEV)
    attn._scale = 0.0
    got = attn(*(t.to(DEV) for t in (q, kp, vp, k, v)), torch.tensor([n], dtype=torch.int32, device=DEV)).cpu().double()
    for b in range(B):
        rows = torch.cat((vp[0], v[b])).double()
        ref, mag = rows.mean(0), rows.abs().mean(0)
        assert bool(((got.view(B, G, 128)[b] - ref).abs() <= output_bound(ref, mag, torch.bfloat16)).all()), b


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("B,P,n", [(2, 100, 20), (60, 5000, 20), (60, 5000, 300), (130, 5000, 7)])
def test_a_key_that_is_no_number_leaves_no_number(dtype, B, P, n):
    """By the list and by the tiles: NaN in a prefix key spoils its KV head for all, in an own key its sequence's head."""
    Hk, G = 2, 2
    q, kp, vp, k, v = inputs(B, Hk, G, P, n, [n] * B, 3, dtype)
    kp[1, P - 2, 5] = float("nan")
    k[1 * Hk + 0, n - 1, 9] = float("nan")
    got = run_plain(q, kp, vp, k, v, B, Hk, G, dtype).view(B, Hk, G, 128).isnan()
    assert bool(got[:, 1].all()) and bool(got[1, 0].all())
    assert not bool(got[0, 0].any()) and not bool(got[2:, 0].any())


@pytest.mark.parametrize("P,extra", [(100, 0), (40000, 1)])
def test_a_captured_step_counts_the_prefixs_own_launch(P, extra):
    """By the list a step has as many launches as over whole caches, by the tiles one more per layer."""
    with torch.device(DEV):
        model = Qwen3Model(Qwen3Config(**{**TINY, "max_position_embeddings": 50000}))
    model = model.to(torch.bfloat16).eval().init_random(seed=3, std=0.05)
    counts = []
    for cache in (model.alloc_cache(64, 4), model.alloc_prefix_cache(P, 8, 4)):
        if isinstance(cache, PrefixKVCache):
            cache.prefix.cur_len = P                       # (rows of zeros)
            cache.cur_len = P
        dec = GraphDecoder(model, cache, mode="dense")
        dec.prepare(cache.cur_len)
        dec.capture()
        counts.append(dec.launches_per_step)
    assert counts[1] == counts[0] + extra * len(model.layers)


def test_a_decoder_over_a_shared_prefix_reports_a_length_beyond_its_rows():
    model, B = tiny_model(), 2
    cache = model.alloc_prefix_cache(20, 6, B)
    with torch.no_grad():
        model.prefill(torch.arange(20, device=DEV).view(1, -1), cache.prefix)
        dec = GraphDecoder(model, cache, mode="dense")
        dec.prepare(20)
        dec.step(torch.zeros(B, 1, dtype=torch.long, device=DEV), 20)
        assert dec.check_status() == 0
        kh, vh = dec._heads(cache.k[0]), dec._heads(cache.v[0])
        q = torch.zeros(B * dec.H, 128, dtype=torch.bfloat16, device=DEV)
        dec.attn[0](q, *cache.prefix_rows(0), kh, vh, torch.tensor([7], dtype=torch.int32, device=DEV))
    assert dec.check_status() == 4


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("B,Hk,G,P,n", [(2, 2, 2, 333, 17), (4, 8, 2, 5000, 100), (40, 4, 2, 5003, 40), (70, 8, 4, 4097, 9),
                                        (9, 1, 8, 20000, 700), (130, 1, 2, 900, 1)])
def test_every_tile_and_partial_counts(dtype, B, Hk, G, P, n):
    """Values that are one in a component of their own for each 1/128 of the rows, weights all alike: an output component is
    the share of its rows, so that one that is lost or counted twice shows."""
    total = P + n
    g = torch.Generator().manual_seed(total)
    q = (torch.randn(B * Hk * G, 128, generator=g) * 0.05).to(dtype)
    kp, k = torch.randn(Hk, P, 128, generator=g).to(dtype), torch.randn(B * Hk, n, 128, generator=g).to(dtype)
    where = torch.arange(total) * 128 // total
    one = torch.eye(128)[where].to(dtype)
    vp, v = one[:P].expand(Hk, -1, -1).contiguous(), one[P:].expand(B * Hk, -1, -1).contiguous()
    got = run_plain(q, kp, vp, k, v, B, Hk, G, dtype).cpu().double().view(B, Hk, G, 128)
    qq = q.double().view(B, Hk, G, 128)
    zp = torch.einsum("bhgd,hpd->bhgp", qq, kp.double())
    zo = torch.einsum("bhgd,bhnd->bhgn", qq, k.double().view(B, Hk, n, 128))
    w = torch.softmax(torch.cat((zp, zo), -1) * SCALE, -1)
    ref = torch.zeros(B, Hk, G, 128, dtype=torch.float64).index_add_(3, where, w)
    # scores well below one: their own error is nothing beside the weights' rounding
    assert bool(((got - ref).abs() <= output_bound(ref, ref, dtype, 2.0 ** -18)).all())
    assert 16 * 128 / total > 4 * 3 * 2.0 ** -8            # (16 rows of a component are far outside the bound)
