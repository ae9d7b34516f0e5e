"""Quantised and shared-prefix caches without a GPU: what the C entry points and the Python classes refuse, the stored
layout, and the caches' bookkeeping."""

from __future__ import annotations

import ctypes
import os
import re

import pytest
import torch

from sparse_kv_reads_b200 import (GraphDecoder, PrefixAttentionGraph, PrefixKVCache, QuantAttentionGraph, QuantKVCache,
                                  Qwen3Config, Qwen3Model)
from sparse_kv_reads_b200 import _lib
from sparse_kv_reads_b200.build import build
from _caches import pack, quantise
from _quant_bounds import attention_bound

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
OK = 0x1000
CPU = torch.device("cpu")


@pytest.fixture(scope="module")
def L():
    build()
    return _lib.lib()


def qcache(**o):
    c = _lib.SkvQCache(OK, OK, OK, None, 2, 4, 64, 128, 8, 0)
    for name, v in o.items():
        setattr(c, name, v)
    return ctypes.byref(c)


@pytest.mark.parametrize("name,mirror,size", [("skv_qcache", _lib.SkvQCache, 4 * 8 + 6 * 4), ("skv_rows", _lib.SkvRows, 10 * 8 + 4 * 4),
                                              ("skv_prefix", _lib.SkvPrefix, 12 * 8 + 8 * 4)])
def test_the_structs_match_the_header(name, mirror, size):
    text = open(os.path.join(ROOT, "include", "skv.h")).read()
    body = text[text.index(f"typedef struct {name} {{"):text.index(f"}} {name};")]
    body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
    names = re.findall(r"[\s*]([A-Za-z_0-9]+)(?=[,;])", body)
    assert names == [f[0] for f in mirror._fields_]
    assert ctypes.sizeof(mirror) == size


BAD_CACHES = [(dict(k=None), -1), (dict(v=None), -1), (dict(scale=None), -1), (dict(d=64), -2), (dict(bits=6), -5),
              (dict(batch=0), -5), (dict(h_kv=-1), -5), (dict(capacity=0), -5), (dict(batch=70000), -5),
              (dict(k=0x1008), -4), (dict(scale=0x1004), -4)]


@pytest.mark.parametrize("name", ["skv_quant_write", "skv_quant_read"])
def test_rows_are_refused_on_the_host(L, name):
    base = dict(k=OK, v=OK, dtype=0, batch=2, tokens=3, kb=4096, kh=1024, kr=128, vb=4096, vh=1024, vr=128, pos=None,
                per=0, pos0=0)

    def call(c=None, **o):
        a = {**base, **o}
        rows = _lib.SkvRows(a["k"], a["v"], a["pos"], a["pos0"], a["kb"], a["kh"], a["kr"], a["vb"], a["vh"], a["vr"], a["per"],
                            a["dtype"], a["batch"], a["tokens"])
        return getattr(L, name)(qcache() if c is None else c, ctypes.byref(rows), None)

    for over, code in BAD_CACHES:
        assert call(qcache(**over)) == code, over
    assert getattr(L, name)(None, ctypes.byref(_lib.SkvRows()), None) == -1
    assert getattr(L, name)(qcache(), None, None) == -1
    assert call(k=None) == -1 and call(v=None) == -1 and call(dtype=3) == -3
    assert call(batch=3) == -5 and call(batch=0) == -5 and call(tokens=-1) == -5 and call(tokens=65) == -5
    assert call(pos0=62) == -5 and call(pos0=-1) == -5
    assert call(k=0x1002) == -4 and call(kr=100) == -4 and call(vh=3) == -4 and call(dtype=1, vb=2) == -4
    assert call(tokens=0) == 0                                                   # nothing to do, nothing launched


def test_the_decode_steps_write_is_refused_on_the_host(L):
    args = dict(qkv=OK, qw=OK, kw=OK, cos=OK, sin=OK, pos=OK, q=OK, batch=2, H=8)

    def call(c=None, **o):
        a = {**args, **o}
        return L.skv_qk_rope_quant(qcache() if c is None else c, a["qkv"], a["qw"], a["kw"], a["cos"], a["sin"], a["pos"],
                                   0, a["q"], a["batch"], a["H"], 1e-6, None)

    for over, code in BAD_CACHES:
        assert call(qcache(**over)) == code, over
    for name in ("qkv", "qw", "kw", "cos", "sin", "pos", "q"):
        assert call(**{name: None}) == -1
    assert call(H=0) == -5 and call(H=6) == -5 and call(batch=3) == -5 and call(q=0x1004) == -4 and call(qw=0x1004) == -4


def test_attention_over_quantised_rows_is_refused_on_the_host(L):
    args = dict(q=OK, dtype=0, G=2, n=OK, ng=0, out=OK, ws=OK, ctas=4)

    def call(c=None, **o):
        a = {**args, **o}
        return L.skv_attend_quant(qcache() if c is None else c, a["q"], a["dtype"], a["G"], a["n"], a["ng"], a["out"],
                                  a["ws"], a["ctas"], 0.1, None)

    for over, code in BAD_CACHES:
        assert call(qcache(**over)) == code, over
    for name in ("q", "n", "out", "ws"):
        assert call(**{name: None}) == -1
    assert call(dtype=2) == -3 and call(G=0) == -2 and call(G=9) == -2 and call(ctas=0) == -5 and call(ng=-1) == -5
    assert call(q=0x1008) == -4 and call(out=0x1002) == -4 and call(ws=0x1008) == -4
    assert L.skv_quant_ctas() == 2 * 148 and L.skv_quant_workspace_bytes(8, 2, 128, 444) == 452 * 2 * 528 + 256
    assert L.skv_quant_workspace_bytes(0, 2, 128, 4) == -5 and L.skv_quant_workspace_bytes(8, 9, 128, 4) == -2


def test_attention_over_a_shared_prefix_is_refused_on_the_host(L):
    args = dict(q=OK, kp=OK, vp=OK, P=100, k=OK, v=OK, n=OK, ng=0, out=OK, ws=OK, batch=2, h=4, G=2, d=128, dtype=0,
                kph=128 * 100, kpr=128, vph=128 * 100, vpr=128, kh=128 * 64, kr=128, vh=128 * 64, vr=128, lim=64, splits=4)

    def call(**o):
        a = {**args, **o}
        c = _lib.SkvPrefix(a["kp"], a["vp"], a["k"], a["v"], a["kph"], a["kpr"], a["vph"], a["vpr"], a["kh"], a["kr"], a["vh"],
                           a["vr"], a["P"], a["lim"], a["batch"], a["h"], a["G"], a["d"], a["dtype"], a["ng"])
        return L.skv_attend_prefix(ctypes.byref(c), a["q"], a["n"], a["out"], a["ws"], a["splits"], None, 0.1, None)

    assert L.skv_attend_prefix(None, OK, OK, OK, OK, 4, None, 0.1, None) == -1
    for name in ("q", "kp", "vp", "k", "v", "n", "out", "ws"):
        assert call(**{name: None}) == -1, name
    assert call(kp=None, vp=None, P=0, d=64) == -2 and call(k=None, v=None, lim=0, d=64) == -2       # no rows: no address
    assert call(d=64) == -2 and call(G=0) == -2 and call(G=9) == -2 and call(dtype=5) == -3
    assert call(batch=0) == -5 and call(h=0) == -5 and call(batch=20000) == -5 and call(P=-1) == -5 and call(lim=-1) == -5
    assert call(P=2 ** 31 - 2) == -5 and call(splits=0) == -5 and call(ng=-1) == -5
    assert call(q=0x1008) == -4 and call(kp=0x1004) == -4 and call(kpr=132) == -4 and call(kpr=64) == -4
    assert call(vr=100) == -4 and call(kh=4) == -4
    assert L.skv_prefix_splits(0, 8, 2, 0) == -5 and L.skv_prefix_splits(2, 8, 9, 0) == -2
    assert L.skv_prefix_splits(2, 8, 2, 9) == -3 and L.skv_prefix_splits(2, 8, 2, 0) >= 1
    assert L.skv_prefix_workspace_bytes(0, 8, 2, 128, 4) == -5 and L.skv_prefix_workspace_bytes(2, 8, 2, 64, 4) == -5


def test_quantised_cache_checks_its_arguments():
    with pytest.raises(ValueError, match="8 or 4 bits"):
        QuantKVCache(1, 1, 2, 16, 128, 6, CPU)
    with pytest.raises(ValueError, match="head_dim"):
        QuantKVCache(1, 1, 2, 16, 64, 8, CPU)
    c = QuantKVCache(2, 3, 2, 16, 128, 4, CPU)
    assert c.k[0].shape == (3, 2, 16, 64) and c.scale[1].shape == (3, 2, 16, 2, 4) and c.check_status() == 0
    x = torch.zeros(3, 2, 4, 128, dtype=torch.bfloat16)
    for bad in (x[..., :64], x[:, :1], torch.zeros(4, 2, 4, 128, dtype=torch.bfloat16), x[0]):
        with pytest.raises(ValueError, match="must be"):
            c.write(0, bad, bad, 0)
    with pytest.raises(ValueError, match="one type"):
        c.write(0, x, x.float(), 0)
    with pytest.raises(ValueError, match="unsupported"):
        c.write(0, x.half(), x.half(), 0)
    for pos in (-1, 13):
        with pytest.raises(ValueError, match="outside"):
            c.write(0, x, x, pos)
        with pytest.raises(ValueError, match="outside"):
            c.read(0, pos, 4)
    for pos in (torch.tensor([0, 1]), torch.tensor([0], dtype=torch.int32), torch.tensor(3)):
        with pytest.raises(ValueError, match="positions are"):
            c.write(0, x, x, pos)
    with pytest.raises(ValueError, match="3 sequences"):
        c.read(0, 0, 1, batch=4)
    with pytest.raises(ValueError, match="no gradient"):
        y = x.clone().requires_grad_()
        c.write(0, y, y, 0)
    c.write(0, x[:, :, :0], x[:, :, :0], 16)                                     # nothing to write: no launch
    assert c.read(0, 3, 0)[0].shape == (3, 2, 0, 128)
    with pytest.raises(ValueError, match="codes must be"):
        QuantKVCache.from_tensors(c.k, c.v, c.scale, 8)
    with pytest.raises(ValueError, match="scales must be"):
        QuantKVCache.from_tensors(c.k, c.v, [s.float() for s in c.scale], 4)
    with pytest.raises(ValueError, match="status must be"):
        QuantKVCache.from_tensors(c.k, c.v, c.scale, 4, c.status[:3])
    with pytest.raises(ValueError, match="CUDA device only"):
        c.write(0, x, x, 0)
    with pytest.raises(ValueError, match="CUDA device only"):
        c.read(0, 0, 1)
    one = c.sequence(2)
    assert one.batch == 1 and one.k[1].data_ptr() == c.k[1][2].data_ptr() and one.status.data_ptr() == c.status[4:].data_ptr()


def test_attention_objects_check_their_arguments(L):
    with pytest.raises(ValueError, match="divide"):
        QuantAttentionGraph(H=5, H_kv=2, d=128, dtype=torch.bfloat16, device=CPU)
    with pytest.raises(ValueError, match="divide"):
        PrefixAttentionGraph(B=1, H=5, H_kv=2, d=128, dtype=torch.bfloat16, device=CPU)
    with pytest.raises(_lib.SkvError):
        QuantAttentionGraph(H=18, H_kv=2, d=128, dtype=torch.bfloat16, device=CPU)
    with pytest.raises(_lib.SkvError):
        PrefixAttentionGraph(B=1, H=18, H_kv=2, d=128, dtype=torch.bfloat16, device=CPU)
    with pytest.raises(ValueError, match="unsupported"):
        QuantAttentionGraph(H=4, H_kv=2, d=128, dtype=torch.float16, device=CPU)
    q, n = torch.zeros(4, 128, dtype=torch.bfloat16), torch.zeros(1, dtype=torch.int32)
    c = QuantKVCache(1, 1, 2, 16, 128, 8, CPU)
    a = QuantAttentionGraph(H=4, H_kv=2, d=128, dtype=torch.bfloat16, device=CPU)
    with pytest.raises(ValueError, match="queries must be"):
        a(q[:3], c, 0, n)
    with pytest.raises(ValueError, match="queries must be"):
        a(q.float(), c, 0, n)
    with pytest.raises(ValueError, match="KV heads"):
        a(q, QuantKVCache(1, 1, 4, 16, 128, 8, CPU), 0, n)
    with pytest.raises(ValueError, match="lengths must be"):
        a(q, c, 0, n.long())
    with pytest.raises(ValueError, match="CUDA device only"):
        a(q, c, 0, n)
    a.n_group = 1
    with pytest.raises(ValueError, match="lengths must be"):
        a(q, c, 0, n)
    p = PrefixAttentionGraph(B=2, H=4, H_kv=2, d=128, dtype=torch.bfloat16, device=CPU)
    q8, kp, k = torch.zeros(8, 128, dtype=torch.bfloat16), torch.zeros(2, 9, 128, dtype=torch.bfloat16), \
        torch.zeros(4, 5, 128, dtype=torch.bfloat16)
    for args, word in (((q8, kp, kp, k, k, n), "CUDA device only"), ((q, kp, kp, k, k, n), "queries must be"), ((q8, kp[:1], kp[:1], k, k, n), "prefix must be"),
                       ((q8, kp, kp[:, :3], k, k, n), "prefix must be"), ((q8, kp, kp, k[:3], k[:3], n), "rows must be"),
                       ((q8, kp.float(), kp.float(), k, k, n), "type and device"),
                       ((q8, kp, kp, k, k, n.long()), "lengths must be"),
                       ((q8, kp, kp, k.transpose(1, 2).contiguous().transpose(1, 2), k, n), "unit last stride")):
        with pytest.raises(ValueError, match=word):
            p(*args)


def test_four_bit_layout_puts_one_run_of_each_group_side_by_side():
    code = torch.arange(128).view(1, 128) // 32 - 2                              # the group's number, less two
    stored = pack(code, 4)
    assert stored.view(8, 8).tolist() == [[0x66, 0x66, 0x77, 0x77, 0x88, 0x88, 0x99, 0x99]] * 8
    code, scale = quantise(torch.zeros(1, 128), 4)
    assert int(pack(code, 4).sum()) == 64 * 0x88 and scale.tolist() == [[0.0] * 4]


TINY = dict(hidden_size=64, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2, head_dim=128,
            intermediate_size=96, vocab_size=200, max_position_embeddings=256)


def test_shared_prefix_prefill_equals_whole_prompts():
    m = Qwen3Model(Qwen3Config(**TINY)).eval().init_random(seed=3, std=0.1)
    g = torch.Generator().manual_seed(0)
    doc = torch.randint(0, 200, (1, 30), generator=g)
    asks = [torch.randint(0, 200, (n,), generator=g) for n in (5, 12)]
    cache = m.alloc_prefix_cache(40, 16, 2)
    with torch.no_grad():
        m.prefill(doc, cache.prefix, chunk=8)
        assert cache.first == 30 and cache.max_seq_len == 46 and cache.cur_len == 30
        got = m.prefill_ragged(asks, cache, chunk=4)
        for b, a in enumerate(asks):
            want = m.prefill(torch.cat((doc[0], a)).view(1, -1), m.alloc_cache(64), chunk=16)
            torch.testing.assert_close(got[b], want, rtol=1e-4, atol=1e-4)       # float32, sums in another order
        assert cache.cur_len == [35, 42]
        # both sequences at once
        cache.cur_len = 30
        two = m(torch.stack([a[:5] for a in asks]), cache, start_pos=30, last_only=True)
        torch.testing.assert_close(two[:1], got[0], rtol=1e-4, atol=1e-4)
    with pytest.raises(ValueError, match="behind the prefix"):
        m(doc, cache, start_pos=3)
    with pytest.raises(ValueError, match="behind the prefix"):
        cache.cur_len = 29
    m.layers[0].attn.decode_attn_op = lambda *a, **k: None
    with pytest.raises(ValueError, match="plain cache"):
        m(doc[:, :1], cache, start_pos=30)
    with pytest.raises(ValueError, match="bits must be"):
        m.alloc_cache(16, bits=5)


def test_the_clustered_mode_refuses_the_new_caches_and_steps_are_checked():
    m = Qwen3Model(Qwen3Config(**TINY)).eval()
    for cache in (m.alloc_cache(16, bits=8), m.alloc_prefix_cache(8, 8, 2)):
        with pytest.raises(ValueError, match="mode='dense'"):
            GraphDecoder(m, cache, mode="cluster")
    cache = m.alloc_prefix_cache(8, 4, 2)
    assert isinstance(cache, PrefixKVCache)
    cache.prefix.cur_len = 6
    dec = GraphDecoder(m, cache, mode="dense")
    dec.prepare(6)
    for pos in (5, 10):
        with pytest.raises(ValueError, match="outside the cache"):
            dec.step(torch.zeros(2, 1, dtype=torch.long), pos)
    cache.prefix.cur_len = 7
    with pytest.raises(ValueError, match="prefix has changed"):
        dec.step(torch.zeros(2, 1, dtype=torch.long), 8)
    long = GraphDecoder(m, m.alloc_cache(600, bits=8), mode="dense")             # the rotary tables have 256 rows
    with pytest.raises(ValueError, match="outside the cache"):
        long.step(torch.zeros(1, 1, dtype=torch.long), 256)


class Replayed:
    """In place of a captured graph."""

    def replay(self):
        raise AssertionError("a step captured for another prefix was replayed")


def test_a_captured_step_is_given_up_when_the_prefix_changes():
    """The length of the prefix is part of a captured step: ``prepare`` and ``load_state_dict`` drop one captured for another."""
    m = Qwen3Model(Qwen3Config(**TINY)).eval()
    cache = m.alloc_prefix_cache(8, 4, 2)
    cache.prefix.cur_len = 6
    dec = GraphDecoder(m, cache, mode="dense")
    dec.prepare(6)
    graph = Replayed()
    dec.graph, dec._captured = graph, (6, False)
    dec.prepare(7)                                         # the same prefix: the step still holds
    assert dec.graph is graph
    cache.prefix.cur_len = 4
    dec.prepare(5)
    assert dec.graph is None
    dec.graph, dec._captured = Replayed(), (6, False)
    dec.load_state_dict({"n": 4, "layers": []})
    assert dec.graph is None and dec.first == 4
    plain = GraphDecoder(m, m.alloc_cache(8), mode="dense")
    plain.graph, plain._captured = Replayed(), (0, False)
    plain.prepare(3)
    assert plain.graph is not None


@pytest.mark.parametrize("kind", ["quantised", "prefix"])
def test_a_captured_ragged_step_keeps_its_buffers_or_is_given_up(kind):
    """A captured step reads positions and lengths where they lay: a second batch of lengths goes to the same place, and the
    first such batch, which needs new buffers, gives up a step captured for equal lengths."""
    m = Qwen3Model(Qwen3Config(**TINY)).eval()
    cache = m.alloc_cache(64, 2, bits=8) if kind == "quantised" else m.alloc_prefix_cache(8, 40, 2)
    dec = GraphDecoder(m, cache, mode="dense")
    dec.fused_dense = True                                 # (of the bf16 model on a GPU; nothing is launched here)
    dec.prepare(5)
    dec.graph, dec._captured = Replayed(), (0, False)
    dec.prepare([5, 9])
    assert dec.graph is None
    where = dec.pos.data_ptr(), dec.n_dev.data_ptr()
    graph = Replayed()
    dec.graph, dec._captured = graph, (0, True)
    dec.prepare([11, 2])
    assert (dec.pos.data_ptr(), dec.n_dev.data_ptr()) == where and dec.graph is graph
    assert dec.pos.tolist() == [11, 2] and dec.n_dev.tolist() == [11, 2]
    with pytest.raises(ValueError, match="one length per sequence"):
        dec.prepare([1])


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("n", [17, 300, 1000])
def test_what_the_attentions_bounds_leave_outside(bits, n):
    """Planted mistakes of the attention over quantised rows: each has a component outside the bound in some head."""
    g = torch.Generator().manual_seed(n)
    heads = []
    for _ in range(4):
        k = (torch.randn(n, 128, generator=g) + 0.7) * torch.randn(128, generator=g).abs()
        (kc, ks), (vc, vs) = quantise(k, bits), quantise(torch.randn(n, 128, generator=g), bits)
        heads.append((kc, ks, vc, vs, (torch.randn(2, 128, generator=g) * 2).to(torch.bfloat16)))

    def found(change):
        bad = []
        for kc, ks, vc, vs, q in heads:
            out, bound = attention_bound(q, kc, ks, vc, vs, bits, 128 ** -0.5)
            wrong = attention_bound(q, *change(kc, ks, vc, vs), bits, 128 ** -0.5)[0]
            bad.append(bool(((wrong - out).abs() > bound).any()))
        return any(bad)

    def exchanged(s, i, j):
        s = s.clone()
        s[:, [i, j]] = s[:, [j, i]]
        return s

    assert found(lambda kc, ks, vc, vs: (kc[:-16], ks[:-16], vc[:-16], vs[:-16]))                # the last tile lost
    assert found(lambda kc, ks, vc, vs: (kc, ks, vc * (torch.arange(n) >= 16).unsqueeze(-1), vs))    # a tile's values lost
    assert found(lambda kc, ks, vc, vs: (kc[n // 4:], ks[n // 4:], vc[n // 4:], vs[n // 4:]))      # a partial lost
    assert found(lambda kc, ks, vc, vs: (kc, ks, vc, vs * 0))                                    # all zeros
    assert found(lambda kc, ks, vc, vs: (kc, ks, vc, vs.float() * 1.1))
    assert found(lambda kc, ks, vc, vs: (kc, ks.float() * 1.1, vc, vs))
    if bits == 4:
        assert found(lambda kc, ks, vc, vs: (kc, exchanged(ks, 0, 1), vc, vs))
        assert found(lambda kc, ks, vc, vs: (kc, ks, vc, exchanged(vs, 2, 3)))
    assert not found(lambda kc, ks, vc, vs: (kc, ks, vc, vs))


def test_the_launches_of_a_shared_prefix_call_are_known_ahead(L):
    c = _lib.SkvPrefix(OK, OK, OK, OK, 128 * 100, 128, 128 * 100, 128, 128 * 64, 128, 128 * 64, 128, 100, 64, 2, 4, 2, 128, 0, 0)
    assert L.skv_prefix_launches(ctypes.byref(c), 4, 0.1) == 1                   # a short prefix: by the list
    c.dtype, c.prefix = 1, 100000
    assert L.skv_prefix_launches(ctypes.byref(c), 4, 0.1) == 1                   # float32: always one
    assert L.skv_prefix_launches(None, 4, 0.1) == -1
    c.d = 64
    assert L.skv_prefix_launches(ctypes.byref(c), 4, 0.1) == -2


def test_the_status_words_of_a_decoder_are_read_together(L):
    m = Qwen3Model(Qwen3Config(**TINY)).eval()
    prefix = GraphDecoder(m, m.alloc_prefix_cache(8, 4, 2), mode="dense")
    assert prefix.check_status() == 0 == prefix.attn[0].check_status()
    prefix.attn[0].status[1], prefix.attn[0].status[3] = 4, 16
    assert prefix.attn[0].check_status() == 20 == prefix.check_status()
    quantised = GraphDecoder(m, m.alloc_cache(16, 2, bits=8), mode="dense")
    assert quantised.check_status() == 0
    quantised.cache.status[2] = 4
    assert quantised.check_status() == 4
    assert GraphDecoder(m, m.alloc_cache(16), mode="dense").check_status() == 0


def test_the_current_stream_of_any_kind_of_device(monkeypatch):
    """A device with its index takes the short way where PyTorch has one; anything else goes to its public function."""
    asked = []
    monkeypatch.setattr(torch.cuda, "current_stream", lambda d=None: asked.append(d) or type("S", (), {"cuda_stream": 77}))
    monkeypatch.setattr(_lib, "_raw_stream", lambda index: 100 + index)
    assert _lib.stream_ptr(torch.device("cuda", 3)) == 103 and asked == []
    for device in (None, 1, "cuda", "cuda:1", torch.device("cuda")):
        assert _lib.stream_ptr(device) == 77 and asked[-1] == device
    monkeypatch.setattr(_lib, "_raw_stream", None)
    assert _lib.stream_ptr(torch.device("cuda", 2)) == 77 and asked[-1] == torch.device("cuda", 2)


@pytest.mark.parametrize("bits", [8, 4])
def test_a_sequence_of_a_cache_of_odd_length_is_taken_from_the_whole(L, bits):
    """The scales of a later sequence may begin off the 16-byte boundary: its struct has the whole cache's addresses and the
    number of sequences ahead of it."""
    c = QuantKVCache(1, 3, 1, 33, 128, bits, CPU)
    one = c.sequence(2).sequence(0)
    st = one._st[0]
    assert st.skip == 2 and st.batch == 1 and st.scale == c.scale[0].data_ptr() and st.k == c.k[0].data_ptr()
    assert one.k[0].data_ptr() == c.k[0][2].data_ptr() and one.scale[0].data_ptr() == c.scale[0][2].data_ptr()
    for b in (-1, 3):
        with pytest.raises(ValueError, match="3 sequences"):
            c.sequence(b)
    assert L.skv_quant_write(qcache(skip=-1), ctypes.byref(_lib.SkvRows(OK, OK, None, 0, 0, 0, 128, 0, 0, 128, 0, 0, 1, 1)), None) == -5


def test_the_rotary_launch_takes_its_tables_by_address(L, monkeypatch):
    """From the position of the cache's first row, without a tensor operation per layer (an eager step has 28 of them)."""
    from torch.utils._python_dispatch import TorchDispatchMode

    from sparse_kv_reads_b200 import graph_decode

    class Nothing(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            raise AssertionError(f"{func} was called")

    got = {}

    class Fake:
        def skv_qk_rope_cache(self, *a):
            got["cos"], got["sin"] = a[3], a[4]
            return 0

        def skv_qk_rope_quant(self, *a):
            got["cos"], got["sin"] = a[4], a[5]
            return 0

    m = Qwen3Model(Qwen3Config(**TINY)).eval()
    prefix = m.alloc_prefix_cache(8, 4, 2)
    prefix.prefix.cur_len = 6
    x = torch.zeros(2, 8 * 128)
    for cache, first in ((m.alloc_cache(8, 2), 0), (m.alloc_cache(8, 2, bits=8), 0), (prefix, 6)):
        dec = GraphDecoder(m, cache, mode="dense")
        dec.prepare(first)
        monkeypatch.setattr(graph_decode, "lib", Fake)
        with Nothing():
            dec._rope(0, x, x, 0)
        monkeypatch.undo()
        row = m.rope_cos[0].numel() * m.rope_cos.element_size()
        assert got == {"cos": m.rope_cos.data_ptr() + first * row, "sin": m.rope_sin.data_ptr() + first * row}


def test_positions_are_whole_numbers_of_any_kind(L):
    np = pytest.importorskip("numpy")
    c = QuantKVCache(1, 1, 2, 16, 128, 8, CPU)
    x = torch.zeros(1, 2, 1, 128, dtype=torch.bfloat16)
    with pytest.raises(TypeError):
        c.write(0, x, x, 2.7)                              # (was taken for 2)
    with pytest.raises(ValueError, match="CUDA device only"):
        c.write(0, x, x, np.int64(3))
    m = Qwen3Model(Qwen3Config(**TINY)).eval()
    cache = m.alloc_prefix_cache(8, 4, 2)
    cache.prefix.cur_len = 6
    dec = GraphDecoder(m, cache, mode="dense")
    dec.prepare(6)
    for pos in (np.int64(10), torch.tensor(10), torch.tensor([10]), [6, 10]):
        with pytest.raises(ValueError, match="position 10 lies outside"):
            dec.step(torch.zeros(2, 1, dtype=torch.long), pos)


def test_a_prefix_prefilled_as_a_ragged_batch_of_one():
    m = Qwen3Model(Qwen3Config(**TINY)).eval().init_random(seed=3, std=0.1)
    cache = m.alloc_prefix_cache(40, 16, 2)
    with torch.no_grad():
        m.prefill_ragged([torch.arange(30)], cache.prefix)
        assert cache.first == 30 and cache.max_seq_len == 46 and cache.cur_len == 30
        got = m.prefill(torch.arange(5).view(1, -1).expand(2, -1), cache)
        want = m.prefill(torch.cat((torch.arange(30), torch.arange(5))).view(1, -1), m.alloc_cache(64))
    torch.testing.assert_close(got[:1], want, rtol=1e-4, atol=1e-4)


def test_the_tensors_of_a_quantised_cache_stay_its_own(L):
    """Their addresses are part of the cache: a layer's tensor cannot be exchanged for another behind its back."""
    c = QuantKVCache(2, 1, 2, 16, 128, 8, CPU)
    for ts in (c.k, c.v, c.scale, c.sequence(0).k):
        with pytest.raises(TypeError):
            ts[0] = torch.zeros_like(ts[0])
    for name in ("k", "v", "scale", "status"):
        with pytest.raises(AttributeError):
            setattr(c, name, getattr(c, name))


def test_another_prefix_in_a_caches_place_is_noticed():
    """A prefix cache exchanged for another of the same length: a step is refused, prepare() drops what was captured."""
    m = Qwen3Model(Qwen3Config(**TINY)).eval()
    cache = m.alloc_prefix_cache(8, 4, 2)
    cache.prefix.cur_len = 6
    dec = GraphDecoder(m, cache, mode="dense")
    dec.prepare(6)
    dec.graph, dec._captured = Replayed(), (6, False)
    cache.prefix = m.alloc_cache(8)
    cache.prefix.cur_len = 6
    with pytest.raises(ValueError, match="prefix has changed"):
        dec.step(torch.zeros(2, 1, dtype=torch.long), 6)
    dec.prepare(6)
    assert dec.graph is None
