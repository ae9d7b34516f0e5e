"""Timed cases of three operators of decoding with long caches.

``rows``    keys and values are quantised to 8 or 4 bits as they are written into a cache, and read back
``attend``  one new token per sequence attends over its quantised cache
``prefix``  one new token per sequence attends over a long prefix that the whole batch shares, kept once, and over the
            tokens of its own behind it

The quantised form: a row (one token of one KV head, 128 values) has one scale in 8 bits, and one for each 32 values in
4 bits.  scale = bf16(largest magnitude / 127 or / 7), code = round(value / scale) clamped to +-127 or +-7, stored with
128 or 8 added.  4-bit codes: the 32 runs of four values of a row lie in the order (run % 8, run // 8), the lower nibble
first.  ``scale[b, h, row]`` holds the scales of the key, then those of the value.
"""

import torch

own = False
D = 128                                   # head dimension


def listed():
    return [
        # a decode step writes one token of each of eight sequences, each at its own position
        {"name": "rows_token_8bit", "op": "rows", "bits": 8, "dtype": "bf16", "B": 8, "H": 8, "T": 1, "at": 4000},
        # a prefill chunk of one prompt
        {"name": "rows_chunk_8bit", "op": "rows", "bits": 8, "dtype": "bf16", "B": 1, "H": 8, "T": 2048, "at": 6144},
        # a prefill chunk of a batch
        {"name": "rows_batch_4bit", "op": "rows", "bits": 4, "dtype": "bf16", "B": 8, "H": 8, "T": 2048, "at": 100},
        # an odd remainder of a prompt, of a model in float32, with the KV heads of a tensor-parallel share
        {"name": "rows_odd_4bit_f32", "op": "rows", "bits": 4, "dtype": "f32", "B": 3, "H": 5, "T": 777, "at": 31},
        # a short prompt, one sequence: latency
        {"name": "attend_short_8bit", "op": "attend", "bits": 8, "B": 1, "H": 8, "G": 2, "n": 300, "ragged": False},
        # the default decode workload's context, one sequence
        {"name": "attend_32k_8bit", "op": "attend", "bits": 8, "B": 1, "H": 8, "G": 2, "n": 32768, "ragged": False},
        # a batch of sequences of different lengths, four query heads per KV head
        {"name": "attend_ragged_8bit", "op": "attend", "bits": 8, "B": 16, "H": 8, "G": 4, "n": 8191, "ragged": True},
        # a batch of long contexts
        {"name": "attend_batch_4bit", "op": "attend", "bits": 4, "B": 8, "H": 8, "G": 2, "n": 32768, "ragged": False},
        # a few answers to a short prompt
        {"name": "prefix_short", "op": "prefix", "B": 4, "H": 8, "G": 2, "P": 333, "n": 17, "ragged": True},
        # eight answers to one prompt
        {"name": "prefix_8k", "op": "prefix", "B": 8, "H": 8, "G": 2, "P": 8192, "n": 256, "ragged": True},
        # 32 samples of one long prompt
        {"name": "prefix_32k", "op": "prefix", "B": 32, "H": 8, "G": 2, "P": 32768, "n": 500, "ragged": True},
        # many short questions about one document
        {"name": "prefix_wide", "op": "prefix", "B": 128, "H": 8, "G": 4, "P": 16383, "n": 64, "ragged": True},
    ]


def draw(rng):
    def log(lo, hi):
        return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))

    op = rng.choice(("rows", "attend", "prefix"))
    H = rng.randint(1, 8)
    if op == "rows":
        B = log(1, 16)
        return {"op": op, "bits": rng.choice((8, 4)), "dtype": rng.choice(("bf16", "bf16", "bf16", "f32")), "B": B, "H": H,
                "T": log(1, min(8192, 131072 // (B * H))), "at": rng.randint(0, 9000)}
    G = rng.choice((1, 2, 2, 3, 4, 4, 5, 8))
    if op == "attend":
        B = log(1, 32)
        return {"op": op, "bits": rng.choice((8, 4)), "B": B, "H": H, "G": G, "n": log(1, min(65536, 2097152 // (B * H))),
                "ragged": rng.random() < 0.5}
    B = log(2, 128)
    return {"op": op, "B": B, "H": H, "G": G, "P": log(16, min(32768, 67108864 // (B * H * G))),
            "n": log(1, min(1024, 262144 // (B * H))), "ragged": rng.random() < 0.7}


def lengths(case):
    """Cached tokens of each sequence."""
    B, n = case["B"], case["n"]
    return [max(1, n - (5 * n * b) // (8 * B)) for b in range(B)] if case["ragged"] else [n] * B


def starts(case):
    """The position each sequence's first new row goes to."""
    return [case["at"] + 7 * b for b in range(case["B"])]


def quantised(x, bits):
    """Rows ``x [..., 128]`` -> ``(stored codes uint8, scales bf16 [..., groups])``."""
    groups, most = (1, 127) if bits == 8 else (4, 7)
    x = x.float().reshape(*x.shape[:-1], groups, D // groups)
    top = x.abs().amax(-1)
    scale = (top / torch.full_like(top, most)).to(torch.bfloat16)     # a quotient, not a product with 1 / most
    s = scale.float().unsqueeze(-1)
    code = torch.where(s > 0, (x / s).round().clamp(-most, most), 0.0).to(torch.int32)
    if bits == 8:
        return (code + 128).to(torch.uint8).flatten(-2), scale
    code = (code + 8).unflatten(-1, (8, 4)).transpose(-3, -2).flatten(-3)
    return (code[..., 0::2] + 16 * code[..., 1::2]).to(torch.uint8), scale


def values(code, scale, bits):
    """Stored codes ``[..., 128 * bits / 8]`` and scales ``[..., groups]`` -> float32 rows ``[..., 128]``."""
    if bits == 8:
        return (code.float() - 128.0) * scale.float()
    code = torch.stack((code & 15, code >> 4), -1).flatten(-2).unflatten(-1, (8, 4, 4)).transpose(-3, -2).flatten(-2)
    return ((code.float() - 8.0) * scale.float().unsqueeze(-1)).flatten(-2)


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device=dev).manual_seed(seed)

    def normal(*shape, dtype=torch.bfloat16, mean=0.0, std=1.0):
        return (torch.randn(*shape, generator=g, device=dev) * std + mean).to(dtype)

    B, H = case["B"], case["H"]
    s = {"case": case}
    if case["op"] == "rows":
        # keys and values as the projections leave them: [B, T, H, 128], seen per head; some channels of a key are large
        dtype = torch.float32 if case["dtype"] == "f32" else torch.bfloat16
        T, cap = case["T"], max(starts(case)) + case["T"]
        s["k"] = (torch.randn(B, T, H, D, generator=g, device=dev) * normal(H, D, dtype=torch.float32).exp()
                  + normal(H, D, dtype=torch.float32)).to(dtype).transpose(1, 2)
        s["v"] = normal(B, T, H, D, dtype=dtype).transpose(1, 2)
        s["pos"] = torch.tensor(starts(case), dtype=torch.long, device=dev)
    elif case["op"] == "attend":
        cap = case["n"]
        s["q"] = normal(B * H * case["G"], D, std=2.0)
        s["n"] = torch.tensor(lengths(case), dtype=torch.int32, device=dev)
    if case["op"] != "prefix":
        bits = case["bits"]
        width = D * bits // 8
        s["kc"] = torch.zeros(B, H, cap, width, dtype=torch.uint8, device=dev)
        s["vc"] = torch.zeros(B, H, cap, width, dtype=torch.uint8, device=dev)
        # what lies behind a sequence's last row has never been written
        s["scale"] = torch.full((B, H, cap, 2, 1 if bits == 8 else 4), float("nan"), dtype=torch.bfloat16, device=dev)
        if case["op"] == "attend":
            for b, n in enumerate(lengths(case)):
                s["kc"][b, :, :n], s["scale"][b, :, :n, 0] = quantised(normal(H, n, D, mean=0.7), bits)
                s["vc"][b, :, :n], s["scale"][b, :, :n, 1] = quantised(normal(H, n, D), bits)
        if own:
            from sparse_kv_reads_b200 import QuantAttentionGraph, QuantKVCache
            s["cache"] = QuantKVCache.from_tensors([s["kc"]], [s["vc"]], [s["scale"]], bits)
            if case["op"] == "attend":
                s["attn"] = QuantAttentionGraph(H=B * H * case["G"], H_kv=B * H, d=D, dtype=torch.bfloat16, device=dev)
                s["attn"].n_group = H
        return s
    lens, cap = lengths(case), case["n"] + 8
    s["q"] = normal(B * H * case["G"], D, std=2.0)
    s["kp"], s["vp"] = normal(H, case["P"], D, mean=0.7), normal(H, case["P"], D)
    s["k"], s["v"] = normal(B * H, cap, D, mean=0.7), normal(B * H, cap, D)
    s["n"] = torch.tensor(lens, dtype=torch.int32, device=dev)
    for b, n in enumerate(lens):
        s["k"][b * H:(b + 1) * H, n:] = float("nan")
        s["v"][b * H:(b + 1) * H, n:] = float("nan")
    if own:
        from sparse_kv_reads_b200 import PrefixAttentionGraph
        s["attn"] = PrefixAttentionGraph(B=B, H=H * case["G"], H_kv=H, d=D, dtype=torch.bfloat16, device=dev)
        s["attn"].n_group = H
    return s


def attended(q, k, v, there, prefix=None):
    """Softmax attention in float32: ``q [B, H, G, 128]`` over ``k, v [B, H, L, 128]`` where ``there [B, 1, 1, L]``, and
    over the rows ``prefix = (kp, vp) [H, P, 128]`` of all sequences."""
    B, H, G, _ = q.shape
    q, rows = q.float() * D ** -0.5, there.squeeze(1).unsqueeze(-1)
    e = (q @ torch.where(rows, k.float(), 0.0).transpose(-1, -2)).masked_fill(~there, -torch.inf)
    v = torch.where(rows, v.float(), 0.0)
    top = e.amax(-1, keepdim=True)
    if prefix is not None:
        kp, vp = prefix[0].float(), prefix[1].float()
        ep = (q.transpose(0, 1).reshape(H, B * G, D) @ kp.transpose(-1, -2)).view(H, B, G, -1).transpose(0, 1)
        top = torch.maximum(top, ep.amax(-1, keepdim=True))
    p = (e - top).exp()
    out, total = p @ v, p.sum(-1, keepdim=True)
    if prefix is not None:
        p = (ep - top).exp()
        out = out + (p.transpose(0, 1).reshape(H, B * G, -1) @ vp).view(H, B, G, D).transpose(0, 1)
        total = total + p.sum(-1, keepdim=True)
    return out / total


def run(state):
    case = state["case"]
    B, H = case["B"], case["H"]
    if case["op"] == "rows":
        if own:
            state["cache"].write(0, state["k"], state["v"], state["pos"])
            return state["cache"].read(0, state["pos"], case["T"], dtype=state["k"].dtype)
        bits = case["bits"]
        seq = torch.arange(B, device=state["pos"].device)[:, None, None]
        head = torch.arange(H, device=seq.device)[None, :, None]
        row = state["pos"][:, None, None] + torch.arange(case["T"], device=seq.device)
        state["kc"][seq, head, row], ks = quantised(state["k"], bits)
        state["vc"][seq, head, row], vs = quantised(state["v"], bits)
        state["scale"][seq, head, row] = torch.stack((ks, vs), -2)
        scale = state["scale"][seq, head, row]
        return (values(state["kc"][seq, head, row], scale[..., 0, :], bits).to(state["k"].dtype),
                values(state["vc"][seq, head, row], scale[..., 1, :], bits).to(state["v"].dtype))
    if case["op"] == "attend":
        if own:
            return state["attn"](state["q"], state["cache"], 0, state["n"])
        k = values(state["kc"], state["scale"][..., 0, :], case["bits"])
        v = values(state["vc"], state["scale"][..., 1, :], case["bits"])
        prefix = None
    else:
        if own:
            return state["attn"](state["q"], state["kp"], state["vp"], state["k"], state["v"], state["n"])
        k, v = state["k"].view(B, H, -1, D), state["v"].view(B, H, -1, D)
        prefix = (state["kp"], state["vp"])
    there = (torch.arange(k.shape[2], device=k.device) < state["n"][:, None]).view(B, 1, 1, -1)
    q = state["q"]
    return attended(q.view(B, H, -1, D), k, v, there, prefix).to(q.dtype).view_as(q)


def work(case):
    B, H = case["B"], case["H"]
    if case["op"] == "rows":
        rows, item = B * H * case["T"], 4 if case["dtype"] == "f32" else 2
        stored = 2 * (D * case["bits"] // 8 + 2 * (1 if case["bits"] == 8 else 4))
        # the rows in, the stored form written and read, the rows out; a maximum, a quotient, a rounding, a product
        return {"bytes": rows * (2 * 2 * D * item + 2 * stored), "flops": rows * 2 * D * 4}
    G, total = case["G"], sum(lengths(case))
    io = 2 * B * H * G * D * 2
    if case["op"] == "attend":
        stored = 2 * (D * case["bits"] // 8 + 2 * (1 if case["bits"] == 8 else 4))
        return {"bytes": total * H * stored + io, "flops": total * H * G * D * 4}
    return {"bytes": (case["P"] + total) * H * 2 * D * 2 + io, "flops": (B * case["P"] + total) * H * G * D * 4}


def exact(case, seed):
    """The operators from their definitions, in float64, one KV head of one sequence at a time."""
    s = prepare(case, seed)
    B, H = case["B"], case["H"]
    f64 = torch.float64

    def restored(x, bits):
        most, size = (127, D) if bits == 8 else (7, 32)
        out = torch.empty(x.shape, dtype=f64, device=x.device)
        for c in range(0, D, size):
            part = x[..., c:c + size].to(f64)
            step = (part.abs().max(-1, keepdim=True).values / most).float().to(torch.bfloat16).to(f64)
            out[..., c:c + size] = torch.round(part / step).clamp(-most, most) * step
        return out

    def decoded(code, scale, bits):
        code = code.to(torch.int64)
        if bits == 8:
            return (code - 128).to(f64) * scale.to(f64)
        out = torch.empty(*code.shape[:-1], D, dtype=f64, device=code.device)
        for d in range(D):
            run_, place = d // 4, d % 4
            nibble = ((run_ % 8) * 4 + run_ // 8) * 4 + place          # where value d lies, in nibbles
            out[..., d] = ((code[..., nibble // 2] >> (4 * (nibble % 2)) & 15) - 8).to(f64) * scale[..., d // 32].to(f64)
        return out

    if case["op"] == "rows":
        return restored(s["k"], case["bits"]), restored(s["v"], case["bits"])
    q = s["q"].to(f64).view(B, H, case["G"], D)
    out = torch.empty_like(q)
    for b, n in enumerate(lengths(case)):
        for h in range(H):
            if case["op"] == "attend":
                k = decoded(s["kc"][b, h, :n], s["scale"][b, h, :n, 0], case["bits"])
                v = decoded(s["vc"][b, h, :n], s["scale"][b, h, :n, 1], case["bits"])
            else:
                k = torch.cat((s["kp"][h], s["k"][b * H + h, :n])).to(f64)
                v = torch.cat((s["vp"][h], s["v"][b * H + h, :n])).to(f64)
            weight = torch.softmax(q[b, h] @ k.T / D ** 0.5, dim=-1)
            out[b, h] = weight @ v
    return out.view(-1, D)
