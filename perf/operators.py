"""The token mixers of a decoder layer, as they are measured: attention over the KV cache, the gated delta rule, and the
gated RMSNorm that follows it.  Every case is one call on data that is already on the GPU.

The plain forms are elementary torch operations in f32; `exact` states the definitions again in 64 bits.  With `own` true the
same inputs go through the C ABI of this repository (`CudaBackend.launch_attention_kv`, `launch_gated_delta_rule`,
`launch_rms_norm_silu_gate`).
"""
import math

import numpy as np
import torch

own = False

# Heads as (query heads, KV heads, head size): the shapes of the repository's benchmark configurations, and one
# with large heads and a small group (generic).
HEADS = ((28, 4, 128), (32, 8, 128), (32, 8, 64), (16, 2, 256))
KV = ("q8_0", "q8_0_words", "f16")   # the three layouts of the KV cache
BLOCK = {"q8_0": 34, "q8_0_words": 36}  # bytes of a block of 32 values


def listed():
    return [
        # The latency of a reply: one token of one conversation, 2048 positions behind it.
        _attn("attend 1 x 2048 q8_0", "decode", "f32", "q8_0", 1, 2048, 2048, 2048, HEADS[0]),
        # A full server: 64 conversations whose lengths are anywhere up to 32768, the quantised cache of the resident path.
        _attn("attend 64 x 32768 words", "decode", "f32", "q8_0_words", 64, 1, 32768, 32768, HEADS[0]),
        # Eight conversations of some length over an f16 cache, activations in f16.
        _attn("attend 8 x 8192 f16", "decode", "f16", "f16", 8, 5000, 8192, 8192, HEADS[1]),
        # A short prompt of a small model from its first token, all in f32.
        _attn("attend prompt 512 f32", "chunk", "f32", "q8_0", 512, 512, 512, 1024, HEADS[2]),
        # A long prompt from its first token, f16 activations.
        _attn("attend prompt 4096 f16", "chunk", "f16", "q8_0", 4096, 4096, 4096, 4096, HEADS[0]),
        # The next piece, of odd length, of a prompt that is already 7001 positions long.
        _attn("attend piece 1001 f16", "chunk", "f16", "q8_0_words", 1001, 8002, 8002, 9000, HEADS[1]),
        # One token of one conversation through the recurrent layer.
        _delta("delta 1 x 1", 1, 1, 1, 16, 32),
        # One token of each of 64 conversations: the states are what has to move.
        _delta("delta 64 x 1", 64, 1, 1, 16, 32),
        # A prompt of 4096 tokens.
        _delta("delta 1 x 4096", 1, 4096, 4096, 16, 32),
        # Eight prompts of odd lengths, with states from earlier pieces.
        _delta("delta 8 x 1500", 8, 100, 1500, 16, 32),
        # The norm of a decode step: one token, 32 heads.
        _norm("gated norm 1 x 32", 1, 32, 128),
        # The norm of a prompt.
        _norm("gated norm 4096 x 32", 4096, 32, 128),
    ]


def _attn(name, form, act, kv, tokens, low, high, slots, heads):
    """decode: `tokens` sequences, one row each, of `low` to `high` visible slots; chunk: rows of one sequence, the last of
    which sees `high` slots."""
    c = {"op": "attention", "form": form, "act": act, "kv": kv, "tokens": tokens, "low": low, "high": high, "slots": slots,
         "q_heads": heads[0], "kv_heads": heads[1], "head": heads[2]}
    return c if name is None else {"name": name, **c}


def _delta(name, sequences, low, high, k_heads, v_heads):
    c = {"op": "delta", "sequences": sequences, "low": low, "high": high, "k_heads": k_heads, "v_heads": v_heads, "head": 128}
    return c if name is None else {"name": name, **c}


def _norm(name, tokens, heads, head):
    c = {"op": "norm", "tokens": tokens, "heads": heads, "head": head}
    return c if name is None else {"name": name, **c}


def draw(rng):
    def size(low, high):  # spread over the logarithm
        return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))

    kind = rng.choice(("decode", "decode", "chunk", "chunk", "delta", "delta", "delta", "norm"))
    if kind == "decode":
        tokens, high = size(1, 64), size(16, 32768)
        return _attn(None, "decode", rng.choice(("f32", "f16")), rng.choice(KV[:2]) if tokens * high > 500000 else rng.choice(KV),
                     tokens, max(1, high // rng.randint(1, 8)), high, high + rng.randint(0, 64), rng.choice(HEADS[:3]))
    if kind == "chunk":
        heads, act = rng.choice(HEADS), rng.choice(("f32", "f16"))
        tokens, before = size(2, 4096), rng.choice((0, size(1, 8192)))
        tokens = min(tokens, max(2, 240 * 10 ** 6 // ((tokens + before) * heads[0] * heads[2] // 128)))
        return _attn(None, "chunk", act, rng.choice(KV), tokens, tokens + before, tokens + before, tokens + before + rng.randint(0, 64), heads)
    if kind == "delta":
        k_heads = rng.choice((4, 8, 16))
        if rng.random() < 0.4:  # decode
            return _delta(None, size(1, 64), 1, rng.choice((1, 1, 4)), k_heads, k_heads * rng.choice((1, 2)))
        high = size(16, 4096)
        return _delta(None, rng.randint(1, max(1, 6000 // high)), max(1, high // rng.randint(1, 16)), high, k_heads, k_heads * rng.choice((1, 2)))
    return _norm(None, size(1, 4096), rng.choice((16, 24, 32)), rng.choice((64, 128)))


# ------------------------------------------------------------------------------------------------- inputs

def _lengths(case):
    """Visible slots of each decode row / tokens of each sequence, up to the upper end of the range: a part of the case, whatever
    the seed."""
    n = case["tokens"] if case["op"] == "attention" else case["sequences"]
    rng = np.random.default_rng((n, case["low"], case["high"]))
    ls = rng.integers(case["low"], case["high"] + 1, n)
    ls[rng.integers(0, n)] = case["high"]
    return [int(x) for x in ls]


def _cache(gen, case, n):
    """One layer's K or V bytes of n sequences [n, slots, bytes]: N(0, 1) values under a scale of their own per channel, packed
    as the cache's write packs them."""
    slots, width = case["slots"], case["kv_heads"] * case["head"]
    per = width * 2 if case["kv"] == "f16" else width // 32 * BLOCK[case["kv"]]
    out = torch.empty(n, slots, per, dtype=torch.uint8, device="cuda")
    channel = torch.rand(width, generator=gen, device="cuda") * 1.5 + 0.25
    for s in range(n):
        x = torch.randn(slots, width, generator=gen, device="cuda") * channel
        if case["kv"] == "f16":
            out[s] = x.half().view(torch.uint8)
            continue
        x = x.view(slots, width // 32, 32)
        d = x.abs().amax(2, keepdim=True) / 127
        q = torch.round(x / d).clamp(-127, 127)
        b = out[s].view(slots, width // 32, BLOCK[case["kv"]])
        if case["kv"] == "q8_0":
            b[..., :2] = d.half().view(torch.uint8)
            b[..., 2:] = q.to(torch.int8).view(torch.uint8)
        else:
            b[..., :4] = d.view(torch.uint8)
            b[..., 4:] = (q + 128).to(torch.uint8)
    return out


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    rand = lambda *shape: torch.randn(*shape, generator=gen, device="cuda")  # noqa: E731
    s = dict(case)
    if case["op"] == "attention":
        decode, T = case["form"] == "decode", case["tokens"]
        n = T if decode else 1
        s["q"] = (rand(T, case["q_heads"], case["head"]) * 1.5).to(_type(case))
        s["k"], s["v"] = _cache(gen, case, n), _cache(gen, case, n)
        s["out"] = torch.empty_like(s["q"])
        s["scale"] = case["head"] ** -0.5
        s["start"] = 0 if decode else case["high"] - T
        s["sequences"] = n
        s["longest"] = case["high"]
        if decode:
            s["pos"] = torch.tensor(_lengths(case), dtype=torch.int32, device="cuda") - 1
            s["seq"] = torch.arange(T, dtype=torch.int32, device="cuda")
        else:
            s["pos"] = s["seq"] = None
    elif case["op"] == "delta":
        ls = _lengths(case)
        T, K, V, D = sum(ls), case["k_heads"], case["v_heads"], case["head"]
        s["lengths"], s["T"] = ls, T
        s["cu"] = torch.tensor([0] + ls, dtype=torch.int32, device="cuda").cumsum(0, dtype=torch.int32)
        s["q"], s["k"] = rand(T, K, D), rand(T, K, D)
        s["v"] = rand(T, V, D)
        # log decays as a softplus of the gate's projection gives them under a rate of its own per head, and write strengths
        rate = torch.rand(V, generator=gen, device="cuda") * 0.5 + 0.02
        s["g"] = -rate * torch.log1p(torch.exp(rand(T, V) - 1))
        s["beta"] = torch.sigmoid(rand(T, V))
        s["state"] = rand(len(ls), V, D, D) * 0.2
        s["state_out"], s["out"] = torch.empty_like(s["state"]), torch.empty_like(s["v"])
        s["scale"] = D ** -0.5
    else:
        shape = (case["tokens"], case["heads"], case["head"])
        s["x"], s["gate"] = rand(*shape), rand(*shape)
        s["w"] = 1 + 0.02 * rand(case["head"])
        s["out"] = torch.empty(shape, device="cuda")
    if own:
        _handle(s)
    return s


def _type(case):
    return torch.float32 if case["act"] == "f32" else torch.float16


def _handle(s):
    """What a program that serves keeps beside its data: the backend and the operator's workspace."""
    import agention_infer_b200 as agn
    s["be"] = be = _backend(agn)
    if s["op"] == "attention":
        s["kv_dtype"] = {"f16": agn.AGN_F16, "q8_0": agn.AGN_Q8_0, "q8_0_words": agn.AGN_KV_Q8_0_WORDS}[s["kv"]]
        s["act_dtype"] = agn.AGN_F32 if s["act"] == "f32" else agn.AGN_F16
        n = be.attention_kv_workspace_bytes(s["tokens"], s["q_heads"], s["kv_heads"], s["head"], s["slots"], s["pos"] is not None)
    elif s["op"] == "delta":
        n = be.gated_delta_rule_workspace_bytes(s["T"], len(s["lengths"]), s["k_heads"], s["v_heads"], s["head"], s["head"])
    else:
        return
    s["workspace"] = torch.empty(max(n, 1), dtype=torch.uint8, device="cuda")


_backends = []


def _backend(agn):
    if not _backends:
        _backends.append(agn.CudaBackend(torch.cuda.current_device()))
        _backends[0].set_stream(torch.cuda.current_stream().cuda_stream or 1)  # 1: CUDA's legacy default stream
    return _backends[0]


# ------------------------------------------------------------------------------------------------- one pass

def run(s):
    if own:
        be = s["be"]
        if s["op"] == "attention":
            be.launch_attention_kv(s["q"], s["k"], s["v"], s["kv_dtype"], s["tokens"], s["q_heads"], s["kv_heads"], s["head"],
                                   s["slots"], pos=s["pos"], pos_start=s["start"], seq=s["seq"], n_seqs=s["sequences"],
                                   scale=s["scale"], act_dtype=s["act_dtype"], out=s["out"], workspace=s["workspace"])
            return s["out"]
        if s["op"] == "delta":
            be.launch_gated_delta_rule(s["q"], s["k"], s["v"], s["g"], s["beta"], s["state"], s["T"], len(s["lengths"]),
                                       s["k_heads"], s["v_heads"], s["head"], s["head"], cu_seqlens=s["cu"], scale=s["scale"],
                                       l2norm_eps=1e-6, state_out=s["state_out"], out=s["out"], workspace=s["workspace"])
            return {"out": s["out"], "state": s["state_out"]}
        return be.launch_rms_norm_silu_gate(s["x"], s["gate"], s["w"], s["tokens"] * s["heads"], s["head"], 1e-6, out=s["out"])
    if s["op"] == "attention":
        return _attention(s)
    if s["op"] == "delta":
        return _delta_rule(s)
    y = s["x"] * torch.rsqrt((s["x"] * s["x"]).mean(2, keepdim=True) + 1e-6) * s["w"]
    return y * (s["gate"] / (1 + torch.exp(-s["gate"])))


def _values(s, cache, longest):
    """[sequences, longest, kv_heads, head] in f32."""
    b = cache[:, :longest]
    if s["kv"] == "f16":
        x = b.view(torch.float16).float()
    else:
        b = b.unflatten(2, (-1, BLOCK[s["kv"]]))
        if s["kv"] == "q8_0":
            x = b[..., :2].contiguous().view(torch.float16).float() * b[..., 2:].contiguous().view(torch.int8).float()
        else:
            x = b[..., :4].contiguous().view(torch.float32) * (b[..., 4:].float() - 128)
    return x.reshape(b.shape[0], longest, s["kv_heads"], s["head"])


def _attention(s):
    T, G, L = s["tokens"], s["q_heads"] // s["kv_heads"], s["longest"]
    n, rows = (T, 1) if s["pos"] is not None else (1, T)
    last = s["pos"].view(T, 1) if s["pos"] is not None else s["start"] + torch.arange(T, device="cuda").view(1, T)
    # [sequence, KV head, row of the group, ...]: the rows of a KV head's group share its keys and values
    q = s["q"].float().view(n, rows, s["kv_heads"], G, s["head"]).permute(0, 2, 3, 1, 4).reshape(n, s["kv_heads"], G * rows, s["head"])
    k, v = _values(s, s["k"], L), _values(s, s["v"], L)
    x = q @ k.permute(0, 2, 3, 1) * s["scale"]
    hidden = torch.arange(L, device="cuda").view(1, 1, 1, L) > last.view(n, 1, rows, 1).expand(n, G, rows, 1).reshape(n, 1, G * rows, 1)
    x.masked_fill_(hidden, -math.inf)
    x -= x.amax(3, keepdim=True)
    x.exp_()
    o = x @ v.permute(0, 2, 1, 3) / x.sum(3, keepdim=True)
    return o.view(n, s["kv_heads"], G, rows, s["head"]).permute(0, 3, 1, 2, 4).reshape(T, s["q_heads"], s["head"]).to(s["q"].dtype)


def _delta_rule(s):
    """In chunks: with the decay summed inside the chunk, the writes of a chunk solve (I + A) D = beta (V - decay K S) for a strictly
    lower triangular A, and the state is carried from chunk to chunk."""
    V, D, n, most = s["v_heads"], s["head"], len(s["lengths"]), max(s["lengths"])
    C = min(64, most)
    N = -(-most // C)
    # the rows of each sequence side by side, padded with rows that write and decay nothing
    at = torch.arange(N * C, device="cuda")
    there = at.view(1, -1) < (s["cu"][1:] - s["cu"][:-1]).view(n, 1)
    index = torch.where(there, s["cu"][:-1].view(n, 1) + at.view(1, -1), 0).long()
    mask = there.view(n, N * C, 1, 1).float()

    def laid(x):  # [n, heads, chunks, C, D]
        return (x[index] * mask).view(n, N, C, x.shape[1], -1).permute(0, 3, 1, 2, 4)

    unit = lambda x: x * torch.rsqrt((x * x).sum(-1, keepdim=True) + 1e-6)  # noqa: E731
    q, k = laid(unit(s["q"]) * s["scale"]), laid(unit(s["k"]))
    q, k = (x.repeat_interleave(V // s["k_heads"], 1) for x in (q, k))
    v, beta = laid(s["v"]), laid(s["beta"].unsqueeze(2))
    g = laid(s["g"].unsqueeze(2)).squeeze(4).double().cumsum(3)
    low = torch.ones(C, C, device="cuda", dtype=torch.bool).tril()
    gap = torch.exp((g.unsqueeze(4) - g.unsqueeze(3)).masked_fill(~low, -math.inf)).float()
    whole, rest = torch.exp(g).float().unsqueeze(4), torch.exp(g[..., -1:] - g).float().unsqueeze(4)
    end = whole[:, :, :, -1:]
    kt = k.transpose(3, 4)
    A = (beta * (k @ kt) * gap).tril(-1)
    R = torch.cat((beta * v, beta * whole * k), 4)
    for i in range(1, C):  # forward substitution, all chunks at once
        R[:, :, :, i] -= (A[:, :, :, i, :i].unsqueeze(3) @ R[:, :, :, :i]).squeeze(3)
    P, qd, kr = (q @ kt) * gap, q * whole, (k * rest).transpose(3, 4)
    S, out = s["state"], []
    for c in range(N):
        d = R[:, :, c, :, :D] - R[:, :, c, :, D:] @ S
        out.append(qd[:, :, c] @ S + P[:, :, c] @ d)
        S = end[:, :, c] * S + kr[:, :, c] @ d
    o = torch.stack(out, 2).permute(0, 2, 3, 1, 4).reshape(n, N * C, V, D)
    return {"out": o[there], "state": S}


# ------------------------------------------------------------------------------------------------- work, 64 bits

def work(case):
    if case["op"] == "attention":
        T, H, d = case["tokens"], case["q_heads"], case["head"]
        width = case["kv_heads"] * d
        slot = 2 * (2 * width if case["kv"] == "f16" else width // 32 * BLOCK[case["kv"]])
        io = 2 * T * H * d * (4 if case["act"] == "f32" else 2)
        if case["form"] == "decode":
            seen = sum(_lengths(case))
            return {"bytes": seen * slot + io, "flops": 4 * seen * H * d}
        return {"bytes": case["high"] * slot + io, "flops": 4 * T * (case["high"] - (T - 1) / 2) * H * d}
    if case["op"] == "delta":
        T, V, D = sum(_lengths(case)), case["v_heads"], case["head"]
        rows = T * 4 * (2 * case["k_heads"] * D + 2 * V * D + 2 * V)
        return {"bytes": rows + 2 * 4 * case["sequences"] * V * D * D, "flops": 6 * T * V * D * D}
    n = case["tokens"] * case["heads"] * case["head"]
    return {"bytes": 12 * n, "flops": 8 * n}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        x, z = s["x"].double(), s["gate"].double()
        return s["w"].double() * x / torch.sqrt((x ** 2).sum(-1, keepdim=True) / case["head"] + 1e-6) * z * torch.sigmoid(z)
    if case["op"] == "delta":  # token by token
        V, D, rep = case["v_heads"], case["head"], case["v_heads"] // case["k_heads"]
        out, S = torch.empty(s["T"], V, D, dtype=torch.float64, device="cuda"), s["state"].double()
        first = torch.tensor(np.cumsum([0] + s["lengths"][:-1]), device="cuda")
        for t in range(max(s["lengths"])):
            on = torch.tensor([i for i, n in enumerate(s["lengths"]) if n > t], device="cuda")
            r = first[on] + t
            q, k = (s[x][r].double() for x in "qk")
            q, k = (x / torch.sqrt((x ** 2).sum(2, keepdim=True) + 1e-6) for x in (q, k))
            q, k = (x[:, torch.arange(V, device="cuda") // rep] for x in (q * s["scale"], k))
            M = S[on] * torch.exp(s["g"][r].double())[:, :, None, None]
            d = s["beta"][r].double()[:, :, None] * (s["v"][r].double() - (M * k[..., None]).sum(2))
            M += k[..., None] * d[:, :, None, :]
            S[on] = M
            out[r] = (M * q[..., None]).sum(2)
        return {"out": out, "state": S}
    T, G, d = case["tokens"], case["q_heads"] // case["kv_heads"], case["head"]
    out = torch.empty(T, case["q_heads"], d, dtype=torch.float64, device="cuda")

    def head(cache, h, upto):  # [upto, d] of KV head h
        if case["kv"] == "f16":
            return cache[:upto].view(torch.float16)[:, h * d:(h + 1) * d].double()
        size = BLOCK[case["kv"]]
        b = cache[:upto, h * (d // 32) * size:(h + 1) * (d // 32) * size].reshape(upto, d // 32, size)
        if case["kv"] == "q8_0":
            return (b[..., 2:].contiguous().view(torch.int8).double() * b[..., :2].contiguous().view(torch.float16).double()).reshape(upto, d)
        return ((b[..., 4:].double() - 128) * b[..., :4].contiguous().view(torch.float32).double()).reshape(upto, d)

    jobs = [(t, t + 1, n, n - 1) for t, n in enumerate(_lengths(case))] if case["form"] == "decode" else \
        [(a, min(T, a + 512), s["start"] + min(T, a + 512), s["start"] + a) for a in range(0, T, 512)]
    for a, b, upto, pos in jobs:
        c = a if case["form"] == "decode" else 0
        seen = torch.arange(upto, device="cuda")[None, :] <= pos + torch.arange(b - a, device="cuda")[:, None]
        for h in range(case["kv_heads"]):
            k, v = head(s["k"][c], h, upto), head(s["v"][c], h, upto)
            for j in range(h * G, (h + 1) * G):
                x = s["q"][a:b, j].double() @ k.T * d ** -0.5
                out[a:b, j] = torch.softmax(torch.where(seen, x, -math.inf), 1) @ v
    return out
