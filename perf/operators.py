"""The attention half of a decoder layer around the ternary projections, operator by operator, for timing and comparison.

Three operators, each in a plain form (elementary torch operations in 32 bits, 64 for angles) and, where `own` is true, as a
program calls the library:

  adapters   low-rank adapters of many requests beside one shared projection:  Y[m] = base[m] + scale_s * B_s (A_s x[m]),  s = slot[m]
  heads      what lies between the q+k+v projection and the attention: norms of the query and key heads, the rotation by
             position, the rounding to 16 bits, and the scatter of keys and values to their cache rows
  attention  causal attention with grouped heads over packed sequences, their keys in a cache of rows (prompts, chunks of
             prompts, single tokens)

Shapes are the decoder layer of the library's benchmark (K=2560: 20 query heads and 5 key/value heads of 128; the q+k+v
projection N=3840, gate+up N=13824, down K=6912 N=2560) or generic.
"""
import math
import random

import torch

own = False

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
CODES = {"f16": 1, "bf16": 2, "f32": 3}


# ------------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # one request decoding one token: its adapter beside the fused q+k+v projection; pure latency
        {"name": "adapters one token", "op": "adapters", "M": 1, "K": 2560, "N": 3840, "slots": 8, "rank_lo": 16, "rank_hi": 16, "type": "bf16",
         "order": "mixed", "none": 0.0, "mix": 1},
        # a decode batch of many requests, ranks and order as they come, some rows without an adapter; the down projection
        {"name": "adapters decode batch", "op": "adapters", "M": 48, "K": 6912, "N": 2560, "slots": 32, "rank_lo": 8, "rank_hi": 64, "type": "f16",
         "order": "mixed", "none": 0.15, "mix": 2},
        # a few hundred rows of many requests (chunks of prompts among decoding rows), odd count, the k/v projection
        {"name": "adapters mixed rows", "op": "adapters", "M": 333, "K": 2560, "N": 640, "slots": 24, "rank_lo": 1, "rank_hi": 100, "type": "bf16",
         "order": "packed", "none": 0.1, "mix": 3},
        # whole prompts of several requests in one packed batch, gate+up projection: the largest read and write of outputs
        {"name": "adapters prompts", "op": "adapters", "M": 3001, "K": 2560, "N": 13824, "slots": 8, "rank_lo": 16, "rank_hi": 64, "type": "bf16",
         "order": "packed", "none": 0.1, "mix": 4},
        # one decoding request: float rows of the projection in, bfloat16 heads out
        {"name": "heads one token", "op": "heads", "T": 1, "q_heads": 20, "kv_heads": 5, "dim": 128, "rotated": 128, "interleaved": False, "norm": True,
         "in": "f32", "out": "bf16", "far": 30000, "capacity": 64, "mix": 5},
        # a prompt of 4096 tokens behind the projection, keys and values to scattered cache rows
        {"name": "heads prompt", "op": "heads", "T": 4096, "q_heads": 20, "kv_heads": 5, "dim": 128, "rotated": 128, "interleaved": False, "norm": True,
         "in": "f32", "out": "bf16", "far": 130000, "capacity": 5000, "mix": 6},
        # a long packed batch, 16-bit rows in, neighbouring pairs, only part of each head rotated
        {"name": "heads packed batch", "op": "heads", "T": 20011, "q_heads": 32, "kv_heads": 8, "dim": 64, "rotated": 48, "interleaved": True, "norm": True,
         "in": "f16", "out": "f16", "far": 8000, "capacity": 20100, "mix": 7},
        # one decoding request, some 1500 tokens in its cache: latency
        {"name": "attention one token", "op": "attention", "kind": "decode", "batch": 1, "lo": 1501, "hi": 1501, "chunk": 1, "q_heads": 20, "kv_heads": 5, "dim": 128,
         "type": "bf16", "tail": 0, "mix": 8},
        # a decode batch whose caches differ in length from nothing to 16384 tokens: bytes
        {"name": "attention decode batch", "op": "attention", "kind": "decode", "batch": 32, "lo": 0, "hi": 16384, "chunk": 1, "q_heads": 20, "kv_heads": 5, "dim": 128,
         "type": "f16", "tail": 3, "mix": 9},
        # one long prompt of 8192 tokens: products
        {"name": "attention prompt", "op": "attention", "kind": "prompt", "batch": 1, "lo": 8192, "hi": 8192, "chunk": 1, "q_heads": 20, "kv_heads": 5, "dim": 128,
         "type": "bf16", "tail": 0, "mix": 10},
        # packed prompts of very different lengths, one head of keys per query head, 64 wide
        {"name": "attention packed prompts", "op": "attention", "kind": "prompt", "batch": 13, "lo": 1, "hi": 2500, "chunk": 1, "q_heads": 16, "kv_heads": 16, "dim": 64,
         "type": "f16", "tail": 5, "mix": 11},
        # chunks of prompts against what their caches hold already
        {"name": "attention chunks", "op": "attention", "kind": "chunk", "batch": 4, "lo": 500, "hi": 20000, "chunk": 256, "q_heads": 20, "kv_heads": 5, "dim": 128,
         "type": "bf16", "tail": 0, "mix": 12},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["adapters", "heads", "attention", "attention"])
    mix = rng.randrange(1 << 30)
    if op == "adapters":
        K, N = 16 * _log(rng, 16, 432), 16 * _log(rng, 4, 864)
        M = _log(rng, 1, max(1, min(4096, 3001 * 13824 // N)))
        hi = _log(rng, 1, 128)
        slots = rng.randint(1, 32)
        return {"op": op, "M": M, "K": K, "N": N, "slots": slots, "rank_lo": rng.randint(1, hi), "rank_hi": hi, "type": rng.choice(["f16", "bf16"]),
                "order": rng.choice(["mixed", "packed"]) if M <= 512 else "packed", "none": rng.choice([0.0, 0.1, 0.3]), "mix": mix}
    if op == "heads":
        dim = rng.choice([32, 64, 80, 96, 128, 256])
        kv = rng.choice([1, 2, 4, 5, 8])
        q = kv * rng.choice([1, 2, 4, 7])
        T = _log(rng, 1, max(1, min(20011, 20011 * 48 * 64 // ((q + 2 * kv) * dim))))
        return {"op": op, "T": T, "q_heads": q, "kv_heads": kv, "dim": dim, "rotated": rng.choice([dim, dim, dim // 2]), "interleaved": rng.random() < 0.4,
                "norm": rng.random() < 0.8, "in": rng.choice(["f32", "f32", "f16", "bf16"]), "out": rng.choice(["f16", "bf16"]), "far": _log(rng, 100, 1000000),
                "capacity": T + rng.randint(0, 300), "mix": mix}
    dim = rng.choice([64, 64, 80, 96, 128, 128, 128, 256])
    kv = rng.choice([1, 2, 4, 5, 8])
    q = kv * rng.choice([1, 2, 4, 8]) if kv <= 4 else kv * rng.choice([1, 2, 4])
    kind = rng.choice(["prompt", "decode", "chunk"])
    if kind == "prompt":
        batch = _log(rng, 1, 16)
        hi = _log(rng, 8, min(4000, int(math.sqrt(2.0e8 / (batch * q)))))
        chunk, lo = 1, rng.randint(0, hi)
    elif kind == "decode":
        batch = _log(rng, 1, 64)
        hi = _log(rng, 16, min(32000, 32 * 16384 * 5 * 128 // (batch * kv * dim)))
        chunk, lo = 1, rng.randint(0, hi)
    else:
        batch, chunk = _log(rng, 1, 8), _log(rng, 2, 600)
        hi = max(chunk, _log(rng, 16, min(20000, int(2.0e8 / (batch * q * chunk)))))
        lo = rng.randint(0, hi)
    return {"op": op, "kind": kind, "batch": batch, "lo": lo, "hi": hi, "chunk": chunk, "q_heads": q, "kv_heads": kv, "dim": dim, "type": rng.choice(["f16", "bf16"]),
            "tail": rng.choice([0, 0, 7]), "mix": mix}


# ------------------------------------------------------------------------------------------------ what a case's "mix" stands for
def _slots(case):
    """Rank and scale of every slot, and the slot of every row (-1: none)."""
    r = random.Random(case["mix"])
    ranks = [r.randint(case["rank_lo"], case["rank_hi"]) for _ in range(case["slots"])]
    scales = [2.0 ** r.randint(-1, 2) / max(1.0, math.sqrt(k)) for k in ranks]
    M, rows = case["M"], []
    while len(rows) < M:
        s = -1 if r.random() < case["none"] else r.randrange(case["slots"])
        rows += [s] * (1 if case["order"] == "mixed" else r.randint(1, max(1, M // 5)))
    return ranks, scales, rows[:M]


def _lengths(case):
    """Queries and keys of every sequence."""
    r = random.Random(case["mix"])
    keys = [r.randint(case["lo"], case["hi"]) for _ in range(case["batch"])]
    if case["batch"] > 1:
        keys[r.randrange(case["batch"])] = case["hi"]
    if case["kind"] == "prompt":
        return keys, keys
    if case["kind"] == "decode":
        return [1] * case["batch"], keys
    return [r.randint(max(1, case["chunk"] // 2), case["chunk"]) for _ in keys], keys  # where the cache is shorter than the chunk, its first rows see nothing


# ------------------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    return {"adapters": _prepare_adapters, "heads": _prepare_heads, "attention": _prepare_attention}[case["op"]](case, seed)


def _prepare_adapters(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    M, K, N, t = case["M"], case["K"], case["N"], TYPES[case["type"]]
    ranks, scales, rows = _slots(case)
    R = max(ranks)
    x = torch.randn(M, K, generator=g, device="cuda")
    x[:, ::7] *= 3.0  # a few channels run larger, as activations do
    A = torch.randn(case["slots"], R, K, generator=g, device="cuda") / math.sqrt(K)
    B = torch.randn(case["slots"], N, R, generator=g, device="cuda") * 0.5
    rank = torch.tensor(ranks, device="cuda")
    lane = torch.arange(R, device="cuda")
    A *= (lane[None, :] < rank[:, None])[:, :, None]  # ranks differ: what lies behind a slot's rank is zero
    B *= (lane[None, :] < rank[:, None])[:, None, :]
    s = {"case": case, "X": x.to(t), "A": A.to(t), "B": B.to(t), "scale": torch.tensor(scales, device="cuda"), "scales": scales, "ranks": ranks,
         "slot": torch.tensor(rows, device="cuda", dtype=torch.int32), "base": torch.randn(M, N, generator=g, device="cuda") * 2.0, "Y": torch.empty(M, N, device="cuda")}
    if own:
        import sptmm_amd as sp

        s["set"] = sp.Adapters(K, N, CODES[case["type"]], case["slots"], R)
        for i, r in enumerate(ranks):
            a, b = s["A"][i, :r].contiguous(), s["B"][i, :, :r].contiguous()
            s["set"].set(i, a.data_ptr(), b.data_ptr(), r, scales[i], torch.cuda.current_stream().cuda_stream)
        s["bytes"] = s["set"].workspace_bytes(M)
        s["ws"] = torch.empty(max(1, s["bytes"]), dtype=torch.uint8, device="cuda")
        torch.cuda.synchronize()
    return s


def _frequencies(case):
    r = case["rotated"]
    return [10000.0 ** (-2.0 * j / r) for j in range(r // 2)]


def _prepare_heads(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    T, q, kv, D = case["T"], case["q_heads"], case["kv_heads"], case["dim"]
    qkv = torch.randn(T, (q + 2 * kv) * D, generator=g, device="cuda") * 1.5
    s = {"case": case, "qkv": qkv.to(TYPES[case["in"]]), "pos": torch.randint(0, case["far"], (T,), generator=g, device="cuda", dtype=torch.int32),
         "row": torch.randperm(case["capacity"], generator=g, device="cuda")[:T].to(torch.int32),
         "gq": 1.0 + 0.2 * torch.randn(D, generator=g, device="cuda"), "gk": 1.0 + 0.2 * torch.randn(D, generator=g, device="cuda"),
         "q": torch.zeros(T, q, D, dtype=TYPES[case["out"]], device="cuda"), "eps": 1e-5,
         "k": torch.randn(case["capacity"], kv, D, generator=g, device="cuda").to(TYPES[case["out"]]),
         "v": torch.randn(case["capacity"], kv, D, generator=g, device="cuda").to(TYPES[case["out"]])}
    s["freq"] = torch.tensor(_frequencies(case), dtype=torch.float64, device="cuda")
    s["k0"], s["v0"] = s["k"].clone(), s["v"].clone()
    if own:
        import sptmm_amd as sp

        w = s["qkv"].element_size()
        at, stride = s["qkv"].data_ptr(), (q + 2 * kv) * D
        s["args"] = sp.HeadsArgs(q=at, k=at + w * q * D, v=at + w * (q + kv) * D, q_stride=stride, k_stride=stride, v_stride=stride, in_type=CODES[case["in"]],
                                 q_out=s["q"].data_ptr(), k_out=s["k"].data_ptr(), v_out=s["v"].data_ptr(), q_out_stride=q * D, k_out_stride=kv * D, v_out_stride=kv * D,
                                 out_type=CODES[case["out"]], tokens=T, q_heads=q, kv_heads=kv, head_dim=D, positions=s["pos"].data_ptr(), kv_rows=s["row"].data_ptr(),
                                 kv_capacity=case["capacity"], q_gain=s["gq"].data_ptr() if case["norm"] else None, k_gain=s["gk"].data_ptr() if case["norm"] else None,
                                 eps=s["eps"], rotation=sp.Rotation(_frequencies(case), case["interleaved"]))
    return s


def _prepare_attention(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    q, kv, D, t = case["q_heads"], case["kv_heads"], case["dim"], TYPES[case["type"]]
    nq, nk = _lengths(case)
    r = random.Random(case["mix"] + 1)
    starts, at = [], 0
    for n in nk:  # every sequence's keys are rows of one cache, with room behind them unless they are packed as the queries are
        starts.append(at)
        at += n + (0 if case["kind"] == "prompt" else r.randint(0, 40))
    total, rows = sum(nq) + case["tail"], max(1, at)
    first = [0]
    for n in nq:
        first.append(first[-1] + n)
    new = lambda *shape: torch.randn(*shape, generator=g, device="cuda")  # noqa: E731
    s = {"case": case, "q": (1.5 * new(total, q, D)).to(t), "k": new(rows, kv, D).to(t), "v": new(rows, kv, D).to(t), "out": new(total, q, D).to(t),
         "first": torch.tensor(first, dtype=torch.int32, device="cuda"), "start": torch.tensor(starts, dtype=torch.int32, device="cuda"),
         "keys": torch.tensor(nk, dtype=torch.int32, device="cuda"), "most_q": max(nq), "most_k": max(nk), "scale": 1.0 / math.sqrt(D)}
    s["out0"] = s["out"].clone()
    if own:
        import sptmm_amd as sp

        packed = case["kind"] == "prompt"  # the keys lie as the queries do
        s["args"] = sp.AttentionArgs(q=s["q"].data_ptr(), k=s["k"].data_ptr(), v=s["v"].data_ptr(), out=s["out"].data_ptr(), type=CODES[case["type"]], q_stride=q * D,
                                     k_stride=kv * D, v_stride=kv * D, out_stride=q * D, kv_rows=rows, q_start=s["first"].data_ptr(),
                                     kv_start=None if packed else s["start"].data_ptr(), kv_len=None if packed else s["keys"].data_ptr(), batch=case["batch"], total_q=total,
                                     max_q=max(nq), max_kv=max(nk), q_heads=q, kv_heads=kv, head_dim=D, scale=s["scale"])
        s["bytes"] = sp.attention_workspace_bytes(s["args"])
        s["ws"] = torch.empty(max(1, s["bytes"]), dtype=torch.uint8, device="cuda")
    return s


# ------------------------------------------------------------------------------------------------ one pass
def run(s):
    op = s["case"]["op"]
    if own:
        import sptmm_amd as sp

        stream = torch.cuda.current_stream().cuda_stream
        if op == "adapters":
            s["set"].apply(s["X"].data_ptr(), s["slot"].data_ptr(), s["case"]["M"], s["base"].data_ptr(), s["Y"].data_ptr(), s["ws"].data_ptr(), s["bytes"], stream)
            return s["Y"]
        if op == "heads":
            sp.heads_norm_rotate(s["args"], stream)
            return {"q": s["q"], "k": s["k"], "v": s["v"]}
        sp.attention(s["args"], s["ws"].data_ptr(), s["bytes"], stream)
        return s["out"]
    return {"adapters": _adapters, "heads": _heads, "attention": _attention}[op](s)


def _adapters(s):
    """All slots' first products side by side, each row keeping its own slot's, then all second products summed."""
    n, R, K = s["A"].shape
    M = s["X"].shape[0]
    h = (s["X"].float() @ s["A"].float().reshape(n * R, K).t()).reshape(M, n, R)
    mine = (s["slot"][:, None] == torch.arange(n, device="cuda")[None, :]).float() * s["scale"][None, :]
    h = (h * mine[:, :, None]).reshape(M, n * R)
    return s["base"] + h @ s["B"].float().permute(0, 2, 1).reshape(n * R, -1)


def _rotate(x, cos, sin, rotated, interleaved):
    """x [T][heads][D]; pairs of the first `rotated` elements turned by the token's angles."""
    a = x[..., 0:rotated:2] if interleaved else x[..., : rotated // 2]
    b = x[..., 1:rotated:2] if interleaved else x[..., rotated // 2: rotated]
    u, w = a * cos[:, None] - b * sin[:, None], b * cos[:, None] + a * sin[:, None]
    turned = torch.stack((u, w), -1).flatten(-2) if interleaved else torch.cat((u, w), -1)
    return torch.cat((turned, x[..., rotated:]), -1)


def _heads(s):
    c = s["case"]
    T, q, kv, D = c["T"], c["q_heads"], c["kv_heads"], c["dim"]
    x = s["qkv"].float().reshape(T, q + 2 * kv, D)
    xq, xk, xv = x[:, :q], x[:, q: q + kv], x[:, q + kv:]
    if c["norm"]:
        xq = xq * torch.rsqrt((xq * xq).mean(-1, keepdim=True) + s["eps"]) * s["gq"]
        xk = xk * torch.rsqrt((xk * xk).mean(-1, keepdim=True) + s["eps"]) * s["gk"]
    angle = s["pos"].double()[:, None] * s["freq"][None, :]
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    s["q"].copy_(_rotate(xq, cos, sin, c["rotated"], c["interleaved"]))
    s["k"][s["row"].long()] = _rotate(xk, cos, sin, c["rotated"], c["interleaved"]).to(s["k"].dtype)
    s["v"][s["row"].long()] = xv.to(s["v"].dtype)
    return {"q": s["q"], "k": s["k"], "v": s["v"]}


def _attention(s):
    """Every sequence padded to the longest, all scores at once."""
    c = s["case"]
    q, kv, D = c["q_heads"], c["kv_heads"], c["dim"]
    nq = s["first"][1:] - s["first"][:-1]
    i, j = torch.arange(s["most_q"], device="cuda"), torch.arange(s["most_k"], device="cuda")
    at_q = (s["first"][:-1, None] + torch.minimum(i[None, :], (nq[:, None] - 1).clamp(min=0))).long().clamp(max=s["q"].shape[0] - 1)  # [batch][most_q]
    at_k = (s["start"][:, None] + torch.minimum(j[None, :], (s["keys"][:, None] - 1).clamp(min=0))).long().clamp(max=s["k"].shape[0] - 1)
    b, g = c["batch"], q // kv
    Q = s["q"][at_q].float().reshape(b, -1, kv, g, D).permute(0, 2, 3, 1, 4).reshape(b, kv, g * s["most_q"], D)
    K = s["k"][at_k].float().permute(0, 2, 3, 1).contiguous()
    V = s["v"][at_k].float().permute(0, 2, 1, 3).contiguous()
    seen = (j[None, None, :] <= (s["keys"] - nq)[:, None, None] + i[None, :, None]) & (j[None, None, :] < s["keys"][:, None, None])  # [batch][most_q][most_k]
    S = (Q.contiguous() @ K).reshape(b, kv, g, s["most_q"], -1) * s["scale"]
    S = S.masked_fill_(~seen[:, None, None], float("-inf"))
    top = S.amax(-1, keepdim=True)
    P = S.sub_(torch.where(torch.isfinite(top), top, torch.zeros_like(top))).exp_()
    total = P.sum(-1, keepdim=True)
    O = (P.reshape(b, kv, g * s["most_q"], -1) @ V).reshape(b, kv, g, s["most_q"], D) / torch.where(total > 0, total, torch.ones_like(total))
    O = O.permute(0, 3, 1, 2, 4).reshape(b, s["most_q"], q, D)
    live = i[None, :] < nq[:, None]
    s["out"][at_q[live]] = O[live].to(s["out"].dtype)
    return s["out"]


# ------------------------------------------------------------------------------------------------ the definition in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "adapters":
        y = s["base"].double()
        rows = _slots(case)[2]
        for i, (r, scale) in enumerate(zip(s["ranks"], s["scale"].double())):
            mine = torch.tensor([m for m, at in enumerate(rows) if at == i], dtype=torch.long, device="cuda")
            if len(mine):
                y[mine] += scale * torch.mm(torch.mm(s["X"][mine].double(), s["A"][i, :r].double().t().contiguous()), s["B"][i, :, :r].double().t().contiguous())
        return y
    if case["op"] == "heads":
        T, q, kv, D, n = case["T"], case["q_heads"], case["kv_heads"], case["dim"], case["rotated"] // 2
        x = s["qkv"].double()
        turn = torch.polar(torch.ones(T, n, dtype=torch.float64, device="cuda"), torch.outer(s["pos"].double(), s["freq"]))

        def head(h, gain):
            v = x[:, h * D: (h + 1) * D].clone()
            if case["norm"]:
                v = v / torch.sqrt(v.square().sum(1, keepdim=True) / D + s["eps"]) * gain.double()
            first, second = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if case["interleaved"] else (slice(0, n), slice(n, 2 * n))
            z = torch.complex(v[:, first].contiguous(), v[:, second].contiguous()) * turn
            v[:, first], v[:, second] = z.real, z.imag
            return v

        k, v = s["k0"].double(), s["v0"].double()
        at = s["row"].long()
        for h in range(kv):
            k[at, h] = head(q + h, s["gk"])
            v[at, h] = x[:, (q + kv + h) * D: (q + kv + h + 1) * D]
        return {"q": torch.stack([head(h, s["gq"]) for h in range(q)], 1), "k": k, "v": v}
    q, kv = case["q_heads"], case["kv_heads"]
    out = s["out0"].double()
    nq, nk = _lengths(case)
    at = 0
    for b, (n, m) in enumerate(zip(nq, nk)):
        start = int(s["start"][b])
        for h in range(q):
            for i0 in range(0, n, 4096):
                i1 = min(n, i0 + 4096)
                Q = s["q"][at + i0: at + i1, h].double()
                end = max(0, m - n + i1)
                K, V = s["k"][start: start + end, h // (q // kv)].double(), s["v"][start: start + end, h // (q // kv)].double()
                w = torch.mm(Q, K.t().contiguous()) * s["scale"]
                last = torch.arange(i0, i1, device="cuda") + (m - n)
                w = torch.where(torch.arange(end, device="cuda")[None, :] <= last[:, None], w, torch.full_like(w, -math.inf))
                some = last >= 0
                o = torch.zeros_like(Q)
                if bool(some.any()):
                    o[some] = torch.mm(torch.softmax(w[some], 1), V)
                out[at + i0: at + i1, h] = o
        at += n
    return out


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    if case["op"] == "adapters":
        ranks, _, rows = _slots(case)
        M, K, N = case["M"], case["K"], case["N"]
        some = sum(r >= 0 for r in rows)
        return {"bytes": 2 * some * K + 8 * M * N + 4 * M + sum(2 * ranks[i] * (K + N) for i in set(rows) if i >= 0),
                "flops": sum(2 * ranks[i] * (K + N) for i in rows if i >= 0)}
    if case["op"] == "heads":
        T, n = case["T"], (case["q_heads"] + 2 * case["kv_heads"]) * case["dim"]
        return {"bytes": T * (n * (4 if case["in"] == "f32" else 2) + 2 * n + 8), "flops": 8 * T * n}
    nq, nk = _lengths(case)
    q, kv, D = case["q_heads"], case["kv_heads"], case["dim"]
    pairs = sum(sum(min(m, max(0, m - n + i + 1)) for i in range(n)) for n, m in zip(nq, nk))
    return {"bytes": 2 * D * (2 * q * sum(nq) + 2 * kv * sum(nk)), "flops": 4 * D * q * pairs}
