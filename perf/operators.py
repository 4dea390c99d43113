"""The serving operators' workloads: keys and values appended to a paged cache with the position
rotation, attention of new tokens over that cache, and sampling from logits.

listed() names twelve cases; draw(rng) makes more of the same ranges. prepare(case, seed) makes what a
serving program holds before the call, run(state) is one call (own: through autokernel_amd.kernels;
otherwise in elementary torch operations), exact(case, seed) the same result in 64 bits, work(case) the
bytes and operations the call cannot do without.

Sizes are this package's model shapes (LlamaModel7B: 32 query and 8 KV heads of 128, vocabulary 32000;
the compact LLaMA: 12 / 4 heads of 64; GPT-2 small: 12 heads of 64, vocabulary 50257) and generic ones.
"""
from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
SIZE = {"f16": 2, "bf16": 2, "f32": 4}
DEVICE = "cuda"
MAX_POSITIONS = 40000
MAX_FLOPS = 1.5e11   # of a drawn attention case
MAX_KEYS = 600000    # cached tokens times KV heads of a drawn attention case (largest listed: about 2 million)


def listed() -> list[dict]:
    return [
        # One user's decode step in half precision: a single new token against about a thousand cached ones.
        {"name": "attn_one_token", "op": "attn", "dtype": "f16", "heads": 32, "kv_heads": 8, "head_dim": 128,
         "page": 16, "chunks": "1", "pasts": "1000"},
        # A server's decode step: 64 sequences of very different lengths, one token each.
        {"name": "attn_decode_ragged", "op": "attn", "dtype": "bf16", "heads": 32, "kv_heads": 8, "head_dim": 128,
         "page": 16, "batch": 64, "chunk_lo": 1, "chunk_hi": 1, "past_lo": 200, "past_hi": 8000},
        # A long document's next piece: 512 new tokens after 16000 cached ones.
        {"name": "attn_chunk", "op": "attn", "dtype": "bf16", "heads": 32, "kv_heads": 8, "head_dim": 128,
         "page": 32, "chunks": "512", "pasts": "16001"},
        # A mixed step of GPT-2's heads (one KV head per query head): chunks of prompts beside single tokens.
        {"name": "attn_mixed", "op": "attn", "dtype": "f16", "heads": 12, "kv_heads": 12, "head_dim": 64,
         "page": 64, "chunks": "333,1,1,129,1,1,1,77,1,1,1,1", "pasts": "0,900,17,400,1023,64,5,946,300,711,0,63"},
        # Prompts read for the first time: four of 2048 tokens, nothing cached before them.
        {"name": "attn_prompts", "op": "attn", "dtype": "bf16", "heads": 32, "kv_heads": 8, "head_dim": 128,
         "page": 16, "chunks": "2048,2048,2048,2048", "pasts": "0,0,0,0"},
        # Full precision, the compact LLaMA's heads: a short chunk and single tokens.
        {"name": "attn_f32", "op": "attn", "dtype": "f32", "heads": 12, "kv_heads": 4, "head_dim": 64,
         "page": 16, "chunks": "40,1,1,1", "pasts": "100,2047,500,1300"},
        # One decode step's keys and values of 48 sequences.
        {"name": "append_decode", "op": "append", "dtype": "f16", "heads": 32, "kv_heads": 8, "head_dim": 128,
         "page": 16, "style": "interleaved", "batch": 48, "chunk_lo": 1, "chunk_hi": 1, "past_lo": 1, "past_hi": 9000},
        # Prompts of odd lengths after cached prefixes, 8000 tokens in all.
        {"name": "append_prompts", "op": "append", "dtype": "bf16", "heads": 32, "kv_heads": 8, "head_dim": 128,
         "page": 16, "style": "halves", "chunks": "4097,1,2047,1855", "pasts": "0,77,3000,19"},
        # Full precision, the compact LLaMA's heads.
        {"name": "append_f32", "op": "append", "dtype": "f32", "heads": 12, "kv_heads": 4, "head_dim": 64,
         "page": 24, "style": "interleaved", "chunks": "300,1,1,45", "pasts": "0,1200,333,800"},
        # One user's next token: top-k and top-p over LLaMA's vocabulary.
        {"name": "sample_one", "op": "sample", "dtype": "f16", "rows": 1, "vocab": 32000, "settings": "topk_topp"},
        # 64 users with settings of their own (greedy rows among them) over GPT-2's odd vocabulary, 32-bit logits.
        {"name": "sample_mixed", "op": "sample", "dtype": "f32", "rows": 64, "vocab": 50257, "settings": "mixed"},
        # A large batch over a large vocabulary, nucleus only: every weight counts.
        {"name": "sample_large", "op": "sample", "dtype": "bf16", "rows": 256, "vocab": 131072, "settings": "topp"},
    ]


def _spread(rng: random.Random, lo: float, hi: float) -> int:
    """A whole number spread over the logarithm of [lo, hi]."""
    return max(1, round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


HEADS = [(32, 8, 128), (12, 4, 64), (12, 12, 64), (32, 32, 128), (16, 2, 128), (8, 8, 64), (20, 4, 64)]


def _draw_lengths(rng: random.Random, kv_heads: int) -> tuple[str, str]:
    kind = rng.choice(["decode", "chunk", "mixed"])
    batch = {"decode": _spread(rng, 1, 128), "chunk": rng.randint(1, 4), "mixed": rng.randint(2, 24)}[kind]
    top = max(64, min(16000, MAX_KEYS // (kv_heads * batch)))
    chunks, pasts = [], []
    for _ in range(batch):
        small = kind == "decode" or (kind == "mixed" and rng.random() < 0.7)
        chunks.append(1 if small else _spread(rng, 2, 1500))
        pasts.append(_spread(rng, 1, top) - 1)
    return ",".join(map(str, chunks)), ",".join(map(str, pasts))


def draw(rng: random.Random) -> dict:
    op = rng.choice(["attn", "attn", "append", "sample"])
    dtype = rng.choice(["f16", "bf16", "f16", "bf16", "f32"])
    if op == "sample":
        rows, vocab = _spread(rng, 1, 300), _spread(rng, 1000, 140000)
        rows = max(1, min(rows, 256 * 131072 // vocab))
        return {"op": op, "dtype": dtype, "rows": rows, "vocab": vocab,
                "settings": rng.choice(["topk_topp", "mixed", "topp", "topk", "minp", "plain"])}
    heads, kv_heads, head_dim = rng.choice(HEADS)
    if op == "append":
        chunks, pasts = _draw_lengths(rng, kv_heads)
        return {"op": op, "dtype": dtype, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim,
                "page": rng.choice([1, 8, 16, 24, 32, 64, 128]), "style": rng.choice(["interleaved", "halves"]),
                "chunks": chunks, "pasts": pasts}
    while True:
        chunks, pasts = _draw_lengths(rng, kv_heads)
        case = {"op": op, "dtype": dtype, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim,
                "page": rng.choice([16, 32, 64, 128]), "chunks": chunks, "pasts": pasts}
        if work(case)["flops"] <= (MAX_FLOPS if dtype != "f32" else MAX_FLOPS / 50):
            return case


def _lengths(case: dict) -> tuple[list[int], list[int]]:
    """Each sequence's new tokens and cached tokens before them."""
    if "chunks" in case:
        return [int(x) for x in case["chunks"].split(",")], [int(x) for x in case["pasts"].split(",")]
    rng = random.Random(case["batch"])
    chunks = [rng.randint(case["chunk_lo"], case["chunk_hi"]) for _ in range(case["batch"])]
    return chunks, [_spread(rng, case["past_lo"], case["past_hi"]) for _ in range(case["batch"])]


def work(case: dict) -> dict:
    e = SIZE[case["dtype"]]
    if case["op"] == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * e + case["rows"] * 12, "flops": 4 * n}
    chunks, pasts = _lengths(case)
    tokens = sum(chunks)
    H, Hk, D = case["heads"], case["kv_heads"], case["head_dim"]
    if case["op"] == "append":
        return {"bytes": tokens * (2 * (H + 2 * Hk) * D * e + D * 4), "flops": 3 * tokens * (H + Hk) * D}
    seen = sum(n * p + n * (n + 1) // 2 for n, p in zip(chunks, pasts))
    cached = sum(n + p for n, p in zip(chunks, pasts))
    return {"bytes": 2 * tokens * H * D * e + 2 * cached * Hk * D * e, "flops": 4 * D * H * seen}


def _rotary_tables(dim: int) -> tuple[torch.Tensor, torch.Tensor]:
    inv = 10000.0 ** (-torch.arange(0, dim, 2, dtype=torch.float64, device=DEVICE) / dim)
    ang = torch.arange(MAX_POSITIONS, dtype=torch.float64, device=DEVICE)[:, None] * inv
    return ang.cos().float(), ang.sin().float()


def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=DEVICE, dtype=torch.float32)

    def rand(*shape):
        return torch.rand(*shape, generator=g, device=DEVICE, dtype=torch.float32)

    if case["op"] == "sample":
        R, V = case["rows"], case["vocab"]
        # word frequencies fall with a power of their rank, each row with an exponent of its own
        logits = (-(1.0 + 1.2 * rand(R, 1)) * (rand(R, V) * V + 1.0).log() + 0.5 * randn(R, V) + 8.0).to(dt)
        st = {"case": case, "logits": logits, "u": rand(R)}
        s = case["settings"]
        st["temperature"], st["top_k"], st["top_p"], st["min_p"] = {
            "topk_topp": (0.8, 50, 0.9, 0.0), "topk": (1.0, 200, 1.0, 0.0), "topp": (1.0, 0, 0.95, 0.0),
            "minp": (1.3, 0, 1.0, 0.05), "plain": (0.9, 0, 1.0, 0.0), "mixed": (None,) * 4}[s]
        if s == "mixed":
            st["temperature"] = torch.where(rand(R) < 0.2, torch.zeros(R, device=DEVICE), 0.5 + rand(R))
            st["top_k"] = torch.where(rand(R) < 0.5, 0.0, 1.0 + 99.0 * rand(R)).to(torch.int32)
            st["top_p"] = torch.where(rand(R) < 0.3, torch.ones(R, device=DEVICE), 0.5 + 0.5 * rand(R))
            st["min_p"] = torch.where(rand(R) < 0.5, torch.zeros(R, device=DEVICE), 0.1 * rand(R))
        return st

    chunks, pasts = _lengths(case)
    B, P = len(chunks), case["page"]
    H, Hk, D = case["heads"], case["kv_heads"], case["head_dim"]
    lens = [n + p for n, p in zip(chunks, pasts)]
    starts = [0]
    for n in chunks:
        starts.append(starts[-1] + n)
    width = max(-(-n // P) for n in lens) + 1
    used = sum(-(-n // P) for n in lens)
    pages = used + 3
    order = torch.randperm(pages, generator=g, device=DEVICE).to(torch.int32)  # pages come in no order
    table = torch.zeros(B, width, dtype=torch.int32, device=DEVICE)
    at = 0
    for b, n in enumerate(lens):
        c = -(-n // P)
        table[b, :c] = order[at:at + c]
        at += c
    kc = randn(pages, Hk, P, D).to(dt)
    vc = randn(pages, Hk, P, D).to(dt)
    # q, k and v are column slices of one projection's output
    qkv = randn(starts[-1], (H + 2 * Hk) * D).to(dt)
    st = {"case": case, "k_cache": kc, "v_cache": vc, "table": table, "chunks": chunks, "pasts": pasts,
          "starts": torch.tensor(starts, dtype=torch.int32, device=DEVICE),
          "lens": torch.tensor(lens, dtype=torch.int32, device=DEVICE),
          "q": qkv[:, :H * D].view(-1, H, D), "k": qkv[:, H * D:(H + Hk) * D].view(-1, Hk, D),
          "v": qkv[:, (H + Hk) * D:].view(-1, Hk, D)}
    if case["op"] == "append":
        st["cos"], st["sin"] = _rotary_tables(D)
    return st


def run(state: dict):
    op = state["case"]["op"]
    if own:
        from autokernel_amd import kernels
        if op == "sample":
            return kernels.get("sample")(state["logits"], state["u"], temperature=state["temperature"],
                                         top_k=state["top_k"], top_p=state["top_p"], min_p=state["min_p"])
        if op == "append":
            q = kernels.get("kv_append")(state["k"], state["v"], state["k_cache"], state["v_cache"], state["table"],
                                         state["starts"], state["lens"], state["cos"], state["sin"], q=state["q"],
                                         interleaved=state["case"]["style"] == "interleaved")
            return q, state["k_cache"], state["v_cache"]
        return kernels.get("paged_attention")(state["q"], state["k_cache"], state["v_cache"], state["table"],
                                              state["starts"], state["lens"])
    return {"sample": _plain_sample, "append": _plain_append, "attn": _plain_attention}[op](state)


# ------------------------------------------------------------------------------ plain forms
def _plain_attention(st: dict) -> torch.Tensor:
    q, kc, vc, table = st["q"], st["k_cache"], st["v_cache"], st["table"]
    H, D = q.shape[1:]
    Hk, P = kc.shape[1:3]
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    t0 = 0
    for b, (n, past) in enumerate(zip(st["chunks"], st["pasts"])):
        if n == 0:
            continue
        L = n + past
        ids = table[b, :-(-L // P)].long()
        K = kc[ids].float().transpose(0, 1).reshape(Hk, -1, D)[:, :L]
        V = vc[ids].float().transpose(0, 1).reshape(Hk, -1, D)[:, :L]
        Q = q[t0:t0 + n].float().transpose(0, 1).reshape(Hk, H // Hk * n, D)
        S = torch.matmul(Q, K.transpose(1, 2).contiguous()) * D ** -0.5
        S = S.view(Hk, H // Hk, n, L)
        hidden = torch.arange(L, device=q.device) > torch.arange(past, L, device=q.device)[:, None]
        S.masked_fill_(hidden, float("-inf"))
        S = (S - S.amax(-1, keepdim=True)).exp_()
        total = S.sum(-1, keepdim=True)
        O = torch.matmul(S.view(Hk, -1, L), V).view(Hk, H // Hk, n, D) / total
        out[t0:t0 + n] = O.reshape(H, n, D).transpose(0, 1).to(q.dtype)
        t0 += n
    return out


def _plain_append(st: dict):
    k, v, q, table = st["k"], st["v"], st["q"], st["table"]
    P, D = st["k_cache"].shape[2:]
    B = table.shape[0]
    starts, lens = st["starts"].long(), st["lens"].long()
    t = torch.arange(k.shape[0], device=k.device)
    b = (t[:, None] >= starts[None, 1:]).sum(1).clamp(max=B - 1)
    pos = lens[b] - (starts[b + 1] - starts[b]) + t - starts[b]
    c, s = st["cos"][pos][:, None], st["sin"][pos][:, None]

    def rotate(x):
        x = x.float()
        if st["case"]["style"] == "interleaved":
            x0, x1 = x[..., 0::2], x[..., 1::2]
            return torch.stack((x0 * c - x1 * s, x0 * s + x1 * c), -1).flatten(-2).to(k.dtype)
        x0, x1 = x[..., :D // 2], x[..., D // 2:]
        return torch.cat((x0 * c - x1 * s, x0 * s + x1 * c), -1).to(k.dtype)

    page, off = table[b, pos // P].long(), pos % P
    st["k_cache"][page, :, off] = rotate(k)
    st["v_cache"][page, :, off] = v
    return rotate(q), st["k_cache"], st["v_cache"]


def _column(value, rows: int, device, dtype=torch.float64) -> torch.Tensor:
    if torch.is_tensor(value):
        return value.to(dtype)[:, None]
    if dtype == torch.float64:  # settings are 32-bit numbers
        value = float(np.float32(value))
    return torch.full((rows, 1), value, dtype=dtype, device=device)


def _plain_sample(st: dict) -> torch.Tensor:
    logits, u = st["logits"], st["u"]
    R, V = logits.shape
    T = _column(st["temperature"], R, logits.device)
    top_k = _column(st["top_k"], R, logits.device, torch.int64)
    top_p = _column(st["top_p"], R, logits.device)
    min_p = _column(st["min_p"], R, logits.device)
    x, order = torch.sort(logits.double(), dim=-1, descending=True, stable=True)
    w = ((x - x[:, :1]) / torch.where(T > 0, T, 1.0)).exp()
    keep = w >= min_p
    rank = torch.arange(V, device=logits.device)
    keep &= (top_k <= 0) | (rank < top_k)
    run_ = torch.cumsum(w * keep, -1)
    before = torch.cat((torch.zeros_like(run_[:, :1]), run_[:, :-1]), -1)
    keep &= (top_p >= 1.0) | (before < top_p * run_[:, -1:]) | (rank == 0)
    total = (run_ * keep).amax(-1, keepdim=True)
    n = keep.sum(-1, keepdim=True)
    pick = ((run_ <= u.double()[:, None] * total) & keep).sum(-1, keepdim=True).minimum(n - 1)
    pick = torch.where(T > 0, pick, 0)
    return order.gather(1, pick)[:, 0]


# ------------------------------------------------------------------------------ 64-bit results
def exact(case: dict, seed: int):
    st = prepare(case, seed)
    if case["op"] == "sample":
        return _exact_sample(st)
    if case["op"] == "append":
        return _exact_append(st)
    return _exact_attention(st)


def _exact_attention(st: dict) -> torch.Tensor:
    H, D = st["q"].shape[1:]
    Hk = st["k_cache"].shape[1]
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device=st["q"].device)
    lens, starts = st["lens"].tolist(), st["starts"].tolist()
    for b, L in enumerate(lens):
        first, end = starts[b], starts[b + 1]
        base = L - (end - first)
        pages = st["table"][b].tolist()
        P = st["k_cache"].shape[2]
        pages = pages[:(L + P - 1) // P]
        keys = torch.cat([st["k_cache"][p] for p in pages], 1)[:, :L]
        values = torch.cat([st["v_cache"][p] for p in pages], 1)[:, :L]
        for h in range(H):
            K, V = keys[h * Hk // H].double(), values[h * Hk // H].double()
            for i0 in range(first, end, 1024):
                i1 = min(end, i0 + 1024)
                logit = st["q"][i0:i1, h].double() @ K.T.contiguous() / math.sqrt(D)
                seen = torch.ones_like(logit, dtype=torch.bool).tril(base + i0 - first)
                weight = torch.where(seen, logit, -math.inf)
                weight = torch.exp(weight - torch.logsumexp(weight, 1, keepdim=True))
                out[i0:i1, h] = weight @ V
    return out


def _exact_append(st: dict):
    kc, vc = st["k_cache"].double(), st["v_cache"].double()
    q_out = st["q"].double().clone()
    lens, starts, table = st["lens"].tolist(), st["starts"].tolist(), st["table"].tolist()
    P, D = kc.shape[2:]
    first = torch.arange(0, D, 2) if st["case"]["style"] == "interleaved" else torch.arange(D // 2)
    second = first + (1 if st["case"]["style"] == "interleaved" else D // 2)
    first, second = first.to(kc.device), second.to(kc.device)
    for b, L in enumerate(lens):
        rows = slice(starts[b], starts[b + 1])
        n = starts[b + 1] - starts[b]
        angle = torch.complex(st["cos"][L - n:L].double(), st["sin"][L - n:L].double())[:, None]

        def turn(x):
            y = x.double().clone()
            z = torch.complex(y[..., first], y[..., second]) * angle
            y[..., first], y[..., second] = z.real, z.imag
            return y

        q_out[rows] = turn(st["q"][rows])
        k_new, v_new = turn(st["k"][rows]), st["v"][rows].double()
        for p in range((L - n) // P, -(-L // P)):
            lo, hi = max(p * P, L - n), min((p + 1) * P, L)
            at = slice(lo - p * P, hi - p * P)
            kc[table[b][p], :, at] = k_new[lo - (L - n):hi - (L - n)].transpose(0, 1)
            vc[table[b][p], :, at] = v_new[lo - (L - n):hi - (L - n)].transpose(0, 1)
    return q_out, kc, vc


def _exact_sample(st: dict) -> torch.Tensor:
    def setting(name, dtype):
        v = st[name]
        v = v.cpu().numpy() if torch.is_tensor(v) else np.full(st["logits"].shape[0], v, np.float32)
        return v.astype(dtype)

    T, top_k = setting("temperature", np.float64), setting("top_k", np.int64)
    top_p, min_p = setting("top_p", np.float64), setting("min_p", np.float64)
    u = st["u"].cpu().numpy().astype(np.float64)
    tokens = []
    for r, row in enumerate(st["logits"].float().cpu().numpy().astype(np.float64)):
        if T[r] == 0:
            tokens.append(int(np.argmax(row)))
            continue
        weight = np.exp((row - row.max()) / T[r])
        ids = np.flatnonzero(weight >= min_p[r])
        ids = ids[np.argsort(-row[ids], kind="stable")]
        if top_k[r] > 0:
            ids = ids[:top_k[r]]
        mass = np.cumsum(weight[ids].astype(np.longdouble))
        if top_p[r] < 1:
            # the shortest prefix that reaches top_p of the mass
            ids = ids[:max(1, 1 + int(np.searchsorted(mass, top_p[r] * mass[-1], side="left")))]
            mass = mass[:len(ids)]
        at = int(np.searchsorted(mass, u[r] * mass[-1], side="right"))
        tokens.append(int(ids[min(at, len(ids) - 1)]))
    return torch.tensor(tokens, device=st["logits"].device)
