"""Workloads of the decoding operators: shared-prefix attention and token sampling.

``listed()`` names the measured cases and ``draw(rng)`` gives more of the same ranges; ``prepare`` makes the inputs of a
case on the GPU, ``run`` makes one pass through its operator (the plain torch expressions, or the framework's kernels
when ``own`` is set), ``work`` counts the bytes and operations that a pass cannot do without and ``exact`` evaluates the
operator's definition in 64 bits.

Shared-prefix attention: ``samples`` continuations of each of ``groups`` prompts decode together. Every continuation
has its own keys and values (the tokens generated so far, ``own_keys`` slots with ``lengths[b]`` in use) and reads its
prompt's keys and values, which are stored once. Query i of continuation b sees the whole prompt and its own positions
j <= lengths[b] - queries + i.

Sampling: one token for each row of logits from one uniform number a row. Weights exp((x - max) / temperature); the
candidates in descending order of x (ties: lowest index first) are cut to the first top_k, then to the shortest
prefix that holds top_p of the weight that is left, then to weights of at least min_p of the largest; the token is the first
kept index whose running weight (in index order) passes u times the kept weight.
"""
import math

import numpy as np
import torch

own = False

_HEADS = {            # (query heads, key / value heads, head dim)
    "tiny": (4, 4, 64),      # yoco_tiny
    "small": (6, 2, 128),    # yoco_small
    "3b": (24, 8, 128),      # yoco_3b
    "mqa": (8, 1, 128),      # one key / value head
}
_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _attn(name, heads, groups, samples, queries, prefix, own_keys, dtype="bf16", ragged=True):
    return {"name": name, "op": "attention", "heads": heads, "groups": groups, "samples": samples, "queries": queries,
            "prefix": prefix, "own_keys": own_keys, "dtype": dtype, "ragged": ragged}


def _samp(name, rows, vocab, mode, dtype="bf16", peaked=True):
    return {"name": name, "op": "sample", "rows": rows, "vocab": vocab, "mode": mode, "dtype": dtype, "peaked": peaked}


def listed():
    return [
        # two continuations of a short prompt on the test model: launch latency
        _attn("attn_tiny_2x37", "tiny", 1, 2, 1, 37, 5),
        # eight samples of a one-page prompt on the one-GPU test model
        _attn("attn_small_8x1000", "small", 1, 8, 1, 1000, 33),
        # 32 samples of a 16k prompt, up to 256 tokens in: the usual decode step of the 3B model
        _attn("attn_3b_32x16384", "3b", 1, 32, 1, 16384, 256),
        # 128 samples of a needle-length prompt: enough rows a head that the matrix products bound it
        _attn("attn_3b_128x32768", "3b", 1, 128, 1, 32768, 512),
        # four prompts of different lengths, 16 samples each, half precision
        _attn("attn_3b_4x16x8191_fp16", "3b", 4, 16, 1, 8191, 200, dtype="fp16"),
        # scoring 20 answers of 24 tokens to one question in a single pass
        _attn("attn_3b_20x24q_2000", "3b", 1, 20, 24, 2000, 24, ragged=False),
        # 16 rows of the test model's vocabulary
        _samp("sample_16x1024_fp32", 16, 1024, "top_p", dtype="fp32"),
        # a single stream: one row of the 3B vocabulary
        _samp("sample_1x100288_top_p", 1, 100288, "top_p"),
        # a batch with the usual top-k and top-p together
        _samp("sample_64x100288_top_k_p", 64, 100288, "top_k_p"),
        # no filter at all: every token keeps its weight (exploration in reinforcement learning)
        _samp("sample_256x100288_plain", 256, 100288, "temperature"),
        # an odd vocabulary in 32 bits, from a model early in training: a flat distribution, min-p
        _samp("sample_96x65537_min_p_fp32", 96, 65537, "min_p", dtype="fp32", peaked=False),
        # requests with settings of their own, rows that start at odd addresses
        _samp("sample_400x50001_mixed", 400, 50001, "mixed"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    if rng.random() < 0.5:
        heads = rng.choice(list(_HEADS))
        hq, _, d = _HEADS[heads]
        groups = rng.choice([1, 1, 2, 4])
        samples = _log_int(rng, 1, 128 // groups)
        queries = 1 if rng.random() < 0.7 else _log_int(rng, 2, 32)
        prefix = _log_int(rng, 1, 32768)
        keys = max(queries, _log_int(rng, 1, 512))
        most = 128 * 24 * (32768 + 512) * 128
        cost = groups * samples * queries * hq * (prefix + keys) * d
        if cost > most:                        # at most the largest listed case
            prefix = max(1, prefix * most // cost - keys)
        c = _attn("", heads, groups, samples, queries, prefix, keys, rng.choice(["bf16", "bf16", "fp16"]),
                  rng.random() < 0.8)
    else:
        vocab = _log_int(rng, 512, 131072)
        rows = _log_int(rng, 1, min(512, 256 * 100288 // vocab))
        c = _samp("", rows, vocab, rng.choice(["top_p", "top_k", "top_k_p", "temperature", "min_p", "mixed"]),
                  rng.choice(["bf16", "bf16", "fp16", "fp32"]), rng.random() < 0.75)
    del c["name"]
    return c


def _lengths(case):
    """(prefix lengths by group, own lengths by row): plain lists that follow from the case alone."""
    G, n, P, S, q = (case[k] for k in ("groups", "samples", "prefix", "own_keys", "queries"))
    if not case["ragged"]:
        return [P] * G, [S] * (G * n)
    pre = [P - (g * 2741) % (P // 2 + 1) for g in range(G)]
    return pre, [S - (b * 7919) % (S - q + 1) // 2 for b in range(G * n)]


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed) * 2 + 1)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    dt = _DTYPES[case["dtype"]]
    if case["op"] == "attention":
        hq, hk, d = _HEADS[case["heads"]]
        G, B, q = case["groups"], case["groups"] * case["samples"], case["queries"]
        pre, lens = _lengths(case)
        # scores with a spread of two, as a trained model's heads have; cache slots past a row's length hold what an
        # unused allocation may hold
        st = {"case": case,
              "q": (2 * normal(B, q, hq, d)).to(dt),
              "prefix_k": normal(G, case["prefix"], hk, d).to(dt), "prefix_v": normal(G, case["prefix"], hk, d).to(dt),
              "k": normal(B, case["own_keys"], hk, d).to(dt), "v": normal(B, case["own_keys"], hk, d).to(dt),
              "prefix_lengths": torch.tensor(pre, dtype=torch.int32, device="cuda"),
              "lengths": torch.tensor(lens, dtype=torch.int32, device="cuda")}
        junk = torch.arange(case["own_keys"], device="cuda")[None, :] >= st["lengths"][:, None]
        st["v"].masked_fill_(junk[:, :, None, None], float("nan"))
        junk = torch.arange(case["prefix"], device="cuda")[None, :] >= st["prefix_lengths"][:, None]
        st["prefix_v"].masked_fill_(junk[:, :, None, None], float("inf"))
        return st
    N, V = case["rows"], case["vocab"]
    if case["peaked"]:                         # a broad floor and a few dozen likely tokens above it
        x = 2.0 * normal(N, V)
        m = min(64, V)
        at = torch.rand(N, V, generator=gen, device="cuda").topk(m, dim=1).indices
        lift = 17.0 - 0.3 * torch.arange(m, device="cuda", dtype=torch.float32) + normal(N, m)
        x.scatter_add_(1, at, lift)
    else:
        x = 0.7 * normal(N, V)
    x = x.to(dt)
    x[:, :2] = float("-inf")                   # begin-of-text and padding are never drawn
    p = {"temperature": torch.full((N,), 0.8), "top_k": torch.zeros(N, dtype=torch.int32),
         "top_p": torch.ones(N), "min_p": torch.zeros(N)}
    mode = case["mode"]
    if mode in ("top_k", "top_k_p"):
        p["top_k"].fill_(50)
    if mode in ("top_p", "top_k_p"):
        p["top_p"].fill_(0.95)
    if mode == "temperature":
        p["temperature"].fill_(1.0)
    if mode == "min_p":
        p["min_p"].fill_(0.05)
    if mode == "mixed":
        r = torch.arange(N)
        p["temperature"] = torch.tensor([0.0, 0.6, 0.8, 1.0, 1.3])[r % 5]
        p["top_k"] = torch.tensor([0, 50, 20, 0, 200, 1, 0], dtype=torch.int32)[r % 7]
        p["top_p"] = torch.tensor([1.0, 0.95, 0.9, 1.0])[r % 4]
        p["min_p"] = torch.tensor([0.0, 0.0, 0.02])[r % 3]
    st = {k: v.to("cuda") for k, v in p.items()}
    st.update(case=case, logits=x, u=torch.rand(N, generator=gen, device="cuda"))
    return st


# ---------------------------------------------------------------------------------------------------------------------
# plain forms


def _attention_plain(q, prefix_k, prefix_v, k, v, lengths, prefix_lengths):
    B, Lq, Hq, D = q.shape
    G, P, Hk = prefix_k.shape[:3]
    S, n, rep = k.shape[1], B // G, Hq // Hk
    qf = q.float().mul(D ** -0.5).view(B, Lq, Hk, rep, D).permute(0, 2, 1, 3, 4)            # [B, Hk, Lq, rep, D]
    own_key = torch.arange(S, device=q.device)
    pre_key = torch.arange(P, device=q.device)
    pre_ok = pre_key < prefix_lengths[:, None]                                              # [G, P]
    own_any = own_key < lengths[:, None]                                                    # [B, S]
    last = lengths[:, None] - Lq + torch.arange(Lq, device=q.device)                        # [B, Lq]
    own_ok = (own_key <= last[:, :, None]) & own_any[:, None, :]                            # [B, Lq, S]
    pk = prefix_k.float().masked_fill(~pre_ok[:, :, None, None], 0).permute(0, 2, 3, 1)     # [G, Hk, D, P]
    pv = prefix_v.float().masked_fill(~pre_ok[:, :, None, None], 0).permute(0, 2, 1, 3)     # [G, Hk, P, D]
    ok = k.float().masked_fill(~own_any[:, :, None, None], 0).permute(0, 2, 3, 1)           # [B, Hk, D, S]
    ov = v.float().masked_fill(~own_any[:, :, None, None], 0).permute(0, 2, 1, 3)           # [B, Hk, S, D]
    grouped = qf.reshape(G, n, Hk, Lq * rep, D).transpose(1, 2).reshape(G, Hk, n * Lq * rep, D)
    s0 = (grouped @ pk).masked_fill(~pre_ok[:, None, None, :], float("-inf"))
    s0 = s0.view(G, Hk, n, Lq * rep, P).transpose(1, 2).reshape(B, Hk, Lq * rep, P)
    s1 = (qf.reshape(B, Hk, Lq * rep, D) @ ok).view(B, Hk, Lq, rep, S)
    s1 = s1.masked_fill(~own_ok[:, None, :, None, :], float("-inf")).view(B, Hk, Lq * rep, S)
    top = torch.maximum(s0.amax(-1, keepdim=True), s1.amax(-1, keepdim=True))
    top = torch.where(top == float("-inf"), torch.zeros_like(top), top)
    s0, s1 = torch.exp(s0 - top), torch.exp(s1 - top)
    total = s0.sum(-1, keepdim=True) + s1.sum(-1, keepdim=True)
    g0 = s0.view(G, n, Hk, Lq * rep, P).transpose(1, 2).reshape(G, Hk, n * Lq * rep, P)
    o = (g0 @ pv).view(G, Hk, n, Lq * rep, D).transpose(1, 2).reshape(B, Hk, Lq * rep, D) + s1 @ ov
    o = torch.where(total > 0, o / total, torch.zeros_like(o))
    return o.view(B, Hk, Lq, rep, D).permute(0, 2, 1, 3, 4).reshape(B, Lq, Hq, D).to(q.dtype)


def _sample_plain(logits, u, temperature, top_k, top_p, min_p):
    # weights and running sums in 64 bits: the token is decided by comparisons between sums over the vocabulary
    N, V = logits.shape
    x = logits.double()
    x = torch.where(torch.isnan(x), torch.full_like(x, float("-inf")), x)
    order = torch.sort(x, dim=-1, descending=True, stable=True).indices
    first = order[:, :1]
    top = x.gather(1, first)
    t = temperature.double()[:, None]
    greedy = t <= 0
    d = torch.where(x == top, torch.zeros_like(x), x - top)
    w = torch.exp(d / torch.where(greedy, torch.ones_like(t), t))
    w = torch.where(greedy, torch.zeros_like(w).scatter(1, first, 1.0), w)
    w = torch.where(x == float("-inf"), torch.zeros_like(w), w)
    ws = w.gather(1, order)
    rank = torch.arange(V, device=x.device)[None, :]
    k = top_k[:, None].long()
    keep = (rank < k) | (k <= 0)
    ws = torch.where(keep, ws, torch.zeros_like(ws))
    run_ = torch.cumsum(ws, -1)
    before = torch.cat([torch.zeros_like(run_[:, :1]), run_[:, :-1]], -1)
    p = top_p.double()[:, None]
    keep &= (before < p * run_[:, -1:]) | (p >= 1) | (rank == 0)
    keep &= ws >= min_p.double()[:, None]
    keep |= rank == 0
    kept = torch.zeros_like(keep).scatter(1, order, keep)
    wk = torch.where(kept, w, torch.zeros_like(w))
    run_ = torch.cumsum(wk, -1)
    total = run_[:, -1:]
    pick = (run_ <= u.double()[:, None] * total).sum(-1, keepdim=True)
    last = torch.where(wk > 0, rank.expand(N, V), torch.zeros_like(order)).amax(-1, keepdim=True)
    pick = torch.minimum(pick, last)
    logprob = torch.log(wk.gather(1, pick) / total)
    empty = top == float("-inf")
    token = torch.where(empty, torch.full_like(pick, -1), pick)
    logprob = torch.where(empty, torch.full_like(logprob, float("-inf")), logprob)
    return token.squeeze(1), logprob.squeeze(1).float()


def run(state):
    if state["case"]["op"] == "attention":
        args = [state[k] for k in ("q", "prefix_k", "prefix_v", "k", "v", "lengths", "prefix_lengths")]
        if own:
            from faster_yoco_b200 import ops
            return ops.shared_prefix_attention(*args[:5], lengths=args[5], prefix_lengths=args[6])
        return _attention_plain(*args)
    args = [state[k] for k in ("logits", "u", "temperature", "top_k", "top_p", "min_p")]
    if own:
        from faster_yoco_b200 import ops
        return ops.sample(*args, return_logprob=True)
    return _sample_plain(*args)


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "attention":
        hq, hk, d = _HEADS[case["heads"]]
        pre, lens = _lengths(case)
        n, q = case["samples"], case["queries"]
        rows = case["groups"] * n * q
        keys = sum(pre) + sum(lens)
        seen = q * n * sum(pre) + sum(q * ln - q * (q - 1) // 2 for ln in lens)
        return {"bytes": size * d * (2 * hk * keys + 2 * hq * rows) + 4 * (len(pre) + len(lens)),
                "flops": 4 * hq * d * seen}
    N, V = case["rows"], case["vocab"]
    # a comparison, a subtraction, a scaling, an exponential and a sum for each logit
    return {"bytes": N * V * size + N * (5 * 4 + 8 + 4), "flops": 5 * N * V}


# ---------------------------------------------------------------------------------------------------------------------
# definitions in 64 bits


def _attention_exact(case, seed):
    st = prepare(case, seed)
    hq, hk, d = _HEADS[case["heads"]]
    pre, lens = _lengths(case)
    q = st["q"].double()
    out = torch.zeros_like(q)
    for g, plen in enumerate(pre):
        for hh in range(hk):
            heads = slice(hh * (hq // hk), (hh + 1) * (hq // hk))
            pk, pv = st["prefix_k"][g, :plen, hh].double(), st["prefix_v"][g, :plen, hh].double()
            for b in range(g * case["samples"], (g + 1) * case["samples"]):
                keys = torch.cat([pk, st["k"][b, :lens[b], hh].double()])
                vals = torch.cat([pv, st["v"][b, :lens[b], hh].double()])
                s = torch.einsum("ihd,jd->hij", q[b, :, heads], keys) / math.sqrt(d)
                end = torch.arange(case["queries"], device=s.device) + plen + lens[b] - case["queries"] + 1
                s[:, torch.arange(keys.shape[0], device=s.device)[None, :] >= end[:, None]] = float("-inf")
                out[b, :, heads] = torch.einsum("hij,jd->ihd", torch.softmax(s, -1), vals)
    return out


def _sample_exact(case, seed):
    st = {k: (v.double() if k == "logits" else v).cpu().numpy() for k, v in prepare(case, seed).items() if k != "case"}
    tokens, logs = [], []
    for r in range(case["rows"]):
        x = st["logits"][r]
        t, k, p = float(st["temperature"][r]), int(st["top_k"][r]), float(st["top_p"][r])
        order = np.argsort(-x, kind="stable")
        if t <= 0:
            tokens.append(int(order[0]))
            logs.append(0.0)
            continue
        w = np.exp((x[order] - x[order[0]]) / t)
        if k > 0:
            order, w = order[:k], w[:k]
        if p < 1:
            n = 1 + int(np.searchsorted(np.cumsum(w), p * math.fsum(w)))
            order, w = order[:n], w[:n]
        fine = w >= float(st["min_p"][r])
        order, w = order[fine], w[fine]
        at = np.argsort(order)
        order, w = order[at], w[at]
        total = math.fsum(w)
        i = min(int(np.searchsorted(np.cumsum(w), float(st["u"][r]) * total, side="right")), len(w) - 1)
        tokens.append(int(order[i]))
        logs.append(math.log(w[i] / total))
    return torch.tensor(tokens), torch.tensor(logs, dtype=torch.float64)


def exact(case, seed):
    return _attention_exact(case, seed) if case["op"] == "attention" else _sample_exact(case, seed)
