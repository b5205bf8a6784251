"""Attention on the two sparse patterns of language models, as cases that can be timed.

  op "prompt"  ``rode_window_attention``: every query sees the ``window`` keys up to its own position and the first ``sinks``
               keys of its sequence; sequences of any lengths are packed one behind the other.  ``past`` keys of each sequence
               come before its first query (a prompt that is worked off in pieces).
  op "train"   the same with the gradients of queries, keys and values.
  op "step"    ``rode_window_attention_step``: one new token per sequence against a cache of keys and values.
  op "prefix"  ``rode_shared_prefix_attention``: one new token per request; all requests share a long prefix (a system prompt, a
               document, samples of one prompt) and have a cache of their own behind it.

A case's lengths follow from the case alone; values are normal, as projections of normalised activations are.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEVICE = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def _packed(op, dtype, tokens, sequences, heads, kv_heads, dim, window, sinks, past=0):
    """tokens: queries of all sequences; past: the most keys that a sequence has before its first query."""
    return {"op": op, "dtype": dtype, "tokens": tokens, "sequences": sequences, "past": past, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "window": window, "sinks": sinks}


def _step(dtype, batch, capacity, heads, kv_heads, dim, window, sinks, heads_first=False):
    """capacity: rows of the cache per sequence; heads_first: the cache lies head by head instead of token by token."""
    return {"op": "step", "dtype": dtype, "batch": batch, "capacity": capacity, "heads": heads, "kv_heads": kv_heads,
            "dim": dim, "window": window, "sinks": sinks, "heads_first": heads_first}


def _prefix(dtype, batch, prefix, capacity, heads, kv_heads, dim):
    return {"op": "prefix", "dtype": dtype, "batch": batch, "prefix": prefix, "capacity": capacity, "heads": heads,
            "kv_heads": kv_heads, "dim": dim}


def listed():
    return [
        # a short question: the call itself is what costs
        {"name": "prompt_tiny", **_packed("prompt", "bf16", 37, 1, 4, 1, 64, 16, 2)},
        # a batch of prompts of uneven lengths
        {"name": "prompt_ragged", **_packed("prompt", "bf16", 8191, 13, 32, 8, 128, 1024, 4)},
        # one long document
        {"name": "prompt_long", **_packed("prompt", "f16", 32768, 1, 16, 4, 128, 4096, 16)},
        # pieces of prompts behind what the cache holds already; a head dimension that is no power of two
        {"name": "prompt_pieces", **_packed("prompt", "bf16", 2045, 4, 16, 2, 96, 4096, 4, past=8000)},
        # training on packed short texts, as many key heads as query heads
        {"name": "train_packed", **_packed("train", "bf16", 4097, 9, 16, 16, 64, 256, 1)},
        # training on long texts, shared key heads
        {"name": "train_long", **_packed("train", "bf16", 16384, 2, 32, 8, 128, 2048, 4)},
        # a small model in single precision, a head dimension that no tile divides, no sinks
        {"name": "train_f32", **_packed("train", "f32", 1500, 3, 8, 8, 80, 200, 0)},
        # one conversation, just begun
        {"name": "step_tiny", **_step("bf16", 1, 64, 8, 2, 64, 32, 4)},
        # a server's batch in mid-answer
        {"name": "step_batch", **_step("bf16", 64, 8192, 32, 8, 128, 4096, 4)},
        # two very long contexts that are seen whole, with a cache that lies head by head
        {"name": "step_long", **_step("f16", 2, 131072, 16, 4, 128, 131072, 0, heads_first=True)},
        # a few samples of one prompt, single precision
        {"name": "prefix_small", **_prefix("f32", 3, 777, 128, 8, 2, 64)},
        # many requests about one long document
        {"name": "prefix_large", **_prefix("bf16", 96, 16384, 1024, 32, 8, 128)},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    """Sizes over their logarithm; head dimensions 64 and 128 mostly, and others of up to 128; both cache layouts."""
    while True:
        op = rng.choice(["prompt", "prompt", "train", "train", "step", "step", "prefix"])
        dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
        dim = rng.choice([64, 128]) if rng.random() < 0.75 else (8 * rng.randint(2, 16) if dtype != "f32" else 4 * rng.randint(4, 32))
        kv_heads = rng.choice([1, 2, 4, 8])
        heads = kv_heads * rng.choice([1, 2, 4, 8])
        sinks = rng.choice([0, 1, 4, 64])
        if op in ("prompt", "train"):
            tokens = _log_int(rng, 40, 16384 if dtype != "f32" else 4096)
            case = _packed(op, dtype, tokens, min(_log_int(rng, 1, 32), tokens), heads, kv_heads, dim,
                           _log_int(rng, 16, 8192), sinks)
            if op == "prompt" and rng.random() < 0.3:
                case["past"] = _log_int(rng, 10, 8000)
            if case["tokens"] * (case["past"] + case["tokens"] / case["sequences"]) * heads > 4e9:
                continue
        elif op == "step":
            batch = _log_int(rng, 1, 128)
            case = _step(dtype, batch, _log_int(rng, 32, 131072), heads, kv_heads, dim, _log_int(rng, 16, 131072), sinks,
                         rng.random() < 0.3)
        else:
            case = _prefix(dtype, _log_int(rng, 1, 96), _log_int(rng, 100, 32768), _log_int(rng, 16, 2048), heads, kv_heads, dim)
        most = {"train": work(listed()[5]), "prompt": work(listed()[2]), "step": work(listed()[8]), "prefix": work(listed()[11])}[op]
        cost = work(case)
        scale = 16 if dtype == "f32" and op in ("prompt", "train") else 1
        cache = case.get("batch", 0) * case.get("capacity", 0) * kv_heads * dim
        if cost["flops"] * scale <= most["flops"] and cost["bytes"] <= most["bytes"] and cache <= 64 * 8192 * 8 * 128:
            return case


def _lengths(n, total=None, most=None, least=0):
    """n uneven lengths that add up to total, or n uneven lengths from least to most."""
    if total is None:
        rng = random.Random(1000003 * n + most)
        return [rng.randint(least, most) for _ in range(n)]
    rng = random.Random(1000003 * n + total)
    weights = [rng.uniform(0.2, 1.0) for _ in range(n)]
    cuts, run = [0], 0.0
    for w in weights:
        run += w
        cuts.append(round(total * run / sum(weights)))
    return [b - a for a, b in zip(cuts, cuts[1:])]


def _sequences(case):
    """Queries and keys of every packed sequence."""
    queries = _lengths(case["sequences"], total=case["tokens"])
    past = _lengths(case["sequences"], most=case["past"], least=case["past"] // 4)
    return queries, [a + b for a, b in zip(queries, past)]


def _cached(case):
    """Tokens in the cache of every sequence of a step (the new one among them) or of every request behind a prefix."""
    if case["op"] == "step":
        return _lengths(case["batch"], most=case["capacity"], least=max(1, case["capacity"] // 2))
    return _lengths(case["batch"], most=case["capacity"], least=0)


def _pairs(queries, keys, window, sinks):
    """Visible (query, key) pairs of one sequence."""
    a, b = keys - queries, keys
    # positions a to b - 1: all p + 1 keys up to the window's size, then the window and the sinks in front of it
    full = max(a, min(b, window))
    total = (full - a) * (a + 1 + full) // 2 + (b - full) * window
    partly = max(full, min(b, window + sinks))
    total += (partly - full) * (full + partly + 1 - 2 * window) // 2
    return total + sinks * (b - partly)


def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    row = case["dim"] * size
    if case["op"] in ("prompt", "train"):
        queries, keys = _sequences(case)
        pairs = sum(_pairs(a, b, case["window"], case["sinks"]) for a, b in zip(queries, keys)) * case["heads"]
        q_bytes, k_bytes = sum(queries) * case["heads"] * row, sum(keys) * case["kv_heads"] * row
        if case["op"] == "prompt":
            return {"bytes": 2 * q_bytes + 2 * k_bytes, "flops": 4 * case["dim"] * pairs}
        return {"bytes": 4 * q_bytes + 4 * k_bytes, "flops": 14 * case["dim"] * pairs}
    q_bytes = case["batch"] * case["heads"] * row
    if case["op"] == "step":
        seen = sum(_pairs(1, n, case["window"], case["sinks"]) for n in _cached(case))
        return {"bytes": 2 * q_bytes + 2 * seen * case["kv_heads"] * row, "flops": 4 * case["dim"] * seen * case["heads"]}
    tokens = sum(_cached(case))
    return {"bytes": 2 * q_bytes + 2 * (tokens + case["prefix"]) * case["kv_heads"] * row,
            "flops": 4 * case["dim"] * (tokens + case["prefix"] * case["batch"]) * case["heads"]}


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, dtype=dtype, device=DEVICE, generator=gen)

    def ints(values):
        return torch.tensor(values, dtype=torch.int32, device=DEVICE)

    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    state = {"case": case}
    if case["op"] in ("prompt", "train"):
        queries, keys = _sequences(case)
        state["queries"], state["keys"] = queries, keys
        state["q"] = normal(sum(queries), heads, dim)
        state["k"], state["v"] = normal(sum(keys), kv_heads, dim), normal(sum(keys), kv_heads, dim)
        state["q_offsets"] = ints([sum(queries[:i]) for i in range(len(queries) + 1)])
        state["k_offsets"] = ints([sum(keys[:i]) for i in range(len(keys) + 1)]) if keys != queries else None
        if case["op"] == "train":
            state["dout"] = normal(sum(queries), heads, dim)
            for name in ("q", "k", "v"):
                state[name].requires_grad_()
        return state
    batch, capacity = case["batch"], case["capacity"]
    state["cached"] = _cached(case)
    state["lengths"] = ints(state["cached"])
    state["q"] = normal(batch, heads, dim)
    for name in ("k_cache", "v_cache"):
        if case.get("heads_first"):
            state[name] = normal(batch, kv_heads, capacity, dim).transpose(1, 2)
        else:
            state[name] = normal(batch, capacity, kv_heads, dim)
    if case["op"] == "prefix":
        state["prefix_k"], state["prefix_v"] = normal(case["prefix"], kv_heads, dim), normal(case["prefix"], kv_heads, dim)
    return state


def _plain_scores(q, k, visible):
    """Softmax over the visible keys: q [kv, group, rows, dim], k [kv, keys, dim], visible [rows, keys] or None."""
    s = torch.matmul(q, k[:, None].transpose(-1, -2)) * (1.0 / math.sqrt(q.shape[-1]))
    if visible is not None:
        s = torch.where(visible, s, torch.full_like(s, -math.inf))
    e = torch.exp(s - s.amax(-1, keepdim=True).clamp_min(torch.finfo(torch.float32).min))
    return e / e.sum(-1, keepdim=True).clamp_min(torch.finfo(torch.float32).tiny)


def _plain_packed(state, train):
    case = state["case"]
    heads, kv_heads, dim, dtype = case["heads"], case["kv_heads"], case["dim"], DTYPES[case["dtype"]]
    group = heads // kv_heads
    q, k, v = (state[n].detach().float() for n in ("q", "k", "v"))
    out = torch.empty_like(q)
    if train:
        dout = state["dout"].float()
        dq, dk, dv = torch.empty_like(q), torch.zeros_like(k), torch.zeros_like(v)
    q0 = k0 = 0
    for nq, nk in zip(state["queries"], state["keys"]):
        ks, vs = k[k0:k0 + nk].transpose(0, 1), v[k0:k0 + nk].transpose(0, 1)
        for a in range(0, nq, 512):
            b = min(nq, a + 512)
            rows = slice(q0 + a, q0 + b)
            end = nk - nq + b

            def by_group(x):
                return x[rows].view(b - a, kv_heads, group, dim).permute(1, 2, 0, 3)

            def by_row(x):
                return x.permute(2, 0, 1, 3).reshape(b - a, heads, dim)

            pos = torch.arange(nk - nq + a, end, device=DEVICE)[:, None]
            key = torch.arange(end, device=DEVICE)
            visible = (key <= pos) & ((key > pos - case["window"]) | (key < case["sinks"]))
            p = _plain_scores(by_group(q), ks[:, :end], visible)
            o = torch.matmul(p, vs[:, None, :end])
            out[rows] = by_row(o)
            if train:
                do = by_group(dout)
                dv[k0:k0 + end] += torch.matmul(p.transpose(-1, -2), do).sum(1).transpose(0, 1)
                ds = torch.matmul(do, vs[:, None, :end].transpose(-1, -2))
                ds = p * (ds - (do * o).sum(-1, keepdim=True)) * (1.0 / math.sqrt(dim))
                dq[rows] = by_row(torch.matmul(ds, ks[:, None, :end]))
                dk[k0:k0 + end] += torch.matmul(ds.transpose(-1, -2), by_group(q)).sum(1).transpose(0, 1)
        q0, k0 = q0 + nq, k0 + nk
    if train:
        return [x.to(dtype) for x in (out, dq, dk, dv)]
    return out.to(dtype)


def _plain_cached(state):
    case = state["case"]
    kv_heads, dim = case["kv_heads"], case["dim"]
    q = state["q"].float().view(case["batch"], kv_heads, -1, dim)
    out = torch.zeros_like(q)
    if case["op"] == "prefix":
        prefix_k, prefix_v = state["prefix_k"].float().transpose(0, 1), state["prefix_v"].float().transpose(0, 1)
    for b, n in enumerate(state["cached"]):
        k, v = state["k_cache"][b, :n].float().transpose(0, 1), state["v_cache"][b, :n].float().transpose(0, 1)
        if case["op"] == "prefix":
            k, v, visible = torch.cat([prefix_k, k], 1), torch.cat([prefix_v, v], 1), None
        else:
            key = torch.arange(n, device=DEVICE)
            visible = (key >= n - case["window"]) | (key < case["sinks"])
        p = _plain_scores(q[b][:, :, None], k, visible)
        out[b] = torch.matmul(p, v[:, None])[:, :, 0]
    return out.reshape(state["q"].shape).to(state["q"].dtype)


def run(state):
    case = state["case"]
    op = case["op"]
    if not own:
        return _plain_packed(state, op == "train") if op in ("prompt", "train") else _plain_cached(state)
    from rode_b200 import rode_attention as A

    if op in ("prompt", "train"):
        out = A.rode_window_attention(state["q"], state["k"], state["v"], case["window"], case["sinks"],
                                      q_offsets=state["q_offsets"], k_offsets=state["k_offsets"])
        if op == "prompt":
            return out
        return [out.detach(), *torch.autograd.grad(out, (state["q"], state["k"], state["v"]), state["dout"])]
    if op == "step":
        return A.rode_window_attention_step(state["q"], state["k_cache"], state["v_cache"], state["lengths"], case["window"],
                                            case["sinks"])
    return A.rode_shared_prefix_attention(state["q"], state["prefix_k"], state["prefix_v"], state["k_cache"], state["v_cache"],
                                          state["lengths"])


def _exact_rows(q, keys, values, seen):
    """Rows q [rows, dim] against keys [n, dim] in 64 bits, seen [rows, n] truth values: probabilities and outputs."""
    logits = (q @ keys.T) / math.sqrt(q.shape[1])
    logits = logits.masked_fill(~seen, -math.inf)
    p = torch.exp(logits - torch.logsumexp(logits, 1, keepdim=True))
    return p, p @ values


def exact(case, seed):
    state = prepare(case, seed)
    group = case["heads"] // case["kv_heads"]
    q = state["q"].detach().double()
    out = torch.zeros_like(q)
    if case["op"] in ("step", "prefix"):
        for b, n in enumerate(state["cached"]):
            if case["op"] == "step":
                index = [j for j in range(n) if j < case["sinks"] or n - j <= case["window"]]
                index = torch.tensor(index, device=DEVICE)
                keys, values = state["k_cache"][b][index].double(), state["v_cache"][b][index].double()
            else:
                keys = torch.cat([state["prefix_k"].double(), state["k_cache"][b][:n].double()])
                values = torch.cat([state["prefix_v"].double(), state["v_cache"][b][:n].double()])
            seen = torch.ones(group, keys.shape[0], dtype=torch.bool, device=DEVICE)
            for h in range(case["kv_heads"]):
                mine = slice(h * group, (h + 1) * group)
                out[b, mine] = _exact_rows(q[b, mine], keys[:, h], values[:, h], seen)[1]
        return out
    train = case["op"] == "train"
    k, v = state["k"].detach().double(), state["v"].detach().double()
    if train:
        dout = state["dout"].double()
        dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    q0 = k0 = 0
    for nq, nk in zip(state["queries"], state["keys"]):
        for a in range(0, nq, 1024):
            b = min(nq, a + 1024)
            # keys that some query of these rows sees: the sinks, and from the first row's window to the last row's position
            lo = max(0, nk - nq + a - case["window"] + 1)
            index = torch.cat([torch.arange(min(case["sinks"], lo), device=DEVICE), torch.arange(lo, nk - nq + b, device=DEVICE)])
            at = torch.arange(nk - nq + a, nk - nq + b, device=DEVICE)
            back = at[:, None] - index[None, :]
            seen = (back >= 0) & ((back < case["window"]) | (index[None, :] < case["sinks"]))
            for h in range(case["heads"]):
                keys, values = k[k0 + index, h // group], v[k0 + index, h // group]
                mine = q[q0 + a:q0 + b, h]
                p, o = _exact_rows(mine, keys, values, seen)
                out[q0 + a:q0 + b, h] = o
                if train:
                    g = dout[q0 + a:q0 + b, h]
                    dv[:, h // group].index_add_(0, k0 + index, p.T @ g)
                    ds = p * (g @ values.T - (g * o).sum(1)[:, None]) / math.sqrt(case["dim"])
                    dq[q0 + a:q0 + b, h] = ds @ keys
                    dk[:, h // group].index_add_(0, k0 + index, ds.T @ mine)
        q0, k0 = q0 + nq, k0 + nk
    return [out, dq, dk, dv] if train else out
