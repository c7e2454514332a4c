"""The work that the operators of a drafted step are measured on.

A server that drafts feeds the target model, for every request, the last token and a few drafted ones (a chain, or a tree
whose branches share their first tokens) in one step, and keeps the part of them that the target agrees with.  Around the
model's products such a step is four operators:

  tables     block tables grown from the requests' lengths, with every token's request, position, place in the pool and
             ancestors (`step_tables`)
  attention  every drafted token over its request's cached context, the tokens above it in its tree and itself
             (`tree_attention`); one layer
  verify     which drafted tokens the target keeps, and the token behind them, from given random numbers (`verify_drafts`)
  keep       the kept tokens' keys and values into the cache pages, all layers at once (`keep_accepted`)

Node 0 of a request is the token that it has already got (the root); its drafted tokens follow, each behind its parent.
`run` computes the plain form, or calls the framework's kernels where `own` is set.
"""
import math
import random

import numpy as np
import torch

own = False
DEVICE = "cuda:0"

# Query heads, key/value heads and head size: the benchmark's 0.5B, 7B and 1.5B-Deep layers, and generic ones.
HEADS = {"8/2x64": (8, 2, 64), "12/2x128": (12, 2, 128), "6/2x128": (6, 2, 128), "32/8x128": (32, 8, 128), "16/16x64": (16, 16, 64),
         "64/8x128": (64, 8, 128), "16/1x64": (16, 1, 64)}


def listed():
    return [
        # one request in a chat, five tokens behind a short context: the step's latency counts
        {"name": "attention-1x700-n5", "op": "attention", "n": 1, "ctx": 700, "ragged": False, "nodes": 5, "chain": True, "heads": "8/2x64",
         "dtype": "bfloat16", "page": 64, "window": 0, "lens": 1},
        # the benchmark's batch and context, small trees
        {"name": "attention-8x4096-n24", "op": "attention", "n": 8, "ctx": 4096, "ragged": False, "nodes": 24, "chain": False, "heads": "12/2x128",
         "dtype": "bfloat16", "page": 64, "window": 0, "lens": 2},
        # a full server: contexts and trees of all lengths; the cache is what is read
        {"name": "attention-32x16384-n32", "op": "attention", "n": 32, "ctx": 16384, "ragged": True, "nodes": 32, "chain": False, "heads": "32/8x128",
         "dtype": "bfloat16", "page": 64, "window": 0, "lens": 3},
        # wide trees of many query heads: the products count
        {"name": "attention-16x8192-n64", "op": "attention", "n": 16, "ctx": 8192, "ragged": False, "nodes": 64, "chain": False, "heads": "64/8x128",
         "dtype": "bfloat16", "page": 64, "window": 0, "lens": 4},
        # the float32 check path behind a window, small pages
        {"name": "attention-f32-4x1000-n12", "op": "attention", "n": 4, "ctx": 1000, "ragged": True, "nodes": 12, "chain": False, "heads": "8/2x64",
         "dtype": "float32", "page": 16, "window": 300, "lens": 5},
        # one request, a drafted chain with its draft's logits
        {"name": "verify-1x5-v32784", "op": "verify", "n": 1, "nodes": 5, "ragged": False, "chain": True, "vocab": 32784, "greedy": 0.0, "lens": 6},
        # a full server with a large vocabulary, chains drawn from a draft model
        {"name": "verify-64x6-v130049", "op": "verify", "n": 64, "nodes": 6, "ragged": False, "chain": True, "vocab": 130049, "greedy": 0.25, "lens": 7},
        # trees of fixed proposals (no draft distribution), some requests greedy
        {"name": "verify-tree-16x16-v65537", "op": "verify", "n": 16, "nodes": 16, "ragged": True, "chain": False, "vocab": 65537, "greedy": 0.25,
         "lens": 8},
        # a small batch of chains
        {"name": "tables-8x5", "op": "tables", "n": 8, "nodes": 5, "ragged": False, "chain": True, "ctx": 4096, "page": 64, "words": 1, "short": False,
         "lens": 9},
        # a full server's trees, long contexts
        {"name": "tables-512x32", "op": "tables", "n": 512, "nodes": 32, "ragged": True, "chain": False, "ctx": 32768, "page": 64, "words": 1,
         "short": False, "lens": 10},
        # one request of the benchmark's 36 layers
        {"name": "keep-1x5-36x128", "op": "keep", "n": 1, "nodes": 5, "ragged": False, "layers": 36, "width": 128, "page": 64, "dtype": "bfloat16",
         "lens": 11},
        # a full server, 32 layers of 8 key/value heads
        {"name": "keep-64x8-32x1024", "op": "keep", "n": 64, "nodes": 8, "ragged": True, "layers": 32, "width": 1024, "page": 64, "dtype": "bfloat16",
         "lens": 12},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["attention", "attention", "verify", "tables", "keep"])
    seed = rng.randrange(1 << 30)
    if op == "attention":
        heads = rng.choice(sorted(HEADS))
        hq, hkv, dh = HEADS[heads]
        f32 = rng.random() < 0.2
        n, nodes = _log(rng, 1, 32), _log(rng, 1, 64)
        most = (1 << 25) // (hkv * dh) if f32 else (1 << 28) // (hkv * dh)                    # cached tokens in all
        most = min(most, (1 << 33) // (nodes * hq * dh))
        ctx = max(1, min(_log(rng, 8, 16384), most // n))
        return {"op": op, "n": n, "ctx": ctx, "ragged": rng.random() < 0.7, "nodes": nodes, "chain": rng.random() < 0.3, "heads": heads,
                "dtype": "float32" if f32 else "bfloat16", "page": rng.choice([16, 64, 64, 128]), "window": rng.choice([0, 0, 0, _log(rng, 2, 4096)]),
                "lens": seed}
    if op == "verify":
        chain = rng.random() < 0.5
        vocab = _log(rng, 1000, 131072)
        nodes = _log(rng, 1, 8 if chain else 32)
        n = max(1, min(_log(rng, 1, 64), 45_000_000 // (vocab * nodes)))
        return {"op": op, "n": n, "nodes": nodes, "ragged": rng.random() < 0.5, "chain": chain, "vocab": vocab,
                "greedy": rng.choice([0.0, 0.25, 1.0]), "lens": seed}
    if op == "tables":
        words = rng.choice([1, 1, 2, 4])
        n, nodes = _log(rng, 1, 512), _log(rng, 1, 32 * words)
        return {"op": op, "n": max(1, min(n, 16384 // nodes)), "nodes": nodes, "ragged": rng.random() < 0.7, "chain": rng.random() < 0.3,
                "ctx": _log(rng, 1, 32768), "page": rng.choice([16, 64, 128]), "words": words, "short": rng.random() < 0.2, "lens": seed}
    return {"op": op, "n": _log(rng, 1, 64), "nodes": _log(rng, 1, 8), "ragged": rng.random() < 0.6, "layers": _log(rng, 1, 32),
            "width": 64 * _log(rng, 1, 16), "page": rng.choice([16, 64, 128]), "dtype": rng.choice(["bfloat16", "float32"]), "lens": seed}


# ----------------------------------------------------------------------------- the requests of a case
def _requests(case):
    """Cached lengths, token counts and parents of a case's requests (the same for every seed)."""
    rng = random.Random(case["lens"])
    n, nodes, ctx = case["n"], case["nodes"], case.get("ctx", 0)
    held = [rng.randint(ctx // 4, ctx) if case["ragged"] else ctx for _ in range(n)]
    new = [rng.randint(1, nodes) if case["ragged"] else nodes for _ in range(n)]
    chain = case.get("chain", True)
    parents = [[-1] + [i - 1 if chain else rng.randint(max(0, i - 6), i - 1) for i in range(1, m)] for m in new]
    return held, new, parents


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def _cu(new):
    return [0] + np.cumsum(new).tolist()


def _words(parents, words):
    """Every token's ancestors and itself as bits of `words` 64-bit integers."""
    rows = np.zeros((sum(len(p) for p in parents), words), dtype=np.uint64)
    t = 0
    for p in parents:
        first = t
        for i, up in enumerate(p):
            if up >= 0:
                rows[t] = rows[first + up]
            rows[t, i // 64] |= np.uint64(1 << (i % 64))
            t += 1
    return torch.from_numpy(rows.view(np.int64)).to(DEVICE)


def _tables(held, page, gen, extra=0):
    """A pool's pages dealt out in random order: block tables of the held tokens, pages in all."""
    blocks = [-(-h // page) + extra for h in held]
    total = max(1, sum(blocks))
    order = torch.randperm(total, generator=gen, device=DEVICE).to(torch.int32)
    table = torch.full((len(held), max(1, max(blocks))), total, dtype=torch.int32, device=DEVICE)
    at = 0
    for s, b in enumerate(blocks):
        table[s, :b] = order[at:at + b]
        at += b
    return table, total


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed * 1000003 + case["lens"] % 1000003)
    held, new, parents = _requests(case)
    n, T = case["n"], sum(new)
    depth = []
    for p in parents:
        for i, up in enumerate(p):
            depth.append(0 if up < 0 else depth[len(depth) - i + up] + 1)
    s = {"case": case, "cu": _i32(_cu(new)), "held": _i32(held)}
    if case["op"] == "attention":
        hq, hkv, dh = HEADS[case["heads"]]
        dt = getattr(torch, case["dtype"])
        table, pages = _tables(held, case["page"], gen)
        s["table"] = table
        s["pool"] = torch.randn(pages + 1, 2, case["page"], hkv * dh, device=DEVICE, generator=gen, dtype=dt)
        s["q"] = torch.randn(T, hq * dh, device=DEVICE, generator=gen, dtype=dt)
        s["k"] = torch.randn(T, hkv * dh, device=DEVICE, generator=gen, dtype=dt)
        s["v"] = torch.randn(T, hkv * dh, device=DEVICE, generator=gen, dtype=dt)
        s["mask"] = None if case["chain"] else _words(parents, 1)
        s["positions"] = _i32(depth) + torch.repeat_interleave(s["held"], s["cu"].diff()).to(torch.int32)
        s["out"] = torch.empty(T, hq * dh, device=DEVICE, dtype=dt)
        s["dense"] = _dense_rows(new)
    elif case["op"] == "verify":
        V = case["vocab"]
        # a target that is sure of a few tokens over a long tail, and a draft that is near it
        base = torch.randn(T, V, device=DEVICE, generator=gen) * 1.5
        top = (torch.randint(0, V, (T, 1), device=DEVICE, generator=gen) + torch.arange(20, device=DEVICE) * (V // 20)) % V
        base.scatter_(1, top, 8.0 + 2.0 * torch.randn(T, 20, device=DEVICE, generator=gen))
        s["logits"] = base
        draft = base + 0.7 * torch.randn(T, V, device=DEVICE, generator=gen)
        s["temperature"] = torch.where(torch.rand(n, device=DEVICE, generator=gen) < case["greedy"], 0.0,
                                       0.5 + torch.rand(n, device=DEVICE, generator=gen))
        temp = torch.repeat_interleave(s["temperature"], s["cu"].diff())[:, None].clamp_min(1e-3)
        up = torch.tensor([max(u, 0) - i for p in parents for i, u in enumerate(p)], device=DEVICE) + torch.arange(T, device=DEVICE)
        if case["chain"]:  # drawn from the draft's distribution behind the parent (Gumbel's rule)
            noise = -torch.log(-torch.log(torch.rand(T, V, device=DEVICE, generator=gen).clamp(1e-7, 1 - 1e-7)))
            s["tokens"] = (draft / temp + noise)[up].argmax(1).to(torch.int32)
            s["draft"] = draft
        else:              # one of the likelier tokens behind the parent, by its place among its siblings
            seen, place = {}, []
            for r, p in enumerate(parents):
                for u in p:
                    seen[(r, u)] = seen.get((r, u), -1) + 1
                    place.append(seen[(r, u)])
            best = draft.topk(8, dim=1).indices
            s["tokens"] = best[up, torch.tensor([min(x, 7) for x in place], device=DEVICE)].to(torch.int32)
            s["draft"] = None
        s["parents"] = None if case["chain"] else _i32([u for p in parents for u in p])
        s["uniforms"] = torch.rand(T, device=DEVICE, generator=gen)
        width = case["nodes"]
        s["tokens_out"], s["path"] = (torch.empty(n, width, dtype=torch.int32, device=DEVICE) for _ in range(2))
        s["count"] = torch.empty(n, dtype=torch.int32, device=DEVICE)
        s["dense"] = _dense_rows(new)
    elif case["op"] == "tables":
        page = case["page"]
        blocks = [-(-h // page) for h in held]
        grow = sum(-(-(h + m) // page) - b for h, m, b in zip(held, new, blocks))
        widest = max(-(-(h + m) // page) for h, m in zip(held, new))
        used, s["spare"] = sum(blocks), sum(blocks) + grow + 1000   # a pool with room for more than this step
        order = torch.randperm(s["spare"], generator=gen, device=DEVICE).to(torch.int32)
        s["table"] = torch.full((n, widest + 1), s["spare"], dtype=torch.int32, device=DEVICE)
        for r, b in enumerate(blocks):
            s["table"][r, :b] = order[sum(blocks[:r]):sum(blocks[:r]) + b]
        s["free"] = order[used:used + (max(1, grow // 2) if case["short"] else grow + 5)].clone()
        s["blocks"], s["new"] = _i32(blocks), _i32(new)
        s["parents"] = None if case["chain"] else _i32([u for p in parents for u in p])
        s["cu"] = torch.full((n + 1,), -7, dtype=torch.int32, device=DEVICE)
        cap = T + case["lens"] % 3                       # a step of a fixed size may hold a few tokens more
        s["seq_of"], s["positions"], s["slots"] = (torch.full((cap,), -7, dtype=torch.int32, device=DEVICE) for _ in range(3))
        s["masks"] = None if case["chain"] else torch.full((cap, case["words"]), -7, dtype=torch.int64, device=DEVICE)
        if s["parents"] is not None:
            s["parents"] = torch.cat([s["parents"], s["parents"].new_full((cap - T,), -1)])
        s["blocks_out"] = torch.empty(n, dtype=torch.int32, device=DEVICE)
        s["taken"] = torch.empty(1, dtype=torch.int32, device=DEVICE)
    else:
        dt = getattr(torch, case["dtype"])
        L, W, page = case["layers"], case["width"], case["page"]
        sizes, rng = random.Random(case["lens"] + 1), random.Random(seed)   # the pool is as large for every seed
        held = [sizes.randint(0, 2 * page) for _ in range(n)]
        table, pages = _tables([h + m for h, m in zip(held, new)], page, gen)
        s["pool"] = torch.randn(L, pages + 1, 2, page, W, device=DEVICE, generator=gen, dtype=dt)
        s["rows"] = torch.randn(L, 2, T, W, device=DEVICE, generator=gen, dtype=dt)
        host = table.cpu().tolist()
        s["slots"] = _i32([host[r][(h + i) // page] * page + (h + i) % page for r, (h, m) in enumerate(zip(held, new)) for i in range(m)])
        count = [max(1, round(m * 0.6)) for m in new]    # root and kept tokens: the same number for every seed
        path = [[0] + sorted(rng.sample(range(1, m), c - 1)) + [-1] * (case["nodes"] - c) for m, c in zip(new, count)]
        s["path"], s["count"] = _i32(path), _i32(count)
    return s


def _dense_rows(new):
    """Token of row i of every request, requests padded to the longest: indices, and which are real."""
    cu, most = _cu(new), max(new)
    at = [[cu[r] + min(i, m - 1) for i in range(most)] for r, m in enumerate(new)]
    return torch.tensor(at, device=DEVICE), torch.tensor([[i < m for i in range(most)] for m in new], device=DEVICE)


# ----------------------------------------------------------------------------- plain forms
def _ancestors(parents, n_rows):
    """[n, N, N] of 0 and 1: row i's ancestors and itself, by (I + A)(I + A^2)(I + A^4)... of the parent matrix A."""
    a = (parents[..., None] == torch.arange(n_rows, device=parents.device)).float()
    r = torch.eye(n_rows, device=parents.device) + a
    a = a @ a
    r = r + a @ r
    a = a @ a
    r = r + a @ r
    a = a @ a
    r = r + a @ r
    a = a @ a
    r = r + a @ r
    a = a @ a
    r = r + a @ r
    a = a @ a
    r = r + a @ r
    a = a @ a
    return r + a @ r


def _plain_attention(s):
    case = s["case"]
    hq, hkv, dh = HEADS[case["heads"]]
    at, real = s["dense"]
    n, N = at.shape
    held, page = s["held"], case["page"]
    ctx = s["pool"][s["table"].long()]                                        # [n, blocks, 2, page, kv]
    L = ctx.shape[1] * page
    key = torch.arange(L, device=DEVICE)
    valid = key < held[:, None]
    keys = torch.cat([ctx[:, :, 0].reshape(n, L, hkv, dh), s["k"][at].view(n, N, hkv, dh)], 1).float()
    values = torch.cat([ctx[:, :, 1].reshape(n, L, hkv, dh), s["v"][at].view(n, N, hkv, dh)], 1).float()
    q = s["q"][at].view(n, N, hkv, hq // hkv, dh).float()
    pos = s["positions"][at]                                                   # [n, N]
    first = pos[..., None] - case["window"] + 1 if case["window"] > 0 else torch.zeros_like(pos)[..., None]
    see_ctx = valid[:, None, :] & (key >= first)
    if s["mask"] is None:
        see_new = torch.ones(N, N, dtype=torch.bool, device=DEVICE).tril().expand(n, N, N)
    else:
        see_new = (s["mask"][at][..., 0, None] >> torch.arange(N, device=DEVICE)) & 1 == 1
    see = torch.cat([see_ctx, see_new & real[:, None, :]], 2)[:, None, None]   # [n, 1, 1, N, L + N]
    score = torch.matmul(q.permute(0, 2, 3, 1, 4), keys.permute(0, 2, 3, 1)[:, :, None]) * dh ** -0.5
    score = score.masked_fill(~see, -math.inf)
    top = score.amax(-1, keepdim=True).clamp_min(torch.finfo(torch.float32).min)
    p = torch.exp(score - top)
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p, values.permute(0, 2, 1, 3)[:, :, None]) / total.clamp_min(1e-30)
    return o.permute(0, 3, 1, 2, 4).reshape(n, N, hq * dh)[real].to(s["q"].dtype)


def _weights(logits, temperature):
    """exp((l - max) / T) in 64 bits, a row's temperature each."""
    x = logits.double()
    return torch.exp((x - x.amax(-1, keepdim=True)) / temperature[:, None])


def _first_above(weights, u):
    """The first index whose running sum of weights passes u times the whole."""
    run = weights.cumsum(-1)
    return (run > (u.double() * run[..., -1])[..., None]).to(torch.int8).argmax(-1)


def _plain_verify(s):
    at, real = s["dense"]
    n, N = at.shape
    rows = torch.arange(n, device=DEVICE)
    temp = torch.repeat_interleave(s["temperature"], s["cu"].diff()).double()
    greedy = s["temperature"] <= 0
    temp = torch.where(temp > 0, temp, 1.0)
    w = _weights(s["logits"], temp)
    best = s["logits"].argmax(-1)
    tokens = s["tokens"].long()[at]                                            # [n, N]
    u = s["uniforms"][at]
    if s["parents"] is None:
        d = _weights(s["draft"], temp)
        w, d = w / w.sum(-1, keepdim=True), d / d.sum(-1, keepdim=True)
        x = tokens[:, 1:, None]
        p, q = (v[at[:, :-1]].gather(2, x)[..., 0] for v in (w, d))
        ok = torch.where(greedy[:, None], best[at[:, :-1]] == x[..., 0], u[:, 1:].double() * q < p)
        ok = (ok & real[:, 1:]).cumprod(1).bool()
        kept = ok.sum(1)                                                       # drafted tokens kept
        last = at[rows, kept]
        f = w[last] - torch.where((kept == real.sum(1) - 1)[:, None], 0.0, d[last])
        f = f.clamp_min(0)
        f = torch.where(f.sum(-1, keepdim=True) > 0, f, w[last])
        end = torch.where(greedy, best[last], _first_above(f, u[:, 0]))
        accepted = torch.cat([torch.ones(n, 1, dtype=torch.bool, device=DEVICE), ok], 1)
        depth = torch.arange(N, device=DEVICE).expand(n, N)
    else:
        drawn = torch.where(torch.repeat_interleave(greedy, s["cu"].diff()), best, _first_above(w, s["uniforms"]))[at]
        up = s["parents"].long()[at]
        same = (up[:, :, None] == up[:, None, :]) & (tokens[:, :, None] == tokens[:, None, :])
        first = ~(same & torch.ones(N, N, dtype=torch.bool, device=DEVICE).tril(-1) & (real[:, None, :])).any(2)
        hit = (drawn.gather(1, up.clamp_min(0)) == tokens) & first & real
        hit[:, 0] = True
        anc = _ancestors(up, N)
        accepted = ((anc * (~hit)[:, None, :]).sum(2) == 0) & real
        depth = anc.sum(2).long() - 1
        kept = accepted.sum(1) - 1
        end = drawn[rows, (accepted * (depth + 1)).argmax(1)]
    place = torch.where(accepted, depth, N)
    path = torch.full((n, N + 1), -1, dtype=torch.int64, device=DEVICE).scatter_(1, place, torch.arange(N, device=DEVICE).expand(n, N))[:, :N]
    out = torch.full((n, N + 2), -1, dtype=torch.int64, device=DEVICE).scatter_(1, torch.where(accepted & (depth > 0), depth - 1, N + 1), tokens)
    out[rows, kept] = end
    return {"tokens": out[:, :N].int(), "path": path.int(), "count": (kept + 1).int()}


def _plain_tables(s):
    held, new, blocks, table, free, page = s["held"], s["new"], s["blocks"], s["table"], s["free"], s["case"]["page"]
    n, cap = held.numel(), s["seq_of"].numel()
    after = torch.maximum(blocks, (held + new + page - 1) // page)
    grow = after - blocks
    start = grow.cumsum(0) - grow
    col = torch.arange(table.shape[1], device=DEVICE)
    take = (start - blocks)[:, None] + col
    fresh = torch.where(take < free.numel(), free[take.clamp(0, free.numel() - 1)], s["spare"])
    table = torch.where(col < blocks[:, None], table, torch.where(col < after[:, None], fresh, s["spare"]))
    ends = new.cumsum(0)
    cu = torch.cat([ends.new_zeros(1), ends])
    t = torch.arange(cap, device=DEVICE)
    seq = torch.searchsorted(ends, t, right=True)
    there = seq < n
    seq = seq.clamp_max(n - 1)
    i = t - cu[seq]
    at = held[seq] + i
    slot = table[seq, at // page]
    slot = torch.where(slot == s["spare"], -1, slot * page + at % page)
    out = {"cu": cu.int(), "table": table.int(), "blocks": after.int(), "taken": grow.sum().int().reshape(1),
           "seq_of": torch.where(there, seq, s["seq_of"]).int(), "slots": torch.where(there, slot, s["slots"]).int()}
    if s["parents"] is None:
        out["positions"] = torch.where(there, at, s["positions"]).int()
        return out
    N = 64 * s["case"]["words"]
    rows = cu[:-1, None] + torch.arange(N, device=DEVICE)
    real = rows < cu[1:, None]
    anc = _ancestors(torch.where(real, s["parents"][rows.clamp_max(cap - 1)], -1).long(), N)
    flat = anc[real].long()                                                    # [T, N]
    bits = (flat.view(-1, s["case"]["words"], 64) << torch.arange(64, device=DEVICE)).sum(-1)
    T = flat.shape[0]
    out["masks"] = torch.cat([bits, s["masks"][T:]])
    out["positions"] = torch.cat([held[seq[:T]] + flat.sum(-1) - 1, s["positions"][T:]]).int()
    return out


def _plain_keep(s):
    pool, rows, path, count = s["pool"], s["rows"], s["path"].long(), s["count"]
    page = pool.shape[3]
    j = torch.arange(path.shape[1], device=DEVICE)
    kept = j < count[:, None]
    src = (s["cu"][:-1, None] + path)[kept]
    slot = s["slots"][(s["cu"][:-1, None] + j).clamp_max(s["slots"].numel() - 1)][kept].long()
    src, slot = src[slot >= 0], slot[slot >= 0]
    pool[:, slot // page, :, slot % page] = rows[:, :, src].permute(2, 0, 1, 3)
    return pool


_PLAIN = {"attention": _plain_attention, "verify": _plain_verify, "tables": _plain_tables, "keep": _plain_keep}


def run(s):
    case = s["case"]
    if not own:
        return _PLAIN[case["op"]](s)
    from poor_mans_mamba_b200.kernels import ops as K
    if case["op"] == "attention":
        hq, hkv, dh = HEADS[case["heads"]]
        if "scratch" not in s:
            s["scratch"] = K.tree_attention_scratch(DEVICE)
        K.tree_attention(s["q"], s["k"], s["v"], s["pool"], s["table"], s["held"], s["cu"], s["out"], hq, hkv, dh, dh ** -0.5, s["scratch"],
                         mask=s["mask"], positions=s["positions"], window=case["window"])
        return s["out"]
    if case["op"] == "verify":
        if "scratch" not in s:
            s["scratch"] = K.verify_drafts_scratch(*s["logits"].shape, DEVICE)
        K.verify_drafts(s["logits"], s["tokens"], s["cu"], s["uniforms"], s["tokens_out"], s["path"], s["count"], s["scratch"],
                        temperature=s["temperature"], parents=s["parents"], draft_logits=s["draft"])
        return {"tokens": s["tokens_out"], "path": s["path"], "count": s["count"]}
    if case["op"] == "tables":
        K.step_tables(s["held"], s["new"], s["blocks"], s["table"], s["free"], case["page"], s["spare"], s["cu"], s["seq_of"], s["positions"],
                      s["slots"], s["blocks_out"], s["taken"], parents=s["parents"], masks=s["masks"])
        out = {"cu": s["cu"], "table": s["table"], "blocks": s["blocks_out"], "taken": s["taken"], "seq_of": s["seq_of"], "slots": s["slots"],
               "positions": s["positions"]}
        return out if s["masks"] is None else {**out, "masks": s["masks"]}
    K.keep_accepted(s["rows"], s["pool"], s["slots"], s["cu"], s["path"], s["count"])
    return s["pool"]


# ----------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    held, new, parents = _requests(case)
    T = sum(new)
    if case["op"] == "attention":
        hq, hkv, dh = HEADS[case["heads"]]
        es = 2 if case["dtype"] == "bfloat16" else 4
        w = case["window"]
        depth, seen, read = [], 0, 0
        for h, p in zip(held, parents):
            d = []
            for up in p:
                d.append(0 if up < 0 else d[up] + 1)
            read += min(h, w - 1) if w > 0 else h
            seen += sum(x + 1 + (max(0, min(h, w - 1 - x)) if w > 0 else h) for x in d)
        return {"bytes": float(es * dh * (2 * hkv * (read + T) + 2 * hq * T)), "flops": float(4 * hq * dh * seen)}
    if case["op"] == "verify":
        rows = T * (2 if case["chain"] else 1) - (case["n"] if case["chain"] else 0)  # the last draft rows are not looked at
        return {"bytes": float(4 * rows * case["vocab"]), "flops": float(4 * rows * case["vocab"])}
    if case["op"] == "tables":
        page = case["page"]
        widest = max(-(-(h + m) // page) for h, m in zip(held, new)) + 1
        grown = sum(-(-(h + m) // page) - -(-h // page) for h, m in zip(held, new))
        beyond = sum(widest - -(-h // page) for h in held)
        tree = 0 if case["chain"] else T * (4 + 8 * case["words"])
        return {"bytes": float(4 * (5 * case["n"] + beyond + grown + 3 * T) + tree), "flops": float(T)}
    es = 2 if case["dtype"] == "bfloat16" else 4
    kept = sum(max(1, round(m * 0.6)) for m in new)
    return {"bytes": float(2 * kept * case["layers"] * 2 * case["width"] * es), "flops": 0.0}


# ----------------------------------------------------------------------------- the definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    held, new, parents = _requests(case)
    return {"attention": _exact_attention, "verify": _exact_verify, "tables": _exact_tables, "keep": _exact_keep}[case["op"]](s, held, new, parents)


def _exact_attention(s, held, new, parents):
    case = s["case"]
    hq, hkv, dh = HEADS[case["heads"]]
    page, rows, t0 = case["page"], [], 0
    for r, (h, p) in enumerate(zip(held, parents)):
        m = len(p)
        pages = s["pool"][s["table"][r, :-(-h // page)].long()].double()
        k = torch.cat([pages[:, 0].reshape(-1, hkv, dh)[:h], s["k"][t0:t0 + m].double().view(m, hkv, dh)])
        v = torch.cat([pages[:, 1].reshape(-1, hkv, dh)[:h], s["v"][t0:t0 + m].double().view(m, hkv, dh)])
        del pages
        see = torch.zeros(m, h + m, dtype=torch.bool)
        depth = []
        for i, up in enumerate(p):
            depth.append(0 if up < 0 else depth[up] + 1)
            see[i, max(0, h + depth[i] - case["window"] + 1) if case["window"] > 0 else 0:h] = True
            j = i
            while j >= 0:
                see[i, h + j] = True
                j = p[j]
        see = see.to(DEVICE)
        q = s["q"][t0:t0 + m].double().view(m, hq, dh)
        heads = []
        for a in range(hq):
            sc = (q[:, a] @ k[:, a // (hq // hkv)].T) / math.sqrt(dh)
            pr = torch.softmax(sc.masked_fill(~see, -math.inf), -1)
            heads.append(pr @ v[:, a // (hq // hkv)])
        rows.append(torch.stack(heads, 1).reshape(m, hq * dh))
        t0 += m
    return torch.cat(rows)


def _exact_verify(s, held, new, parents):
    n, width, cu = len(new), s["case"]["nodes"], _cu(new)
    tokens, temp, u = s["tokens"].tolist(), s["temperature"].tolist(), s["uniforms"].double().tolist()
    out, path = [[-1] * width for _ in range(n)], [[-1] * width for _ in range(n)]
    count = []

    def dist(rows, t):
        z = rows.double() / t
        return torch.softmax(z, -1)

    def pick(f, x):
        run = torch.cumsum(f, 0)
        return int(torch.searchsorted(run, float(x) * run[-1:], right=True))

    for r in range(n):
        t0, p, now, kept = cu[r], parents[r], 0, 0
        path[r][0] = 0
        rest = None
        while True:
            row = s["logits"][t0 + now]
            f = None if temp[r] <= 0 else dist(row, temp[r])
            children = [i for i in range(now + 1, len(p)) if p[i] == now]
            nxt = None
            if s["draft"] is None:
                end = int(row.argmax()) if f is None else pick(f, u[t0 + now])
                nxt = next((i for i in children if tokens[t0 + i] == end), None)
            elif children:
                x = tokens[t0 + children[0]]
                if f is None:
                    nxt = children[0] if int(row.argmax()) == x else None
                else:
                    g = dist(s["draft"][t0 + now], temp[r])
                    if u[t0 + children[0]] * float(g[x]) < float(f[x]):
                        nxt = children[0]
                    else:
                        rest = (f - g).clamp_min(0)
            if nxt is None:
                if s["draft"] is not None:
                    end = int(row.argmax()) if f is None else pick(f if rest is None or float(rest.sum()) <= 0 else rest, u[t0])
                out[r][kept] = end
                count.append(kept + 1)
                break
            out[r][kept] = tokens[t0 + nxt]
            kept += 1
            path[r][kept] = now = nxt
    return {"tokens": _i32(out), "path": _i32(path), "count": _i32(count)}


def _exact_tables(s, held, new, parents):
    page, spare, free = s["case"]["page"], s["spare"], s["free"].tolist()
    table, given = s["table"].tolist(), 0
    seq, pos, slots = s["seq_of"].tolist(), s["positions"].tolist(), s["slots"].tolist()
    masks = None if s["masks"] is None else s["masks"].cpu().clone()
    blocks, t = [], 0
    bits = None if masks is None else _words(parents, masks.shape[1]).cpu()
    for r, (h, p) in enumerate(zip(held, parents)):
        had, want = -(-h // page), -(-(h + len(p)) // page)
        for b in range(had, len(table[r])):
            table[r][b] = spare
            if b < want:
                table[r][b] = free[given] if given < len(free) else spare
                given += 1
        blocks.append(max(had, want))
        depth = []
        for i, up in enumerate(p):
            depth.append(0 if up < 0 else depth[up] + 1)
            seq[t], pos[t] = r, h + depth[i]
            to = table[r][(h + i) // page]
            slots[t] = -1 if to == spare else to * page + (h + i) % page
            if masks is not None:
                masks[t] = bits[t]
            t += 1
    out = {"cu": _i32(_cu(new)), "table": _i32(table), "blocks": _i32(blocks), "taken": _i32([given]), "seq_of": _i32(seq), "slots": _i32(slots),
           "positions": _i32(pos)}
    return out if masks is None else {**out, "masks": masks.to(DEVICE)}


def _exact_keep(s, held, new, parents):
    pool, page, t0 = s["pool"].double(), s["case"]["page"], 0
    slots, path, count = s["slots"].tolist(), s["path"].tolist(), s["count"].tolist()
    for r, m in enumerate(new):
        for j in range(count[r]):
            to = slots[t0 + j]
            pool[:, to // page, :, to % page] = s["rows"][:, :, t0 + path[r][j]].double()
        t0 += m
    return pool
