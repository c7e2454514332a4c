"""Plain forms of the operators of a drafted step, in 64 bits and one request at a time."""
import math

import torch


def ancestors(parents):
    """Per token of a request: the places of its ancestors and itself, and its depth.  A parent that does not lie in front of its
    child is none."""
    out, depth = [], []
    for i, up in enumerate(parents):
        ok = 0 <= up < i
        out.append((out[up] if ok else []) + [i])
        depth.append(depth[up] + 1 if ok else 0)
    return out, depth


def step_tables(held, new, blocks, table, free, page_size, spare, cap, parents=None, words=0, fill=-7):
    table = [list(r) for r in table]
    width, cu, given = len(table[0]), [0], 0
    seq, pos, slots = [fill] * cap, [fill] * cap, [fill] * cap
    masks = [[fill] * words for _ in range(cap)] if parents is not None else None
    after = []
    for s, (h, m, b) in enumerate(zip(held, new, blocks)):
        a = max(b, -(-(h + m) // page_size))
        pages = []
        for j in range(a):
            if j < b:
                pages.append(table[s][j] if j < width else spare)
            else:
                page = free[given] if given < len(free) else spare
                given += 1
                pages.append(page if j < width else spare)
        for j in range(b, width):
            table[s][j] = pages[j] if j < a else spare
        after.append(a)
        t0 = cu[-1]
        up = parents[t0:t0 + m] if parents is not None else None
        anc, depth = ancestors(up) if up is not None else (None, list(range(m)))
        for i in range(m):
            t = t0 + i
            if t >= cap:
                break
            page = pages[(h + i) // page_size]
            seq[t], pos[t] = s, h + depth[i]
            slots[t] = -1 if page in (-1, spare) else page * page_size + (h + i) % page_size
            if masks is not None:
                for w in range(words):
                    bits = sum(1 << (j - 64 * w) for j in anc[i] if 64 * w <= j < 64 * w + 64)
                    masks[t][w] = bits - (1 << 64) if bits >= 1 << 63 else bits
        cu.append(t0 + m)
    return dict(cu=cu, table=table, blocks=after, taken=[given], seq_of=seq, positions=pos, slots=slots, masks=masks)


def tree_attention(q, k, v, ctx_k, ctx_v, see_ctx, see_new, scale, sink=None):
    """One request: q [m, Hq, d], k, v [m, Hkv, d], cached keys and values [h, Hkv, d], truth values [m, h] and [m, m].
    Returns the rows [m, Hq, d], the weighted sums of |v| (for tolerances), and the largest sum of |q||k| scale of a row."""
    m, hq, d = q.shape
    g = hq // k.shape[1]
    q, k, v = q.double(), torch.cat([ctx_k, k]).double(), torch.cat([ctx_v, v]).double()
    see = torch.cat([see_ctx, see_new], 1)
    out, mag, size = (torch.zeros(m, hq, d, dtype=torch.float64) for _ in range(3))
    for h in range(hq):
        for i in range(m):
            at = see[i].nonzero()[:, 0]
            if len(at) == 0:
                continue
            kk, vv = k[at, h // g], v[at, h // g]
            s = (kk @ q[i, h]) * scale
            top = float(s.max()) if sink is None else max(float(s.max()), float(sink[h]))
            p = torch.exp(s - top)
            total = p.sum() + (math.exp(float(sink[h]) - top) if sink is not None else 0.0)
            out[i, h] = p @ vv / total
            mag[i, h] = p @ vv.abs() / total
            size[i, h] = float((kk.abs() @ q[i, h].abs()).max()) * scale
    return out, mag, size


def _weights(row, t):
    """exp((l - max) / T): NaN as -inf, +inf shares the weight among its like; None: no weight at all."""
    x = torch.nan_to_num(row.double(), nan=-math.inf, posinf=math.inf, neginf=-math.inf)
    top = x.max()
    if top == -math.inf:
        return None
    if top == math.inf:
        return (x == math.inf).double()
    return torch.exp((x - top) / t)


def _best(row):
    x = torch.nan_to_num(row.double(), nan=-math.inf, posinf=math.inf, neginf=-math.inf)
    return None if x.max() == -math.inf else int((x == x.max()).nonzero()[0, 0])


def pick(f, u):
    run = torch.cumsum(f, 0)
    return int((run > u * run[-1]).nonzero()[0, 0])


def verify(logits, tokens, cu, uniforms, width, temperature=None, parents=None, draft=None):
    n = len(cu) - 1
    out, path = [[-1] * width for _ in range(n)], [[-1] * width for _ in range(n)]
    count = [0] * n
    for s in range(n):
        t0, m = cu[s], cu[s + 1] - cu[s]
        if m == 0:
            continue
        temp = 0.0 if temperature is None else float(temperature[s])
        greedy = not temp > 0
        up = list(range(-1, m - 1)) if parents is None else parents[t0:t0 + m]
        now, kept, rest = 0, 0, None
        path[s][0] = 0
        while True:
            row = logits[t0 + now]
            children = [i for i in range(now + 1, m) if up[i] == now] if kept + 1 < width else []
            nxt = None
            w = None if greedy else _weights(row, temp)
            empty = _best(row) is None
            if draft is None:
                end = 0 if empty else _best(row) if greedy else pick(w, float(uniforms[t0 + now]))
                if not empty:
                    nxt = next((i for i in children if int(tokens[t0 + i]) == end), None)
            else:
                if children and not empty:
                    x = int(tokens[t0 + children[0]])
                    if greedy:
                        nxt = children[0] if _best(row) == x else None
                    else:
                        d = _weights(draft[t0 + now], temp)
                        p = w / w.sum()
                        qq = torch.zeros_like(p) if d is None else d / d.sum()
                        if 0 <= x < len(p) and d is not None and float(uniforms[t0 + children[0]]) * float(qq[x]) < float(p[x]):
                            nxt = children[0]
                        else:
                            rest = (p - qq).clamp_min(0)
                if nxt is None:
                    f = w if rest is None or float(rest.sum()) <= 0 else rest
                    end = 0 if empty else _best(row) if greedy else pick(f, float(uniforms[t0]))
            if nxt is None:
                out[s][kept] = end
                count[s] = kept + 1
                break
            out[s][kept] = int(tokens[t0 + nxt])
            kept += 1
            path[s][kept] = now = nxt
    return dict(tokens=out, path=path, count=count)


def keep(rows, pool, slots, cu, path, count):
    """rows [L, planes, T, W] into a copy of pool [L, pages, planes, P, W]."""
    pool = pool.clone()
    page = pool.shape[3]
    for s in range(len(count)):
        t0, m = cu[s], cu[s + 1] - cu[s]
        for j in range(min(count[s], len(path[s]), m)):
            node, slot = path[s][j], slots[t0 + j]
            if 0 <= node < m and 0 <= slot < pool.shape[1] * page:
                pool[:, slot // page, :, slot % page] = rows[:, :, t0 + node]
    return pool
