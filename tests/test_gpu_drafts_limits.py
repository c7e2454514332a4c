"""The operators of a drafted step at the ends of what they take: temperatures, scores and lengths of every size, tensors that lie in one
another, bounds beyond the step; against the plain forms in 64 bits."""
import math
import random

import pytest
import torch

from plain import drafts_plain as P
from test_gpu_drafts import DEV, K, Case, cumulate, drafts_of, i32, verify  # noqa: F401

pytestmark = pytest.mark.gpu


def f32(x):
    """The float32 nearest to x (what a temperature tensor holds)."""
    return torch.tensor(x, dtype=torch.float32).item()


# ----------------------------------------------------------------------------- verification
@pytest.mark.parametrize("temperature", [1e-38, 1e-36, 1e-30, 1e-10, 1e-9, 2e-8, 1e-8, 1e-6, 1e-5, 1e-3, 1e4, 1e30, 1e36])
@pytest.mark.parametrize("mode", ["tree", "chain", "drawn"])
def test_verify_drafts_at_any_temperature(temperature, mode):
    """Logits of deviations 3 to 1,000 and one row shifted by 1e10; vocabularies that end inside a piece of 1,024."""
    lens = [4, 1, 6, 3, 5]
    temps = [f32(temperature)] * 5
    for V, spread in ((50, 1.5), (4097, 5.0), (5000, 150.0), (2500, 500.0)):
        # (proposals are drawn in 32 bits, where a logit over 1e-38 is no number)
        logits, draft, parents, tokens, u = drafts_of(lens, V, V, [max(t, 1e-36) for t in temps], mode == "tree")
        logits, draft = logits * spread, draft * spread
        logits[4] += 1e10
        logits[0, 3::7] = logits[0].max()      # ties: they share the weight
        logits[1, 5::9] = math.nan
        logits[2, 1::5] = -math.inf
        for s in range(2, 6):                  # drafts that can be kept: the largest logit behind their parent
            tokens[5 + s] = int(torch.nan_to_num(logits[5 + s - 1], nan=-math.inf).argmax())
        verify(logits, tokens, lens, u, 6, temps, parents if mode == "tree" else None, draft if mode == "drawn" else None)


@pytest.mark.parametrize("mode", ["tree", "chain", "drawn"])
@pytest.mark.parametrize("V", [50, 1024, 3000])
def test_verify_drafts_rows_of_very_negative_logits(mode, V):
    """Masks of the type's lowest value, alone, beside -inf and beside NaN, in rows that a walk reaches: every token that is
    not masked deeper has its share."""
    low = torch.finfo(torch.float32).min
    logits = torch.full((6, V), low)
    logits[1, ::2] = -math.inf
    logits[2, 1::3] = math.nan
    logits[3] = -1e30
    logits[3, ::4] = -math.inf
    logits[4, 20:] = -3e38
    logits[5, 9] = -1e-30
    lens, draft = [1] * 6, torch.zeros(6, V)
    for u in (0.0, 0.3, 0.7, 1 - 2.0 ** -24):
        for temps in ([1.0] * 6, [f32(1e-3)] * 6, [f32(1e30)] * 6):
            verify(logits.to(DEV), [0] * 6, lens, torch.full((6,), u), 2, temps, [-1] * 6 if mode == "tree" else None,
                   draft.to(DEV) if mode == "drawn" else None)


def test_verify_drafts_infinite_temperature():
    """Every token that is not masked weighs as much as any other."""
    logits = torch.randn(3, 100, generator=torch.Generator().manual_seed(1))
    logits[:, 50:] = -math.inf
    for draft in (None, torch.zeros(3, 100, device=DEV)):
        for u in (0.0, 0.31, 0.99):
            out, path = (torch.full((3, 1), -9, dtype=torch.int32, device=DEV) for _ in range(2))
            K().verify_drafts(logits.to(DEV), i32([0] * 3), i32([0, 1, 2, 3]), torch.full((3,), u, device=DEV), out, path, i32([0] * 3),
                              K().verify_drafts_scratch(3, 100, DEV), temperature=torch.full((3,), math.inf, device=DEV), draft_logits=draft)
            assert out[:, 0].tolist() == [int(u * 50)] * 3


# ----------------------------------------------------------------------------- attention
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("heads", [(2, 1, 512), (2, 1, 256), (8, 2, 64), (6, 2, 128)])
def test_tree_attention_bounds_beyond_the_step(dtype, heads):
    """Bounds that pass the step's rows (`step_tables` leaves them so where the tokens have no room), masks that name the tokens that are
    not there: nothing behind the rows of q, k and v is read."""
    c = Case([70, 130], [5, 7], heads, dtype, 64, seed=21, extra_rows=24)
    T = c.cu[-1]
    c.mask = torch.full_like(c.mask, -1)
    for see in c.see:
        see[:] = True
    for t in (c.q, c.k, c.v):
        t[T:] = math.nan
    whole, held, cu = c.out, i32(c.held), i32([0, 5, T + 17])
    q, k, v, c.out = (t[:T] for t in (c.q, c.k, c.v, whole))
    K().tree_attention(q, k, v, c.pool, c.table, held, cu, c.out, c.hq, c.hkv, c.d, c.scale, K().tree_attention_scratch(DEV), mask=c.mask[:T])
    c.out = whole
    c.check()


# ----------------------------------------------------------------------------- tables
@pytest.mark.parametrize("page", [1, 64])
@pytest.mark.parametrize("tree", [False, True])
def test_step_tables_of_lengths_beyond_32_bits(page, tree):
    """Lengths whose sums pass 32 bits: bounds and counts stay at the largest number, places that there cannot be are -1, and
    nothing is written or read outside the tables."""
    most, cap, n = 2 ** 31 - 1, 9, 5
    held, new, blocks = [3, most, 0, most - 1, 5], [4, most, most, 2, 6], [4, most, 0, 1, most]
    rows = [[7, 8, 9, 6], [0, 1, 2, 3], [30, 30, 30, 30], [4, 30, 30, 30], [10, 11, 12, 13]]
    guard = 300

    def framed(size, fill=-7, dtype=torch.int32):
        whole = torch.full((size + 2 * guard,), fill, dtype=dtype, device=DEV)
        return whole, whole[guard:guard + size]

    out = {k: framed(m) for k, m in dict(cu=n + 1, seq=cap, pos=cap, slots=cap, blocks=n, taken=1, table=4 * n).items()}
    out["masks"] = framed(cap, dtype=torch.int64)
    out["table"][1].copy_(i32(rows).view(-1))
    parents = i32([-1, 0, 0, 2] + [-1, 0, 1, 2, 3])
    K().step_tables(i32(held), i32(new), i32(blocks), out["table"][1].view(n, 4), i32([20, 21]), page, 30, out["cu"][1], out["seq"][1], out["pos"][1],
                    out["slots"][1], out["blocks"][1], out["taken"][1], parents=parents if tree else None,
                    masks=out["masks"][1].view(cap, 1) if tree else None)
    for whole, inside in out.values():
        assert (whole[:guard] == -7).all() and (whole[-guard:] == -7).all()
    got = {k: v[1].tolist() for k, v in out.items()}
    need = [max(b, min(-(-(h + m) // page), most)) for h, m, b in zip(held, new, blocks)]
    assert got["cu"] == [0, 4, most, most, most, most] and got["blocks"] == need
    assert got["taken"] == [min(most, sum(a - b for a, b in zip(need, blocks)))]
    assert got["seq"] == [0] * 4 + [1] * 5
    assert got["pos"] == [3 + d for d in ((0, 1, 1, 2) if tree else range(4))] + [most] * 5
    # pages of 1: request 0 needs seven of a table of four (three are counted as taken and have no place), so the others find none left;
    # of 64: it needs none, and the two free ones go to request 2
    assert got["slots"] == ([6, -1, -1, -1] if page == 1 else [7 * 64 + 3 + i for i in range(4)]) + [-1] * 5
    third = [30] * 4 if page == 1 else [20, 21, 30, 30]
    assert [got["table"][4 * s:4 * s + 4] for s in range(n)] == [rows[0], rows[1], third, [4, 30, 30, 30], rows[4]]
    if tree:
        assert got["masks"] == [1, 3, 5, 13, 1, 3, 7, 15, 31]


# ----------------------------------------------------------------------------- bounds
@pytest.mark.parametrize("cu", [[-4, 2, 6], [0, 2, 9], [5, -2 ** 31, 6], [-2 ** 31, -5, 6], [3, 2 ** 31 - 1, 2 ** 31 - 1]])
@pytest.mark.parametrize("mode", ["tree", "drawn"])
def test_verify_drafts_bounds_outside_the_rows(cu, mode):
    """Bounds below the first row or beyond the last are cut to the rows; a request that ends before it begins has none."""
    V, T = 300, 6
    logits, draft, _, tokens, u = drafts_of([3, 3], V, 4, [1.0, 1.0], False)
    parents = [-1, 0, 0, 1, 2, 3]
    out, path, count = i32([[-9] * 4] * 2), i32([[-9] * 4] * 2), i32([-9] * 2)
    K().verify_drafts(logits, i32(tokens), i32(cu), u.to(DEV), out, path, count, K().verify_drafts_scratch(T, V, DEV), temperature=torch.ones(2, device=DEV),
                      parents=i32(parents) if mode == "tree" else None, draft_logits=draft if mode == "drawn" else None)
    for s in range(2):
        first = min(max(cu[s], 0), T)
        cut = [first, max(first, min(max(cu[s + 1], 0), T))]
        want = P.verify(logits.cpu(), tokens, cut, u, 4, [1.0], parents if mode == "tree" else None, draft.cpu() if mode == "drawn" else None)
        assert dict(tokens=[out[s].tolist()], path=[path[s].tolist()], count=[int(count[s])]) == want


@pytest.mark.parametrize("cu", [[-4, 2, 6], [0, 2, 9], [5, -2 ** 31, 6], [-2 ** 31, -5, 6], [3, 2 ** 31 - 1, 2 ** 31 - 1]])
def test_keep_accepted_bounds_outside_the_rows(cu):
    rows, pool = torch.randn(2, 2, 6, 64, device=DEV), torch.randn(2, 3, 2, 8, 64, device=DEV)
    slots, path, count = [3, 20, 7, 11, 1, 16], [[0, 1, 3], [0, 2, 1]], [3, 3]
    want = P.keep(rows.cpu(), pool.cpu(), slots, [min(max(x, 0), 6) for x in cu], path, count)
    K().keep_accepted(rows, pool, i32(slots), i32(cu), i32(path), i32(count))
    assert torch.equal(pool.cpu(), want)


# ----------------------------------------------------------------------------- attention of rows that see nothing
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("heads", [(8, 2, 64), (6, 2, 128), (16, 1, 64), (32, 2, 128), (2, 1, 256), (2, 1, 512)])
@pytest.mark.parametrize("held,new", [([0, 0, 0], [40, 1, 64]), ([200], [64]), ([0], [130]), ([0] * 200, [3] * 200)])
def test_tree_attention_sinks_of_minus_infinity(dtype, heads, held, new):
    """Heads without a sink (-inf) beside heads with one: rows that see nothing are zero, whether their unit is one block's or was cut,
    and no row is harmed by keys of its request that it does not see."""
    c = Case(held, new, heads, dtype, 64, seed=31, words=3 if max(new) > 64 else 1)
    for see in c.see:
        see[:, :32] = False
        see[::3] = False
    c.write_mask()
    sink = torch.randn(heads[0], generator=torch.Generator().manual_seed(3))
    sink[::2] = -math.inf
    for s in (torch.full_like(sink, -math.inf), sink):
        c.run(1, s.to(DEV))
        c.check(1, s.to(DEV))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("heads", [(8, 2, 64), (12, 2, 128), (2, 1, 256)])
def test_tree_attention_of_one_row_of_any_stride(dtype, heads):
    """A step of one token in slices of rows whose length is odd: the only row begins where it has to."""
    c = Case([200], [1], heads, dtype, 64, seed=5)
    w = c.hq * c.d
    for name in ("q", "k", "v"):
        t = getattr(c, name)
        wide = torch.zeros(2, w + 515 if w % 2 == 0 else w + 516, dtype=dtype, device=DEV)
        wide[:1, :t.shape[1]] = t
        setattr(c, name, wide[:1, :t.shape[1]])
        assert getattr(c, name).stride(0) % 2 == 1
    c.run()
    c.check()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("heads", [(8, 2, 64), (16, 1, 128), (2, 1, 256), (2, 1, 512)])
def test_tree_attention_in_the_place_of_the_queries(dtype, heads):
    """Results written over q: units of one block, units that shares cut, wide ones."""
    for held, new in (([3000, 40], [33, 9]), ([20] * 300, [5] * 300), ([0], [1])):
        c = Case(held, new, heads, dtype, 64, seed=17)
        first = c.q.clone()
        c.out = c.q
        c.run()
        c.q = first
        c.check()


# ----------------------------------------------------------------------------- launches directly behind
def test_launches_directly_behind_find_tables_and_kept_rows():
    """Attention of a decode step reads positions, block tables and cached keys ahead of its wait for the launch before it: directly behind
    the tables' launch, and behind the kept rows', it reads what those have written."""
    ops, n, page, hq, hkv, d, P_ = K(), 64, 64, 8, 2, 64, 600
    g = torch.Generator(device=DEV).manual_seed(1)
    bf = dict(dtype=torch.bfloat16, device=DEV)
    pool = torch.randn(1, P_ + 1, 2, page, hkv * d, generator=g, **bf)
    q, k, v = torch.randn(n, hq * d, generator=g, **bf), torch.randn(n, hkv * d, generator=g, **bf), torch.randn(n, hkv * d, generator=g, **bf)
    one, free = i32([1] * n), torch.randperm(P_, device=DEV, generator=g).int()
    cu, seq, pos, slots, blocks, taken = i32([0] * (n + 1)), i32([0] * n), i32([0] * n), i32([0] * n), i32([0] * n), i32([0])
    table, zero = i32([[P_] * 9] * n), i32([0] * n)

    def attend(to):
        ops.flash_decode_attention(q, k, v, 1.0, 1.0, 1.0, None, pool[0], table, pos, to, hq, hkv, d, d ** -0.5)

    for i in range(60):
        held = torch.randint(0, 8 * page, (n,), generator=g, device=DEV, dtype=torch.int32)
        free = free[torch.randperm(P_, generator=g, device=DEV)]
        got, again = (torch.zeros(n, hq * d, **bf) for _ in range(2))
        torch.cuda.synchronize()
        ops.step_tables(held, one, zero, table, free, page, P_, cu, seq, pos, slots, blocks, taken)
        attend(got)
        torch.cuda.synchronize()
        assert torch.equal(pos, held)
        attend(again)
        assert torch.equal(got, again), i
        # kept rows: a token of every request, into places that the step behind them reads
        rows = torch.randn(1, 2, n, hkv * d, generator=g, **bf)
        place = (table[torch.arange(n, device=DEV), 0] * page + held.clamp_max(page - 1) // 2).int()
        path, count = i32([[0]] * n), one
        torch.cuda.synchronize()
        ops.keep_accepted(rows, pool, place, cu, path, count)
        attend(got)
        torch.cuda.synchronize()
        attend(again)
        assert torch.equal(got, again), i


# ----------------------------------------------------------------------------- windows over the step's own tokens
def windowed(c, window):
    """Keeps the mask, and takes what `window` hides among the step's own tokens out of what the plain form sees."""
    pos = c.positions.tolist()
    for s, see in enumerate(c.see):
        own = torch.tensor(pos[c.cu[s]:c.cu[s + 1]])
        first = own - window + 1 if window > 0 else own - own % -window
        see &= own[None, :] >= first[:, None]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("heads", [(8, 2, 64), (6, 2, 128), (16, 1, 128), (16, 1, 64), (2, 1, 256), (2, 1, 512)])
@pytest.mark.parametrize("window", [1, 5, 200, -8, -64])
@pytest.mark.parametrize("parents", ["tree", None])
def test_tree_attention_window_over_the_step(dtype, heads, window, parents):
    """Paths deeper than the window, chunks whose border lies among the step's tokens; hidden values that are not numbers harm nobody."""
    c = Case([300, 62, 0, 130], [14, 9, 40, 61], heads, dtype, 64, seed=23, parents=parents, extra_rows=2)
    sink = torch.randn(heads[0], generator=torch.Generator().manual_seed(2)).to(DEV)
    windowed(c, window)
    c.run(window, sink, window_step=True)
    c.check(window, sink)
    hidden = [(s, j) for s, see in enumerate(c.see) for j in range(see.shape[0]) if int(see[:, j].sum()) <= 1]
    for s, j in hidden[::3]:   # (a token that sees itself alone may spoil its own row)
        c.v[c.cu[s] + j, ::3] = math.inf
    c.run(window, None, window_step=True)
    c.check(window)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("window", [7, 64, 300, -16, -64])
def test_tree_attention_window_over_long_chains(dtype, window):
    c = Case([100, 0, 700], [300, 513, 1], (4, 2, 64), dtype, 64, parents=None, seed=3)
    windowed(c, window)
    c.run(window, window_step=True)
    c.check(window)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("window", [3, 40, -8, -64])
def test_tree_attention_with_a_window_is_paged_attention_along_every_path(dtype, window):
    """Every node of a tree against the framework's attention of single tokens: the path down to it is put into the cache, and the
    node's row attends over it there."""
    hq, hkv, d, page = 8, 2, 64, 16
    held, new = [57, 6], [12, 9]
    c = Case(held, new, (hq, hkv, d), dtype, page, seed=41, extra_pages=12)
    c.run(window, window_step=True)
    for s, m in enumerate(new):
        t0, h = c.cu[s], held[s]
        depth = [int(x) - h for x in c.positions[t0:t0 + m]]
        table = torch.full((1, 8), c.pages - 1, dtype=torch.int32, device=DEV)
        used = -(-h // page)
        table[0, :used] = c.table[s, :used]
        spare = sorted(set(range(c.pages - 1)) - set(c.table[:, :].flatten().tolist()))
        table[0, used:used + 2] = i32(spare[:2])
        for i in range(m):
            path = [i]
            while c.parents[s][path[0]] >= 0:
                path.insert(0, c.parents[s][path[0]])
            assert len(path) == depth[i] + 1
            pool = c.pool.clone()
            for at, node in enumerate(path):
                p = int(table[0, (h + at) // page])
                pool[p, 0, (h + at) % page], pool[p, 1, (h + at) % page] = c.k[t0 + node], c.v[t0 + node]
            one = torch.zeros(1, hq * d, dtype=dtype, device=DEV)
            K().paged_attention(c.q[t0 + i:t0 + i + 1].contiguous(), pool, table, i32([h + depth[i]]), i32([0]), one, hq, hkv, d, c.scale, window=window)
            got, want = c.out[t0 + i].double(), one[0].double()
            # both are within their sums' errors of the formula (float32: some 100 terms, scores of size 4); bfloat16: the probabilities and
            # the result are rounded to 2^-8 on one side, the result on both
            size = c.v[t0:t0 + m].abs().max().double().clamp_min(4.0)
            off = 3 * 2.0 ** -8 * size if dtype == torch.bfloat16 else 200 * 2.0 ** -24 * 4 * size
            assert float((got - want).abs().max()) <= float(off), (s, i)


# ----------------------------------------------------------------------------- units of 256 rows
# 16 query heads a key/value head: 9 tokens fill the second set of 128 rows with 16, 20 leave a last unit whose second set has none.
WIDE = [([333, 1500, 0, 70], [20, 9, 17, 40]), ([(37 * s) % 300 for s in range(90)], [(9, 20, 8, 16)[s % 4] for s in range(90)])]


def wide(held, new, d, page=64, **kw):
    c = Case(held, new, (16, 1, d), torch.bfloat16, page, **kw)
    assert sum(new) * 16 > 128 * len(new)
    return c


def some(new):
    """Of many requests every seventh is looked at."""
    return set(range(0, len(new), 7)) if len(new) > 8 else None


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("held,new", WIDE)
@pytest.mark.parametrize("window", [0, 5, 100, -64])
def test_wide_units_windows_and_sinks(d, held, new, window):
    c = wide(held, new, d, seed=51, extra_rows=3)
    sink = torch.randn(16, generator=torch.Generator().manual_seed(4)).to(DEV)
    for s in (None, sink):
        c.run(window, s)
        c.check(window, s, some(new))


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("held,new", WIDE)
@pytest.mark.parametrize("window", [0, 1])
def test_wide_units_empty_rows_and_any_mask(d, held, new, window):
    """(A window of 1 hides the whole cache: rows that see nothing at all.)"""
    c = wide(held, new, d, seed=52)
    g = torch.Generator().manual_seed(1)
    for see in c.see:
        see[:] = torch.rand(see.shape, generator=g) < 0.4
        see[::3] = False
        see[:, 2:4] = False
    c.write_mask()
    for s in (None, torch.randn(16, generator=g).to(DEV)):
        c.run(window, s)
        c.check(window, s, some(new))


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("held,new", WIDE)
@pytest.mark.parametrize("window", [0, 90])
def test_wide_units_values_that_are_not_numbers(d, held, new, window):
    """Both sets of rows take what is not finite out of the one tile of values that they share."""
    c = wide(held, new, d, seed=53)
    for s, m in enumerate(new):
        t0 = c.cu[s]
        if m > 8:
            c.k[t0 + 3] = math.nan
            c.v[t0 + 5, :3] = math.inf
            c.v[t0 + 7, d // 2:] = -math.inf
            c.v[t0 + m - 1, 1::2] = math.nan
        if held[s] > 80:    # a cached value and a cached key
            for place, plane, row in ((70, 1, slice(4, 6)), (held[s] - 2, 0, slice(0, d))):
                c.pool[int(c.table[s, place // 64]), plane, place % 64, row] = math.inf if plane else math.nan
                c.ctx[s][plane, place, row] = math.inf if plane else math.nan
    c.q[c.cu[1] + 4, :d] = math.nan
    c.run(window)
    c.check(window, only=some(new))


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("page", [8, 24, 48, 200, 256])
@pytest.mark.parametrize("window", [0, 70])
def test_wide_units_page_sizes(d, page, window):
    for held, new in (WIDE[0], ([301, 64, 17], [33, 16, 5])):
        c = wide(held, new, d, page, seed=page, extra_pages=2)
        c.run(window)
        c.check(window)


@pytest.mark.parametrize("d", [64, 128])
def test_wide_units_of_as_many_requests_as_there_may_be(d):
    """1,024 requests: the most whose lengths lie in shared memory beside the tiles."""
    n = 1024
    c = wide([s % 7 for s in range(n)], [10 - s % 2 for s in range(n)], d, 8, seed=6)
    c.run()
    c.check(only=set(range(0, n, 60)))


# ----------------------------------------------------------------------------- the operators together
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("window", [0, 3, 20, -8])
def test_drafted_steps_row_by_row(dtype, tree, window):
    """A layer of attention whose tokens come from 16 columns of its rows, greedy: drafted steps against one token a step through the
    framework's paged attention.  Every kept node's attention row is the single step's within both sides' roundings, and every token is
    the single step's wherever its two best logits are further apart than those roundings can move them."""
    hq, hkv, d, V, page, n, total = 4, 2, 64, 97, 16, 3, 30
    ops, w, rng = K(), hkv * d, random.Random(3)
    g = torch.Generator(device=DEV).manual_seed(5)
    E = torch.randn(V, 64, generator=g, device=DEV, dtype=torch.float64)
    W = torch.randn(64, (hq + 2 * hkv) * d, generator=g, device=DEV, dtype=torch.float64) / 8
    columns = torch.randperm(hq * d, generator=g, device=DEV)[:16]
    R = torch.randn(16, V, generator=g, device=DEV, dtype=torch.float64)
    inv = (1e4 ** (-torch.arange(0, d, 2) / d)).to(DEV)
    prompts = [[rng.randrange(V) for _ in range(m)] for m in (5, 30, 17)]
    rows_of = (E @ W).to(dtype)                                      # a token's q, k and v, the same whoever asks
    half = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -24
    # (a rotation keeps a row's length up to its rounding; |q||k| bounds a score's sum of magnitudes)
    norm = lambda x: float(x.double().view(V, -1, d).norm(dim=-1).max()) * 1.02
    size = norm(rows_of[:, :hq * d]) * norm(rows_of[:, hq * d:hq * d + w]) * d ** -0.5
    vmax = rows_of[:, hq * d + w:].double().abs().amax(0).view(hkv, 1, d).expand(hkv, hq // hkv, d).reshape(-1)
    # per side: scores, exponentials and sums in float; in bfloat16 the probabilities (one side's) and both results are rounded
    err = 2 * (2 * (d + 2) * 2.0 ** -24 * size + 100 * 2.0 ** -24 + 2.0 ** -21) * vmax + (3 if dtype == torch.bfloat16 else 2) * half * vmax
    move = float((err[columns][:, None] * R.abs()).sum(0).max())     # of a logit

    # ---- one token a step
    pool, table = torch.zeros(40, 2, page, w, dtype=dtype, device=DEV), torch.arange(n * 10, device=DEV).view(n, 10).int()
    lens, want, best = [0] * n, [{} for _ in range(n)], [{} for _ in range(n)]   # by place: the row, (token behind it, gap)

    def plain(tokens):
        seq, pos = [s for s in range(n) for _ in tokens[s]], [lens[s] + i for s in range(n) for i in range(len(tokens[s]))]
        x = rows_of[torch.tensor([t for f in tokens for t in f], device=DEV)]
        q, o = torch.empty(len(seq), hq * d, dtype=dtype, device=DEV), torch.empty(len(seq), hq * d, dtype=dtype, device=DEV)
        ops.qkv_rope_store(x[:, :hq * d], x[:, hq * d:hq * d + w], x[:, hq * d + w:], 1, 1, 1, inv, i32(pos), i32(seq), table, pool, q, None, None, hq, hkv, d)
        ops.paged_attention(q, pool, table, i32(pos), i32(seq), o, hq, hkv, d, d ** -0.5, window=window, use_tensor_cores=False)
        top = (o.double()[:, columns] @ R).topk(2)
        for i, (s, p) in enumerate(zip(seq, pos)):
            want[s][p] = o[i].double()
            best[s][p] = (int(top.indices[i, 0]), float(top.values[i, 0] - top.values[i, 1]))
        for s in range(n):
            lens[s] += len(tokens[s])
        return [[best[s][lens[s] - 1][0]] for s in range(n)]

    nxt = plain(prompts)
    out = [list(x) for x in nxt]                                     # out[s][i]: the token at place len(prompt) + i
    for _ in range(total + 6):
        nxt = plain(nxt)
        for s in range(n):
            out[s] += nxt[s]

    # ---- drafted steps
    pages, room, width = 40, 64, 8
    pool = torch.zeros(1, pages + 1, 2, page, w, dtype=dtype, device=DEV)
    free, blocks, blocks_out = rng.sample(range(pages), pages), i32([0] * n), i32([0] * n)
    table = torch.full((n, 10), pages, dtype=torch.int32, device=DEV)
    held, got = [0] * n, [0] * n                                     # got: tokens of out that are known
    scratch, vscratch = ops.tree_attention_scratch(DEV), ops.verify_drafts_scratch(room, V, DEV)
    feed, parents = [list(p) for p in prompts], [list(range(-1, len(p) - 1)) for p in prompts]
    steps = compared = close = 0
    while min(got) < total:
        steps += 1
        new = [len(f) for f in feed]
        first = steps == 1
        cu, taken, seq = i32([0] * (n + 1)), i32([0]), i32([0] * room)
        pos, slots, masks = torch.zeros_like(seq), torch.full_like(seq, -1), torch.zeros(room, 1, dtype=torch.int64, device=DEV)
        up = i32([p for f in parents for p in f] + [-1] * (room - sum(new)))
        ops.step_tables(i32(held), i32(new), blocks, table, i32(free), page, pages, cu, seq, pos, slots, blocks_out, taken, parents=up, masks=masks)
        blocks.copy_(blocks_out)
        free = free[int(taken):]
        tokens = i32([x for f in feed for x in f] + [0] * (room - sum(new)))
        x, rows = rows_of[tokens.long()], torch.zeros(1, 2, room, w, dtype=dtype, device=DEV)
        q, o = torch.empty(room, hq * d, dtype=dtype, device=DEV), torch.zeros(room, hq * d, dtype=dtype, device=DEV)
        ops.qkv_rope_store(x[:, :hq * d], x[:, hq * d:hq * d + w], x[:, hq * d + w:], 1, 1, 1, inv, pos, seq, None, None, q, rows[0, 0], rows[0, 1], hq, hkv, d)
        ops.tree_attention(q, rows[0, 0], rows[0, 1], pool[0], table, i32(held), cu, o, hq, hkv, d, d ** -0.5, scratch, mask=None if first else masks,
                           positions=pos, window=window, window_step=True)
        logits = (o.double()[:, columns] @ R).float()
        tokens_out, path, count = (torch.full(size_, -1, dtype=torch.int32, device=DEV) for size_ in ((n, width), (n, width), (n,)))
        if first:                                                    # a prompt: all of it is kept
            path, count = i32([list(range(m)) + [-1] * (30 - m) for m in new]), i32(new)
        else:
            ops.verify_drafts(logits, tokens, cu, torch.zeros(room, device=DEV), tokens_out, path, count, vscratch, parents=up)
        kept, nodes, said = count.tolist(), path.tolist(), tokens_out.tolist()
        for s in range(n):
            t0 = int(cu[s])
            for j in range(kept[s]):
                node, place = nodes[s][j], held[s] + j
                assert ((o[t0 + node].double() - want[s][place]).abs() <= err).all(), (steps, s, j)
                compared += 1
                token, gap = best[s][place]
                if first and j < kept[s] - 1:
                    continue
                mine = int(logits[t0 + node].argmax())
                assert first or mine == said[s][j]
                if mine != token:
                    assert gap <= 2 * move + 1e-6, (steps, s, j, gap, move)
                    close += 1
                    kept[s] = j + 1                                  # the single steps' token goes on
                    break
        ops.keep_accepted(rows, pool, slots, cu, path, i32(kept))
        feed, parents = [], []
        for s in range(n):
            got[s] += 1 if first else kept[s]
            held[s] += kept[s]
            assert held[s] == len(prompts[s]) + got[s] - 1
            if got[s] >= total:                                      # a request that has got all: no tokens in the steps left
                feed.append([])
                parents.append([])
                continue
            coming = out[s][got[s]:got[s] + 4]
            f, p, at = [out[s][got[s] - 1]], [-1], 0
            right = rng.randint(0, len(coming))
            for i, c in enumerate(coming):
                if tree:                                             # a wrong token beside every right one
                    f.append((c + 1) % V)
                    p.append(at)
                f.append(c if i < right else (c + 2) % V)
                p.append(at)
                at = len(f) - 1
            feed.append(f)
            parents.append(p)
    assert compared >= n * total and steps < total and close <= compared // 4


# ----------------------------------------------------------------------------- kept rows of many layers and requests
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("layers,planes,n", [(7, 2, 42), (5, 1, 130), (7, 1, 100), (3, 2, 200), (5, 1, 301), (7, 2, 150)])
@pytest.mark.parametrize("width", [8, 72])
def test_keep_accepted_of_many_requests(dtype, layers, planes, n, width):
    """One, two and four planes a block, also where they do not divide the planes."""
    rng, g = random.Random(n), torch.Generator().manual_seed(n)
    lens = [rng.choice([0, 1, 5, 8]) for _ in range(n)]
    T, page, pages = sum(lens), 8, 3 * n
    pool = torch.randn(layers, pages, planes, page, width, generator=g).to(dtype).to(DEV)
    rows = torch.randn(layers, planes, T, width, generator=g).to(dtype).to(DEV)
    slots = rng.sample(range(pages * page), T)
    count = [rng.randint(0, m) for m in lens]
    path = [sorted(rng.sample(range(m), c)) + [-1] * (8 - c) for m, c in zip(lens, count)]
    want = P.keep(rows.cpu(), pool.cpu(), slots, cumulate(lens), path, count)
    K().keep_accepted(rows, pool, i32(slots), i32(cumulate(lens)), i32(path), i32(count))
    assert torch.equal(pool.cpu(), want)


# ----------------------------------------------------------------------------- the largest and the smallest calls
@pytest.mark.parametrize("V", [600001, 1500000, 2097152])
@pytest.mark.parametrize("mode", ["tree", "drawn"])
def test_verify_drafts_of_the_largest_vocabularies(V, mode):
    """Up to 2,048 pieces of a row, whose sums take 64 KB of every block's shared memory."""
    lens, temps = [3, 1], [0.75, 1.0]
    logits, draft, parents, tokens, u = drafts_of(lens, V, 3, temps, mode == "tree", near=0.3)
    if mode == "drawn":   # (a draft that is refused, and one that is not)
        tokens[1], u[1], u[2] = int(logits[0].argmax()), 0.0, 1 - 2.0 ** -24
    verify(logits, tokens, lens, u, 3, temps, parents if mode == "tree" else None, draft if mode == "drawn" else None)
    with pytest.raises(K().KernelError):
        wide = torch.zeros(1, 2097153, device=DEV)
        K().verify_drafts(wide, i32([0]), i32([0, 1]), u[:1].to(DEV), i32([[0]]), i32([[0]]), i32([0]), torch.empty(1 << 20, dtype=torch.uint8, device=DEV))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("heads", [(300, 1, 64), (129, 1, 128), (1, 1, 64), (33, 33, 64)])
def test_tree_attention_groups_of_any_size(dtype, heads):
    """Groups of more rows than a unit or a block holds: a token's rows lie in several."""
    c = Case([70, 0, 200], [3, 1, 2], heads, dtype, 64, seed=9, extra_rows=1)
    c.run()
    c.check()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("page", [1024, 4096, 4104])
def test_tree_attention_large_pages(dtype, page):
    c = Case([5000, 17, 0], [20, 3, 1], (8, 2, 64), dtype, page, seed=8)
    c.run(300, window_step=True)
    windowed(c, 300)
    c.check(300)


def test_calls_without_tokens():
    """No rows at all: nothing is written but counts of zero, bounds and tables."""
    ops, none = K(), torch.zeros(0, dtype=torch.int32, device=DEV)
    out, path, count = i32([[7, 7]] * 2), i32([[7, 7]] * 2), i32([7, 7])
    for draft in (None, torch.zeros(0, 50, device=DEV)):
        ops.verify_drafts(torch.zeros(0, 50, device=DEV), none, i32([0, 0, 0]), torch.zeros(0, device=DEV), out, path, count, ops.verify_drafts_scratch(0, 50, DEV),
                          draft_logits=draft)
        assert out.tolist() == path.tolist() == [[-1, -1]] * 2 and count.tolist() == [0, 0]
        out.fill_(7), path.fill_(7), count.fill_(7)
    for d in (64, 512):
        q, kv = torch.zeros(0, 2 * d, dtype=torch.bfloat16, device=DEV), torch.zeros(0, d, dtype=torch.bfloat16, device=DEV)
        ops.tree_attention(q, kv, kv, torch.zeros(2, 2, 8, d, dtype=torch.bfloat16, device=DEV), i32([[0]]), i32([3]), i32([0, 0]), torch.empty_like(q), 2, 1, d, 0.1,
                           ops.tree_attention_scratch(DEV))
    pool = torch.ones(1, 2, 2, 8, 64, device=DEV)
    ops.keep_accepted(torch.zeros(1, 2, 0, 64, device=DEV), pool, none, i32([0, 0]), i32([[0]]), i32([1]))
    assert (pool == 1).all()
    cu, table, taken, after = i32([5] * 3), i32([[4, 9], [9, 9]]), i32([5]), i32([5, 5])
    ops.step_tables(i32([8, 0]), i32([0, 0]), i32([1, 0]), table, none, 8, 9, cu, none, none.clone(), none.clone(), after, taken)
    assert cu.tolist() == [0, 0, 0] and table.tolist() == [[4, 9], [9, 9]] and taken.tolist() == [0] and after.tolist() == [1, 0]
    ops.step_tables(i32([8, 3]), i32([1, 9]), i32([1, 1]), table, none, 8, 9, cu, none, none.clone(), none.clone(), after, taken)   # no room, no page
    assert cu.tolist() == [0, 1, 10] and table.tolist() == [[4, 9], [9, 9]] and taken.tolist() == [2] and after.tolist() == [2, 2]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_verify_and_keep_side_by_side_on_two_streams(dtype):
    """Two requests' batches at once, tensors of their own each."""
    sets = []
    for seed in (1, 2):
        lens, temps = [5, 3, 8], [0.8, 0.0, 1.1]
        logits, draft, _, tokens, u = drafts_of(lens, 33000, seed, temps, False)
        rows, pool = torch.randn(4, 2, 16, 64, device=DEV).to(dtype), torch.zeros(4, 9, 2, 8, 64, dtype=dtype, device=DEV)
        out = [i32([[0] * 8] * 3), i32([[0] * 8] * 3), i32([0] * 3)]
        sets.append((lens, temps, logits, draft, tokens, u, rows, pool, random.Random(seed).sample(range(72), 16), out, K().verify_drafts_scratch(16, 33000, DEV),
                     i32(tokens), i32(cumulate(lens)), u.to(DEV), torch.tensor(temps, device=DEV), torch.cuda.Stream()))
    places = [i32(s[8]) for s in sets]
    torch.cuda.synchronize()
    for _ in range(20):
        for (lens, temps, logits, draft, tokens, u, rows, pool, slots, out, scratch, tok, cu, uni, temp, stream), at in zip(sets, places):
            with torch.cuda.stream(stream):
                K().verify_drafts(logits, tok, cu, uni, *out, scratch, temperature=temp, draft_logits=draft)
                K().keep_accepted(rows, pool, at, cu, out[1], out[2])
    torch.cuda.synchronize()
    for lens, temps, logits, draft, tokens, u, rows, pool, slots, out, *_ in sets:
        want = P.verify(logits.cpu(), tokens, cumulate(lens), u, 8, temps, None, draft.cpu())
        assert dict(tokens=out[0].tolist(), path=out[1].tolist(), count=out[2].tolist()) == want
        assert torch.equal(pool.cpu(), P.keep(rows.cpu(), torch.zeros_like(pool).cpu(), slots, cumulate(lens), want["path"], want["count"]))
