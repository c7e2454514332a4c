"""What the launchers of a drafted step's operators refuse before they touch a device (no GPU needed), and the plain forms that
the GPU tests compare with, against formulas of their own."""
import math

import pytest
import torch

from plain import drafts_plain as P
from poor_mans_mamba_b200.kernels import ops as K

BAD = K.PMM_ERR_BAD_ARGUMENT
A = 1 << 20  # a pointer that nothing follows


def refused(name, good, **bad):
    """The launcher's arguments `good` with some replaced."""
    args = dict(good)
    for key, value in bad.items():
        assert key in args
        args[key] = value
    return K._fn(name)(*args.values()) == BAD


TABLES = dict(held=A, new=A, blocks=A, table=A, width=8, free=A, n_free=4, n=2, page_size=64, spare=100, cu=A, seq_of=A, positions=A, slots=A,
              cap=10, blocks_out=A, taken=A, parents=None, masks=None, words=0, stream=None)
KEEP = dict(rows=A, ld_layer=100, ld_plane=100, ld_row=100, n_rows=4, pool=A, layers=1, pages=4, planes=2, page_size=64, width=64, item=2,
            slots=A, cu=A, path=A, path_width=4, count=A, n=2, stream=None)
VERIFY = dict(logits=A, ld=100, draft=None, ld_draft=0, tokens=A, parents=None, cu=A, n=2, uniforms=A, temperature=None, V=100, n_rows=4,
              scratch=A, tokens_out=A, path=A, width=4, count=A, sms=148, stream=None)


@pytest.mark.parametrize("bad", [dict(width=0), dict(page_size=0), dict(spare=-1), dict(spare=1 << 26), dict(parents=A), dict(masks=A),
                                 dict(parents=A, masks=A, words=0), dict(parents=A, masks=A, words=5), dict(cap=-1), dict(n_free=-1)])
def test_step_tables_refuses(bad):
    assert refused("pmm_step_tables", TABLES, **bad)


@pytest.mark.parametrize("bad", [dict(pages=0), dict(page_size=0), dict(width=0), dict(item=1), dict(item=8), dict(path_width=0), dict(n_rows=-1),
                                 dict(n=70000)])
def test_keep_accepted_refuses(bad):
    assert refused("pmm_keep_accepted", KEEP, **bad)


@pytest.mark.parametrize("bad", [dict(V=0), dict(V=1 << 30), dict(n_rows=-1), dict(width=0), dict(scratch=None), dict(scratch=A + 8), dict(sms=0),
                                 dict(draft=A, parents=A)])
def test_verify_drafts_refuses(bad):
    assert refused("pmm_verify_drafts", VERIFY, **bad)


def test_tensors_of_the_host_are_refused():
    i = torch.zeros(2, dtype=torch.int32)
    f = torch.zeros(2, 16)
    with pytest.raises(K.KernelError):
        K.step_tables(i, i, i, i.view(2, 1), i, 64, 1, i, i, i, i, i, i)
    with pytest.raises(K.KernelError):
        K.verify_drafts(f, i, i, f[0], i.view(2, 1), i.view(2, 1), i, f)
    with pytest.raises(K.KernelError):
        K.keep_accepted(f[None], f.view(1, 1, 2, 16), i, i, i.view(2, 1), i)
    with pytest.raises(K.KernelError):
        K.tree_attention(f, f, f, f.view(1, 2, 1, 16), i.view(2, 1), i, i, f, 1, 1, 16, 1.0, f)


# ----------------------------------------------------------------------------- the plain forms themselves
def test_plain_verification_leaves_tokens_distributed_as_the_target():
    """The first token of a step over many uniforms: chains from a draft and fixed proposals both leave p."""
    g = torch.Generator().manual_seed(3)
    V, n = 5, 4000
    logits, draft = torch.randn(3, V, generator=g), torch.randn(3, V, generator=g)
    p, q = torch.softmax(logits[0].double() / 0.8, 0), torch.softmax(draft[0].double() / 0.8, 0)
    for drawn in (True, False):
        got = torch.zeros(V)
        for _ in range(n):
            x = int(torch.multinomial(q, 1, generator=g))
            u = torch.rand(3, generator=g)
            r = P.verify(logits, [0, x, 1], [0, 3], u, 3, [0.8], None, draft if drawn else None)
            got[r["tokens"][0][0]] += 1
        # (a count of n draws is off by more than five of its standard deviations once in a million)
        assert ((got / n - p).abs() <= 5 * (p * (1 - p) / n).sqrt()).all()


def test_plain_tree_attention_of_a_chain_is_causal_attention():
    g = torch.Generator().manual_seed(1)
    k, v, q = torch.randn(9, 2, 16, generator=g), torch.randn(9, 2, 16, generator=g), torch.randn(9, 4, 16, generator=g)
    out, _, _ = P.tree_attention(q[5:], k[5:], v[5:], k[:5], v[:5], torch.ones(4, 5, dtype=torch.bool), torch.ones(4, 4, dtype=torch.bool).tril(), 0.25)
    ref = torch.nn.functional.scaled_dot_product_attention(q.double().transpose(0, 1), k.double().transpose(0, 1).repeat_interleave(2, 0),
                                                           v.double().transpose(0, 1).repeat_interleave(2, 0), is_causal=True, scale=0.25)
    assert (out - ref.transpose(0, 1)[5:]).abs().max() < 1e-12


def test_plain_tables_of_a_small_step():
    t = P.step_tables([3, 0, 8], [2, 1, 0], [1, 0, 2], [[5, 9], [9, 9], [6, 7]], [1, 2], 4, 9, 5, parents=[-1, 0, -1, -1, -1], words=1)
    assert t["cu"] == [0, 2, 3, 3] and t["table"] == [[5, 1], [2, 9], [6, 7]] and t["blocks"] == [2, 1, 2] and t["taken"] == [2]
    assert t["seq_of"] == [0, 0, 1, -7, -7] and t["positions"] == [3, 4, 0, -7, -7] and t["slots"] == [5 * 4 + 3, 1 * 4, 2 * 4, -7, -7]
    assert t["masks"] == [[1], [3], [1], [-7], [-7]]
    assert math.isclose(sum(t["cu"]), 8)


# ----------------------------------------------------------------------------- tensors that lie in one another
def overlaps(name, good, **other):
    args = dict(good)
    for key, value in other.items():
        assert key in args
        args[key] = value
    return K._fn(name)(*args.values()) == K.PMM_ERR_OVERLAP


def test_keep_accepted_refuses_rows_in_the_pool():
    """The pool has 1 MiB here; two planes of four rows of 128 bytes, 200 bytes apart."""
    pool = 1 << 30
    good = dict(KEEP, pool=pool, pages=64, page_size=64, planes=2, width=64, item=2, ld_plane=400, ld_layer=800, ld_row=100, slots=A, n=2)
    size = 64 * 2 * 64 * 64 * 2
    last = (400 + 3 * 100 + 64) * 2     # bytes from the first row to the end of the last
    for at, bad in [(pool, True), (pool + 500, True), (pool - 2, True), (pool - last, False), (pool - last + 2, True), (pool + size - 2, True),
                    (pool + size, False), (pool - 8 * last, False)]:
        assert overlaps("pmm_keep_accepted", good, rows=at) == bad, at - pool
    # rows around a pool: layers in front of it and behind it, none in it
    wide = dict(good, layers=2, pages=16, ld_layer=(size + 4096) // 2)
    assert not overlaps("pmm_keep_accepted", wide, rows=pool - 4096)
    assert overlaps("pmm_keep_accepted", dict(wide, ld_layer=size // 4), rows=pool - 4096)
    assert not overlaps("pmm_keep_accepted", dict(good, n_rows=0), rows=pool)


def test_step_tables_refuses_outputs_in_its_inputs():
    """Two requests of ten tokens: lengths of 8 bytes, a table of 64, tokens' tensors of 40."""
    names = ["held", "new", "blocks", "free", "table", "cu", "seq_of", "positions", "slots", "blocks_out", "taken", "parents", "masks"]
    apart = dict(TABLES, words=1, **{k: A + 4096 * i for i, k in enumerate(names)})
    assert not overlaps("pmm_step_tables", apart)
    size = dict(held=8, new=8, blocks=8, parents=40)
    for out in ("cu", "blocks_out", "taken", "table", "seq_of", "positions", "slots", "masks"):
        for name, bytes_of in size.items():
            for at, bad in ((0, True), (bytes_of - 4, True), (bytes_of, False)):
                assert overlaps("pmm_step_tables", apart, **{out: apart[name] + at}) == bad, (out, name, at)
    assert overlaps("pmm_step_tables", apart, cu=apart["blocks"] - 8) and not overlaps("pmm_step_tables", apart, cu=apart["blocks"] - 12)
    assert overlaps("pmm_step_tables", apart, table=apart["free"] - 60) and not overlaps("pmm_step_tables", apart, table=apart["free"] - 64)


def test_verify_drafts_refuses_outputs_in_its_inputs():
    """Two requests of four tokens over 100 entries, outputs four wide."""
    names = ["logits", "tokens", "cu", "uniforms", "temperature", "scratch", "tokens_out", "path", "count"]
    apart = dict(VERIFY, **{k: A + 8192 * i for i, k in enumerate(names)})
    assert not overlaps("pmm_verify_drafts", apart)
    size = dict(tokens=16, cu=12, uniforms=16, temperature=8, scratch=4 * 2 * 16 + 16, tokens_out=32, path=32, count=8)
    for out in ("tokens_out", "path", "count"):
        for name, bytes_of in size.items():
            if name != out:
                for at, bad in ((0, True), (bytes_of - 4, True), (bytes_of, False)):
                    assert overlaps("pmm_verify_drafts", apart, **{out: apart[name] + at}) == bad, (out, name, at)
    # rows of 100 entries, 150 apart: between them there is room
    for rows in (dict(logits=A, ld=150), dict(draft=A + 8192 * 20, ld_draft=150)):
        base = rows.get("draft", A)
        for at, bad in ((0, True), (396, True), (400, False), (600 - 32, False), (600 - 28, True), (3 * 600 + 399, True), (3 * 600 + 400, False)):
            assert overlaps("pmm_verify_drafts", apart, **rows, path=base + at) == bad, at
    assert overlaps("pmm_verify_drafts", apart, **{"parents": apart["path"]})


TREE = dict(q=A, ldq=512, k=A, ldk=128, v=A, ldv=128, pool=A, pages=4, block_table=A, max_blocks=2, held=A, cu=A, positions=None, mask=None, words=0,
            sink=None, out=A, scale=0.125, window=0, window_step=0, page_size=64, n_seq=2, T=6, Hq=8, Hkv=2, Dh=64)


@pytest.mark.parametrize("name,elem,last", [("pmm_tree_attention", 4, dict(dtype=0, sms=148, stream=None)), ("pmm_tree_attention", 2, dict(dtype=1, sms=148, stream=None)),
                                            ("pmm_tree_attention_tc", 2, dict(wide=0, scratch=A, sms=148, status=A, stream=None))])
def test_tree_attention_refuses_outputs_in_its_inputs(name, elem, last):
    """Six rows of 512 values beside keys and values of 128."""
    M = 1 << 24
    apart = {**TREE, **last, "q": M, "k": 2 * M, "v": 3 * M, "pool": 4 * M, "out": 5 * M}
    if "scratch" in last:
        apart["scratch"] = 6 * M
    assert not overlaps(name, apart)
    row, kv = 512 * elem, 128 * elem
    for at, bad in ((4 * M, True), (4 * M + 4 * 2 * 64 * kv - 16, True), (4 * M + 4 * 2 * 64 * kv, False), (4 * M - 6 * row + 16, True), (4 * M - 6 * row, False),
                    (2 * M + 6 * kv - 16, True), (2 * M + 6 * kv, False), (3 * M, True), (M, False), (M + row, True), (M - 16, True), (M + 6 * row, False)):
        assert overlaps(name, apart, out=at) == bad, (at / M, at % M)
    # q a slice of rows twice as wide: not in place
    assert overlaps(name, apart, ldq=1024, out=M) and not overlaps(name, apart, ldq=1024, out=M, T=1)
    # one row: its neighbours in the same row are free
    assert not overlaps(name, apart, T=1, q=M, ldq=4096, k=M + row, ldk=4096, v=M + row + kv, ldv=4096, out=M + row + 2 * kv)
    assert overlaps(name, apart, T=1, q=M, ldq=4096, k=M + row, ldk=4096, v=M + row + kv, ldv=4096, out=M + row + kv)


def test_sizes_of_scratch_are_not_remembered_without_end():
    for rows in range(1, 3 * K._SIZES_KEPT):
        assert K._sized("pmm_verify_scratch", rows, 5000) == 2 * rows * 5 * 16 + 4 * rows
        assert len(K._SIZES) <= K._SIZES_KEPT
