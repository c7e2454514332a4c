"""The operators of a drafted step at the ends of what they take: temperatures, scores and lengths of every size, tensors that lie in one
another, bounds beyond the step; against the plain forms in 64 bits."""
import math

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
