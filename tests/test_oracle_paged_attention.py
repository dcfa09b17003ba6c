"""Pins of oracle/paged_attention.py (CPU): torch's attention over dense keys,
and the join of two parts by their lse."""
import math

import torch
import torch.nn.functional as F

from oracle import paged_attention as opa


def _paged(k, page):
    """[n, Hkv, D] as a cache whose pages lie in reverse, and its table row."""
    n, hkv, d = k.shape
    pages = -(-n // page)
    c = torch.full((pages + 1, page, hkv, d), math.nan, dtype=k.dtype)
    row = torch.arange(pages - 1, -1, -1, dtype=torch.int32)
    for j in range(n):
        c[row[j // page], j % page] = k[j]
    return c, row[None]


def _case(n, hq, hkv, d, t, seed=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64).float()  # noqa: E731
    return r(1, t, hq, d), r(n, hkv, d), r(n, hkv, d)


def test_matches_torch_attention_with_drafts_and_window():
    for window in (0, 5):
        q, k, v = _case(37, 6, 2, 8, 3)
        kc, row = _paged(k, 4)
        vc, _ = _paged(v, 4)
        got = opa.attention(q, kc, vc, row, torch.tensor([37]), window=window)
        at = 34 + torch.arange(3)[:, None]
        mask = (torch.arange(37) <= at) & ((torch.arange(37) > at - window) if window else True)
        want = F.scaled_dot_product_attention(
            q[0].transpose(0, 1).double(), k.repeat_interleave(3, 1).transpose(0, 1).double(),
            v.repeat_interleave(3, 1).transpose(0, 1).double(), mask)
        torch.testing.assert_close(got["o"][0], want.transpose(0, 1))


def test_parts_join_by_their_lse():
    q, k, v = _case(40, 4, 4, 8, 1, 3)
    whole = opa.attention(q, *[_paged(x, 8)[0] for x in (k, v)], _paged(k, 8)[1], torch.tensor([40]))
    parts = [opa.attention(q, *[_paged(x[s], 8)[0] for x in (k, v)], _paged(k[s], 8)[1],
                           torch.tensor([n])) for s, n in ((slice(0, 16), 16), (slice(16, 40), 24))]
    w = torch.softmax(torch.stack([p["lse"] for p in parts]), 0)
    torch.testing.assert_close(sum(w[i][..., None] * parts[i]["o"] for i in range(2)), whole["o"])
    torch.testing.assert_close(torch.logsumexp(torch.stack([p["lse"] for p in parts]), 0),
                               whole["lse"])


def test_rows_that_see_nothing_are_zero():
    q, k, v = _case(5, 2, 1, 8, 3)
    kc, row = _paged(k, 4)
    vc, _ = _paged(v, 4)
    o = opa.attention(q, kc, vc, row, torch.tensor([2]))
    assert (o["o"][0, 0] == 0).all() and (o["lse"][0, 0] == -math.inf).all()
    assert o["lse"][0, 1:].isfinite().all()
    o = opa.attention(q, kc, vc, torch.full_like(row, -1), torch.tensor([5]))
    assert (o["o"] == 0).all()
