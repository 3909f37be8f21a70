"""prefix_attn (simlingo_amd/paged.py) with values that are not finite, in every own key in turn: they reach the rows that see the
key, all of them and no others, in every form of the kernel, wherever the new tokens begin and beside keys whose page there is not."""
import pytest
import torch

from simlingo_amd import paged as PG

pytestmark = pytest.mark.gpu
BF16, I32 = torch.bfloat16, torch.int32
NAN, INF = float("nan"), float("inf")

FORMS = {  # heads, kv heads, d, new tokens, prefix keys, own page: rows of a sequence's kv head -> how they are taken
    "direct": (14, 2, 64, 2, 0, 8),              # 14
    "direct-small-pages": (14, 2, 64, 5, 0, 2),  # 35
    "direct-single-slots": (4, 1, 128, 3, 0, 1),
    "tiles-64": (14, 2, 64, 4, 0, 8),            # 28
    "tiles-128": (14, 2, 64, 24, 0, 16),         # 168
    "tiles-64-wide": (8, 2, 128, 5, 0, 8),       # 20
    "tiles-128-wide": (8, 2, 128, 24, 0, 8),     # 96
    "whole": (14, 2, 64, 24, 70, 8),             # 64-row tiles of few sequences, 128-row tiles of many
    "whole-wide": (8, 2, 128, 24, 70, 16),
    "beside-a-long-prefix": (14, 2, 64, 4, 3000, 8),
}


@pytest.mark.parametrize("bad_page", (False, True), ids=("pages", "bad-page"))
@pytest.mark.parametrize("form", FORMS)
def test_values_that_are_not_finite_reach_their_rows(dev, form, bad_page):
    """A call for each count X of own keys before the new tokens: sequence i of it has such a value in its key i. Clean and poisoned
    call differ in that value alone, so every other number has to come out the same to the bit."""
    hq, hkv, d, n_q, plen, page = FORMS[form]
    g = torch.Generator(device=dev).manual_seed(3)
    noise = lambda *s: torch.randn(*s, generator=g, device=dev).to(BF16)  # noqa: E731
    prefix = None
    if plen:
        pages = -(-plen // 16)
        prefix = (noise(pages, 16, hkv, d), noise(pages, 16, hkv, d), torch.arange(pages, dtype=I32, device=dev).view(1, -1),
                  torch.tensor([plen], dtype=I32, device=dev))
    wrong = []
    for X in range(131):
        n = X + n_q
        cols = -(-n // page)
        k, v = noise(n * cols, page, hkv, d), noise(n * cols, page, hkv, d)
        table = torch.randperm(n * cols, generator=g, device=dev).to(I32).view(n, cols)
        key = torch.arange(n, device=dev)
        if bad_page:  # the neighbour of the key's page, so in the same 32 keys
            other = (key // page) ^ 1
            table[key[other < cols], other[other < cols]] = -1
        lens = torch.full((n,), n, dtype=I32, device=dev)
        q = noise(n * n_q, hq * d)
        kw = dict(prefix=prefix, n_heads=hq, n_q=n_q)
        clean = PG.prefix_attn(q, own=(k, v, table, lens), **kw).view(n, n_q, hkv, hq // hkv, d)
        head, at = key % hkv, (key * 7) % d
        value = torch.tensor([NAN, INF, -INF], device=dev)[key % 3]
        v[table[key, key // page].long(), key % page, head, at] = value.to(BF16)
        got = PG.prefix_attn(q, own=(k, v, table, lens), **kw).view(n, n_q, hkv, hq // hkv, d)
        want = clean.clone()
        sees = key[:, None] <= X + torch.arange(n_q, device=dev)[None]  # [n, n_q]
        part = want[key, :, head, :, at]                                 # [n, n_q, heads of the kv head]
        want[key, :, head, :, at] = torch.where(sees[..., None], value.to(BF16)[:, None, None].expand_as(part), part)
        same = (got == want) | (torch.isnan(got) & torch.isnan(want))
        assert torch.isfinite(clean).all()
        if not same.all():
            wrong += [(X, i) for i in (~same).flatten(1).any(1).nonzero().view(-1).tolist()]
    assert not wrong, (len(wrong), wrong[:20])


@pytest.mark.parametrize("form", FORMS)
def test_scores_of_minus_infinity_alone_count_as_none(dev, form):
    """A sequence whose keys all score -inf gives zeros and a log sum of -inf, like one without keys; its neighbours are not touched."""
    hq, hkv, d, n_q, plen, page = FORMS[form]
    g = torch.Generator(device=dev).manual_seed(4)
    n, length = 5, 40 + n_q
    cols = -(-length // page)
    k, v = (torch.randn(n * cols, page, hkv, d, generator=g, device=dev).to(BF16) for _ in range(2))
    table = torch.arange(n * cols, dtype=I32, device=dev).view(n, cols)
    lens = torch.full((n,), length, dtype=I32, device=dev)
    q = torch.rand(n * n_q, hq * d, generator=g, device=dev).add_(0.1).to(BF16)
    prefix = None
    if plen:  # the second sequence's group alone has a prefix of -inf
        pages = -(-plen // 16)
        pk, pv = (torch.randn(2 * pages, 16, hkv, d, generator=g, device=dev).to(BF16) for _ in range(2))
        prefix = (pk, pv, torch.stack([torch.arange(pages, device=dev) + i * pages for i in (0, 1, 0, 0, 0)]).to(I32),
                  torch.full((n,), plen, dtype=I32, device=dev))
    call = lambda lse: PG.prefix_attn(q, own=(k, v, table, lens), prefix=prefix, n_heads=hq, n_q=n_q, lse=lse).view(n, n_q, hq * d)  # noqa: E731
    lse = [torch.full((n * n_q, hq), 3.0, device=dev) for _ in range(2)]
    before = call(lse[0])
    k[table[1].long()] = -INF
    if plen:
        pk[pages:] = -INF
    after = call(lse[1])
    assert not after[1].any() and (lse[1].view(n, -1)[1] == -INF).all()
    rest = [0, 2, 3, 4]
    assert torch.equal(after[rest], before[rest]) and torch.equal(lse[0].view(n, -1)[rest], lse[1].view(n, -1)[rest])
