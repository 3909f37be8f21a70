"""Paged cache operators (simlingo_amd/paged.py: kv_append, prefix_attn) against plain 64-bit forms (paged_ref.py)."""
import pytest
import torch

import paged_ref as R
from simlingo_amd import kernels as K
from simlingo_amd import paged as PG

pytestmark = pytest.mark.gpu
BF16, I32 = torch.bfloat16, torch.int32


def gen(seed):
    return torch.Generator().manual_seed(seed)


def noise(g, *shape, scale=1.0):
    return (torch.randn(*shape, generator=g) * scale).to(BF16)


def pools(g, n_pages, page, heads, d, layout="slots"):
    """k, v on the CPU with garbage everywhere; layout: slot-major, head-major, or both interleaved in one allocation."""
    if layout == "heads":
        return tuple(noise(g, n_pages, heads, page, d).permute(0, 2, 1, 3) for _ in range(2))
    if layout == "pair":
        x = noise(g, n_pages, page, 2, heads, d)
        return x[:, :, 0], x[:, :, 1]
    return tuple(noise(g, n_pages, page, heads, d) for _ in range(2))


def to(t, dev):
    """On the device with the same strides."""
    if t is None:
        return None
    if t.is_contiguous():
        return t.to(dev)
    base = t._base if t._base is not None else t
    return base.to(dev).as_strided(t.shape, t.stride(), t.storage_offset())


def tables(g, lens, page, extra=0):
    cols = max(1, max(-(-n // page) for n in lens)) + extra
    n = len(lens) * cols
    return torch.randperm(n, generator=g).to(I32).view(len(lens), cols), n


# ---- kv_append ----------------------------------------------------------------------------------------------------
APPEND = [  # heads, kv heads, d, page, lengths before, new rows each, layout
    (14, 2, 64, 1, [40, 40, 40, 40], 1, "slots"),
    (14, 2, 64, 16, [0], 133, "pair"),
    (2, 1, 64, 64, [63, 0, 64], 3, "heads"),
    (32, 8, 128, 16, [5, 31, 100], 17, "slots"),
    (3, 3, 128, 256, [0, 255], 2, "heads"),
    (1, 1, 64, 2, [0], 1, "slots"),
]


@pytest.mark.parametrize("hq,hkv,d,page,before,new,layout", APPEND)
def test_kv_append(dev, hq, hkv, d, page, before, new, layout):
    g = gen(hq * 7 + page)
    table, n_pages = tables(g, [b + new for b in before], page, extra=1)
    k, v = pools(g, n_pages + 1, page, hkv, d, layout)
    seq = torch.tensor([i for i in range(len(before)) for _ in range(new)], dtype=I32)
    pos = torch.tensor([b + t for b in before for t in range(new)], dtype=I32)
    order = torch.randperm(len(pos), generator=g)
    seq, pos = seq[order], pos[order]
    wide = noise(g, len(pos), (hq + 2 * hkv) * d + 24)  # rows with a stride of their own
    cos, sin = K.rope_tables(int(pos.max()) + 1, 1e6, "cpu", d)
    dk, dv, dq = to(k, dev), to(v, dev), torch.full((len(pos), hq * d + 8), 7.0, dtype=BF16, device=dev)
    dw = wide.to(dev)
    PG.kv_append(dw[:, :-24], dk, dv, table.to(dev), pos.to(dev), dq[:, :-8], n_heads=hq, cos=cos.to(dev), sin=sin.to(dev), seq=seq.to(dev))
    q, ko, vo, _ = R.append(wide[:, :-24].contiguous(), k, v, table, pos, seq, hq, cos, sin)
    # rotation in f32 (three roundings of terms of at most |x| + |y|), then one rounding to bf16
    big = wide.double().abs().max() * 2
    for got, want in ((dq[:, :-8], q), (dk, ko)):
        assert ((got.cpu().double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -22 * big).all()
    assert torch.equal(dv.cpu().double(), vo)
    assert (dq[:, -8:] == 7.0).all() and torch.equal(dw.cpu(), wide)


def test_kv_append_leaves_padding(dev):
    """Positions below 0, behind the table or the rotation's rows, sequences and pages that there are not: nothing is written."""
    g = gen(1)
    hq, hkv, d, page = 2, 1, 64, 4
    k, v = pools(g, 6, page, hkv, d)
    table = torch.tensor([[0, 1, 2], [3, -1, 6], [2**31 - 1, -2**31, 5]], dtype=I32)
    seq = torch.tensor([0, 0, 0, 1, 1, 1, 2, 2, 2, 3, -1, 0, 0], dtype=I32)
    pos = torch.tensor([0, -1, 12, 3, 4, 8, 0, 4, 9, 0, 0, 10, 2**31 - 1], dtype=I32)
    qkv = noise(g, len(pos), (hq + 2 * hkv) * d)
    cos, sin = K.rope_tables(10, 1e4, "cpu", d)  # position 10 has no row
    dk, dv, dq = k.to(dev), v.to(dev), torch.full((len(pos), hq * d), 7.0, dtype=BF16, device=dev)
    PG.kv_append(qkv.to(dev), dk, dv, table.to(dev), pos.to(dev), dq, n_heads=hq, cos=cos.to(dev), sin=sin.to(dev), seq=seq.to(dev))
    q, ko, vo, done = R.append(qkv, k, v, table, pos, seq, hq, cos, sin)
    assert done.tolist() == [True, False, False, True, False, False, False, False, True, False, False, False, False]
    assert (dq.cpu()[~done] == 7.0).all() and torch.equal(dv.cpu().double(), vo)
    assert ((dk.cpu().double() - ko).abs() <= 2.0 ** -8 * ko.abs() + 2.0 ** -20).all()
    assert ((dq.cpu().double() - q)[done].abs() <= 2.0 ** -8 * q[done].abs() + 2.0 ** -20).all()


def test_kv_append_in_place_and_without(dev):
    """q rotated in the rows themselves equals q rotated elsewhere; without tables it is a copy; without q_out q is not touched."""
    g = gen(2)
    hq, hkv, d, n = 14, 2, 64, 9
    qkv = noise(g, n, (hq + 2 * hkv) * d).to(dev)
    table, pos = torch.arange(n, dtype=I32, device=dev).view(n, 1), torch.zeros(n, dtype=I32, device=dev)
    cos, sin = K.rope_tables(4, 1e6, dev)
    pos.fill_(3)
    table = torch.arange(n, dtype=I32, device=dev).view(n, 1)
    outs = []
    for inside in (False, True):
        x = qkv.clone()
        k, v = (torch.zeros(n, 4, hkv, d, dtype=BF16, device=dev) for _ in range(2))
        q = x[:, :hq * d] if inside else torch.empty(n, hq * d, dtype=BF16, device=dev)
        PG.kv_append(x, k, v, table, pos, q, n_heads=hq, cos=cos, sin=sin)
        outs.append((q.clone(), k, v))
        assert torch.equal(x[:, hq * d:], qkv[:, hq * d:])
    for a, b in zip(*outs):
        assert torch.equal(a, b)
    k, v = (torch.zeros(n, 4, hkv, d, dtype=BF16, device=dev) for _ in range(2))
    x = qkv.clone()
    PG.kv_append(x, k, v, table, pos, n_heads=hq)
    assert torch.equal(x, qkv)
    assert torch.equal(k[:, 3].reshape(n, -1), qkv[:, hq * d:(hq + hkv) * d]) and not k[:, :3].any()
    assert torch.equal(v[:, 3].reshape(n, -1), qkv[:, (hq + hkv) * d:])
    PG.kv_append(x[:0], k, v, table, pos[:0], n_heads=hq)  # no rows


# ---- prefix_attn --------------------------------------------------------------------------------------------------
def case(seed, hq, hkv, d, groups, width, n_q, plens, ppage, olens, opage, layout="slots", scale=1.5):
    g = gen(seed)
    n = groups * width
    prefix = None
    if plens is not None:
        ptab, np_ = tables(g, plens, ppage)
        pk, pv = pools(g, np_, ppage, hkv, d, layout)
        prefix = (pk, pv, ptab, torch.tensor(plens, dtype=I32))
    otab, no = tables(g, olens, opage)
    ok, ov = pools(g, no, opage, hkv, d, layout)
    own = (ok, ov, otab, torch.tensor(olens, dtype=I32))
    return noise(g, n * n_q, hq * d, scale=scale), own, prefix


def on(dev, kv):
    return None if kv is None else tuple(to(t, dev) for t in kv)


def run(dev, q, own, prefix, hq, n_q, **kw):
    lse = torch.full((q.shape[0], hq), 3.0, device=dev)
    out = PG.prefix_attn(q.to(dev), own=on(dev, own), prefix=on(dev, prefix), n_heads=hq, n_q=n_q, lse=lse, **kw)
    return out.cpu(), lse.cpu()


def check(dev, q, own, prefix, hq, n_q, **kw):
    out, lse = run(dev, q, own, prefix, hq, n_q, **kw)
    want, wl, spread = R.attn(q, own, prefix, hq, n_q, **kw)
    ok = R.close_attn(out, want, spread)
    assert ok.all(), (out.double() - want).abs().max()
    none = torch.isinf(wl)
    assert torch.equal(none, torch.isinf(lse)) and (lse[none] < 0).all()
    # the sum of probabilities rounded to bf16: its log moves by at most 2^-8
    assert ((lse.double() - wl)[~none].abs() <= 2.0 ** -8 * 1.05).all()
    return out


ATTN = [  # heads, kv heads, d, groups, width, n_q, prefixes, page, own lengths, page, layout
    (2, 1, 64, 1, 1, 1, [1], 1, [1], 1, "slots"),
    (14, 2, 64, 1, 4, 1, [70], 64, [5, 5, 5, 5], 1, "slots"),
    (14, 2, 64, 2, 3, 1, [33, 257], 16, [1, 15, 16, 17, 31, 129], 16, "heads"),
    (14, 2, 64, 1, 16, 1, [300], 32, [3] * 16, 2, "pair"),
    (32, 8, 128, 1, 2, 1, [131], 8, [40, 7], 4, "heads"),
    (32, 8, 128, 2, 5, 1, [97, 128], 256, [1, 2, 3, 4, 5, 160, 33, 32, 31, 64], 16, "slots"),
    (4, 4, 128, 1, 3, 1, None, 0, [1, 200, 64], 8, "pair"),
    (14, 2, 64, 3, 1, 1, None, 0, [700, 1, 129], 64, "heads"),
    (14, 2, 64, 1, 3, 9, [45], 16, [9, 30, 12], 4, "slots"),
    (2, 1, 64, 2, 2, 40, [64, 5], 8, [40, 47, 100, 41], 16, "slots"),
    (8, 1, 128, 1, 2, 5, [19], 1, [5, 70], 2, "slots"),
    (16, 1, 64, 1, 2, 3, [200], 128, [3, 4], 32, "slots"),
    # more rows than a wave holds: tiles shared by the workgroup
    (14, 2, 64, 1, 8, 1, [1], 8, [1] * 8, 8, "slots"),
    (14, 2, 64, 2, 7, 1, [127, 300], 8, [5] * 14, 16, "heads"),
    (14, 2, 64, 1, 40, 1, [161], 64, [2] * 40, 1, "pair"),
    (32, 8, 128, 1, 12, 1, [419], 8, [9] * 12, 16, "slots"),
    (32, 8, 128, 2, 19, 1, [33, 290], 32, [3] * 38, 4, "pair"),
    (8, 2, 128, 1, 2, 21, [77], 16, [21, 150], 8, "heads"),
    (14, 2, 64, 1, 2, 6, [0], 16, [6, 333], 32, "slots"),
    (4, 1, 64, 1, 1, 37, None, 0, [300], 16, "slots"),
    (3, 3, 64, 1, 2, 50, [64], 16, [50, 20], 16, "slots"),
    (5, 1, 128, 1, 3, 13, [40], 64, [13, 14, 64], 8, "slots"),
    (16, 1, 128, 1, 2, 20, [9], 2, [25, 40], 64, "slots"),
]


@pytest.mark.parametrize("c", ATTN, ids=lambda c: "h%d-%d-d%d-g%dx%d-q%d-p%s-o%s" % (c[0], c[1], c[2], c[3], c[4], c[5], c[7], c[9]))
def test_prefix_attn(dev, c):
    hq, hkv, d, groups, width, n_q, plens, ppage, olens, opage, layout = c
    q, own, prefix = case(sum(olens) + hq, hq, hkv, d, groups, width, n_q, plens, ppage, olens, opage, layout)
    check(dev, q, own, prefix, hq, n_q)


@pytest.mark.parametrize("d", (64, 128))
@pytest.mark.parametrize("n,n_q", ((6, 40), (9, 61), (12, 33), (3, 97)))
def test_prefix_attn_whole_rows(dev, d, n, n_q):
    """32 kv heads x n sequences of 64-row tiles, in one part: 8 waves or 4 a tile, and tiles of 128 rows; own keys that end in and
    between tiles, a prefix that ends in one, a query of NaN and its neighbours, and the output in the queries' place."""
    q, own, prefix = case(n, 32, 32, d, 1, n, n_q, [77], 16, [n_q + i * 23 % 70 for i in range(n)], 8)
    q[5, d:2 * d] = 0.0
    out = check(dev, q, own, prefix, 32, n_q)
    x = q.clone()
    x[5, d:2 * d] = float("nan")
    x = x.to(dev)
    got = PG.prefix_attn(x, x, own=on(dev, own), prefix=on(dev, prefix), n_heads=32, n_q=n_q).cpu()
    assert torch.isnan(got[5, d:2 * d]).all()
    got[5, d:2 * d] = out[5, d:2 * d]
    assert torch.equal(got, out)


def test_prefix_attn_many_ranges(dev):
    """Long keys, few rows: many ranges a row, and a second call with short lengths in the same tables."""
    q, own, prefix = case(3, 2, 1, 64, 1, 2, 1, [2100], 64, [1500, 40], 16)
    check(dev, q, own, prefix, 2, 1)
    short = (own[0], own[1], own[2], torch.tensor([1, 0], dtype=I32))
    check(dev, q, short, (*prefix[:3], torch.tensor([3], dtype=I32)), 2, 1)


def test_prefix_attn_peaked(dev):
    """Scores that rise along the keys, far apart: the running maximum moves again and again, and terms vanish."""
    for sign in (1, -1):
        q, own, prefix = case(4, 2, 1, 64, 1, 2, 1, [600], 64, [140, 33], 16)
        q = (q.float().abs() * 3).to(BF16)
        ramp = torch.linspace(-6, 6, 640).view(10, 64, 1, 1) * sign
        pk = torch.empty_like(prefix[0])
        pk[prefix[2][0].long()] = (prefix[0][prefix[2][0].long()].float().abs() * 0.2 + ramp).to(BF16)
        check(dev, q, own, (pk, *prefix[1:]), 2, 1)


def test_prefix_attn_empty_rows(dev):
    """No key at all gives zeros and -inf; lengths below 0 count as 0; new tokens before the first own key see the prefix only."""
    q, own, prefix = case(5, 14, 2, 64, 2, 3, 4, [40, 30], 16, [9] * 6, 4)
    own = (*own[:3], torch.tensor([0, 2, -5, 0, 9, 1], dtype=I32))
    prefix = (*prefix[:3], torch.tensor([0, 17], dtype=I32))
    out = check(dev, q, own, prefix, 14, 4)
    assert not out[0:4].any() and not out[4:6].any() and not out[8:12].any() and out[12:].any()
    out = check(dev, q, own, None, 14, 4)
    assert not out[12:16].any()


def test_prefix_attn_masked_values(dev):
    """NaN and infinities in slots behind the lengths, in other pages and in keys that a token does not see yet stay out."""
    q, own, prefix = case(6, 14, 2, 64, 1, 2, 3, [41], 16, [5, 37], 8)
    for kv, lens in ((own, [5, 37]), (prefix, [41])):
        used = torch.zeros(kv[0].shape[:2], dtype=torch.bool)
        for i, n in enumerate(lens):
            for j in range(n):
                used[kv[2][i, j // kv[0].shape[1]], j % kv[0].shape[1]] = True
        kv[0][~used] = float("nan")
        kv[1][~used] = float("inf")
    check(dev, q, own, prefix, 14, 3)
    # the last own key's value is not finite: the last token's rows only
    clean, _ = run(dev, q, own, prefix, 14, 3)
    pg, sl = own[2][1, 36 // 8], 36 % 8
    own[1][pg, sl, 0, 5] = float("nan")
    own[1][pg, sl, 1, 9] = -float("inf")
    got, _ = run(dev, q, own, prefix, 14, 3)
    bad = torch.zeros_like(got, dtype=torch.bool).view(2, 3, 14, 64)
    bad[1, 2, :7, 5] = True
    bad[1, 2, 7:, 9] = True
    bad = bad.view_as(got)
    assert torch.equal(got[~bad], clean[~bad])
    assert torch.isnan(got.view(2, 3, 14, 64)[1, 2, :7, 5]).all() and (got.view(2, 3, 14, 64)[1, 2, 7:, 9] == -float("inf")).all()


def test_prefix_attn_masked_values_many_rows(dev):
    """The same with tiles that a workgroup shares: garbage behind the lengths, non-finite values in keys seen by some rows."""
    for d, hq, hkv in ((64, 14, 2), (128, 8, 2)):
        q, own, prefix = case(17, hq, hkv, d, 1, 2, 24, [41], 16, [30, 90], 8)
        for kv, lens in ((own, [30, 90]), (prefix, [41])):
            used = torch.zeros(kv[0].shape[:2], dtype=torch.bool)
            for i, n in enumerate(lens):
                for j in range(n):
                    used[kv[2][i, j // kv[0].shape[1]], j % kv[0].shape[1]] = True
            kv[0][~used] = float("nan")
            kv[1][~used] = float("nan")
        clean = check(dev, q, own, prefix, hq, 24).view(2, 24, hq, d)
        for i, key, head, at, val in ((0, 29, 0, 5, float("nan")), (1, 80, 1, 9, float("inf")), (1, 70, 0, d - 1, -float("inf"))):
            own[1][own[2][i, key // 8], key % 8, head, at] = val
        got = run(dev, q, own, prefix, hq, 24)[0].view(2, 24, hq, d)
        r = hq // hkv
        bad = torch.zeros_like(got, dtype=torch.bool)
        for i, key, head, at, val, n in ((0, 29, 0, 5, float("nan"), 30), (1, 80, 1, 9, float("inf"), 90), (1, 70, 0, d - 1, -float("inf"), 90)):
            part = got[i, key - (n - 24):, head * r:(head + 1) * r, at]
            assert torch.isnan(part).all() if val != val else (part == val).all()
            bad[i, key - (n - 24):, head * r:(head + 1) * r, at] = True
        assert torch.equal(got[~bad], clean[~bad])


def test_prefix_attn_nan_reaches_the_output(dev):
    """A query that is NaN, and a sequence whose only key is: NaN in those rows and no others, in one part or split, few rows or many."""
    nan = float("nan")
    for hq, hkv, d, width, n_q, plens, olens in ((14, 2, 64, 2, 1, None, [1, 40]), (14, 2, 64, 2, 1, [300], [1, 140]), (14, 2, 64, 6, 1, [300], [5] * 6),
                                                 (14, 2, 64, 20, 1, [300], [1] * 20), (32, 8, 128, 20, 1, [200], [7] * 20), (8, 2, 64, 26, 30, [70], [31] * 26),
                                                 (8, 2, 128, 26, 30, [70], [31] * 26), (6, 2, 64, 2, 40, None, [40, 60])):
        q, own, prefix = case(23, hq, hkv, d, 1, width, n_q, plens, 16, olens, 8)
        q[-1, :d] = nan                                       # the last token's first head
        if olens[0] == 1:
            own[0][int(own[2][0, 0]), 0, hkv - 1] = nan       # sequence 0's only own key, last kv head
        out, lse = run(dev, q, own, prefix, hq, n_q)
        out = out.view(-1, hq, d)
        want = torch.zeros(out.shape[0], hq, dtype=torch.bool)
        want[-1, 0] = True
        if olens[0] == 1:
            want[0, hq - hq // hkv:] = True
        assert torch.equal(torch.isnan(out).all(-1), want) and torch.equal(torch.isnan(out).any(-1), want)
        assert torch.equal(torch.isnan(lse), want)


def test_prefix_attn_bad_pages(dev):
    """Keys on page numbers outside the cache are masked, in both caches and at every page size."""
    for ppage, opage in ((16, 8), (64, 1), (2, 32)):
        q, own, prefix = case(7, 4, 2, 64, 1, 3, 1, [150], ppage, [40, 9, 70], opage)
        own[2][0, 0], own[2][2, -1], prefix[2][0, 1] = -1, own[0].shape[0], 2**31 - 1
        check(dev, q, own, prefix, 4, 1)
    for d, hq, hkv, n_q in ((64, 14, 2, 1), (128, 8, 2, 20)):
        q, own, prefix = case(18, hq, hkv, d, 1, 9, n_q, [290], 8, [40] * 9, 8)
        own[2][0, 0], own[2][2, -1], prefix[2][0, 1], prefix[2][0, 30] = -1, own[0].shape[0], 2**31 - 1, -2**31
        check(dev, q, own, prefix, hq, n_q)
    q, own, prefix = case(7, 4, 2, 64, 1, 3, 1, [150], 2, [40, 9, 70], 32)
    own[2].fill_(-1)
    prefix[2].fill_(-7)
    assert not check(dev, q, own, prefix, 4, 1).any()


def test_prefix_attn_bounds_cut_lengths(dev):
    q, own, prefix = case(8, 2, 1, 64, 1, 2, 1, [90], 16, [40, 20], 8)
    check(dev, q, own, prefix, 2, 1, max_own=25, max_prefix=33)
    check(dev, q, own, prefix, 2, 1, max_own=0, max_prefix=0)
    long = (*own[:3], torch.tensor([2**31 - 1, 20], dtype=I32))  # cut to the table
    check(dev, q, long, prefix, 2, 1)
    check(dev, q, own, prefix, 2, 1, scale=0.3)


def test_prefix_attn_strided_rows(dev):
    """q and out as column slices of wider rows; the rest of out is left as it was."""
    q, own, prefix = case(9, 14, 2, 64, 1, 3, 2, [50], 16, [5, 2, 9], 4)
    wide = torch.zeros(6, 14 * 64 + 256, dtype=BF16)
    wide[:, :14 * 64] = q
    buf = torch.full((8, 14 * 64 + 64), 5.0, dtype=BF16, device=dev)
    out = PG.prefix_attn(wide.to(dev)[:, :14 * 64], buf[1:7, 64:], own=on(dev, own), prefix=on(dev, prefix), n_heads=14, n_q=2)
    want, _, spread = R.attn(q, own, prefix, 14, 2)
    assert out.data_ptr() == buf[1:, 64:].data_ptr() and R.close_attn(out.cpu(), want, spread).all()
    assert (buf[0] == 5).all() and (buf[7] == 5).all() and (buf[:, :64] == 5).all()


def test_prefix_attn_in_the_queries_place(dev):
    """out = q, in every form: split and joined, direct, whole rows; and out in other columns of q's rows."""
    for hq, hkv, d, width, n_q, plens, olens in ((14, 2, 64, 5, 1, [300], [5] * 5), (14, 2, 64, 3, 1, None, [90, 1, 3]), (8, 2, 64, 26, 30, [70], [31] * 26),
                                                 (32, 8, 128, 20, 1, [200], [7] * 20), (6, 2, 128, 2, 40, None, [40, 60])):
        q, own, prefix = case(19, hq, hkv, d, 1, width, n_q, plens, 16, olens, 8)
        want = PG.prefix_attn(q.to(dev), own=on(dev, own), prefix=on(dev, prefix), n_heads=hq, n_q=n_q)
        buf = torch.zeros(q.shape[0], 2 * hq * d, dtype=BF16, device=dev)
        x = buf[:, :hq * d]
        x.copy_(q)
        got = PG.prefix_attn(x, buf[:, hq * d:], own=on(dev, own), prefix=on(dev, prefix), n_heads=hq, n_q=n_q)
        assert torch.equal(got, want) and torch.equal(x.cpu(), q)
        assert torch.equal(PG.prefix_attn(x, x, own=on(dev, own), prefix=on(dev, prefix), n_heads=hq, n_q=n_q), want)


def test_tensors_elsewhere(dev):
    q, own, prefix = case(20, 2, 1, 64, 1, 1, 1, [9], 4, [3], 4)
    for i in range(4):
        mixed = tuple(x if j == i else to(x, dev) for j, x in enumerate(own))
        with pytest.raises(RuntimeError, match="tensors on"):
            PG.prefix_attn(q.to(dev), own=mixed, n_heads=2)
    k, v = to(own[0], dev), to(own[1], dev)
    with pytest.raises(RuntimeError, match="tensors on"):
        PG.kv_append(torch.zeros(1, 256, dtype=BF16, device=dev), k, v, own[2], torch.zeros(1, dtype=I32, device=dev), n_heads=2)


def test_prefix_attn_offsets_past_32_bits(dev):
    """Pages more than 2^31 elements apart."""
    heads, d, page = 1, 64, 16
    step = 1 << 30
    base = [torch.zeros(3 * step + 2048, dtype=BF16, device=dev) for _ in range(2)]
    k, v = (b.as_strided((4, page, heads, d), (step, d, d, 1)) for b in base)
    g = gen(10)
    small = pools(g, 4, page, heads, d)
    k.copy_(small[0].to(dev))
    v.copy_(small[1].to(dev))
    table, lens = torch.tensor([[3, 0, 2, 1]], dtype=I32), torch.tensor([59], dtype=I32)
    q = noise(g, 1, 2 * d, scale=1.5)
    out = PG.prefix_attn(q.to(dev), own=(k, v, table.to(dev), lens.to(dev)), n_heads=2)
    want, _, spread = R.attn(q, (*small, table, lens), None, 2, 1)
    assert R.close_attn(out.cpu(), want, spread).all()
    qkv = noise(g, 1, 4 * d)
    PG.kv_append(qkv.to(dev), k, v, table.to(dev), torch.tensor([7], dtype=I32, device=dev), n_heads=2)
    assert torch.equal(k[3, 7, 0].cpu(), qkv[0, 2 * d:3 * d]) and torch.equal(v[3, 7, 0].cpu(), qkv[0, 3 * d:])


def test_same_answer_for_equal_rows_and_repeats(dev):
    """No atomics: the same call gives the same bits, and sequences that are alike get the same rows."""
    q, own, prefix = case(11, 14, 2, 64, 1, 4, 1, [900], 64, [50] * 4, 16)
    q = q[:1].expand(4, -1).contiguous()
    own = (own[0], own[1], own[2][:1].expand(4, -1).contiguous(), own[3])
    a, la = run(dev, q, own, prefix, 14, 1)
    b, lb = run(dev, q, own, prefix, 14, 1)
    assert torch.equal(a, b) and torch.equal(la, lb) and all(torch.equal(a[0], a[i]) for i in range(4))


def test_graph_follows_lengths(dev):
    """A captured append and attention replay with other lengths, positions and tables; eager work goes on in between."""
    hq, hkv, d = 14, 2, 64
    q, own, prefix = case(12, hq, hkv, d, 1, 4, 1, [500], 64, [200] * 4, 16)
    do, dp = on(dev, own), on(dev, prefix)
    qkv = noise(gen(13), 4, (hq + 2 * hkv) * d).to(dev)
    cos, sin = K.rope_tables(1024, 1e6, dev)
    dq, out = torch.empty(4, hq * d, dtype=BF16, device=dev), torch.empty(4, hq * d, dtype=BF16, device=dev)
    pos, seq = torch.zeros(4, dtype=I32, device=dev), torch.arange(4, dtype=I32, device=dev)

    def step():
        PG.kv_append(qkv, do[0], do[1], do[2], pos, dq, n_heads=hq, cos=cos, sin=sin, seq=seq)
        PG.prefix_attn(dq, out, own=do, prefix=dp, n_heads=hq)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    g = gen(14)
    for n, pl in ((1, 500), (200, 1), (33, 0), (64, 333)):
        lens = torch.tensor([n, max(1, n - 1), 1, n], dtype=I32)
        do[3].copy_(lens)
        pos.copy_(lens - 1)
        dp[3].fill_(pl)
        do[2].copy_(do[2].cpu()[torch.randperm(4, generator=g)])
        qkv.copy_(noise(g, *qkv.shape))
        step()
        want = out.clone(), dq.clone(), do[0].clone(), do[1].clone()
        out.zero_()
        torch.cuda.synchronize()
        for _ in range(2):
            graph.replay()
            torch.cuda.synchronize()
            for x, y in zip((out, dq, do[0], do[1]), want):
                assert torch.equal(x, y)
            torch.randn(1000, device=dev).sum().item()


def test_other_stream(dev):
    """Two streams at once, each with its own workspace."""
    sets = []
    for seed in (15, 16):
        q, own, prefix = case(seed, 14, 2, 64, 1, 4, 1, [1500], 64, [100] * 4, 16)
        sets.append((q.to(dev), on(dev, own), on(dev, prefix)))
    want = [PG.prefix_attn(q, own=o, prefix=p, n_heads=14) for q, o, p in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [[], []]
    for _ in range(10):
        for i, (q, o, p) in enumerate(sets):
            with torch.cuda.stream(streams[i]):
                got[i].append(PG.prefix_attn(q, own=o, prefix=p, n_heads=14))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want[i]) for i in range(2) for x in got[i])
