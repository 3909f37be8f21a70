"""prefix_attn (simlingo_amd/paged.py) keeps probabilities, sums and partial outputs to 32 bits' worth until the output is rounded.

What a row's output may be off by, with S the largest sum_i |q_i k_i| * scale of its keys and n their number:
  its own rounding                                          2^-8 |out|
  a score in units of e: d roundings of the dot product's sums, 8 of the scale, the difference from the maximum (up to 2 S) and the
  parts' maxima, 2^-24 S each                               e_s = (d + 8) 2^-24 S
  a probability: e_s, exp2 (2 units, 2^-22), its two bf16 terms (2^-15)     e_p = e_s + 2^-22 + 2^-15
  which moves the output by at most 2 e_p sum p |v - out|   (numerator and sum both)
  sums of n products and up to 256 joined parts             (n + 256) 2^-24 sum p |v|, of which sum p |v| <= |out| + sum p |v - out|
A probability rounded to bf16 once is off by up to 2^-8: some output near 0 shows it in every call.

The log of the sum: e_p, the sum's n + 256 roundings, and 4 roundings of numbers of at most 2 S + log n + 1."""
import math

import pytest
import torch

import paged_ref as R
from test_paged_gpu import ATTN, case, on
from simlingo_amd import paged as PG

pytestmark = pytest.mark.gpu

MORE = [  # many ranges, whole rows of 64 and 128, wide tiles
    (2, 1, 64, 1, 2, 1, [2100], 64, [700, 40], 16, "slots"),
    (14, 2, 64, 1, 9, 20, [130], 16, [20 + 7 * i for i in range(9)], 8, "slots"),
    (32, 32, 64, 1, 12, 33, [77], 16, [33 + i for i in range(12)], 8, "slots"),
    (32, 32, 128, 1, 9, 40, [77], 16, [40 + i for i in range(9)], 8, "slots"),
    (14, 2, 64, 1, 16, 1, [1500], 128, [5] * 16, 16, "slots"),
    (32, 8, 128, 1, 20, 1, [900], 16, [3] * 20, 16, "slots"),
    (32, 8, 128, 1, 3, 1, [500], 16, [3, 40, 9], 16, "slots"),       # 12, 16 and 20 rows of a prefix
    (32, 8, 128, 2, 4, 1, [500, 77], 16, [3] * 8, 8, "heads"),
    (32, 8, 128, 1, 5, 1, [500], 16, [3] * 5, 16, "pair"),
]


def magnitudes(q, own, prefix, hq, n_q):
    """-> (S [rows, heads], the most keys a row has)."""
    ok, _, otab, olen = own
    hkv, d = ok.shape[2:]
    n_seq, most = otab.shape[0], 0
    qq = q.double().abs().view(n_seq, n_q, hq, d)
    S = torch.zeros(n_seq, n_q, hq, dtype=torch.float64)
    for i in range(n_seq):
        k = R.keys_of(ok, otab[i], int(olen[i]))[0]
        if prefix is not None:
            g = i // (n_seq // prefix[2].shape[0])
            k = torch.cat([R.keys_of(prefix[0], prefix[2][g], int(prefix[3][g]))[0], k])
        most = max(most, len(k))
        for h in range(hq):
            S[i, :, h] = (qq[i, :, h] @ k[:, h // (hq // hkv)].abs().t()).amax(1) / math.sqrt(d)
    return S.view(-1, hq), most


@pytest.mark.parametrize("c", ATTN + MORE, ids=lambda c: "h%d-%d-d%d-g%dx%d-q%d-p%s-o%s" % (c[0], c[1], c[2], c[3], c[4], c[5], c[7], c[9]))
def test_off_by_its_rounding(dev, c):
    hq, hkv, d, groups, width, n_q, plens, ppage, olens, opage, layout = c
    q, own, prefix = case(sum(olens) + hq + 1, hq, hkv, d, groups, width, n_q, plens, ppage, olens, opage, layout)
    lse = torch.full((q.shape[0], hq), 3.0, device=dev)
    out = PG.prefix_attn(q.to(dev), own=on(dev, own), prefix=on(dev, prefix), n_heads=hq, n_q=n_q, lse=lse).cpu().double()
    lse = lse.cpu().double()
    want, wl, spread = R.attn(q, own, prefix, hq, n_q)
    S, n = magnitudes(q, own, prefix, hq, n_q)
    e_p = (d + 8) * 2.0 ** -24 * S + 2.0 ** -22 + 2.0 ** -15  # [rows, heads]
    wide = lambda x: x.repeat_interleave(d, 1)  # noqa: E731
    tol = 2.0 ** -8 * want.abs() + 2 * wide(e_p) * spread + (n + 256) * 2.0 ** -24 * (want.abs() + spread) + 1e-30
    assert ((out - want).abs() <= tol).all(), ((out - want).abs() / tol).max()
    seen = torch.isfinite(wl)
    near = (lse - wl).abs() <= e_p + (n + 256) * 2.0 ** -24 + 4 * 2.0 ** -24 * (2 * S + math.log(n + 1) + 1)
    assert near[seen].all(), (lse - wl)[seen].abs().max()
