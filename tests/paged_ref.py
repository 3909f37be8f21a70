"""Plain 64-bit forms of the paged decode operators (simlingo_amd/paged.py), on the CPU."""
import math

import torch

NEG = -math.inf


def rotate(x, cos, sin):
    """rotate_half RoPE of [rows, heads, d] by per-row tables [rows, d / 2]."""
    a, b = x.chunk(2, dim=-1)
    c, s = cos[:, None], sin[:, None]
    return torch.cat([a * c - b * s, b * c + a * s], -1)


def append(qkv, k, v, table, pos, seq, n_heads, cos, sin):
    """-> (rotated q [rows, heads * d] f64, k, v pools f64 after, mask of the rows written)."""
    n_pages, page, hkv, d = k.shape
    x = qkv.double().view(qkv.shape[0], n_heads + 2 * hkv, d)
    ko, vo, q = k.double().clone(), v.double().clone(), torch.zeros(qkv.shape[0], n_heads * d, dtype=torch.float64)
    done = torch.zeros(qkv.shape[0], dtype=torch.bool)
    for i in range(qkv.shape[0]):
        p, s = int(pos[i]), int(seq[i])
        if p < 0 or p // page >= table.shape[1] or not 0 <= s < table.shape[0] or (cos is not None and p >= cos.shape[0]):
            continue
        pg = int(table[s, p // page])
        if not 0 <= pg < n_pages:
            continue
        done[i] = True
        y = x[i:i + 1, :n_heads + hkv]
        if cos is not None:
            y = rotate(y, cos[p:p + 1].double(), sin[p:p + 1].double())
        q[i] = y[0, :n_heads].reshape(-1)
        ko[pg, p % page] = y[0, n_heads:]
        vo[pg, p % page] = x[i, n_heads + hkv:]
    return q, ko, vo, done


def keys_of(k, table, n):
    """(rows [n, heads, d] f64, mask of those on a page that exists) of one sequence."""
    n_pages, page = k.shape[:2]
    out = torch.zeros(n, *k.shape[2:], dtype=torch.float64)
    ok = torch.zeros(n, dtype=torch.bool)
    for j in range(n):
        pg = int(table[j // page])
        if 0 <= pg < n_pages:
            ok[j] = True
            out[j] = k[pg, j % page].double()
    return out, ok


def attn(q, own, prefix, n_heads, n_q, scale=None, max_own=None, max_prefix=None):
    """-> (out [rows, heads * d], lse [rows, heads], spread [rows, heads * d] = sum p |v - out|), all f64."""
    ok, ov, otab, olen = own
    hkv, d = ok.shape[2:]
    n, r = otab.shape[0], n_heads // hkv
    groups = n if prefix is None else prefix[2].shape[0]
    scale = d ** -0.5 if scale is None else scale
    out = torch.zeros(n, n_q, n_heads, d, dtype=torch.float64)
    spread, lse = torch.zeros_like(out), torch.full((n, n_q, n_heads), NEG, dtype=torch.float64)
    qq = q.double()[:, :n_heads * d].reshape(n, n_q, n_heads, d)

    def cut(length, bound, cols, page):
        most = cols * page if bound is None else min(bound, cols * page)
        return max(0, min(int(length), most))

    for i in range(n):
        m = cut(olen[i], max_own, otab.shape[1], ok.shape[1])
        kk, good = keys_of(ok, otab[i], m)
        vv, _ = keys_of(ov, otab[i], m)
        pl = 0
        if prefix is not None:
            g = i // (n // groups)
            pl = cut(prefix[3][g], max_prefix, prefix[2].shape[1], prefix[0].shape[1])
            pk, pgood = keys_of(prefix[0], prefix[2][g], pl)
            pv, _ = keys_of(prefix[1], prefix[2][g], pl)
            kk, vv, good = torch.cat([pk, kk]), torch.cat([pv, vv]), torch.cat([pgood, good])
        for t in range(n_q):
            seen = (torch.arange(pl + m) <= pl + m - n_q + t) & good
            seen |= (torch.arange(pl + m) < pl) & good
            if not seen.any():
                continue
            for h in range(n_heads):
                s = kk[seen][:, h // r] @ qq[i, t, h] * scale
                p = torch.softmax(s, 0)
                x = vv[seen][:, h // r]
                o = (p[:, None] * x).sum(0)
                out[i, t, h], lse[i, t, h] = o, torch.logsumexp(s, 0)
                spread[i, t, h] = (p[:, None] * (x - o).abs()).sum(0)
    return out.view(n * n_q, -1), lse.view(n * n_q, -1), spread.view(n * n_q, -1)


def close_attn(got, want, spread):
    """The kernel rounds each probability to bf16 (relative error at most 2^-8, and the sum is of the rounded ones): the
    output moves by at most 2^-8 sum p |v - out|; it is itself rounded to bf16 (2^-8 |out|). 5 % more covers the scores' own
    f32 error (below 2^-24 * 128 * 25 = 2e-4 of a probability) and second-order terms; 1e-6 the f32 sums of values of order 1."""
    return (got.double() - want).abs() <= 2.0 ** -8 * 1.05 * (spread + want.abs()) + 1e-6


def select(logits, scores, width, k, finished=None, pad=0):
    """-> (scores f64, parent, token) by the definition: a stable sort of all width * V scores."""
    n, v = logits.shape
    scores = torch.where(torch.isfinite(scores), scores, torch.full_like(scores, NEG))
    score = scores.double().view(n, 1) + torch.log_softmax(logits.double(), 1)
    if finished is not None:
        for i in range(n):
            if finished[i]:
                score[i] = NEG
                score[i, pad] = scores[i].double()
    score = torch.where(torch.isnan(score), torch.full_like(score, NEG), score) + 0.0
    best, at = torch.sort(score.view(n // width, width * v), dim=1, descending=True, stable=True)
    return best[:, :k], at[:, :k] // v, at[:, :k] % v


# log of the row sum: exp(x - max) of |x - max| <= 24 where it counts carries (24 + 2) 2^-24, the sum of a chunk's up to 8192
# terms in 32 (a thread's own) + 6 (its wave) + 4 (the waves) additions 42 * 2^-24; then one rounding of the score to f32
LSE_TOL = 68 * 2.0 ** -24


def check_select(got, want, exact_order=False):
    gs, gp, gt = (x.cpu() for x in got)
    ws, wp, wt = want
    fin = torch.isfinite(ws)
    assert torch.equal(fin, torch.isfinite(gs)), (gs, ws)
    tol = LSE_TOL + 2.0 ** -24 * ws[fin].abs()
    assert ((gs.double()[fin] - ws[fin]).abs() <= tol).all(), (gs.double()[fin] - ws[fin]).abs().max()
    # where two candidates are closer than both errors, either order is right
    gap = (ws[:, 1:] - ws[:, :-1]).abs()
    near = torch.zeros_like(fin)
    if not exact_order:
        close = fin[:, 1:] & (gap <= 2 * LSE_TOL) & (gap > 0)
        near[:, 1:] |= close
        near[:, :-1] |= close
    assert torch.equal(gp.long()[~near], wp[~near]) and torch.equal(gt.long()[~near], wt[~near]), (gp, wp, gt, wt)
