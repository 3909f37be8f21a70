"""BeamDecoder: kv_append, prefix_attn, beam_select and beam_reorder together, through the language half, against the CPU
oracle's logits (oracle/vla_oracle.py) and a plain beam search over them.

The HIP path runs bf16 weights with LoRA merged, the oracle f32: a token's log probability differs by bf16 rounding. Gate per
token: 6e-2 x std(logits), twice the greedy test's gate on one logit (a log probability is a difference of two)."""
import pytest
import torch

from golden_util import load_case
from oracle import vla_oracle as O

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def setup(dev):
    from simlingo_amd.engine import VLAEngine
    cfg, P, ex, _ = load_case("leftpad")
    return cfg, P, ex, VLAEngine(cfg, dev, P)


def prompts(cfg, P, ex, eng):
    from simlingo_amd.plan import plan_from_example
    plan = plan_from_example(cfg, ex, inference=True)
    X = eng.encode_inputs(ex.driving_input.camera_images.to(eng.device), plan, plan.to_device(eng.device), {})
    pix = ex.driving_input.camera_images
    vit = O.extract_feature(P, cfg, pix.reshape(-1, *pix.shape[3:]))
    lang, valid = O.language_inputs(P, cfg, ex, vit, inference=True)
    out = []
    for b in range(plan.B):
        n = int(plan.seqlens[b]) - cfg.n_queries
        out.append((X[b * plan.S:b * plan.S + n], lang[b][valid[b]]))
    return out


def oracle_logprobs(P, cfg, emb, rows):
    """log probabilities [n, V] at each of the tokens of several rows of ids, teacher forced, one row at a time."""
    out, spread = [], 0.0
    for ids in rows:
        x = torch.cat([emb, P["llm.embed"][torch.tensor(ids, dtype=torch.long)]], 0)
        _, logits = O.llm_forward(P, cfg, x[None], torch.ones(1, x.shape[0], dtype=torch.bool))
        lg = logits[0, emb.shape[0] - 1:emb.shape[0] - 1 + max(1, len(ids))]
        spread = max(spread, float(lg.std()))
        out.append(torch.log_softmax(lg.double(), -1))
    return out, spread


def test_scores_are_the_oracles(setup):
    """Every beam's score is the sum of its own tokens' log probabilities: keys, tables and tokens moved together."""
    from simlingo_amd.decode import BeamDecoder
    cfg, P, ex, eng = setup
    n = 10
    for W in (1, 2, 5, 16):
        dec = BeamDecoder(eng, num_beams=W, max_len=512, max_new_tokens=n, eos_id=-1)
        for prefix, emb in prompts(cfg, P, ex, eng):
            ids, scores = dec.search(prefix)
            assert ids.shape == (W, n) and len({tuple(r) for r in ids.tolist()}) == W
            assert (scores[:-1] >= scores[1:]).all()
            lp, spread = oracle_logprobs(P, cfg, emb, ids.tolist())
            for w in range(W):
                want = lp[w].gather(1, ids[w][:, None]).sum().item()
                assert abs(want - scores[w].item()) <= 6e-2 * spread * n, (W, w, want, scores[w].item())


def test_every_step_takes_the_best(setup):
    """Each step's beams are extensions of the step before, and by the oracle's scores none is worse than the num_beams-th best
    extension by more than both scores' rounding. (The end result of a beam search is no continuous function of the logits: a
    beam that rounding drops may have led to the best one. So it is held to the oracle step by step, from its own beams.)"""
    from simlingo_amd.decode import BeamDecoder
    cfg, P, ex, eng = setup
    n, W = 6, 3
    dec = BeamDecoder(eng, num_beams=W, max_len=512, max_new_tokens=n, eos_id=-1)
    for prefix, emb in prompts(cfg, P, ex, eng):
        beams = [()]
        for i in range(n):
            ids, scores = dec.search(prefix, i + 1)
            lp, spread = oracle_logprobs(P, cfg, emb, [list(b) + [0] for b in beams])
            cand = {}
            for j, b in enumerate(beams):
                so_far = float(sum(lp[j][t, tok] for t, tok in enumerate(b)))
                cand.update({b + (t,): so_far + float(lp[j][i, t]) for t in range(cfg.vocab)})
            order = sorted(cand.values(), reverse=True)
            tol = 6e-2 * spread * (i + 1)
            beams = [tuple(r) for r in ids.tolist()]
            for w, b in enumerate(beams):
                assert b in cand and cand[b] >= order[W - 1] - 2 * tol, (i, w, b)
                assert abs(cand[b] - scores[w].item()) <= tol


def test_one_beam_is_the_greedy_loop(setup):
    """One beam picks what GreedyDecoder picks, wherever the oracle's two best logits are apart (0.2 x std: the greedy test's)."""
    from simlingo_amd.decode import BeamDecoder, GreedyDecoder
    cfg, P, ex, eng = setup
    kw = dict(max_len=512, max_new_tokens=12, eos_id=-1)
    beam, greedy = BeamDecoder(eng, num_beams=1, **kw), GreedyDecoder(eng, **kw)
    for prefix, emb in prompts(cfg, P, ex, eng):
        a, b = beam.generate(prefix), greedy.generate(prefix)
        same = a == b
        if not same.all():
            i = int((~same).nonzero()[0])
            lp, spread = oracle_logprobs(P, cfg, emb, [b[:i + 1].tolist()])
            top = lp[0][i].topk(2).values
            assert float(top[0] - top[1]) <= 0.2 * spread, (i, a, b)


def test_ends_and_drives(setup):
    """An ended beam stays as it is, fills up with the end token and keeps its score; the decoder goes where GreedyDecoder goes."""
    from simlingo_amd.decode import BeamDecoder, infer_example
    cfg, P, ex, eng = setup
    prefix, emb = prompts(cfg, P, ex, eng)[0]
    free = BeamDecoder(eng, num_beams=4, max_len=512, max_new_tokens=8, eos_id=-1)
    ids, _ = free.search(prefix)
    eos = int(ids[1, 2])
    dec = BeamDecoder(eng, num_beams=4, max_len=512, max_new_tokens=8, eos_id=eos, check_every=2)
    got, scores = dec.search(prefix)
    ended = 0
    lp, spread = oracle_logprobs(P, cfg, emb, got.tolist())
    for w in range(4):
        at = (got[w] == eos).nonzero().view(-1)
        stop = int(at[0]) + 1 if at.numel() else 8
        assert (got[w, stop:] == eos).all()
        ended += at.numel() > 0
        want = lp[w].gather(1, got[w][:, None])[:stop].sum().item()
        assert abs(want - scores[w].item()) <= 6e-2 * spread * 8
    assert ended
    best = dec.generate(prefix)
    assert best.tolist() == got[0, : best.numel()].tolist() and (best.numel() == 8 or best[-1] == eos)
    sp, rp, toks = infer_example(eng, dec, ex)
    assert torch.isfinite(sp).all() and torch.isfinite(rp).all() and toks[0] == best.tolist()
    assert dec.search(prefix, 0)[0].shape == (4, 0) and dec.search(prefix, 1)[0].shape == (4, 1)
    with pytest.raises(ValueError, match="exceeds the cache"):
        BeamDecoder(eng, num_beams=2, max_len=prefix.shape[0] + 7, max_new_tokens=8).search(prefix)
    with pytest.raises(ValueError, match="num_beams"):
        BeamDecoder(eng, num_beams=0)
