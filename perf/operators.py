"""What the paged decode operators (`simlingo_amd.paged`) are measured on: their cases, inputs, plain forms and values in 64 bits.

    kv_append     rotates the queries and keys of new tokens and puts keys and values into a paged cache
    prefix_attn   attention of few new tokens per sequence over a prefix that a group of sequences shares and over their own keys
    beam_select   the best continuations over all beams and the whole vocabulary
    beam_reorder  rows of a state follow the beams that were chosen

Heads, lengths and the vocabulary are the Qwen2 half's (14 query heads on 2 of 64, 151655 tokens, prompts of 798 rows), the tiny configuration's,
and a generic wider model's (32 heads on 8 of 128).
"""
import math

import torch

own = False

QWEN, TINY, WIDE = (14, 2, 64), (2, 1, 64), (32, 8, 128)  # query heads, key/value heads, head size
VOCAB = 151655
THETA = 1e6


# ---- cases ----------------------------------------------------------------------------------------------------------------------------------
def _append(name, heads, n_seq, rows, page, start, spread):
    """`rows` new tokens of each of n_seq sequences, of which the i-th holds start + (i * 7919) % (spread + 1) already."""
    return {"name": name, "op": "append", "hq": heads[0], "hkv": heads[1], "d": heads[2], "n_seq": n_seq, "rows": rows, "page": page,
            "start": start, "spread": spread}


def _attn(name, heads, groups, width, n_q, prefix, prefix_page, own_len, spread, own_page):
    """groups x width sequences with n_q new tokens each; the prefix of group g has prefix - (g * 37) % 64 keys, and the i-th sequence has
    own_len + (i * 7919) % (spread + 1) keys of its own, the new tokens' among them."""
    return {"name": name, "op": "attn", "hq": heads[0], "hkv": heads[1], "d": heads[2], "groups": groups, "width": width, "n_q": n_q,
            "prefix": prefix, "prefix_page": prefix_page, "own_len": own_len, "spread": spread, "own_page": own_page}


def _select(name, batch, width, k, vocab, dtype, done):
    """The k best of width * vocab continuations for each of `batch` inputs; `done` of each input's beams have ended."""
    return {"name": name, "op": "select", "batch": batch, "width": width, "k": k, "vocab": vocab, "dtype": dtype, "done": done}


def _reorder(name, outer, batch, width, used, row, dtype, in_place):
    """State [outer, batch * width, row]; the first `used` of each row move."""
    return {"name": name, "op": "reorder", "outer": outer, "batch": batch, "width": width, "used": used, "row": row, "dtype": dtype,
            "in_place": in_place}


def listed():
    return [
        # one step of four beams on one image: the new token's keys go to single slots
        _append("append-step", QWEN, 4, 1, 1, 40, 0),
        # a prompt of the training length enters the cache
        _append("append-prompt", QWEN, 1, 798, 64, 0, 0),
        # chunks of many sequences of the wide model, at odd positions
        _append("append-chunks", WIDE, 61, 211, 16, 5, 977),
        # the agent's prompt shared by four beams, 40-odd tokens in
        _attn("attn-beam", QWEN, 1, 4, 1, 798, 64, 41, 0, 1),
        # eight images, eight questions about each, answers of different lengths
        _attn("attn-serve", QWEN, 8, 8, 1, 1086, 64, 1, 254, 16),
        # long shared histories
        _attn("attn-long", QWEN, 2, 16, 1, 32771, 128, 300, 700, 64),
        # the wide model over a long document, small pages
        _attn("attn-wide", WIDE, 1, 32, 1, 16411, 16, 5, 1999, 16),
        # the instructions' tokens after the image's, all at once
        _attn("attn-chunk", QWEN, 1, 12, 77, 640, 64, 77, 20, 16),
        # one step of four beams over the whole vocabulary
        _select("select-step", 1, 4, 4, VOCAB, "float32", 0),
        # a served batch: eight inputs of eight beams, twice as many candidates, some beams at their end
        _select("select-serve", 8, 8, 16, VOCAB, "bfloat16", 2),
        # the table of cache slots after a step
        _reorder("reorder-table", 1, 8, 8, 101, 128, "int32", False),
        # a dense cache of 24 layers moved in place, the survivors stay where they are
        _reorder("reorder-cache", 24, 4, 8, 16256, 32768, "bfloat16", True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("append", "attn", "attn", "select", "reorder"))
    most = [work(c) for c in listed() if c["op"] == op]
    while True:
        if op == "append":
            total = _log(rng, 1, 12000)
            n_seq = min(total, _log(rng, 1, 256))
            c = _append("", rng.choice((QWEN, TINY, WIDE)), n_seq, max(1, total // n_seq), 2 ** rng.randint(0, 8), rng.randint(0, 700),
                        rng.randint(0, 900))
        elif op == "attn":
            n_q = rng.choice((1, 1, 1, _log(rng, 2, 100)))
            c = _attn("", rng.choice((QWEN, QWEN, TINY, WIDE)), _log(rng, 1, 8), _log(rng, 1, 32), n_q, _log(rng, 1, 32768), 2 ** rng.randint(0, 8),
                      n_q + _log(rng, 1, 700) - 1, rng.randint(0, 700), 2 ** rng.randint(0, 7))
        elif op == "select":
            width = rng.randint(1, 16)
            c = _select("", _log(rng, 1, 8), width, rng.randint(1, 2 * width), rng.choice((256, _log(rng, 300, VOCAB), VOCAB)),
                        rng.choice(("float32", "bfloat16")), rng.randint(0, width // 2))
        else:
            row = _log(rng, 16, 32768)
            c = _reorder("", _log(rng, 1, 24), _log(rng, 1, 8), rng.randint(2, 16), rng.randint(1, row), row, rng.choice(("int32", "bfloat16")),
                         rng.random() < 0.5)
        del c["name"]
        if all(work(c)[m] <= max(x[m] for x in most) for m in ("bytes", "flops")):
            return c


# ---- inputs ---------------------------------------------------------------------------------------------------------------------------------
def _starts(c):
    return [c["start"] + (i * 7919) % (c["spread"] + 1) for i in range(c["n_seq"])]


def _lengths(c):
    plen = [max(1, c["prefix"] - (g * 37) % 64) for g in range(c["groups"])]
    olen = [c["own_len"] + (i * 7919) % (c["spread"] + 1) for i in range(c["groups"] * c["width"])]
    return plen, olen


def _table(lengths, page, gen):
    """Page numbers in a random order: [sequences, the longest's pages] and how many pages there are."""
    cols = max(-(-n // page) for n in lengths)
    n = len(lengths) * cols
    return torch.randperm(n, generator=gen, device=gen.device).to(torch.int32).view(len(lengths), cols), n


def _rotation(rows, d, dev):
    angle = torch.outer(torch.arange(rows, dtype=torch.float64), THETA ** (-torch.arange(0, d, 2, dtype=torch.float64) / d))
    return angle.cos().float().to(dev), angle.sin().float().to(dev)


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    c = case

    def noise(*shape, dtype=torch.bfloat16, scale=1.0):
        return (torch.randn(*shape, generator=gen, device=dev) * scale).to(dtype)

    def ints(values):
        return torch.tensor(values, dtype=torch.int32, device=dev)

    s = {"case": c}
    if c["op"] == "append":
        starts, rows, d = _starts(c), c["rows"], c["d"]
        s["table"], n_pages = _table([n + rows for n in starts], c["page"], gen)
        s["seq"] = ints([i for i in range(c["n_seq"]) for _ in range(rows)])
        s["pos"] = ints([n + t for n in starts for t in range(rows)])
        s["cos"], s["sin"] = _rotation(max(starts) + rows, d, dev)
        s["qkv"] = noise(c["n_seq"] * rows, (c["hq"] + 2 * c["hkv"]) * d)
        s["q"] = torch.empty(c["n_seq"] * rows, c["hq"] * d, dtype=torch.bfloat16, device=dev)
        s["k"], s["v"] = noise(n_pages, c["page"], c["hkv"], d), noise(n_pages, c["page"], c["hkv"], d)
    elif c["op"] == "attn":
        plen, olen = _lengths(c)
        s["ptab"], n_prefix = _table(plen, c["prefix_page"], gen)
        s["otab"], n_own = _table(olen, c["own_page"], gen)
        s["plen"], s["olen"] = ints(plen), ints(olen)
        s["pk"], s["pv"] = (noise(n_prefix, c["prefix_page"], c["hkv"], c["d"]) for _ in range(2))
        s["ok"], s["ov"] = (noise(n_own, c["own_page"], c["hkv"], c["d"]) for _ in range(2))
        s["q"] = noise(len(olen) * c["n_q"], c["hq"] * c["d"], scale=1.5)
        s["out"] = torch.empty_like(s["q"])
    elif c["op"] == "select":
        n = c["batch"] * c["width"]
        s["logits"] = noise(n, c["vocab"], dtype=getattr(torch, c["dtype"]), scale=3.0)
        s["scores"] = noise(n, dtype=torch.float32).abs().mul_(-4.0)
        s["finished"] = (torch.arange(n, device=dev) % c["width"]) >= c["width"] - c["done"]
    else:
        n, w = c["batch"] * c["width"], c["width"]
        if c["dtype"] == "int32":
            s["x"] = torch.randint(0, 1 << 30, (c["outer"], n, c["row"]), generator=gen, device=dev, dtype=torch.int32)
        else:
            s["x"] = noise(c["outer"], n, c["row"])
        parent = torch.randint(0, w, (c["batch"], w), generator=gen, device=dev)
        if c["in_place"]:  # who is chosen stays, the others take a survivor's state: a second pass on the same state changes nothing
            stays = torch.randint(0, 2, (c["batch"], w), generator=gen, device=dev).bool()
            stays[:, 0] = True
            at = torch.where(stays, torch.arange(w, device=dev), torch.zeros_like(parent))
            parent = torch.where(stays, at, torch.gather(at, 1, parent))
        s["parent"] = parent.to(torch.int32)
        s["to"] = s["x"] if c["in_place"] else s["x"].clone()
    return s


# ---- one pass -------------------------------------------------------------------------------------------------------------------------------
def run(state):
    s, c = state, state["case"]
    if own:
        from simlingo_amd import paged
        if c["op"] == "append":
            paged.kv_append(s["qkv"], s["k"], s["v"], s["table"], s["pos"], s["q"], n_heads=c["hq"], cos=s["cos"], sin=s["sin"], seq=s["seq"])
            return s["q"], s["k"], s["v"]
        if c["op"] == "attn":
            return paged.prefix_attn(s["q"], s["out"], own=(s["ok"], s["ov"], s["otab"], s["olen"]),
                                     prefix=(s["pk"], s["pv"], s["ptab"], s["plen"]), n_heads=c["hq"], n_q=c["n_q"])
        if c["op"] == "select":
            return paged.beam_select(s["logits"], s["scores"], width=c["width"], k=c["k"], finished=s["finished"], pad_id=0)
        return paged.beam_reorder(s["x"][..., :c["used"]], s["parent"], dim=1, out=s["to"][..., :c["used"]])
    return {"append": _plain_append, "attn": _plain_attn, "select": _plain_select, "reorder": _plain_reorder}[c["op"]](s, c)


def _plain_append(s, c):
    hq, hkv, d = c["hq"], c["hkv"], c["d"]
    x = s["qkv"].float().view(-1, hq + 2 * hkv, d)
    pos, seq = s["pos"].long(), s["seq"].long()
    cos, sin = s["cos"][pos][:, None], s["sin"][pos][:, None]
    a, b = x[:, :hq + hkv].split(d // 2, dim=2)
    turned = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=2)
    s["q"].copy_(turned[:, :hq].reshape(len(pos), hq * d))
    at = s["table"][seq, pos // c["page"]].long(), pos % c["page"]
    s["k"][at] = turned[:, hq:].to(torch.bfloat16)
    s["v"][at] = x[:, hq + hkv:].to(torch.bfloat16)
    return s["q"], s["k"], s["v"]


def _plain_attn(s, c):
    g, w, t, hkv, d = c["groups"], c["width"], c["n_q"], c["hkv"], c["d"]
    r = c["hq"] // hkv
    q = s["q"].float().view(g, w, t, hkv, r, d) / math.sqrt(d)

    def rows(pages, table):  # [sequences, heads, keys, d]
        return pages[table.long()].float().flatten(1, 2).transpose(1, 2).contiguous()

    pk, pv, ok, ov = rows(s["pk"], s["ptab"]), rows(s["pv"], s["ptab"]), rows(s["ok"], s["otab"]), rows(s["ov"], s["otab"])
    sp = torch.matmul(q.permute(0, 3, 1, 2, 4, 5).reshape(g, hkv, w * t * r, d), pk.transpose(2, 3).contiguous())
    so = torch.matmul(q.flatten(0, 1).transpose(1, 2).reshape(g * w, hkv, t * r, d), ok.transpose(2, 3).contiguous())
    sp = sp.masked_fill(torch.arange(pk.shape[2], device=q.device) >= s["plen"].view(g, 1, 1, 1), -math.inf)
    last = s["olen"].view(-1, 1) - t + torch.arange(t, device=q.device)
    hidden = torch.arange(ok.shape[2], device=q.device) > last.view(g * w, 1, t, 1, 1)
    so = so.view(g * w, hkv, t, r, -1).masked_fill(hidden, -math.inf)
    sp = sp.view(g, hkv, w, t, r, -1).transpose(1, 2).reshape(g * w, hkv, t, r, -1)
    top = torch.maximum(sp.amax(-1, keepdim=True), so.amax(-1, keepdim=True))
    ep, eo = torch.exp(sp - top), torch.exp(so - top)
    total = ep.sum(-1, keepdim=True) + eo.sum(-1, keepdim=True)
    op = torch.matmul(ep.view(g, w, hkv, t * r, -1).transpose(1, 2).reshape(g, hkv, w * t * r, -1), pv)
    op = op.view(g, hkv, w, t, r, d).transpose(1, 2).reshape(g * w, hkv, t, r, d)
    oo = torch.matmul(eo.view(g * w, hkv, t * r, -1), ov).view(g * w, hkv, t, r, d)
    out = (op + oo) / total
    return s["out"].copy_(out.transpose(1, 2).reshape(g * w * t, c["hq"] * d))


def _plain_select(s, c):
    n, v, w, k = c["batch"] * c["width"], c["vocab"], c["width"], c["k"]
    x = s["logits"].double()  # in 64 bits: the order of candidates whose scores are close
    top = x.amax(1, keepdim=True)
    score = s["scores"].double().view(n, 1) + (x - top - torch.log(torch.exp(x - top).sum(1, keepdim=True)))
    held = torch.full_like(score, -math.inf)
    held[:, 0] = s["scores"].double()
    score = torch.where(s["finished"].view(n, 1), held, score)
    best, at = torch.sort(score.view(c["batch"], w * v), dim=1, descending=True, stable=True)
    at = at[:, :k]
    return best[:, :k].float(), (at // v).to(torch.int32), (at % v).to(torch.int32)


def _plain_reorder(s, c):
    n, w, used = c["batch"] * c["width"], c["width"], c["used"]
    row = s["parent"].long().view(-1) + torch.arange(n, device=s["parent"].device) // w * w
    s["to"][..., :used] = s["x"][:, row, :used]
    return s["to"][..., :used]


# ---- the work, and the values in 64 bits ------------------------------------------------------------------------------------------------------
def work(case):
    c = case
    if c["op"] == "append":
        t = c["n_seq"] * c["rows"]
        return {"bytes": t * ((c["hq"] + 2 * c["hkv"]) * c["d"] * 4 + 12) + min(t, max(_starts(c)) + c["rows"]) * c["d"] * 4,
                "flops": 3 * t * (c["hq"] + c["hkv"]) * c["d"]}
    if c["op"] == "attn":
        plen, olen = _lengths(c)
        kv, n = c["hkv"] * c["d"] * 4, len(olen) * c["n_q"]
        pairs = sum(plen) * c["width"] * c["n_q"] + sum(c["n_q"] * m - c["n_q"] * (c["n_q"] - 1) // 2 for m in olen)
        return {"bytes": (sum(plen) + sum(olen)) * kv + 2 * n * c["hq"] * c["d"] * 2, "flops": 4 * pairs * c["hq"] * c["d"]}
    if c["op"] == "select":
        n = c["batch"] * (c["width"] - c["done"]) * c["vocab"]
        return {"bytes": n * (4 if c["dtype"] == "float32" else 2) + c["batch"] * (c["width"] * 5 + c["k"] * 12), "flops": 3 * n}
    return {"bytes": 2 * c["outer"] * c["batch"] * c["width"] * c["used"] * (4 if c["dtype"] == "int32" else 2), "flops": 0}


def exact(case, seed):
    """From the definitions, one sequence at a time."""
    s, c = prepare(case, seed), case
    if c["op"] == "append":
        hq, hkv, d = c["hq"], c["hkv"], c["d"]
        angle = s["pos"].double()[:, None] * torch.exp(-math.log(THETA) * torch.arange(d // 2, device="cuda", dtype=torch.float64) * 2 / d)
        turn = torch.polar(torch.ones_like(angle), angle)[:, None]
        x = s["qkv"].double().view(len(angle), hq + 2 * hkv, 2, d // 2)
        z = torch.complex(x[:, :hq + hkv, 0], x[:, :hq + hkv, 1]) * turn
        z = torch.cat([z.real, z.imag], 2)
        k, v = s["k"].double(), s["v"].double()
        for i, n in enumerate(_starts(c)):
            t0 = i * c["rows"]
            p = torch.arange(n, n + c["rows"], device="cuda")
            slot = s["table"][i].long()[p // c["page"]] * c["page"] + p % c["page"]
            k.view(-1, hkv, d)[slot] = z[t0:t0 + c["rows"], hq:]
            v.view(-1, hkv, d)[slot] = x[t0:t0 + c["rows"], hq + hkv:].reshape(-1, hkv, d)
        return z[:, :hq].reshape(len(angle), hq * d), k, v
    if c["op"] == "attn":
        plen, olen = _lengths(c)
        r, t, d = c["hq"] // c["hkv"], c["n_q"], c["d"]
        if len(olen) * c["hkv"] > 4000:
            return None
        out = torch.empty(len(olen), t, c["hq"], d, dtype=torch.float64, device="cuda")
        q = s["q"].double().view(len(olen), t, c["hq"], d)
        for i, m in enumerate(olen):
            g = i // c["width"]

            def keys(pages, table, n):
                return pages[table.long()].flatten(0, 1)[:n].double()

            kk = torch.cat([keys(s["pk"], s["ptab"][g], plen[g]), keys(s["ok"], s["otab"][i], m)])
            vv = torch.cat([keys(s["pv"], s["ptab"][g], plen[g]), keys(s["ov"], s["otab"][i], m)])
            seen = torch.arange(plen[g] + m, device="cuda") <= plen[g] + m - t + torch.arange(t, device="cuda")[:, None]
            for h in range(c["hkv"]):
                part = slice(h * r, (h + 1) * r)
                a = q[i, :, part].reshape(t * r, d) @ kk[:, h].t().contiguous() * d ** -0.5
                a = a.masked_fill(~seen.repeat_interleave(r, 0), -math.inf)
                out[i, :, part] = (torch.softmax(a, -1) @ vv[:, h].contiguous()).view(t, r, d)
        return out.view(len(olen) * t, c["hq"] * d)
    if c["op"] == "select":
        b, w, v = c["batch"], c["width"], c["vocab"]
        score = s["scores"].double().view(-1, 1) + torch.log_softmax(s["logits"].double(), 1)
        for i in range(b * w):
            if bool(s["finished"][i]):
                score[i] = -math.inf
                score[i, 0] = s["scores"][i].double()
        best, parent, token = [], [], []
        for rows in score.view(b, w * v):
            bar = torch.topk(rows, c["k"]).values[-1]
            at = torch.nonzero(rows >= bar).view(-1).tolist()
            found = sorted(zip(rows[at].tolist(), at), key=lambda e: (-e[0], e[1]))[:c["k"]]
            best.append([e[0] for e in found])
            parent.append([e[1] // v for e in found])
            token.append([e[1] % v for e in found])
        whole = dict(dtype=torch.int32, device="cuda")
        return torch.tensor(best, dtype=torch.float64, device="cuda"), torch.tensor(parent, **whole), torch.tensor(token, **whole)
    w, used = c["width"], c["used"]
    to = s["to"][..., :used].clone()
    for i, p in enumerate(s["parent"].view(-1).tolist()):
        to[:, i] = s["x"][:, i // w * w + p, :used]
    return to.double() if c["dtype"] != "int32" else to
