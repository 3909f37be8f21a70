"""Decoding many sequences over a paged key/value cache: the operators behind `decode.BeamDecoder`, for any caller.

The agent's greedy loop (simlingo_training/models/language_model/llm.py:178-250) runs one sequence; the questions and
instructions about one frame and the beams of one answer share the image prompt, whose keys these operators read once:

  kv_append     rotates new tokens' queries and keys and puts keys and values into their pages
  prefix_attn   attention of new tokens over a prefix shared by a group of sequences and over their own keys
  beam_select   the k best continuations over all beams and the whole vocabulary
  beam_reorder  the rows of a state follow the beams chosen

A cache is a pair of bf16 tensors k, v [pages, page, kv heads, head size], any strides with the last dimension
contiguous (page a power of two, head size 64 or 128); a table [sequences, columns] int32 names the pages of each
sequence in order. Everything runs on the current stream of the current device and can be captured in a graph; lengths,
positions and tables are read on the device, so a captured call follows their contents.
"""
from __future__ import annotations

import ctypes
import math

import torch

from . import kernels as K

BF16, F32, I32 = torch.bfloat16, torch.float32, torch.int32


class KVPoolDesc(ctypes.Structure):  # slx_kv_pool
    _fields_ = [("k", K.c_vp), ("v", K.c_vp), ("page_stride", K.c_i64), ("slot_stride", K.c_i64), ("head_stride", K.c_i64),
                ("n_pages", K.c_int), ("page", K.c_int), ("heads", K.c_int), ("head_dim", K.c_int)]


class KVAppendDesc(ctypes.Structure):  # slx_kv_append_desc
    _fields_ = [("pool", KVPoolDesc), ("qkv", K.c_vp), ("ldqkv", K.c_i64), ("q_out", K.c_vp), ("ldq", K.c_i64),
                ("table", K.c_vp), ("ldt", K.c_i64), ("n_seq", K.c_int), ("cols", K.c_int), ("seq", K.c_vp), ("pos", K.c_vp),
                ("rows_per_seq", K.c_int), ("Hq", K.c_int), ("rows", K.c_i64), ("cos_tab", K.c_vp), ("sin_tab", K.c_vp),
                ("rope_rows", K.c_int)]


class PrefixAttnDesc(ctypes.Structure):  # slx_prefix_attn_desc
    _fields_ = [("prefix_pool", KVPoolDesc), ("own_pool", KVPoolDesc), ("q", K.c_vp), ("ldq", K.c_i64), ("out", K.c_vp),
                ("ldo", K.c_i64), ("lse", K.c_vp), ("ptab", K.c_vp), ("ldpt", K.c_i64), ("plen", K.c_vp), ("otab", K.c_vp),
                ("ldot", K.c_i64), ("olen", K.c_vp), ("max_prefix", K.c_int), ("max_own", K.c_int), ("pcols", K.c_int),
                ("ocols", K.c_int), ("groups", K.c_int), ("width", K.c_int), ("n_q", K.c_int), ("Hq", K.c_int),
                ("scale", K.c_float), ("ws", K.c_vp), ("ws_floats", K.c_i64)]


class BeamSelectDesc(ctypes.Structure):  # slx_beam_select_desc
    _fields_ = [("logits", K.c_vp), ("ldx", K.c_i64), ("logits_bf16", K.c_int), ("batch", K.c_int), ("width", K.c_int),
                ("vocab", K.c_int), ("k", K.c_int), ("score", K.c_vp), ("finished", K.c_vp), ("pad", K.c_int),
                ("score_out", K.c_vp), ("parent", K.c_vp), ("token", K.c_vp), ("finished_out", K.c_vp), ("eos", K.c_int),
                ("ws", K.c_vp), ("ws_bytes", K.c_i64)]


class BeamReorderDesc(ctypes.Structure):  # slx_beam_reorder_desc
    _fields_ = [("src", K.c_vp), ("dst", K.c_vp), ("s0", K.c_i64), ("s1", K.c_i64), ("src_row", K.c_i64), ("d0", K.c_i64),
                ("d1", K.c_i64), ("dst_row", K.c_i64), ("row_bytes", K.c_i64), ("n0", K.c_int), ("n1", K.c_int),
                ("batch", K.c_int), ("width", K.c_int), ("parent", K.c_vp)]


K.register("slx_kv_append", [ctypes.POINTER(KVAppendDesc), K.c_vp])
K.register("slx_prefix_attn", [ctypes.POINTER(PrefixAttnDesc), K.c_vp])
K.register("slx_prefix_attn_ws_floats", [ctypes.POINTER(PrefixAttnDesc)], K.c_i64)
K.register("slx_beam_select", [ctypes.POINTER(BeamSelectDesc), K.c_vp])
K.register("slx_beam_select_ws_bytes", [ctypes.POINTER(BeamSelectDesc)], K.c_i64)
K.register("slx_beam_reorder", [ctypes.POINTER(BeamReorderDesc), K.c_vp])

MAX_WIDTH = MAX_K = 64      # beam_select, beam_reorder
MAX_VOCAB = 262144          # beam_select


def _need(ok, msg):
    if not ok:
        raise ValueError(msg)


def _on_device(who, first, *rest):
    """Every tensor on the current device, where the launch goes."""
    d = first.device
    for t in rest:
        if t is not None and t.device != d:
            raise RuntimeError(f"{who}: tensors on {d} and {t.device}")
    if d.type != "cuda":
        raise RuntimeError(f"{who}: SimLingo MI355X kernels need device tensors (no CPU fallback)")
    if d.index != torch.cuda.current_device():
        raise RuntimeError(f"{who}: tensors on {d}, current device cuda:{torch.cuda.current_device()}")


def _i32(who, name, t, shape):
    _need(t.dtype is I32 and t.shape == shape and t.is_contiguous(), f"{who}: {name} must be contiguous int32 {list(shape)}")


def _rows(who, name, t, cols):
    """A bf16 matrix view whose rows are contiguous and 16-B aligned -> its row stride."""
    _need(t.dtype is BF16 and t.dim() == 2 and t.shape[1] >= cols, f"{who}: {name} must be bf16 [rows, >= {cols}]")
    s0, s1 = t.stride()
    _need(s1 == 1 and s0 % 8 == 0 and t.data_ptr() % 16 == 0, f"{who}: rows of {name} must be contiguous and 16-B aligned")
    return s0


def _pool(who, k, v, written=False):
    """slx_kv_pool of a cache k, v [pages, page, heads, head size]."""
    _need(k.dtype is BF16 and v.dtype is BF16 and k.dim() == 4, f"{who}: k and v must be bf16 [pages, page, heads, head size]")
    st, sh = k.stride(), k.shape
    _need(sh == v.shape and st == v.stride(), f"{who}: k and v must have the same shape and strides")
    n, page, heads, d = sh
    _need(n > 0 and page > 0 and page & (page - 1) == 0 and heads > 0 and (d == 64 or d == 128),
          f"{who}: pages and heads > 0, page a power of two, head size 64 or 128 (got {list(sh)})")
    kp, vp = k.data_ptr(), v.data_ptr()
    _need(st[3] == 1 and (st[0] | st[1] | st[2]) % 8 == 0 and (kp | vp) % 16 == 0,
          f"{who}: heads of k and v must be contiguous and 16-B aligned")
    if written:
        _need(all(s or m == 1 for s, m in zip(st, sh)), f"{who}: k and v must not be expanded")
    return KVPoolDesc(kp, vp, st[0], st[1], st[2], n, page, heads, d)


def _table(who, name, t):
    _need(t.dtype is I32 and t.dim() == 2 and t.shape[1] > 0 and t.stride(1) == 1, f"{who}: {name} must be int32 [sequences, columns], rows contiguous")
    # rows of a one-row table may have any stride
    return max(t.stride(0), t.shape[1])


def kv_append(qkv, k, v, table, pos, q_out=None, *, n_heads, cos=None, sin=None, seq=None, rows_per_seq=1):
    """Rows of the fused projection, q (n_heads) | k | v, into a paged cache: row i is token `pos[i]` of sequence `seq[i]`
    (i // rows_per_seq without seq). q and k are rotated (rotate_half RoPE, tables [positions, head size / 2] f32 as
    kernels.rope_tables gives; no tables: no rotation) in f32 and rounded once; rotated q goes to q_out, which may be
    qkv's own q columns; without q_out q is not read.

    A row with pos < 0, or one that names no slot (behind the table or the rotation's rows, a sequence or page that there
    is not), is padding: nothing of it is written. Two rows of one call must not name the same slot."""
    who = "kv_append"
    pool = _pool(who, k, v, written=True)
    hkv, d = pool.heads, pool.head_dim
    _need(n_heads >= 0 and (q_out is None or n_heads > 0), f"{who}: n_heads")
    rows = qkv.shape[0]
    ld = _rows(who, "qkv", qkv, (n_heads + 2 * hkv) * d)
    ldt = _table(who, "table", table)
    _need(table.shape[0] > 0 and rows_per_seq > 0, f"{who}: an empty table, or rows_per_seq < 1")
    _i32(who, "pos", pos, (rows,))
    if seq is not None:
        _i32(who, "seq", seq, (rows,))
    ldq = 0
    if q_out is not None:
        ldq = _rows(who, "q_out", q_out, n_heads * d)
        _need(q_out.shape[0] == rows, f"{who}: q_out has {q_out.shape[0]} rows, qkv {rows}")
    rope = 0
    _need((cos is None) == (sin is None), f"{who}: cos and sin go together")
    if cos is not None:
        rope = cos.shape[0]
        for t in (cos, sin):
            _need(t.dtype is F32 and t.shape == (rope, d // 2) and t.is_contiguous() and rope > 0 and t.data_ptr() % 16 == 0,
                  f"{who}: cos and sin must be contiguous f32 [positions, {d // 2}]")
    _on_device(who, qkv, k, v, table, pos, q_out, cos, sin, seq)
    desc = KVAppendDesc(pool, qkv.data_ptr(), ld, q_out.data_ptr() if q_out is not None else 0, ldq, table.data_ptr(), ldt,
                        table.shape[0], table.shape[1], seq.data_ptr() if seq is not None else 0, pos.data_ptr(), rows_per_seq,
                        n_heads, rows, cos.data_ptr() if rope else 0, sin.data_ptr() if rope else 0, rope)
    K.check(K.lib().slx_kv_append(ctypes.byref(desc), K.stream_ptr()), "slx_kv_append")


def prefix_attn(q, out=None, *, own, prefix=None, n_heads, n_q=1, scale=None, max_own=None, max_prefix=None, lse=None):
    """Attention of n_q new tokens per sequence. own = (k, v, table [N, columns], lengths [N]): each sequence's keys, its new
    tokens' among them as the last; prefix = (k, v, table [G, columns], lengths [G]): keys that sequences g * N/G ...
    share, before their own. q rows [N * n_q, n_heads * head size], a sequence's tokens together, already rotated; the
    kv heads are the caches'. Token t sees the whole prefix and own keys up to length - n_q + t; a row without any key
    gives zeros. scale: 1 / sqrt(head size) by default. max_own, max_prefix: bounds of the lengths where they are known
    to be lower than the tables' columns (longer ones are cut to them); the split of the work goes by them.
    Keys on a page number outside the cache are masked. lse: optional f32 [N * n_q, n_heads], natural log of the softmax
    sum (-inf without keys). Returns out (bf16, like q)."""
    who = "prefix_attn"
    ok, ov, otab, olen = own
    opool = _pool(who, ok, ov)
    d = opool.head_dim
    n = otab.shape[0]
    _need(n_heads > 0 and n_heads % opool.heads == 0, f"{who}: n_heads must be a multiple of the cache's {opool.heads} heads")
    _need(n_q > 0 and q.dim() == 2 and q.shape[0] == n * n_q, f"{who}: q must have {n} x {n_q} rows")
    ldq = _rows(who, "q", q, n_heads * d)
    ldot = _table(who, "own table", otab)
    _i32(who, "own lengths", olen, (n,))
    groups = n
    ppool, ptab, ldpt, plen, pcols, pmax = KVPoolDesc(), None, 0, None, 0, 0
    pk = pv = None
    if prefix is not None:
        pk, pv, ptab, plen = prefix
        ppool = _pool(who, pk, pv)
        _need(ppool.heads == opool.heads and ppool.head_dim == d, f"{who}: the two caches differ in heads or head size")
        ldpt = _table(who, "prefix table", ptab)
        groups, pcols = ptab.shape
        _i32(who, "prefix lengths", plen, (groups,))
        _need(groups > 0 and n % groups == 0, f"{who}: {n} sequences do not make {groups} groups of one size")
        pmax = min(pcols * ppool.page, 2**31 - 1) if max_prefix is None else max_prefix
    omax = min(otab.shape[1] * opool.page, 2**31 - 1) if max_own is None else max_own
    _need(omax >= 0 and pmax >= 0, f"{who}: bounds must not be negative")
    if out is None:
        out = torch.empty(q.shape[0], n_heads * d, dtype=BF16, device=q.device)
    ldo = _rows(who, "out", out, n_heads * d)
    _need(out.shape[0] == q.shape[0], f"{who}: out has {out.shape[0]} rows, q {q.shape[0]}")
    if lse is not None:
        _need(lse.dtype is F32 and lse.shape == (q.shape[0], n_heads) and lse.is_contiguous(),
              f"{who}: lse must be contiguous f32 [{q.shape[0]}, {n_heads}]")
    _on_device(who, q, ok, ov, otab, olen, out, pk, pv, ptab, plen, lse)
    if n == 0:
        return out
    desc = PrefixAttnDesc(ppool, opool, q.data_ptr(), ldq, out.data_ptr(), ldo, lse.data_ptr() if lse is not None else 0,
                          ptab.data_ptr() if ptab is not None else 0, ldpt, plen.data_ptr() if plen is not None else 0,
                          otab.data_ptr(), ldot, olen.data_ptr(), pmax, omax, pcols, otab.shape[1], groups, n // groups, n_q,
                          n_heads, 1.0 / math.sqrt(d) if scale is None else scale, 0, 0)
    lib = K.lib()
    need = lib.slx_prefix_attn_ws_floats(ctypes.byref(desc))
    if need < 0:
        K.check(need, "slx_prefix_attn")
    if need:
        ws = torch.empty(need, dtype=F32, device=q.device)  # of this call alone, from the current stream's pool
        desc.ws, desc.ws_floats = ws.data_ptr(), need
    K.check(lib.slx_prefix_attn(ctypes.byref(desc), K.stream_ptr()), "slx_prefix_attn")
    return out


def beam_select(logits, scores, *, width, k=None, finished=None, pad_id=0, eos_id=None, out=None, finished_out=None):
    """The k (default: width) best continuations of each batch entry by scores[b, w] + log_softmax(logits[b, w])[t], in
    descending order, ties to the lowest w * V + t. logits [batch * width, V] f32 or bf16, rows contiguous; scores
    [batch * width] f32 (-inf: the beam is out). finished [batch * width] bool / uint8: such a row offers `pad_id` alone,
    its score unchanged. A score that is not a number (rows of -inf, rows with a NaN or +inf) counts as -inf.

    Returns (scores f32, parent int32, token int32), each [batch, k] (out: the three to write to; the scores may be
    `scores` itself if k == width). finished_out [batch, k], with eos_id: finished[parent] or token == eos_id."""
    who = "beam_select"
    k = width if k is None else k
    _need(0 < width <= MAX_WIDTH and 0 < k <= MAX_K, f"{who}: width and k must be 1 .. {MAX_WIDTH}")
    _need(logits.dim() == 2 and logits.dtype in (F32, BF16) and logits.stride(1) == 1, f"{who}: logits must be f32 or bf16 [rows, V], rows contiguous")
    n, vocab = logits.shape
    _need(0 < vocab <= MAX_VOCAB and n % width == 0 and k <= width * vocab, f"{who}: 1 .. {MAX_VOCAB} logits a row, rows a multiple of width, k <= width * V")
    b = n // width
    _need(scores.dtype is F32 and scores.numel() == n and scores.is_contiguous(), f"{who}: scores must be contiguous f32 [{n}]")
    if finished is not None:
        _need(finished.dtype in (torch.bool, torch.uint8) and finished.numel() == n and finished.is_contiguous(), f"{who}: finished must be contiguous bool [{n}]")
        _need(0 <= pad_id < vocab, f"{who}: pad_id outside the vocabulary")
    if finished_out is not None:
        _need(finished_out.dtype in (torch.bool, torch.uint8) and finished_out.numel() == b * k and finished_out.is_contiguous(),
              f"{who}: finished_out must be contiguous bool [{b}, {k}]")
    if out is None:
        dev = logits.device
        out = (torch.empty(b, k, dtype=F32, device=dev), torch.empty(b, k, dtype=I32, device=dev), torch.empty(b, k, dtype=I32, device=dev))
    else:
        for t, dt in zip(out, (F32, I32, I32)):
            _need(t.dtype is dt and t.numel() == b * k and t.is_contiguous(), f"{who}: out must be contiguous f32, int32, int32 [{b}, {k}]")
    for t, given, what in ((out[0], scores, "scores"), (finished_out, finished, "finished")):
        _need(t is None or given is None or t.data_ptr() != given.data_ptr() or k == width, f"{who}: {what} in place needs k == width")
    _on_device(who, logits, scores, finished, finished_out, *out)
    if b == 0:
        return out
    desc = BeamSelectDesc(logits.data_ptr(), max(logits.stride(0), vocab), int(logits.dtype is BF16), b, width, vocab, k, scores.data_ptr(),
                          finished.data_ptr() if finished is not None else 0, pad_id, out[0].data_ptr(), out[1].data_ptr(),
                          out[2].data_ptr(), finished_out.data_ptr() if finished_out is not None else 0,
                          -1 if eos_id is None else eos_id, 0, 0)
    lib = K.lib()
    need = lib.slx_beam_select_ws_bytes(ctypes.byref(desc))
    if need < 0:
        K.check(need, "slx_beam_select")
    ws = torch.empty(need, dtype=torch.uint8, device=logits.device)  # of this call alone, from the current stream's pool
    desc.ws, desc.ws_bytes = ws.data_ptr(), need
    K.check(lib.slx_beam_select(ctypes.byref(desc), K.stream_ptr()), "slx_beam_select")
    return out


def _span(t):
    """Bytes [from, to) that a view touches."""
    return t.data_ptr(), t.data_ptr() + (sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1) * t.element_size()


def beam_reorder(x, parent, *, dim=0, out=None):
    """out[..., b * W + w, ...] = x[..., b * W + parent[b, w], ...] along `dim` of a state of any type; parent int32 [batch, W]
    as beam_select returns it. Without out (or with x itself) in place, for any parents. The other dimensions may be
    strided as long as they make at most two runs of rows. A parent outside 0 .. W - 1 stands for w itself.
    Returns out."""
    who = "beam_reorder"
    out = x if out is None else out
    _need(parent.dtype is I32 and parent.dim() == 2 and parent.is_contiguous(), f"{who}: parent must be contiguous int32 [batch, W]")
    b, w = parent.shape
    _need(0 < w <= MAX_WIDTH, f"{who}: W must be 1 .. {MAX_WIDTH}")
    _need(-x.dim() <= dim < x.dim() and x.shape == out.shape and x.dtype is out.dtype, f"{who}: dim, or out unlike x")
    dim %= x.dim()
    _need(x.shape[dim] == b * w, f"{who}: dimension {dim} of x has {x.shape[dim]} rows, parent {b} x {w}")
    if x.numel() == 0:
        return out
    es, ss, ds = x.element_size(), x.stride(), out.stride()
    run, outer = 1, []  # a row's contiguous elements; the other dimensions (extent, stride in x, stride in out), inner first
    for i in range(x.dim() - 1, -1, -1):
        m = x.shape[i]
        if i == dim or m == 1:
            continue
        if not outer and ss[i] == ds[i] == run:
            run *= m
        elif outer and ss[i] == outer[-1][0] * outer[-1][1] and ds[i] == outer[-1][0] * outer[-1][2]:
            outer[-1] = (outer[-1][0] * m, outer[-1][1], outer[-1][2])
        else:
            outer.append((m, ss[i], ds[i]))
    _need(len(outer) <= 2, f"{who}: the state's strides make more than two runs of rows")
    _need(all(s for m, _, s in outer) and (ds[dim] or b * w == 1), f"{who}: out must not be expanded")
    same = x.data_ptr() == out.data_ptr()
    if not same or ss != ds:
        (a0, a1), (c0, c1) = _span(x), _span(out)
        _need(a1 <= c0 or c1 <= a0, f"{who}: out overlaps x")
    _on_device(who, x, out, parent)
    outer += [(1, 0, 0)] * (2 - len(outer))
    (n1, s1, d1), (n0, s0, d0) = outer
    desc = BeamReorderDesc(x.data_ptr(), out.data_ptr(), s0 * es, s1 * es, ss[dim] * es, d0 * es, d1 * es, ds[dim] * es, run * es,
                           n0, n1, b, w, parent.data_ptr())
    K.check(K.lib().slx_beam_reorder(ctypes.byref(desc), K.stream_ptr()), "slx_beam_reorder")
    return out
