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
import functools
import math
import struct

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


for _name in ("slx_kv_append", "slx_prefix_attn", "slx_beam_select", "slx_beam_reorder"):
    K.register(_name, [K.c_vp, K.c_vp])
K.register("slx_prefix_attn_ws_floats", [K.c_vp], K.c_i64)
K.register("slx_beam_select_ws_bytes", [K.c_vp], K.c_i64)

MAX_WIDTH = MAX_K = 64      # beam_select, beam_reorder
MAX_VOCAB = 262144          # beam_select

# The calls below are a token's step many times over, on small tensors: descriptors are packed in one go (native sizes and
# alignment, the structures' own layout) and a check builds its message only when it fails.
_POOL = "PPqqqiiii"
_APPEND = struct.Struct("@" + _POOL + "PqPqPqiiPPiiqPPi0q")
_ATTN = struct.Struct("@" + _POOL + _POOL + "PqPqPPqPPqPiiiiiiiifPq")
_SELECT = struct.Struct("@PqiiiiiPPiPPPPiPq")
_REORDER = struct.Struct("@PPqqqqqqqiiiiP")
_NO_POOL = (0,) * 9
_raw_stream, _current = torch._C._cuda_getCurrentRawStream, torch._C._cuda_getDevice


def _bad(msg):
    raise ValueError(msg)


def _device(who, first, *rest):
    """The device of every tensor given (None: not given), which has to be the current one, where the launch goes."""
    d = first.get_device()
    for t in rest:
        if t is not None and t.get_device() != d:
            raise RuntimeError(f"{who}: tensors on {first.device} and {t.device}")
    if d < 0:
        raise RuntimeError(f"{who}: SimLingo MI355X kernels need device tensors (no CPU fallback)")
    if d != _current():
        raise RuntimeError(f"{who}: tensors on cuda:{d}, current device cuda:{torch.cuda.current_device()}")
    return d


def _i32(who, name, t, n):
    if t.dtype is not I32 or t.numel() != n or t.dim() != 1 or not t.is_contiguous():
        _bad(f"{who}: {name} must be contiguous int32 [{n}]")


def _rows(who, name, t, n, cols):
    """A bf16 matrix view of n rows that are contiguous and 16-B aligned -> its address and row stride."""
    sh, st, p = t.shape, t.stride(), t.data_ptr()
    if t.dtype is not BF16 or len(sh) != 2:
        _bad(f"{who}: {name} must be a bf16 matrix")
    if sh[0] != n or sh[1] < cols:
        _bad(f"{who}: {name} must have {n} rows of at least {cols}, got {list(sh)}")
    s0, s1 = st
    if s1 != 1 or (s0 * 2 | p) & 15:
        _bad(f"{who}: rows of {name} must be contiguous and 16-B aligned")
    return p, s0


def _pool(who, k, v, written=False):
    """The fields of slx_kv_pool for a cache k, v [pages, page, heads, head size]."""
    sh, st, kp, vp = k.shape, k.stride(), k.data_ptr(), v.data_ptr()
    if k.dtype is not BF16 or v.dtype is not BF16 or len(sh) != 4:
        _bad(f"{who}: k and v must be bf16 [pages, page, heads, head size]")
    if sh != v.shape or st != v.stride():
        _bad(f"{who}: k and v must have the same shape and strides")
    n, page, heads, d = sh
    s0, s1, s2, s3 = st
    if n < 1 or page < 1 or page & (page - 1) or heads < 1 or d != 64 and d != 128:
        _bad(f"{who}: pages and heads > 0, page a power of two, head size 64 or 128 (got {list(sh)})")
    if s3 != 1 or ((s0 | s1 | s2) * 2 | kp | vp) & 15:
        _bad(f"{who}: heads of k and v must be contiguous and 16-B aligned")
    if written and not ((s0 or n == 1) and (s1 or page == 1) and (s2 or heads == 1)):
        _bad(f"{who}: k and v must not be expanded")
    return kp, vp, s0, s1, s2, n, page, heads, d


def _table(who, name, t):
    """Address, row stride, rows and columns of a page table."""
    sh, st = t.shape, t.stride()
    if t.dtype is not I32 or len(sh) != 2:
        _bad(f"{who}: {name} must be int32 [sequences, columns]")
    n, cols = sh
    s0, s1 = st
    if cols < 1 or s1 != 1 and cols > 1 or s0 < cols and n > 1:
        _bad(f"{who}: {name} must have columns, its rows contiguous and apart")
    return t.data_ptr(), s0 if s0 > cols else cols, n, cols


def kv_append(qkv, k, v, table, pos, q_out=None, *, n_heads, cos=None, sin=None, seq=None, rows_per_seq=1):
    """Rows of the fused projection, q (n_heads) | k | v, into a paged cache: row i is token `pos[i]` of sequence `seq[i]`
    (i // rows_per_seq without seq). q and k are rotated (rotate_half RoPE, tables [positions, head size / 2] f32 as
    kernels.rope_tables gives; no tables: no rotation) in f32 and rounded once; rotated q goes to q_out, which may be
    qkv's own q columns; without q_out q is not read.

    A row with pos < 0, or one that names no slot (behind the table or the rotation's rows, a sequence or page that there
    is not), is padding: nothing of it is written. Two rows of one call must not name the same slot."""
    who = "kv_append"
    pool = _pool(who, k, v, True)
    hkv, d = pool[7], pool[8]
    if n_heads < 0 or (q_out is not None and n_heads == 0):
        _bad(f"{who}: n_heads {n_heads}")
    rows = qkv.shape[0]
    x, ldx = _rows(who, "qkv", qkv, rows, (n_heads + 2 * hkv) * d)
    tab, ldt, n_seq, cols = _table(who, "table", table)
    if n_seq < 1 or rows_per_seq < 1:
        _bad(f"{who}: an empty table, or rows_per_seq < 1")
    _i32(who, "pos", pos, rows)
    if seq is not None:
        _i32(who, "seq", seq, rows)
    q, ldq = _rows(who, "q_out", q_out, rows, n_heads * d) if q_out is not None else (0, 0)
    c = s = rope = 0
    if cos is None or sin is None:
        if cos is not sin:
            _bad(f"{who}: cos and sin go together")
    else:
        sh, c, s = cos.shape, cos.data_ptr(), sin.data_ptr()
        rope = sh[0]
        if not (cos.dtype is F32 and sin.dtype is F32 and sh == sin.shape and len(sh) == 2 and sh[1] == d // 2 and rope > 0
                and cos.is_contiguous() and sin.is_contiguous() and not (c | s) & 15):
            _bad(f"{who}: cos and sin must be contiguous f32 [positions, {d // 2}]")
    desc = _APPEND.pack(*pool, x, ldx, q, ldq, tab, ldt, n_seq, cols, seq.data_ptr() if seq is not None else 0, pos.data_ptr(),
                        rows_per_seq, n_heads, rows, c, s, rope)
    dev = _device(who, qkv, k, v, table, pos, q_out, cos, sin, seq)
    rc = K.lib().slx_kv_append(desc, _raw_stream(dev))
    if rc:
        K.check(rc, "slx_kv_append")


@functools.lru_cache(maxsize=1024)
def _attn_ws(ppool, opool, has_prefix, pmax, omax, pcols, ocols, groups, width, n_q, n_heads):
    """Floats of workspace for these sizes (the C entry's own rule; no address goes into it)."""
    ptab = 16 if has_prefix else 0
    need = K.lib().slx_prefix_attn_ws_floats(_ATTN.pack(*_fake(ppool), *_fake(opool), 0, 0, 0, 0, 0, ptab, pcols, ptab, 0, ocols, 0, pmax, omax,
                                                        pcols, ocols, groups, width, n_q, n_heads, 1.0, 0, 0))
    if need < 0:
        K.check(need, "slx_prefix_attn")
    return need


def _fake(pool):
    """slx_kv_pool's fields from its sizes alone."""
    n, page, heads, d = pool
    return (16, 16, 0, 0, 0, n, page, heads, d) if n else _NO_POOL


def prefix_attn(q, out=None, *, own, prefix=None, n_heads, n_q=1, scale=None, max_own=None, max_prefix=None, lse=None):
    """Attention of n_q new tokens per sequence. own = (k, v, table [N, columns], lengths [N]): each sequence's keys, its new
    tokens' among them as the last; prefix = (k, v, table [G, columns], lengths [G]): keys that sequences g * N/G ...
    share, before their own. q rows [N * n_q, n_heads * head size], a sequence's tokens together, already rotated; the
    kv heads are the caches'. Token t sees the whole prefix and own keys up to length - n_q + t; a row without any key
    gives zeros. scale > 0: 1 / sqrt(head size) by default. max_own, max_prefix: bounds of the lengths where they are known
    to be lower than the tables' columns (longer ones are cut to them); the split of the work goes by them.
    Keys on a page number outside the cache are masked. lse: optional f32 [N * n_q, n_heads], natural log of the softmax
    sum (-inf without keys). Returns out (bf16, like q)."""
    who = "prefix_attn"
    ok, ov, otab, olen = own
    opool = _pool(who, ok, ov)
    heads, d = opool[7], opool[8]
    ot, ldot, n, ocols = _table(who, "own table", otab)
    if n_heads < 1 or n_heads % heads:
        _bad(f"{who}: n_heads must be a multiple of the cache's {heads} heads")
    if n_q < 1:
        _bad(f"{who}: n_q {n_q}")
    scale = d ** -0.5 if scale is None else scale
    if not 0 < scale < math.inf:
        _bad(f"{who}: scale must be positive")
    rows, cols = n * n_q, n_heads * d
    x, ldq = _rows(who, "q", q, rows, cols)
    _i32(who, "own lengths", olen, n)
    ppool, pk, pv, ptab, plen, pt, ldpt, groups, pcols, pmax, pl = _NO_POOL, None, None, None, None, 0, 0, n, 0, 0, 0
    if prefix is not None:
        pk, pv, ptab, plen = prefix
        ppool = _pool(who, pk, pv)
        if ppool[7] != heads or ppool[8] != d:
            _bad(f"{who}: the two caches differ in heads or head size")
        pt, ldpt, groups, pcols = _table(who, "prefix table", ptab)
        _i32(who, "prefix lengths", plen, groups)
        if groups < 1 or n % groups:
            _bad(f"{who}: {n} sequences do not make {groups} groups of one size")
        pl = plen.data_ptr()
        pmax = min(pcols * ppool[6], 2**31 - 1) if max_prefix is None else max_prefix
    omax = min(ocols * opool[6], 2**31 - 1) if max_own is None else max_own
    if not (0 <= omax < 2**31 and 0 <= pmax < 2**31):
        _bad(f"{who}: bounds must be 0 .. 2^31 - 1")
    if out is None:
        out = torch.empty(rows, cols, dtype=BF16, device=q.device)
    o, ldo = _rows(who, "out", out, rows, cols)
    if lse is not None and not (lse.dtype is F32 and lse.shape == (rows, n_heads) and lse.is_contiguous()):
        _bad(f"{who}: lse must be contiguous f32 [{rows}, {n_heads}]")
    dev = _device(who, q, ok, ov, otab, olen, out, pk, pv, ptab, plen, lse)
    if not n:
        return out
    width = n // groups
    need = _attn_ws(ppool[5:], opool[5:], pt != 0, pmax, omax, pcols, ocols, groups, width, n_q, n_heads)
    ws = torch.empty(need, dtype=F32, device=q.device) if need else None  # of this call alone, from the current stream's memory
    desc = _ATTN.pack(*ppool, *opool, x, ldq, o, ldo, lse.data_ptr() if lse is not None else 0, pt, ldpt, pl, ot, ldot, olen.data_ptr(),
                      pmax, omax, pcols, ocols, groups, width, n_q, n_heads, scale, ws.data_ptr() if need else 0, need)
    rc = K.lib().slx_prefix_attn(desc, _raw_stream(dev))
    if rc:
        K.check(rc, "slx_prefix_attn")
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
    if not (0 < width <= MAX_WIDTH and 0 < k <= MAX_K):
        _bad(f"{who}: width and k must be 1 .. {MAX_WIDTH}")
    bf = logits.dtype is BF16
    if logits.dim() != 2 or not (bf or logits.dtype is F32):
        _bad(f"{who}: logits must be f32 or bf16 [rows, V]")
    (n, vocab), (ldx, s1) = logits.shape, logits.stride()
    if s1 != 1 and vocab > 1 or ldx < vocab and n > 1:
        _bad(f"{who}: rows of logits must be contiguous and apart")
    if not (0 < vocab <= MAX_VOCAB and n % width == 0 and k <= width * vocab):
        _bad(f"{who}: 1 .. {MAX_VOCAB} logits a row, rows a multiple of width, k <= width * V")
    b = n // width
    if not (scores.dtype is F32 and scores.numel() == n and scores.is_contiguous()):
        _bad(f"{who}: scores must be contiguous f32 [{n}]")
    sp, fp, fo = scores.data_ptr(), 0, 0
    if finished is not None:
        if not (finished.dtype in (torch.bool, torch.uint8) and finished.numel() == n and finished.is_contiguous()):
            _bad(f"{who}: finished must be contiguous bool [{n}]")
        if not 0 <= pad_id < vocab:
            _bad(f"{who}: pad_id outside the vocabulary")
        fp = finished.data_ptr()
    if finished_out is not None:
        if not (finished_out.dtype in (torch.bool, torch.uint8) and finished_out.numel() == b * k and finished_out.is_contiguous()):
            _bad(f"{who}: finished_out must be contiguous bool [{b}, {k}]")
        fo = finished_out.data_ptr()
    if out is None:
        s_out, (p_out, t_out) = torch.empty(b, k, dtype=F32, device=logits.device), torch.empty(2, b, k, dtype=I32, device=logits.device).unbind()
        out = s_out, p_out, t_out
    s_out, p_out, t_out = out
    if not (s_out.dtype is F32 and p_out.dtype is I32 and t_out.dtype is I32 and s_out.numel() == p_out.numel() == t_out.numel() == b * k
            and s_out.is_contiguous() and p_out.is_contiguous() and t_out.is_contiguous()):
        _bad(f"{who}: out must be contiguous f32, int32, int32 [{b}, {k}]")
    so = s_out.data_ptr()
    if k != width and n and (so == sp or fo and fo == fp):
        _bad(f"{who}: scores or finished in place need k == width")
    dev = _device(who, logits, scores, s_out, p_out, t_out, finished, finished_out)
    if not b:
        return out
    need = _select_ws(b, width, vocab, k)
    ws = torch.empty(need, dtype=torch.uint8, device=logits.device)  # of this call alone, from the current stream's memory
    rc = K.lib().slx_beam_select(_SELECT.pack(logits.data_ptr(), max(ldx, vocab), bf, b, width, vocab, k, sp, fp, pad_id if fp else 0, so,
                                              p_out.data_ptr(), t_out.data_ptr(), fo, -1 if eos_id is None else eos_id, ws.data_ptr(), need),
                                 _raw_stream(dev))
    if rc:
        K.check(rc, "slx_beam_select")
    return out


@functools.lru_cache(maxsize=1024)
def _select_ws(b, width, vocab, k):
    need = K.lib().slx_beam_select_ws_bytes(_SELECT.pack(0, vocab, 0, b, width, vocab, k, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0))
    if need < 0:
        K.check(need, "slx_beam_select")
    return need


def _span(t):
    """Bytes [from, to) that a view touches."""
    return t.data_ptr(), t.data_ptr() + (sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1) * t.element_size()


def beam_reorder(x, parent, *, dim=0, out=None):
    """out[..., b * W + w, ...] = x[..., b * W + parent[b, w], ...] along `dim` of a state of any type; parent int32 [batch, W]
    as beam_select returns it. Without out (or with x itself) in place, for any parents. The other dimensions may be
    strided as long as they make at most two runs of rows. A parent outside 0 .. W - 1 stands for w itself.
    Returns out."""
    who = "beam_reorder"
    if parent.dtype is not I32 or parent.dim() != 2 or not parent.is_contiguous():
        _bad(f"{who}: parent must be contiguous int32 [batch, W]")
    b, w = parent.shape
    if not 0 < w <= MAX_WIDTH:
        _bad(f"{who}: W must be 1 .. {MAX_WIDTH}")
    if out is None:
        out = x
    sh, ss, ds, nd = x.shape, x.stride(), out.stride(), x.dim()
    if not -nd <= dim < nd or sh != out.shape or x.dtype is not out.dtype:
        _bad(f"{who}: dim, or out unlike x")
    dim %= nd
    if sh[dim] != b * w:
        _bad(f"{who}: dimension {dim} of x has {sh[dim]} rows, parent {b} x {w}")
    es, run, outer, empty = x.element_size(), 1, [], False
    for i in range(nd - 1, -1, -1):  # a row's contiguous elements; the other dimensions (extent, stride in x, in out), inner first
        m, s, t = sh[i], ss[i], ds[i]
        empty = empty or m == 0
        if i == dim or m == 1:
            continue
        if not outer and s == t == run:
            run *= m
        elif outer and s == outer[-1][0] * outer[-1][1] and t == outer[-1][0] * outer[-1][2]:
            outer[-1] = (outer[-1][0] * m, outer[-1][1], outer[-1][2])
        else:
            outer.append((m, s, t))
    if empty:
        return out
    if len(outer) > 2:
        _bad(f"{who}: the state's strides make more than two runs of rows")
    if any(not t for _, _, t in outer) or (not ds[dim] and b * w > 1):
        _bad(f"{who}: out must not be expanded")
    xp, op = x.data_ptr(), out.data_ptr()
    if xp != op or ss != ds:
        (a0, a1), (c0, c1) = _span(x), _span(out)
        if a0 < c1 and c0 < a1:
            _bad(f"{who}: out overlaps x")
    outer += ((1, 0, 0), (1, 0, 0))
    (n1, s1, d1), (n0, s0, d0) = outer[:2]
    desc = _REORDER.pack(xp, op, s0 * es, s1 * es, ss[dim] * es, d0 * es, d1 * es, ds[dim] * es, run * es, n0, n1, b, w, parent.data_ptr())
    rc = K.lib().slx_beam_reorder(desc, _raw_stream(_device(who, x, out, parent)))
    if rc:
        K.check(rc, "slx_beam_reorder")
    return out
