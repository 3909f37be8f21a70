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
positions and tables are read on the device, so a captured call follows their contents. These are operators for serving: they have no
gradients, and what they return is detached.
"""
from __future__ import annotations

import ctypes

import torch

from . import kernels as K


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

_native = None


def _bind():
    """simlingo_amd/_paged.so (csrc/paged_bind.cpp), which reads and checks the tensors and calls the library: these calls are a
    token's step many times over, on a few small tensors each. No fallback: an error if it is not built."""
    global _native
    try:
        from . import _paged
    except ImportError as e:
        raise RuntimeError("simlingo_amd/_paged.so is not built (or for another torch): run `python -m simlingo_amd.build`. "
                           "There is no CPU/eager fallback for the SimLingo MI355X kernels.") from e
    lib = K.lib()
    names = ("slx_kv_append", "slx_prefix_attn", "slx_prefix_attn_ws_floats", "slx_beam_select", "slx_beam_select_ws_bytes",
             "slx_beam_reorder", "slx_last_error")
    _paged.setup(tuple(ctypes.cast(getattr(lib, n), K.c_vp).value for n in names), torch._C._cuda_getCurrentRawStream,
                 torch._C._cuda_getDevice)
    _native = _paged
    return _paged


def kv_append(qkv, k, v, table, pos, q_out=None, *, n_heads, cos=None, sin=None, seq=None, rows_per_seq=1):
    """Rows of the fused projection, q (n_heads) | k | v, into a paged cache: row i is token `pos[i]` of sequence `seq[i]`
    (i // rows_per_seq without seq). q and k are rotated (rotate_half RoPE, tables [positions, head size / 2] f32 as
    kernels.rope_tables gives; no tables: no rotation) in f32 and rounded once; rotated q goes to q_out, which may be
    qkv's own q columns; without q_out q is not read.

    A row with pos < 0, or one that names no slot (behind the table or the rotation's rows, a sequence or page that there
    is not), is padding: nothing of it is written. Two rows of one call must not name the same slot. k and v are apart from
    each other and from qkv and q_out, and what is written from what is read beside; columns or slots of one buffer may be."""
    (_native or _bind()).kv_append(qkv, k, v, table, pos, q_out, n_heads, cos, sin, seq, rows_per_seq)


def prefix_attn(q, out=None, *, own, prefix=None, n_heads, n_q=1, scale=None, max_own=None, max_prefix=None, lse=None):
    """Attention of n_q new tokens per sequence. own = (k, v, table [N, columns], lengths [N]): each sequence's keys, its new
    tokens' among them as the last; prefix = (k, v, table [G, columns], lengths [G]): keys that sequences g * N/G ...
    share, before their own (groups of one size: a smaller one is filled up with sequences of length 0, which cost what the
    others do). q rows [N * n_q, n_heads * head size], a sequence's tokens together, already rotated; the kv heads are the
    caches'. Token t sees the whole prefix and own keys up to length - n_q + t; a row without any key, or with scores of -inf
    alone, gives zeros. scale > 0: 1 / sqrt(head size) by default. max_own, max_prefix: bounds of the lengths where they are
    known to be lower than the tables' columns (longer ones are cut to them), at most 2^30; the split of the work goes by
    them. Keys on a page number outside the cache are masked. lse: optional f32 [N * n_q, n_heads], natural log of the softmax
    sum (-inf without keys). Returns out (bf16, like q); it may be q itself, or other columns of its rows. out and lse are
    apart from the caches, tables and lengths.

    Scores, softmax, sums and partial outputs are held in f32 (probabilities enter the product with V as two bf16 terms,
    2^-15); the output is rounded once."""
    ok, ov, otab, olen = own
    pk, pv, ptab, plen = prefix if prefix is not None else (None, None, None, None)
    return (_native or _bind()).prefix_attn(q, out, ok, ov, otab, olen, pk, pv, ptab, plen, n_heads, n_q, scale, max_own, max_prefix, lse)


def beam_select(logits, scores, *, width, k=None, finished=None, pad_id=0, eos_id=None, out=None, finished_out=None):
    """The k (default: width) best continuations of each batch entry by scores[b, w] + log_softmax(logits[b, w])[t], in
    descending order, ties to the lowest w * V + t. logits [batch * width, V] f32 or bf16, rows contiguous, V up to MAX_VOCAB
    and fewer than 2^24 pieces of 4096 in all the rows; width, k up to MAX_WIDTH, MAX_K; scores
    [batch * width] f32 (not finite: the beam is out). finished [batch * width] bool / uint8: such a row offers `pad_id` alone,
    its score unchanged. The scores of a row that is out, is -inf throughout or holds a NaN or +inf count as -inf.

    Returns (scores f32, parent int32, token int32), each [batch, k] (out: the three to write to; the scores may be
    `scores` itself if k == width, and finished_out `finished`). finished_out [batch, k], with eos_id: finished[parent] or token == eos_id."""
    return (_native or _bind()).beam_select(logits, scores, width, k, finished, pad_id, eos_id, out, finished_out)


def beam_reorder(x, parent, *, dim=0, out=None):
    """out[..., b * W + w, ...] = x[..., b * W + parent[b, w], ...] along `dim` of a state of any type; parent int32 [batch, W]
    as beam_select returns it. Without out (or with x itself) in place, for any parents. The other dimensions may be
    strided as long as they make at most two runs of rows. A parent outside 0 .. W - 1 stands for w itself.
    out is apart from x (or x itself) and from parent. Returns out."""
    return (_native or _bind()).beam_reorder(x, parent, dim, out)
