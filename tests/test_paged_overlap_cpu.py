"""What the paged decode operators (simlingo_amd/paged.py) write must lie apart from itself and from what they read: calls that do not
keep to that are refused before a launch, calls that do are taken, however their memory is interleaved. Without a GPU."""
import ctypes

import pytest
import torch

from simlingo_amd import kernels as K
from simlingo_amd import paged as PG
from test_paged_cpu import append_args, attn_args

BF16, F32, I32 = torch.bfloat16, torch.float32, torch.int32


def taken(call, ok, text):
    """A good call ends at the device (there is none here), a bad one at the check named."""
    with pytest.raises(RuntimeError if ok else ValueError, match="no CPU" if ok else text):
        call()


@pytest.mark.parametrize("stride,ok", ((0, False), (64, False), (248, False), (256, True), (264, True), (1024, True)))
def test_rows_written_lie_apart(stride, ok):
    buf = torch.zeros(8192, dtype=BF16)
    out = buf.as_strided((4, 256), (stride, 1))
    taken(lambda: PG.prefix_attn(**attn_args(out=out)), ok, "out overlap each other")
    taken(lambda: PG.kv_append(**append_args(q_out=out[:3])), ok, "q_out overlap each other")
    taken(lambda: PG.prefix_attn(**attn_args(q=out)), True, "")  # rows that are read may be one row


def test_one_row_has_no_stride():
    one = torch.zeros(256, dtype=BF16).expand(1, -1)
    own = tuple(x[:1] if x.dim() < 3 else x for x in attn_args()["own"])
    taken(lambda: PG.prefix_attn(**attn_args(q=one, out=torch.zeros(256, dtype=BF16).expand(1, -1), own={f"_{i}": t for i, t in enumerate(own)}, prefix={}) | dict(prefix=None)), True, "")


def test_c_entries_refuse_rows_that_overlap():
    lib = K.lib()
    pool = PG.KVPoolDesc(4096, 8192, 1024, 128, 64, 4, 8, 2, 64)
    ap = PG.KVAppendDesc(pool=pool, rows=2, n_seq=1, cols=1, ldt=1, rows_per_seq=1, Hq=4, qkv=4096, ldqkv=512, table=4096, pos=4096, q_out=1 << 20, ldq=248)
    assert lib.slx_kv_append(ctypes.byref(ap), None) == -22 and b"q_out overlap" in lib.slx_last_error()
    at = PG.PrefixAttnDesc(own_pool=pool, q=4096, ldq=256, out=4096, ldo=248, otab=4096, ldot=2, olen=4096, max_own=16, ocols=2, groups=1, width=2, n_q=1, Hq=4, scale=1.0)
    assert lib.slx_prefix_attn(ctypes.byref(at), None) == -22 and b"out overlap" in lib.slx_last_error()


def touched(t):
    """The elements of its storage that a view covers, each as often as it does."""
    at = torch.full(t.shape, t.storage_offset(), dtype=torch.int64)
    for i, (n, s) in enumerate(zip(t.shape, t.stride())):
        at = at + (torch.arange(n) * s).view([n if j == i else 1 for j in range(t.dim())])
    return at.reshape(-1).tolist()


def share(a, b):
    return bool(set(touched(a)) & set(touched(b)))


LAYOUTS = {  # k and v of one allocation, side by side at every level
    "tokens": lambda n, p, h, d: torch.zeros(n, p, 2, h, d, dtype=BF16).unbind(2),
    "heads": lambda n, p, h, d: torch.zeros(n, p, h, 2, d, dtype=BF16).unbind(3),
    "pages": lambda n, p, h, d: torch.zeros(n, 2, p, h, d, dtype=BF16).unbind(1),
    "head-major": lambda n, p, h, d: [x.transpose(1, 2) for x in torch.zeros(n, 2, h, p, d, dtype=BF16).unbind(1)],
    "head-pairs": lambda n, p, h, d: [x.transpose(1, 2) for x in torch.zeros(n, h, 2, p, d, dtype=BF16).unbind(2)],
    "slots-of-heads": lambda n, p, h, d: [x.transpose(1, 2) for x in torch.zeros(n, h, p, 2, d, dtype=BF16).unbind(3)],
    "halves": lambda n, p, h, d: torch.zeros(2, n, p, h, d, dtype=BF16).unbind(0),
}


@pytest.mark.parametrize("layout", LAYOUTS)
def test_caches_side_by_side_are_taken(layout):
    for n, p, h in ((4, 8, 2), (1, 1, 1), (3, 16, 1), (1, 4, 3), (5, 1, 2)):
        k, v = LAYOUTS[layout](n, p, h, 64)
        assert not share(k, v)
        taken(lambda: PG.kv_append(**append_args(k=k, v=v, qkv=torch.zeros(3, (4 + 2 * h) * 64, dtype=BF16))), True, "")


def test_caches_that_overlap_are_refused():
    b = torch.zeros(1 << 16, dtype=BF16)
    view = lambda at, *st: b.as_strided((4, 8, 2, 64), (*st, 1), at)  # noqa: E731
    for st in ((1024, 128, 64), (2048, 256, 128), (1024, 64, 512)):
        k = view(0, *st)
        for at in range(0, 4096, 40):
            v = view(at, *st)
            if at:
                taken(lambda: PG.kv_append(**append_args(k=k, v=v)), not share(k, v), "k and v overlap")
    for st in ((1024, 128, 56), (1024, 64, 64), (512, 128, 64), (64, 512, 128), (40, 400, 16)):  # heads, slots, pages over each other
        k, v = view(0, *st), view(1 << 15, *st)
        assert len(set(touched(k))) < k.numel()
        taken(lambda: PG.kv_append(**append_args(k=k, v=v)), False, "overlap each other")


def test_any_strides():
    """Against the sets of elements themselves, for strides drawn at random (some of them apart by chance alone)."""
    g = torch.Generator().manual_seed(0)
    pick = lambda lo, hi: int(torch.randint(lo, hi, (1,), generator=g))  # noqa: E731
    b = torch.zeros(1 << 18, dtype=BF16)
    seen = {True: 0, False: 0}
    for _ in range(600):
        shape = (pick(1, 5), 2 ** pick(0, 3), pick(1, 4), 64)
        st = [8 * pick(1, 2 ** pick(2, 8)) for _ in range(3)]
        k, v = b.as_strided(shape, (*st, 1), 0), b.as_strided(shape, (*st, 1), 8 * pick(1, 600))
        own = len(set(touched(k))) == k.numel()
        ok = own and not share(k, v)
        seen[ok] += 1
        taken(lambda: PG.kv_append(**append_args(k=k, v=v, qkv=torch.zeros(3, (4 + 2 * shape[2]) * 64, dtype=BF16))), ok, "overlap")
    assert min(seen.values()) > 50


def test_cache_apart_from_the_rows():
    """One buffer of fused rows q | k | v: its k and v columns as the cache, a row a slot. Its q columns may be written; qkv may not be in it."""
    S, hq, hkv, d = 32, 4, 2, 64
    b = torch.zeros(S, (hq + 2 * hkv) * d, dtype=BF16)
    pages = lambda at: b.as_strided((4, 8, hkv, d), (8 * b.stride(0), b.stride(0), d, 1), at)  # noqa: E731
    k, v, q = pages(hq * d), pages((hq + hkv) * d), b[:, :hq * d]
    new = torch.zeros(3, (hq + 2 * hkv) * d, dtype=BF16)
    taken(lambda: PG.kv_append(**append_args(k=k, v=v, qkv=new, q_out=q[5:8])), True, "")
    taken(lambda: PG.kv_append(**append_args(k=k, v=v, qkv=new, q_out=b[5:8, 64:320])), False, "cache overlaps")
    taken(lambda: PG.kv_append(**append_args(k=k, v=v, qkv=b[5:8])), False, "cache overlaps")
    taken(lambda: PG.kv_append(**append_args(k=k, v=v, qkv=new, q_out=b[5:8, 64:320])), False, "cache overlaps")
    own = dict(_0=k, _1=v)
    taken(lambda: PG.prefix_attn(**attn_args(own=own, q=q[:4], out=q[:4])), True, "")
    taken(lambda: PG.prefix_attn(**attn_args(own=own, q=q[:4], out=q[9:13])), True, "")
    taken(lambda: PG.prefix_attn(**attn_args(own=own, out=b[:4, 64:320])), False, "out overlaps a cache")
    taken(lambda: PG.prefix_attn(**attn_args(own=own, out=b[28:32, hq * d:])), False, "out overlaps a cache")
    taken(lambda: PG.prefix_attn(**attn_args(prefix=own, out=b[28:32, hq * d:])), False, "out overlaps a cache")
    taken(lambda: PG.prefix_attn(**attn_args(own=own, lse=b.view(-1)[256:288].view(F32).view(4, 4))), False, "lse overlaps a cache")


def test_tables_apart_from_what_is_written():
    b = torch.zeros(4096, dtype=torch.int32)
    ints = lambda at, *shape: b[at:at + torch.Size(shape).numel()].view(shape)  # noqa: E731
    out = b[:512].view(BF16).view(4, 256)
    for kw in (dict(own=dict(_2=ints(500, 4, 3))), dict(own=dict(_3=ints(0, 4))), dict(prefix=dict(_2=ints(511, 2, 3))), dict(prefix=dict(_3=ints(300, 2)))):
        taken(lambda: PG.prefix_attn(**attn_args(out=out, **kw)), False, "out overlaps a table")
    taken(lambda: PG.prefix_attn(**attn_args(out=out, own=dict(_2=ints(512, 4, 3)))), True, "")
    lse = b[600:616].view(F32).view(4, 4)
    taken(lambda: PG.prefix_attn(**attn_args(lse=lse, own=dict(_3=ints(615, 4)))), False, "lse overlaps a table")
    q_out = out[:3]
    for kw in (dict(table=ints(383, 2, 2)), dict(pos=ints(7, 3)), dict(seq=ints(100, 3)), dict(cos=b[:512].view(F32).view(16, 32))):
        taken(lambda: PG.kv_append(**append_args(q_out=q_out, **kw)), False, "q_out overlaps the table")
    pool = b.view(BF16)
    k, v = pool[:4096].view(4, 8, 2, 64), pool[4096:].view(4, 8, 2, 64)
    for at in (0, 2047, 2048, 4092):
        taken(lambda: PG.kv_append(**append_args(k=k, v=v, pos=ints(at, 3))), False, "the cache overlaps the table")


def test_reorder_out_apart():
    """Rows of out that overlap each other, or the parents, are refused; other columns or rows of x's own buffer are not."""
    parent = torch.zeros(2, 2, dtype=I32)
    b = torch.zeros(256)
    x = torch.zeros(4, 6)
    for st in ((5, 1), (6, 1), (1, 4), (1, 3), (2, 4), (2, 8), (2, 9), (4, 17), (5, 21), (4, 6), (3, 5)):
        out = b.as_strided((4, 6), st)
        ok = len(set(touched(out))) == 24
        taken(lambda: PG.beam_reorder(x, parent, out=out), ok, "rows of out overlap")
        taken(lambda: PG.beam_reorder(out, parent), ok, "rows of out overlap")
    buf = torch.zeros(8, 20)
    for out, ok in ((buf[:4, 6:12], True), (buf[4:, :6], True), (buf[:4, 5:11], False), (buf[1:5, :6], False), (buf[1:5, 6:12], True), (buf[::2, :6], False), (buf[:4, :6], True)):
        taken(lambda: PG.beam_reorder(buf[:4, :6], parent, out=out), ok, "out overlaps x")
    taken(lambda: PG.beam_reorder(buf[::2, :6], parent, out=buf[1::2, :6]), True, "")
    taken(lambda: PG.beam_reorder(buf[:, :6], torch.zeros(4, 2, dtype=I32), out=buf[:, 6:18:2]), True, "")
    ints = torch.zeros(4, 3, dtype=I32)
    ints4 = ints.view(-1)[2:6].view(2, 2)
    taken(lambda: PG.beam_reorder(ints, ints4), False, "out overlaps parent")
    taken(lambda: PG.beam_reorder(ints[:, :1], ints.view(-1)[1:3].view(1, 2).expand(2, 2).contiguous()), True, "")
    taken(lambda: PG.beam_reorder(ints4.view(4, 1), ints4, out=torch.zeros(4, 1, dtype=I32)), True, "")


def test_one_row_in_place_whatever_its_stride():
    """A single row's stride says nothing: x and out of one memory are in place."""
    b = torch.zeros(64)
    taken(lambda: PG.beam_reorder(b.as_strided((1, 8), (3, 1)), torch.zeros(1, 1, dtype=I32), out=b.as_strided((1, 8), (8, 1))), True, "")


def test_lazily_negated_views():
    """The memory of a view that torch negates or conjugates on reading holds other numbers: refused, but where it moves as it is."""
    z = torch.zeros(4, 9, dtype=torch.complex64)
    neg = z.conj().imag  # the imaginary part with its sign to be turned
    parent = torch.zeros(2, 2, dtype=I32)
    assert neg.is_neg() and z.conj().is_conj()
    logits = torch.zeros(8, 18).view(4, 2, 18)[:, 0, :9]
    taken(lambda: PG.beam_select(logits, torch.zeros(4), width=2), True, "")
    taken(lambda: PG.beam_select(torch._neg_view(logits), torch.zeros(4), width=2), False, "negated")
    taken(lambda: PG.beam_select(logits, torch._neg_view(torch.zeros(4)), width=2), False, "negated")
    taken(lambda: PG.prefix_attn(**attn_args(q=torch._neg_view(torch.zeros(4, 256, dtype=BF16)))), False, "negated")
    taken(lambda: PG.prefix_attn(**attn_args(out=torch._neg_view(torch.zeros(4, 256, dtype=BF16)))), False, "negated")
    taken(lambda: PG.kv_append(**append_args(cos=torch._neg_view(torch.zeros(16, 32)))), False, "negated")
    for x in (neg, z.conj()):
        taken(lambda: PG.beam_reorder(x, parent), True, "")
        taken(lambda: PG.beam_reorder(x, parent, out=torch.empty(4, 9, dtype=x.dtype)), False, "negated")
    taken(lambda: PG.beam_reorder(z.conj(), parent, out=torch.empty(4, 9, dtype=z.dtype).conj()), True, "")


def test_long_buffers_are_told_apart():
    """Many rows of a fused buffer whose other columns are the cache: the search stays short, whatever the number of rows and pages."""
    S, hkv, d = 1 << 17, 1, 64
    b = torch.empty(S, 3 * hkv * d, dtype=BF16)  # not touched
    table, lens = torch.zeros(S, 1, dtype=I32), torch.zeros(S, dtype=I32)
    for page in (1, 16, 4096):
        k, v = (b.as_strided((S // page, page, hkv, d), (page * b.stride(0), b.stride(0), d, 1), at) for at in (d, 2 * d))
        call = lambda out: PG.prefix_attn(b[:, :d], out, own=(k, v, table, lens), n_heads=1)  # noqa: E731
        taken(lambda: call(b[:, :d]), True, "")
        taken(lambda: call(b[:, 8:72]), False, "overlaps")
        taken(lambda: call(b[:, d:2 * d]), False, "overlaps a cache")
        taken(lambda: PG.kv_append(torch.zeros(S, 192, dtype=BF16), k, v, table, lens, b[:, :d], n_heads=1), True, "")
