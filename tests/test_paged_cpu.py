"""Refusals of the paged decode operators (simlingo_amd/paged.py) and of their C entries, without a GPU: every bad call ends in
an error before a launch. The plain 64-bit forms (paged_ref.py) are checked against each other's definitions here too."""
import ctypes
import os
import shutil
import subprocess

import pytest
import torch

import paged_ref as R
from simlingo_amd import kernels as K
from simlingo_amd import paged as PG

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BF16, F32, I32 = torch.bfloat16, torch.float32, torch.int32


def pool(n=4, page=8, heads=2, d=64, dtype=BF16):
    return torch.zeros(n, page, heads, d, dtype=dtype), torch.zeros(n, page, heads, d, dtype=dtype)


def append_args(**kw):
    k, v = pool()
    a = dict(qkv=torch.zeros(3, 8 * 64, dtype=BF16), k=k, v=v, table=torch.zeros(2, 2, dtype=I32), pos=torch.zeros(3, dtype=I32),
             q_out=torch.zeros(3, 4 * 64, dtype=BF16), n_heads=4, cos=torch.zeros(16, 32), sin=torch.zeros(16, 32), seq=torch.zeros(3, dtype=I32))
    a.update(kw)
    return a


def test_good_calls_stop_at_the_device_only():
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        PG.kv_append(**append_args())
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        PG.prefix_attn(**attn_args())
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        PG.beam_select(torch.zeros(4, 9), torch.zeros(4), width=2)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        PG.beam_reorder(torch.zeros(4, 9), torch.zeros(2, 2, dtype=I32))


@pytest.mark.parametrize("kw", [
    dict(qkv=torch.zeros(3, 8 * 64)), dict(qkv=torch.zeros(3, 7 * 64, dtype=BF16)), dict(qkv=torch.zeros(3, 8 * 64 + 4, dtype=BF16)[:, :512]),
    dict(qkv=torch.zeros(3, 8 * 64 + 8, dtype=BF16)[:, 1:513]), dict(k=pool()[0][:, :, :, ::2]), dict(k=pool(dtype=F32)[0]), dict(k=pool(n=5)[0]),
    dict(zip("kv", pool(page=6))), dict(zip("kv", pool(d=96))), dict(zip("kv", pool(d=32))), dict(zip("kv", pool(n=0))),
    dict(k=torch.zeros(1, 8, 2, 64, dtype=BF16).expand(4, -1, -1, -1), v=torch.zeros(1, 8, 2, 64, dtype=BF16).expand(4, -1, -1, -1)),
    dict(table=torch.zeros(2, 2)), dict(table=torch.zeros(2, 0, dtype=I32)), dict(table=torch.zeros(0, 2, dtype=I32)), dict(table=torch.zeros(2, 4, dtype=I32)[:, ::2]),
    dict(pos=torch.zeros(2, dtype=I32)), dict(pos=torch.zeros(3, dtype=torch.int64)), dict(seq=torch.zeros(6, dtype=I32)[::2]),
    dict(q_out=torch.zeros(2, 256, dtype=BF16)), dict(q_out=torch.zeros(3, 192, dtype=BF16)), dict(n_heads=0), dict(n_heads=-1), dict(sin=None),
    dict(cos=torch.zeros(16, 32, dtype=BF16)), dict(cos=torch.zeros(15, 32)), dict(rows_per_seq=0),
], ids=lambda kw: "-".join(kw))
def test_kv_append_refuses(kw):
    with pytest.raises(ValueError, match="kv_append"):
        PG.kv_append(**append_args(**kw))


def attn_args(**kw):
    own, prefix = (*pool(), torch.zeros(4, 3, dtype=I32), torch.zeros(4, dtype=I32)), (*pool(page=16), torch.zeros(2, 3, dtype=I32), torch.zeros(2, dtype=I32))
    a = dict(q=torch.zeros(4, 4 * 64, dtype=BF16), own=own, prefix=prefix, n_heads=4)
    for name, t in kw.pop("own", {}).items():
        a["own"] = tuple(t if i == int(name[1]) else x for i, x in enumerate(a["own"]))
    for name, t in kw.pop("prefix", {}).items():
        a["prefix"] = tuple(t if i == int(name[1]) else x for i, x in enumerate(a["prefix"]))
    a.update(kw)
    return a


@pytest.mark.parametrize("kw", [
    dict(q=torch.zeros(3, 256, dtype=BF16)), dict(q=torch.zeros(4, 256)), dict(q=torch.zeros(4, 128, dtype=BF16)), dict(n_heads=3), dict(n_heads=0), dict(n_q=0), dict(n_q=2),
    dict(own=dict(_2=torch.zeros(4, 3))), dict(own=dict(_2=torch.zeros(4, 0, dtype=I32))), dict(own=dict(_3=torch.zeros(3, dtype=I32))), dict(own=dict(_0=pool(n=3)[0])),
    dict(prefix=dict(_2=torch.zeros(3, 3, dtype=I32), _3=torch.zeros(3, dtype=I32))), dict(prefix=dict(_3=torch.zeros(2, dtype=torch.int64))),
    dict(prefix=dict(_0=pool(heads=1)[0], _1=pool(heads=1)[1])), dict(prefix=dict(_0=pool(d=128)[0], _1=pool(d=128)[1])),
    dict(max_own=-1), dict(max_prefix=-1), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(out=torch.zeros(4, 192, dtype=BF16)), dict(out=torch.zeros(5, 256, dtype=BF16)), dict(lse=torch.zeros(4, 3)),
], ids=lambda kw: "-".join(kw))
def test_prefix_attn_refuses(kw):
    with pytest.raises(ValueError, match="prefix_attn"):
        PG.prefix_attn(**attn_args(**kw))


@pytest.mark.parametrize("kw", [
    dict(width=0), dict(width=65), dict(width=3), dict(k=0), dict(k=65), dict(logits=torch.zeros(4, 9, dtype=torch.float16)), dict(logits=torch.zeros(4, 18)[:, ::2]),
    dict(logits=torch.zeros(4, 0)), dict(logits=torch.zeros(4, 262145, dtype=BF16)), dict(logits=torch.zeros(4, 1), k=3), dict(scores=torch.zeros(3)), dict(scores=torch.zeros(4, dtype=BF16)),
    dict(finished=torch.zeros(4)), dict(finished=torch.zeros(3, dtype=torch.bool)), dict(finished=torch.zeros(4, dtype=torch.bool), pad_id=9),
    dict(finished=torch.zeros(4, dtype=torch.bool), pad_id=-1), dict(finished_out=torch.zeros(3, dtype=torch.bool)), dict(out=(torch.zeros(2, 2), torch.zeros(2, 2), torch.zeros(2, 2))),
    dict(k=4, inplace=True),
], ids=lambda kw: "-".join(kw))
def test_beam_select_refuses(kw):
    a = dict(logits=torch.zeros(4, 9), scores=torch.zeros(4), width=2)
    if kw.pop("inplace", False):
        a["scores"] = torch.zeros(8)[:4]
        a["out"] = (a["scores"].as_strided((2, 4), (4, 1)), torch.zeros(2, 4, dtype=I32), torch.zeros(2, 4, dtype=I32))
    a.update(kw)
    with pytest.raises(ValueError, match="beam_select"):
        PG.beam_select(**a)


@pytest.mark.parametrize("x,parent,kw", [
    (torch.zeros(4, 3), torch.zeros(2, 2), {}), (torch.zeros(4, 3), torch.zeros(4, dtype=I32), {}), (torch.zeros(5, 3), torch.zeros(2, 2, dtype=I32), {}),
    (torch.zeros(4, 3), torch.zeros(2, 2, dtype=I32), dict(dim=2)), (torch.zeros(4, 3), torch.zeros(2, 2, dtype=I32), dict(out=torch.zeros(4, 2))),
    (torch.zeros(4, 3), torch.zeros(2, 2, dtype=I32), dict(out=torch.zeros(4, 3, dtype=BF16))), (torch.zeros(65, 3), torch.zeros(1, 65, dtype=I32), {}),
    (torch.zeros(2, 4, 5, 6, 7)[:, :, ::2, ::2, ::2], torch.zeros(2, 2, dtype=I32), dict(dim=1)), (torch.zeros(1, 3).expand(4, 3), torch.zeros(2, 2, dtype=I32), {}),
    (torch.zeros(4, 1).expand(4, 3), torch.zeros(2, 2, dtype=I32), {}),
])
def test_beam_reorder_refuses(x, parent, kw):
    with pytest.raises(ValueError, match="beam_reorder"):
        PG.beam_reorder(x, parent, **kw)


def test_writing_over_what_is_read():
    """Outputs in the place of the queries, or in other columns of their rows, are taken; anything else that overlaps is not."""
    buf = torch.zeros(6, 1024, dtype=BF16)
    for q_out, ok in ((buf[:3, :256], True), (buf[:3, 512:768], True), (buf[3:, :256], True), (buf[:3, 64:320], False), (buf[1:4, :256], False), (buf[:3, 256:512], False)):
        with pytest.raises(RuntimeError if ok else ValueError, match="no CPU" if ok else "overlaps qkv"):
            PG.kv_append(**append_args(qkv=buf[:3, :512], q_out=q_out))
    for out, ok in ((buf[:4, :256], True), (buf[:4, 256:512], True), (buf[1:5, :256], False), (buf[:4, 128:384], False)):
        with pytest.raises(RuntimeError if ok else ValueError, match="no CPU" if ok else "overlaps q"):
            PG.prefix_attn(**attn_args(q=buf[:4, :256], out=out))
    k = pool()[0]
    with pytest.raises(ValueError, match="same memory"):
        PG.kv_append(**append_args(k=k, v=k))
    with pytest.raises(ValueError, match="lse overlaps"):
        PG.prefix_attn(**attn_args(q=buf[:4, :256], lse=buf.view(-1)[512:].view(torch.float32)[:16].view(4, 4)))


@pytest.mark.parametrize("at,k,ok", (((0, 100, 200, 300), 4, True), ((400, 100, 200, 500), 4, True), ((404, 100, 200, 300), 4, False), ((0, 100, 200, 502), 4, False),
                                     ((400, 100, 200, 300), 2, False), ((0, 100, 200, 500), 2, False), ((0, 400, 200, 300), 4, False), ((0, 16, 200, 300), 4, False),
                                     ((0, 32, 64, 96), 4, True), ((0, 32, 64, 92), 4, False)))
def test_select_outputs_apart(at, k, ok):
    """scores at byte 400 (8 of 4 B), finished at 500 (8 of 1 B); outputs of 2 x k at the bytes given."""
    b = torch.zeros(512, dtype=torch.uint8)
    v = lambda o, t: b[o:o + 2 * k * t.itemsize].view(t).view(2, k)
    out, fout = (v(at[0], torch.float32), v(at[1], torch.int32), v(at[2], torch.int32)), v(at[3], torch.uint8)
    with pytest.raises(RuntimeError if ok else ValueError, match="no CPU" if ok else "overlap|in place"):
        PG.beam_select(torch.zeros(8, 9), b[400:432].view(torch.float32), width=4, k=k, finished=b[500:508], out=out, finished_out=fout)


def test_beam_reorder_refuses_overlap():
    x = torch.zeros(6, 4)
    with pytest.raises(ValueError, match="overlaps"):
        PG.beam_reorder(x[:4], torch.zeros(2, 2, dtype=I32), out=x[2:])


def test_c_entries_refuse():
    """The C entries check what they are given themselves: -22 and a message, nothing launched."""
    lib = K.lib()

    def refused(name, desc, text):
        assert getattr(lib, name)(ctypes.byref(desc) if desc is not None else None, None) == -22
        assert text in lib.slx_last_error(), lib.slx_last_error()

    good = PG.KVPoolDesc(4096, 8192, 1024, 128, 64, 4, 8, 2, 64)
    for field, value, text in (("k", 4104, b"16-B aligned"), ("v", 0, b"16-B aligned"), ("head_dim", 96, b"head_dim"), ("page", 6, b"power of two"), ("n_pages", 0, b"n_pages"),
                               ("page", 0, b"power of two"), ("page", -8, b"power of two"), ("slot_stride", 12, b"multiples of 8"), ("page_stride", -8, b"multiples of 8")):
        bad = PG.KVPoolDesc.from_buffer_copy(good)
        setattr(bad, field, value)
        refused("slx_kv_append", PG.KVAppendDesc(pool=bad, rows=1, n_seq=1, cols=1, ldt=1, rows_per_seq=1), text)
        refused("slx_prefix_attn", PG.PrefixAttnDesc(own_pool=bad, groups=1, width=1, n_q=1, Hq=2, ocols=1, ldot=1), text)
    ap = dict(pool=good, rows=1, n_seq=1, cols=1, ldt=1, rows_per_seq=1, Hq=4, qkv=4096, ldqkv=512, table=4096, pos=4096)
    for kw, text in ((dict(rows=-1), b"rows"), (dict(cols=2), b"ldt"), (dict(rows_per_seq=0), b"rows_per_seq"), (dict(cos_tab=4096), b"go together"), (dict(qkv=0), b"null"),
                     (dict(qkv=4098), b"16-B"), (dict(ldqkv=516), b"16-B"), (dict(pos=0), b"null")):
        refused("slx_kv_append", PG.KVAppendDesc(**{**ap, **kw}), text)
    refused("slx_kv_append", None, b"null")
    assert lib.slx_kv_append(ctypes.byref(PG.KVAppendDesc(**{**ap, "rows": 0})), None) == 0
    at = dict(own_pool=good, q=4096, ldq=256, out=4096, ldo=256, otab=4096, ldot=2, olen=4096, max_own=16, ocols=2, groups=1, width=2, n_q=1, Hq=4, scale=1.0)
    pre = dict(prefix_pool=good, ptab=4096, ldpt=64, plen=4096, max_prefix=512, pcols=64)
    for kw, text in ((dict(Hq=3), b"multiple"), (dict(width=0), b"width"), (dict(n_q=0), b"n_q"), (dict(ocols=3), b"ocols"), (dict(max_own=-1), b"max_own"), (dict(q=0), b"null"),
                     (dict(q=4104), b"16-B"), (dict(ldo=12), b"16-B"), ({**pre, "plen": 0}, b"plen"), ({**pre, "ldpt": 3}, b"pcols"), (pre, b"workspace"),
                     (dict(groups=1 << 20, width=1 << 10, n_q=4), b"too many"), (dict(scale=0.0), b"scale"), (dict(Hq=1 << 14, width=64), b"too many")):
        refused("slx_prefix_attn", PG.PrefixAttnDesc(**{**at, **kw}), text)
    other = PG.KVPoolDesc.from_buffer_copy(good)
    other.heads = 1
    refused("slx_prefix_attn", PG.PrefixAttnDesc(**{**at, **pre, "prefix_pool": other}), b"differ")
    d = PG.PrefixAttnDesc(**{**at, **pre})
    need = lib.slx_prefix_attn_ws_floats(ctypes.byref(d))
    assert need > 0 and need % (2 * 4 * 66) == 0
    d.max_own, d.ocols = (1 << 30) + 1, 1 << 30
    d.ldot = d.ocols
    refused("slx_prefix_attn", d, b"2^30")
    assert lib.slx_prefix_attn_ws_floats(ctypes.byref(d)) < 0
    d.max_own, d.ocols, d.ldot = 16, 2, 2
    d.ws, d.ws_floats = 4096, need - 1
    refused("slx_prefix_attn", d, b"workspace")
    refused("slx_prefix_attn", None, b"null")
    se = dict(logits=4096, ldx=9, batch=1, width=2, vocab=9, k=2, score=4096, score_out=4096, parent=4096, token=4096, ws=4096, ws_bytes=1 << 20)
    for kw, text in ((dict(width=65), b"width"), (dict(batch=1 << 25), b"batch"), (dict(vocab=262145, ldx=262145), b"vocab"), (dict(k=65), b"k <="), (dict(k=19), b"k <="), (dict(ldx=8), b"ldx"),
                     (dict(finished=4096, pad=9), b"pad"), (dict(token=0), b"null"), (dict(ws=0), b"workspace"), (dict(ws_bytes=16), b"workspace"), (dict(ws=4100), b"workspace")):
        refused("slx_beam_select", PG.BeamSelectDesc(**{**se, **kw}), text)
    refused("slx_beam_select", None, b"null")
    assert lib.slx_beam_select(ctypes.byref(PG.BeamSelectDesc(**{**se, "batch": 0})), None) == 0
    re_ = dict(src=4096, dst=4096, src_row=64, dst_row=64, row_bytes=64, n0=1, n1=1, batch=1, width=2, parent=4096)
    for kw, text in ((dict(width=0), b"width"), (dict(width=65), b"width"), (dict(batch=-1), b"extents"), (dict(row_bytes=-4), b"extents"), (dict(parent=0), b"null"),
                     (dict(dst_row=128), b"equal strides"), (dict(n0=1 << 16, n1=1 << 15), b"2^31")):
        refused("slx_beam_reorder", PG.BeamReorderDesc(**{**re_, **kw}), text)
    refused("slx_beam_reorder", None, b"null")


def test_struct_layouts_match_header(tmp_path):
    if shutil.which("gcc") is None:
        pytest.skip("gcc not available")
    structs = {"slx_kv_pool": PG.KVPoolDesc, "slx_kv_append_desc": PG.KVAppendDesc, "slx_prefix_attn_desc": PG.PrefixAttnDesc,
               "slx_beam_select_desc": PG.BeamSelectDesc, "slx_beam_reorder_desc": PG.BeamReorderDesc}
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "slx.h"', "int main(void){"]
    for name, cls in structs.items():
        lines.append(f'printf("{name} size %zu\\n", sizeof({name}));')
        lines += [f'printf("{name} {f[0]} %zu\\n", offsetof({name}, {f[0]}));' for f in cls._fields_]
    src, exe = tmp_path / "probe.c", tmp_path / "probe"
    src.write_text("\n".join(lines + ["return 0;}"]))
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    for line in filter(None, subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split("\n")):
        name, field, val = line.split()
        assert int(val) == (ctypes.sizeof(structs[name]) if field == "size" else getattr(structs[name], field).offset), line


def test_reference_forms():
    """The 64-bit attention equals a softmax over the joined keys; select equals a sort of all scores."""
    g = torch.Generator().manual_seed(0)
    k, v = (torch.randn(3, 4, 1, 64, generator=g).to(BF16) for _ in range(2))
    q = torch.randn(2, 128, generator=g).to(BF16)
    own = (k, v, torch.tensor([[2, 0]], dtype=I32), torch.tensor([6], dtype=I32))
    out, lse, _ = R.attn(q, own, (k, v, torch.tensor([[1]], dtype=I32), torch.tensor([3], dtype=I32)), 2, 2)
    keys = torch.cat([k[1, :3, 0], k[2, :, 0], k[0, :2, 0]]).double()
    vals = torch.cat([v[1, :3, 0], v[2, :, 0], v[0, :2, 0]]).double()
    for t in range(2):
        for h in range(2):
            s = keys[:8 + t] @ q[t].double()[h * 64:h * 64 + 64] / 8
            assert torch.allclose(out[t, h * 64:h * 64 + 64], torch.softmax(s, 0) @ vals[:8 + t])
            assert torch.allclose(lse[t, h], torch.logsumexp(s, 0))
    x = torch.tensor([[1.0, 3.0, 3.0], [float("-inf")] * 3])
    s, p, t = R.select(x, torch.zeros(2), 2, 5)
    assert p.tolist() == [[0, 0, 0, 1, 1]] and t.tolist() == [[1, 2, 0, 0, 1]] and torch.isinf(s[0, 3:]).all()
