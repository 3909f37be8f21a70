"""Sizes and numbers at which the paged decode operators (simlingo_amd/paged.py) end: refused before a launch, with the reason. Without a GPU."""
import ctypes

import pytest
import torch

from simlingo_amd import kernels as K
from simlingo_amd import paged as PG
from test_paged_cpu import append_args, attn_args

POOL = PG.KVPoolDesc(4096, 8192, 1024, 128, 64, 4, 8, 2, 64)


def answer(name, desc):
    """What the C entry says, with made-up addresses: a call that its checks let through ends at the launch, as there is no device here."""
    if torch.cuda.is_available():
        pytest.skip("made-up addresses: for machines without a GPU")
    lib = K.lib()
    rc = getattr(lib, name)(ctypes.byref(desc), None)
    return rc, lib.slx_last_error()


def launched(name, desc):
    rc, text = answer(name, desc)
    return rc < -1000 and b"launch failed" in text


def refused(name, desc, reason):
    rc, text = answer(name, desc)
    return rc == -22 and reason in text


def test_launches_of_2_to_the_32_threads():
    """A launch holds fewer than 2^32 threads: one workgroup less is launched, one more is refused and not cut off."""
    most = (1 << 24) - 1
    append = dict(pool=POOL, n_seq=1, cols=1, ldt=1, rows_per_seq=1, Hq=64, qkv=4096, ldqkv=1 << 13, table=4096, pos=4096, q_out=4096, ldq=4096)  # a row a workgroup
    assert launched("slx_kv_append", PG.KVAppendDesc(rows=most, **append))
    assert refused("slx_kv_append", PG.KVAppendDesc(rows=most + 1, **append), b"too many rows")
    select = dict(logits=4096, width=1, k=1, score=4096, score_out=4096, parent=4096, token=4096, ws=4096, ws_bytes=1 << 60)
    for vocab, rows in ((40, most), (4097, most // 2), (262144, most // 64)):
        assert launched("slx_beam_select", PG.BeamSelectDesc(batch=rows, vocab=vocab, ldx=vocab, **select))
        assert refused("slx_beam_select", PG.BeamSelectDesc(batch=rows + 1, vocab=vocab, ldx=vocab, **select), b"2^24")
        assert K.lib().slx_beam_select_ws_bytes(ctypes.byref(PG.BeamSelectDesc(batch=rows + 1, vocab=vocab, ldx=vocab, **select))) == -22
    attn = dict(own_pool=POOL, q=4096, ldq=256, out=4096, ldo=256, otab=4096, ldot=2, olen=4096, max_own=16, ocols=2, width=1, n_q=1, Hq=2, scale=1.0, ws=4096, ws_floats=1 << 60)
    assert launched("slx_prefix_attn", PG.PrefixAttnDesc(groups=most // 2, **attn))
    assert refused("slx_prefix_attn", PG.PrefixAttnDesc(groups=most // 2 + 1, **attn), b"too many rows")
    small = PG.KVPoolDesc(4096, 8192, 512, 128, 64, 4, 4, 2, 64)  # pages of 4: own keys and prefix in parts, joined 16 rows a workgroup
    join = {**attn, **dict(own_pool=small, prefix_pool=POOL, ptab=4096, ldpt=64, plen=4096, max_prefix=512, pcols=64, groups=1, width=1 << 17)}
    assert launched("slx_prefix_attn", PG.PrefixAttnDesc(**{**join, "n_q": 1023}))
    assert refused("slx_prefix_attn", PG.PrefixAttnDesc(**{**join, "n_q": 1024}), b"too many rows")
    reorder = dict(src=4096, dst=1 << 40, src_row=1, dst_row=1, n0=1, n1=1, batch=1, width=1, parent=4096)
    for size in (1, 2, 4, 16):
        r = {**reorder, "src_row": size << 33, "dst_row": size << 33}
        assert launched("slx_beam_reorder", PG.BeamReorderDesc(**{**r, "row_bytes": size * ((1 << 32) - 256 - (size < 16))}))
        assert refused("slx_beam_reorder", PG.BeamReorderDesc(**{**r, "row_bytes": size * ((1 << 32) - 255 + 2 * (size < 16))}), b"too long")


@pytest.mark.parametrize("scale,ok", ((1e-50, False), (1e-46, False), (1e-44, True), (0.125, True), (2e38, True), (2.4e38, False), (3e38, False), (1e39, False)))
def test_scales(scale, ok):
    """The scale and its product with log2(e) are held in 32 bits: one that becomes 0 or infinite there is refused."""
    with pytest.raises(RuntimeError if ok else ValueError, match="no CPU" if ok else "scale"):
        PG.prefix_attn(**attn_args(scale=scale))
    d = PG.PrefixAttnDesc(own_pool=POOL, q=4096, ldq=256, out=4096, ldo=256, otab=4096, ldot=2, olen=4096, max_own=16, ocols=2, groups=1, width=2, n_q=1, Hq=4, scale=scale)
    assert launched("slx_prefix_attn", d) if ok else refused("slx_prefix_attn", d, b"scale")
