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
