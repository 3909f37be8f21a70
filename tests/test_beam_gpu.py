"""Beam search operators (simlingo_amd/paged.py: beam_select, beam_reorder) against plain 64-bit forms (paged_ref.py)."""
import pytest
import torch

import paged_ref as R
from simlingo_amd import paged as PG

pytestmark = pytest.mark.gpu
BF16, F32, I32 = torch.bfloat16, torch.float32, torch.int32
INF, NAN = float("inf"), float("nan")


def gen(seed):
    return torch.Generator().manual_seed(seed)


def pick(dev, logits, scores, width, k, finished=None, pad=0, **kw):
    return PG.beam_select(logits.to(dev), scores.to(dev), width=width, k=k, finished=None if finished is None else finished.to(dev), pad_id=pad, **kw)


def check(dev, logits, scores, width, k, finished=None, pad=0, exact_order=False):
    R.check_select(pick(dev, logits, scores, width, k, finished, pad), R.select(logits, scores, width, k, finished, pad), exact_order)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("b,w,k,v", [(1, 1, 1, 1), (1, 1, 5, 5), (1, 4, 4, 151655), (2, 3, 6, 256), (3, 8, 16, 4097), (1, 16, 32, 8191), (2, 5, 64, 300),
                                     (1, 64, 64, 4096), (1, 2, 3, 262144), (5, 1, 2, 12289), (2, 64, 7, 65),
                                     (4, 16, 32, 66001), (8, 8, 64, 151655), (64, 8, 3, 5001),
                                     (3, 12, 25, 256), (1, 16, 32, 20011), (2, 16, 64, 70000), (1, 8, 40, 28675)])
def test_beam_select(dev, b, w, k, v, dtype):
    g = gen(b + w + k + v)
    logits = (torch.randn(b * w, v, generator=g) * 3).to(dtype)
    scores = -torch.rand(b * w, generator=g) * 6
    check(dev, logits, scores, w, k)


def test_odd_row_strides(dev):
    """Rows at any alignment of their type, with NaN between them."""
    for dtype in (F32, BF16):
        for v, ld in ((4099, 4101), (1000, 1001), (151655, 151657)):
            g = gen(v)
            logits = (torch.randn(6, v, generator=g) * 3).to(dtype)
            wide = torch.full((6, ld), NAN, dtype=dtype)
            wide[:, 1:v + 1] = logits
            scores = -torch.rand(6, generator=g)
            got = PG.beam_select(wide.to(dev)[:, 1:v + 1], scores.to(dev), width=3, k=5)
            R.check_select(got, R.select(logits, scores, 3, 5))


def test_ties_take_the_lowest(dev):
    """Equal logits, within a row, over chunks, between beams; every logit equal; +0 and -0."""
    for dtype in (F32, BF16):
        x = torch.zeros(4, 9000, dtype=dtype)
        s = torch.zeros(4)
        check(dev, x, s, 2, 30, exact_order=True)
        x[:, 8999] = 1
        x[:, 4096] = 1
        x[1, 4095] = 1
        check(dev, x, s, 4, 9, exact_order=True)
        x = torch.zeros(2, 700, dtype=dtype)
        x[:, ::2] = -0.0
        check(dev, x, s[:2], 2, 64, exact_order=True)
        g = gen(3)
        row = torch.randn(1, 20000, generator=g).to(dtype)
        check(dev, row.expand(8, -1).contiguous(), torch.full((8,), -1.25), 8, 16, exact_order=True)  # beams alike: the first ones'
        many = torch.randint(0, 3, (64, 66000), generator=g).to(dtype)  # the form with 8192 columns a workgroup
        check(dev, many, torch.zeros(64), 16, 40, exact_order=True)
        few = torch.randint(0, 3, (3, 5000), generator=g).to(dtype)
        check(dev, few, torch.zeros(3), 1, 40, exact_order=True)
        up = torch.arange(5000, dtype=F32).view(1, -1).div(64).to(dtype)  # rising: every thread's last is its largest
        check(dev, up, torch.zeros(1), 1, 64, exact_order=True)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_masked_logits(dev, dtype):
    g = gen(4)
    low = torch.finfo(dtype).min
    x = (torch.randn(6, 5000, generator=g) * 2).to(dtype)
    s = -torch.rand(6, generator=g)
    x[0] = -INF                      # nothing left: the row offers nothing
    x[1] = low                       # all at the type's lowest: all alike
    x[2, 7:] = -INF
    x[3, 100:] = low
    x[4, 11] = NAN
    x[5, 12] = INF
    check(dev, x, s, 6, 20)
    check(dev, x, s, 3, 9)           # the second entry: only rows 3 and (lost) 4, 5
    check(dev, x, s, 1, 20)          # rows that offer nothing: -inf, the lowest tokens
    x[2, :] = -INF
    x[2, 4500] = 0
    check(dev, x[2:3], s[2:3], 1, 6)  # one continuation, then -inf in the order of the tokens
    y = torch.full((2, 300), -INF, dtype=dtype)
    y[1, 250:252] = 1
    check(dev, y, s[:2], 2, 12)


def test_dead_and_finished_beams(dev):
    g = gen(5)
    x = torch.randn(12, 3001, generator=g) * 2
    s = -torch.rand(12, generator=g) * 3
    s[1] = s[2] = s[3] = -INF        # the first step: one beam alive
    s[6] = NAN
    s[5] = INF                       # as good as out
    fin = torch.zeros(12, dtype=torch.bool)
    fin[4] = fin[7] = True
    fin[8:] = True
    s[9] = -INF
    x[4] = NAN                       # an ended row's logits are not looked at
    for pad in (0, 5, 3000):
        check(dev, x, s, 4, 4, fin, pad)
        check(dev, x, s, 4, 9, fin, pad)
    check(dev, x, s, 4, 8, fin.to(torch.uint8), 2)
    s[:] = -INF
    check(dev, x, s, 4, 6)
    check(dev, x[:, :2].contiguous(), torch.zeros(12), 4, 8, fin, 1)  # fewer continuations than asked for, -inf in order


def test_many_batch_entries(dev):
    g = gen(9)
    x, s = torch.randn(70000, 40, generator=g), -torch.rand(70000, generator=g)
    check(dev, x, s, 1, 2)


def test_tensors_elsewhere(dev):
    x, s = torch.randn(4, 40), torch.zeros(4)
    with pytest.raises(RuntimeError, match="tensors on"):
        PG.beam_select(x.to(dev), s, width=2)
    with pytest.raises(RuntimeError, match="tensors on"):
        PG.beam_reorder(x.to(dev), torch.zeros(2, 2, dtype=I32))
    with pytest.raises(TypeError, match="must be a tensor"):
        PG.beam_select(x.to(dev), 0.0, width=2)


def test_in_place_and_finished_out(dev):
    g = gen(6)
    x, s = torch.randn(8, 500, generator=g), -torch.rand(8, generator=g)
    fin = torch.tensor([0, 0, 1, 0, 0, 0, 0, 1], dtype=torch.bool)
    ws, wp, wt = R.select(x, s, 4, 4, fin, 9)
    eos = int(wt[0, 1])
    ds, df = s.to(dev), fin.to(dev)
    out = (ds, torch.empty(2, 4, dtype=I32, device=dev), torch.empty(2, 4, dtype=I32, device=dev))
    PG.beam_select(x.to(dev), ds, width=4, finished=df, pad_id=9, eos_id=eos, out=out, finished_out=df)
    R.check_select((ds.view(2, 4), out[1], out[2]), (ws, wp, wt))
    want = torch.gather(fin.view(2, 4), 1, wp) | (wt == eos)
    assert torch.equal(df.cpu().view(2, 4), want)


REORDER = [  # shape, dim, batch, width, dtype
    ((8, 101), 0, 2, 4, I32), ((4, 6, 33), 1, 3, 2, BF16), ((3, 2, 5, 7, 64), 1, 1, 2, BF16), ((64, 40), 0, 1, 64, F32), ((17, 9), 0, 1, 17, torch.uint8),
    ((10,), 0, 2, 5, torch.int64), ((2, 3, 30, 9), 2, 5, 6, torch.float64), ((33, 16), 0, 1, 33, F32), ((5, 1), 0, 5, 1, BF16),
]


@pytest.mark.parametrize("shape,dim,b,w,dtype", REORDER)
def test_beam_reorder(dev, shape, dim, b, w, dtype):
    g = gen(sum(shape))
    x = torch.randint(0, 250, shape, generator=g).to(dtype)
    parent = torch.randint(0, w, (b, w), generator=g).to(I32)
    rows = (parent.long() + torch.arange(b)[:, None] * w).view(-1)
    want = x.index_select(dim, rows)
    dx, dp = x.to(dev), parent.to(dev)
    assert torch.equal(PG.beam_reorder(dx, dp, dim=dim, out=torch.empty_like(dx)).cpu(), want) and torch.equal(dx.cpu(), x)
    got = PG.beam_reorder(dx, dp, dim=dim - len(shape))
    assert got is dx and torch.equal(dx.cpu(), want)


def test_beam_reorder_slices(dev):
    """The used part of a dense cache [layers, sequences, heads, slots, d], and odd columns of a table."""
    g = gen(7)
    x = torch.randn(3, 6, 2, 20, 8, generator=g).to(BF16)
    parent = torch.tensor([[2, 2, 0], [1, 0, 1]], dtype=I32)
    rows = torch.tensor([2, 2, 0, 4, 3, 4])
    dx = x.to(dev)
    PG.beam_reorder(dx[:, :, :, :13], parent.to(dev), dim=1)
    want = x.clone()
    want[:, :, :, :13] = x[:, rows, :, :13]
    assert torch.equal(dx.cpu(), want)
    t = torch.arange(6 * 33, dtype=I32).view(6, 33)
    dt, to = t.to(dev), torch.zeros(6, 33, dtype=I32, device=dev)
    PG.beam_reorder(dt[:, 1:8], parent.to(dev), out=to[:, 3:10])
    assert torch.equal(to.cpu()[:, 3:10], t[rows][:, 1:8]) and not to[:, :3].any() and not to[:, 10:].any()
    PG.beam_reorder(dt[:, ::2], parent.to(dev))
    want = t.clone()
    want[:, ::2] = t[rows][:, ::2]
    assert torch.equal(dt.cpu(), want)
    PG.beam_reorder(dt[:, :0], parent.to(dev))


def test_beam_reorder_bad_parents(dev):
    x = torch.arange(24, dtype=F32).view(4, 6)
    parent = torch.tensor([[-1, 4, 2**31 - 1, 0]], dtype=I32)
    want = x[[0, 1, 2, 0]]
    assert torch.equal(PG.beam_reorder(x.to(dev), parent.to(dev), out=torch.empty(4, 6, device=dev)).cpu(), want)
    assert torch.equal(PG.beam_reorder(x.to(dev), parent.to(dev)).cpu(), want)


def test_many_outer_rows(dev):
    """More outer rows than a grid's second axis has workgroups."""
    x = torch.randint(0, 100, (70000, 2), dtype=I32)
    parent = torch.tensor([[1, 0]], dtype=I32)
    assert torch.equal(PG.beam_reorder(x.to(dev), parent.to(dev), dim=1).cpu(), x.flip(1))


def test_beam_graph(dev):
    """Select, then reorder the table, captured and replayed over changing logits."""
    g = gen(8)
    x, s = torch.randn(8, 6000, generator=g).to(dev), torch.zeros(8, device=dev)
    out = (torch.empty(2, 4, device=dev), torch.empty(2, 4, dtype=I32, device=dev), torch.empty(2, 4, dtype=I32, device=dev))
    table = torch.arange(8 * 50, dtype=I32, device=dev).view(8, 50)

    def step():
        PG.beam_select(x, s, width=4, out=out)
        PG.beam_reorder(table, out[1])

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    torch.cuda.synchronize()
    for i in range(4):
        x.copy_(torch.randn(8, 6000, generator=g))
        s.copy_(-torch.rand(8, generator=g))
        table.copy_(torch.randint(0, 1000, (8, 50), generator=g, dtype=I32))
        before = table.cpu().clone()
        graph.replay()
        torch.cuda.synchronize()
        want = R.select(x.cpu(), s.cpu(), 4, 4)
        R.check_select(out, want)
        rows = (out[1].cpu().long() + torch.tensor([[0], [4]])).view(-1)
        assert torch.equal(table.cpu(), before[rows])
        torch.randn(1000, device=dev).sum().item()


def test_widest_in_a_graph(dev):
    """64 rows, 64 chosen, which takes the most shared memory: captured, and replayed between eager calls."""
    g = gen(11)
    x, s = torch.randn(64, 5000, generator=g).to(dev), torch.zeros(64, device=dev)
    out = (torch.empty(1, 64, device=dev), torch.empty(1, 64, dtype=I32, device=dev), torch.empty(1, 64, dtype=I32, device=dev))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        PG.beam_select(x, s, width=64, out=out)
    for i in range(3):
        x.copy_(torch.randn(64, 5000, generator=g))
        s.copy_(-torch.rand(64, generator=g))
        graph.replay()
        R.check_select(out, R.select(x.cpu(), s.cpu(), 64, 64))
        for a, b in zip(PG.beam_select(x, s, width=64), out):
            assert torch.equal(a, b)
