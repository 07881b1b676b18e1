"""Embedding lookup and its gradient by sorted tokens.

A lookup is one product in fp32 and one rounding.  A gradient row is a sum of n rows in fp32 in some fixed order, off by at most
n 2^-24 sum |terms|, then a product and a rounding to the table's type."""

import pytest
import torch

from torchure_b200 import ops
from torchure_b200.ops import debug, kernels
from torchure_b200.ops.embedding import embedding

GPU = pytest.param("cuda", marks=pytest.mark.gpu)
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float64: 2.0 ** -53}


@pytest.fixture(autouse=True)
def _check_kernel_errors():
    yield
    if torch.cuda.is_available():
        kernels.check_error()


def problem(T, V, D, table_type=torch.float32, hot=0.0, seed=0, ids_type=torch.int64):
    g = torch.Generator().manual_seed(seed)
    ids = torch.randint(0, V, (T,), generator=g)
    ids = torch.where(torch.rand(T, generator=g) < hot, torch.full_like(ids, V // 3), ids).to(ids_type)
    return ids, torch.randn(V, D, generator=g).to(table_type)


def check(ids, table, dout, out, dtable, scale, padding=None):
    """Against the definition in 64 bits, element by element."""
    ids, table, dout = ids.cpu().long().reshape(-1), table.detach().cpu().double(), dout.cpu().double()
    want = table[ids] * scale
    got = out.detach().cpu().double().reshape(want.shape)
    assert ((got - want).abs() <= want.abs() * (HALF[out.dtype] + 2.0 ** -24)).all()
    keep = torch.ones_like(ids, dtype=torch.bool) if padding is None else ids != padding
    rows = dout.reshape(-1, table.shape[1])[keep]
    total = torch.zeros_like(table).index_add_(0, ids[keep], rows) * scale
    size = torch.zeros_like(table).index_add_(0, ids[keep], rows.abs()) * abs(scale)
    n = torch.bincount(ids[keep], minlength=table.shape[0])[:, None].double()
    bound = size * n * 2.0 ** -24 + total.abs() * (HALF[dtable.dtype] + 2.0 ** -23) + 1e-40
    assert ((dtable.detach().cpu().double() - total).abs() <= bound).all()


CASES = [      # T, V, D, table, rows, hot, scale
    (1, 1, 1, torch.float32, torch.float32, 0.0, 1.0),
    (1, 50, 8, torch.bfloat16, torch.float32, 0.0, 2.0),
    (2, 2, 4, torch.float32, torch.bfloat16, 1.0, 1.0),
    (15, 700, 33, torch.bfloat16, torch.bfloat16, 0.5, 0.3),
    (17, 3, 12, torch.float32, torch.float32, 0.0, -1.5),
    (33, 511, 64, torch.float32, torch.float32, 0.2, 1.0),
    (1000, 512, 100, torch.float32, torch.bfloat16, 0.1, 1.0),
    (1025, 513, 260, torch.bfloat16, torch.bfloat16, 0.9, 22.6),
    (2500, 40000, 36, torch.float32, torch.float32, 0.3, 1.0),
    (5000, 7, 1000, torch.float32, torch.float32, 0.0, 1.0),
    (4096, 262143, 8, torch.float32, torch.float32, 0.1, 1.0),          # 18 bits of key with the one behind the table
    (3000, 262144, 8, torch.float32, torch.bfloat16, 0.1, 1.0),         # 19: three digits
    (20011, 1500, 1031, torch.bfloat16, torch.bfloat16, 0.6, 1.0),
    (70001, 9, 5, torch.float32, torch.float32, 0.5, 1.0),
    (160000, 1, 3, torch.float32, torch.float32, 0.0, 1.0),             # one row takes all
]


@pytest.mark.parametrize("device", ["cpu", GPU])
@pytest.mark.parametrize("T, V, D, table_type, out_type, hot, scale", CASES)
def test_against_the_definition(device, T, V, D, table_type, out_type, hot, scale):
    ids, table = problem(T, V, D, table_type, hot, seed=T)
    w = table.to(device, copy=True).requires_grad_()
    out = embedding(ids.to(device), w, scale, out_dtype=out_type)
    dout = torch.randn(T, D, generator=torch.Generator().manual_seed(1)).to(out_type)
    dtable, = torch.autograd.grad(out, w, dout.to(device))
    assert out.dtype == out_type and out.shape == (T, D) and dtable.dtype == table_type and dtable.shape == (V, D)
    check(ids, table, dout, out, dtable, scale)


@pytest.mark.parametrize("device", ["cpu", GPU])
@pytest.mark.parametrize("ids_type", [torch.int64, torch.int32])
@pytest.mark.parametrize("padding", [0, -1, 17])
def test_padding_shapes_and_strides(device, ids_type, padding):
    ids, table = problem(600, 64, 24, hot=0.4, ids_type=ids_type, seed=2)
    ids = ids.view(20, 30)
    room = torch.randn(64, 40, generator=torch.Generator().manual_seed(5)).to(device)
    room[:, 3:27] = table.to(device)
    wide = room.clone().requires_grad_()
    out = embedding(ids.to(device).t(), wide[:, 3:27], 1.5, padding)          # ids in columns, rows 40 apart
    assert out.shape == (30, 20, 24)
    big = torch.randn(30, 20, 48, generator=torch.Generator().manual_seed(3)).to(device)
    dwide, = torch.autograd.grad(out, wide, big[..., ::2])                    # a gradient with gaps
    assert (dwide[:, :3] == 0).all() and (dwide[:, 27:] == 0).all() and (dwide[padding] == 0).all()
    check(ids.t(), table, big[..., ::2], out, dwide[:, 3:27], 1.5, padding % 64)


@pytest.mark.parametrize("device", ["cpu", GPU])
def test_nothing_to_look_up(device):
    for shape, V, D in (((0,), 5, 8), ((3, 0), 5, 8), ((4,), 5, 0)):
        w = torch.randn(V, D, device=device, requires_grad=True)
        ids = torch.zeros(shape, dtype=torch.int64, device=device)
        out = embedding(ids, w)
        assert out.shape == (*shape, D)
        d, = torch.autograd.grad(out, w, torch.ones_like(out))
        assert d.shape == (V, D) and (d == 0).all()


@pytest.mark.parametrize("device", ["cpu", GPU])
def test_refusals(device):
    ids, w = torch.zeros(3, dtype=torch.int64, device=device), torch.randn(5, 8, device=device)
    for bad in (lambda: embedding(ids.to(torch.int16), w), lambda: embedding(ids, w.half()) if device == "cuda" else embedding(ids.float(), w),
                lambda: embedding(ids, w[0]), lambda: embedding(ids, w[:0]), lambda: embedding(ids, w, padding_idx=5),
                lambda: embedding(ids, w, padding_idx=-6), lambda: embedding(ids, w, float("nan")), lambda: embedding(ids, w, out_dtype=torch.half)):
        with pytest.raises((ValueError, TypeError)):
            bad()


def test_ids_outside_the_table_on_the_cpu():
    for ids in ([0, 5], [-1, 0]):
        with pytest.raises(IndexError):
            embedding(torch.tensor(ids), torch.randn(5, 8))


@pytest.mark.parametrize("device", ["cpu", GPU])
@pytest.mark.parametrize("D", [1, 7, 8, 33])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_broadcast_rows_and_gradients(device, D, dtype):
    """One row expanded to a table, and gradients that are one row, or one number, for all tokens."""
    ids, table = problem(70, 12, D, dtype, seed=3)
    row = table[:1].to(device, copy=True).requires_grad_()
    wide = row.expand(12, D)
    one = torch.randn(D, generator=torch.Generator().manual_seed(4)).to(dtype)
    for dout in (one.expand(70, D), one[:1].expand(70, D)):
        out = embedding(ids.to(device), wide, 2.0)
        w = table.to(device, copy=True).requires_grad_()
        full = embedding(ids.to(device), w, 2.0)
        dtable, = torch.autograd.grad(full, w, dout.to(device))
        check(ids, table, dout, full, dtable, 2.0)
        check(ids, table[:1].expand(12, D), dout, out, dtable, 2.0)
        drow, = torch.autograd.grad(out, row, dout.to(device))
        assert drow.shape == (1, D)
    # (strides that a reshape keeps)
    assert torch.equal(embedding(ids.to(device)[:0], wide), wide[:0])


@pytest.mark.gpu
def test_operands_on_one_gpu():
    with pytest.raises(ValueError):
        embedding(torch.zeros(3, dtype=torch.int64), torch.randn(5, 8, device="cuda"))
    with pytest.raises(ValueError):
        embedding(torch.zeros(3, dtype=torch.int64, device="cuda"), torch.randn(5, 8))


@pytest.mark.gpu
def test_ids_outside_the_table():
    """Rows of NaN that no loss can miss, and no gradient; the rest is as without them."""
    ids, table = problem(300, 40, 36, seed=6)
    ids[::7], ids[3::50], ids[5::60] = -1, 40, 2 ** 40
    w = table.cuda().requires_grad_()
    out = embedding(ids.cuda(), w)
    bad = (ids < 0) | (ids >= 40)
    assert torch.isnan(out[bad.cuda()]).all()
    dout = torch.randn(300, 36, generator=torch.Generator().manual_seed(1))
    d, = torch.autograd.grad(out, w, dout.cuda())
    check(ids[~bad], table, dout[~bad], out[~bad.cuda()], d, 1.0)


@pytest.mark.gpu
def test_same_bits_every_time_and_next_to_other_work():
    """No order of arrival decides a sum: repeated, on another stream beside itself, and captured."""
    ids, table = problem(30000, 5000, 520, torch.bfloat16, hot=0.3, seed=7)
    ids, w = ids.cuda(), table.cuda().requires_grad_()
    dout = torch.randn(30000, 520, device="cuda", dtype=torch.bfloat16)

    def both():
        out = embedding(ids, w, 2.0, 11)
        return out.detach(), torch.autograd.grad(out, w, dout)[0]

    first = both()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        there = [both() for _ in range(3)]
    here = [both() for _ in range(3)]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for run in here + there for a, b in zip(run, first))
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = both()
        graphs.append((graph, got))
    ids.copy_(problem(30000, 5000, 520, hot=0.6, seed=8)[0].cuda())
    want = both()
    for graph, got in graphs:
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for _, got in graphs for a, b in zip(got, want))


@pytest.mark.gpu
def test_every_row_is_written():
    debug.enable()
    try:
        for T, V, D in ((3, 1000, 64), (5000, 3001, 77)):
            ids, table = problem(T, V, D, seed=9)
            w = table.cuda().requires_grad_()
            out = embedding(ids.cuda(), w)
            torch.autograd.grad(out, w, torch.ones_like(out))
            assert debug.verify() == 2
    finally:
        debug.enable(False)


@pytest.mark.gpu
def test_gradient_against_a_difference():
    """The loss is linear in the table: a difference along the gradient is its square, but for the roundings of the lookups."""
    ids, table = problem(900, 200, 128, hot=0.2, seed=10)
    w = table.cuda().requires_grad_()
    dout = torch.randn(900, 128, device="cuda", generator=torch.Generator(device="cuda").manual_seed(0))
    d, = torch.autograd.grad(embedding(ids.cuda(), w, 3.0), w, dout)
    h = 0.5
    value = [float((embedding(ids.cuda(), w.detach() + sign * h * d, 3.0).double() * dout.double()).sum()) for sign in (1, -1)]
    slope, want = (value[0] - value[1]) / (2 * h), float(d.double().square().sum())
    assert abs(slope - want) < 1e-5 * want


@pytest.mark.gpu
def test_large_table_offsets():
    """Rows behind the 2^31st element of the table and of its gradient."""
    V, D = 70000, 32768
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 24 GB")
    w = torch.zeros(V, D, device="cuda", dtype=torch.bfloat16)
    w[V - 1], w[65536], w[0] = 1.0, 2.0, 3.0
    w.requires_grad_()
    ids = torch.tensor([V - 1, 65536, V - 1, 0], device="cuda")
    out = embedding(ids, w)
    assert [float(out[i].detach().float().mean()) for i in range(4)] == [1.0, 2.0, 1.0, 3.0]
    d, = torch.autograd.grad(out, w, torch.ones_like(out))
    sums = d.float().sum(1) if False else torch.stack([d[i].float().mean() for i in (V - 1, 65536, 0, 1, 65535, V - 2)])
    assert sums.tolist() == [2.0, 1.0, 1.0, 0.0, 0.0, 0.0] and int(torch.count_nonzero(d)) == 3 * D
    del w, d, out
    torch.cuda.empty_cache()


@pytest.mark.gpu
def test_forward_mode_and_second_gradients_are_refused():
    import torch.autograd.forward_ad as fwd

    ids, w = torch.zeros(3, dtype=torch.int64, device="cuda"), torch.randn(5, 8, device="cuda", requires_grad=True)
    dout = torch.ones(3, 8, device="cuda", requires_grad=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(embedding(ids, w), w, dout, create_graph=True)
    with fwd.dual_level(), pytest.raises(NotImplementedError):
        embedding(ids, fwd.make_dual(w.detach(), torch.ones(5, 8, device="cuda")))


@pytest.mark.gpu
def test_launches_are_counted():
    ids, table = problem(5000, 3000, 64)
    w = table.cuda().requires_grad_()
    before = ops.launches()
    out = embedding(ids.cuda(), w)
    assert ops.launches() == before + 1
    torch.autograd.grad(out, w, torch.ones_like(out))
    assert ops.launches() > before + 2


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 2, 3, 69, 70])
@pytest.mark.parametrize("D, gap", [(1, 0), (1, 1), (1, 2), (2, 1), (3, 0), (3, 2), (7, 0), (7, 4), (8, 1), (513, 2), (600, 1)])
def test_rows_of_16_bits_that_end_in_the_middle_of_a_word(T, D, gap):
    """Tables and gradients of odd widths and odd strides, the last row at the very end of its storage: rows are read as 32-bit words, and of one
    column an odd number of them leaves no word for the last."""
    g = torch.Generator().manual_seed(T)
    V, scale, wide = 9, 0.7, D + gap

    def rows(n):
        room = torch.full((n * wide - gap,), float("nan"), dtype=torch.bfloat16)
        x = room.as_strided((n, D), (wide, 1))
        x.copy_(torch.randn(n, D, generator=g))
        return x, room.cuda().as_strided((n, D), (wide, 1))

    ids = torch.randint(0, V, (T,), generator=g)
    ids[0] = V - 1
    table, there = rows(V)
    dout, dthere = rows(T)
    out = embedding(ids.cuda(), there.requires_grad_(), scale)
    dtable, = torch.autograd.grad(out, there, dthere)
    check(ids, table, dout, out, dtable, scale)


def check_sparse(ids, table, dout, dtable, scale, padding):
    """As ``check`` for tables too large to widen: the rows that have tokens, in 64 bits, and zeros everywhere else."""
    keep = (ids >= 0) & (ids < table.shape[0]) & (ids != padding)
    rows, place = torch.unique(ids[keep], return_inverse=True)
    terms = dout[keep].double()
    total = torch.zeros(len(rows), dout.shape[1], dtype=torch.float64, device=ids.device).index_add_(0, place, terms) * scale
    size = torch.zeros_like(total).index_add_(0, place, terms.abs()) * abs(scale)
    n = torch.bincount(place, minlength=len(rows))[:, None].double()
    got = dtable[rows]
    bound = size * n * 2.0 ** -24 + total.abs() * (HALF[dtable.dtype] + 2.0 ** -23) + 1e-40
    assert ((got.double() - total).abs() <= bound).all()
    assert int(torch.count_nonzero(dtable)) == int(torch.count_nonzero(got))


# T, V, D, table: one CTA sorts up to 8192 tokens with its lists in shared memory, and up to 16384 with them in scratch memory where the gradient has 18000
# bytes a token or more; two, three or four digits, so that the lists end in the same place after an even and an odd number of passes.
SORTS = [
    (8192, 40000, 64, torch.float32, True),
    (8192, 300000, 64, torch.float32, True),
    (8193, 40000, 921, torch.float32, False),          # 147.36 MB, 18000 a token are 147.47
    (8193, 40000, 924, torch.float32, True),
    (8193, 40000, 1845, torch.bfloat16, True),
    (16384, 40000, 1844, torch.float32, True),
    (16384, 300000, 248, torch.float32, True),
    (12345, 300000, 186, torch.float32, True),
    (16384, 140000000, 2, torch.bfloat16, True),
    (16384, 300000, 244, torch.float32, False),
    (16385, 40000, 1900, torch.float32, False),
    (16385, 300000, 256, torch.float32, False),
]


@pytest.mark.gpu
@pytest.mark.parametrize("T, V, D, table_type, whole", SORTS)
@pytest.mark.parametrize("hot", [0.0, 0.4])
def test_sorts_at_the_borders_of_their_rule(T, V, D, table_type, whole, hot):
    g = torch.Generator(device="cuda").manual_seed(T + V)
    ids = torch.randint(0, V, (T,), device="cuda", generator=g)
    skewed = (V * torch.rand(T, device="cuda", generator=g, dtype=torch.float64) ** 8).long()       # a few ids many times
    ids = torch.where(torch.rand(T, device="cuda", generator=g) < hot, skewed, ids)
    ids[::97], ids[5::301], ids[7::1000] = V - 1, 3, V // 2
    ids[11::500], ids[13::700] = -1, V                                                             # outside: no gradient
    w = torch.zeros(V, D, dtype=table_type, device="cuda").requires_grad_()
    dout = torch.randn(T, D, device="cuda", generator=g).to(table_type)
    before = ops.launches()
    dtable, = torch.autograd.grad(embedding(ids, w, 0.5, 3), w, dout)
    digits = -(-V.bit_length() // 9)
    assert ops.launches() - before == 1 + (1 if whole else 2 * digits) + 2
    check_sparse(ids, w, dout, dtable, 0.5, 3)
    again, = torch.autograd.grad(embedding(ids.int(), w, 0.5, 3), w, dout)
    assert torch.equal(again, dtable)
