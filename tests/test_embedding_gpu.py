"""The embedding lookup and its gradient. The lookup is one float32 product rounded once, so equality is the tolerance; a
gradient row that is the sum of n rows is off by at most (n + 2) float32 half steps of the sum of the magnitudes (row_bounds.py)
and the rounding to its type."""
import math

import pytest
import torch

from row_bounds import U, check

pytestmark = pytest.mark.gpu

KINDS = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
IDS = {"u8": torch.uint8, "i32": torch.int32, "i64": torch.int64}


def values(shape, kind, seed=0):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    return torch.randn(shape, generator=gen, device="cuda").to(kind)


def indices(shape, low, high, kind=torch.int32, seed=0):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed + 1000)
    return torch.randint(low, high, shape, generator=gen, device="cuda").to(kind)


def lookup(ids, table, scale, kind):
    ids = ids.long()
    here = (ids >= 0) & (ids < table.shape[0])
    s = torch.tensor(scale, dtype=torch.float32, device="cuda")
    y = table.float()[torch.where(here, ids, 0)] * s if table.shape[0] else torch.zeros((*ids.shape, table.shape[1]), device="cuda")
    return torch.where(here.unsqueeze(-1), y, 0.0).to(kind)


def check_grad(got, g, ids, scale, padding=None, before=None, what=""):
    rows, cols = got.shape
    ids, g = ids.reshape(-1).long(), g.reshape(-1, cols).double()
    keep = (ids >= 0) & (ids < rows)
    if padding is not None:
        keep &= ids != padding
    ids, g = ids[keep], g[keep]
    scale = float(torch.tensor(scale, dtype=torch.float32))
    want = torch.zeros((rows, cols), dtype=torch.float64, device="cuda").index_add_(0, ids, g) * scale
    mag = torch.zeros((rows, cols), dtype=torch.float64, device="cuda").index_add_(0, ids, g.abs()) * abs(scale)
    n = torch.zeros(rows, dtype=torch.float64, device="cuda").index_add_(0, ids, torch.ones(len(ids), dtype=torch.float64, device="cuda"))
    bound = U * (n[:, None] + 2) * mag
    if before is not None:
        want = want + before.double()
        bound = bound + U * want.abs()
    check(got, want, bound, what)
    return n


COLS = [1, 2, 3, 4, 5, 7, 8, 9, 16, 31, 32, 33, 64, 100, 255, 256, 257, 333, 512, 1000, 1024, 2050, 4096, 5001]


@pytest.mark.parametrize("cols", COLS)
@pytest.mark.parametrize("table,dst,ids", [("f32", "f32", "i32"), ("bf16", "bf16", "i64"), ("f16", "f32", "u8"), ("f32", "f16", "i64"),
                                           ("bf16", "bf16", "u8")])
def test_lookup(pkg, cols, table, dst, ids):
    t = values((211, cols), KINDS[table], cols)
    for shape in ((1,), (7,), (3, 130), (2049,)):
        i = indices(shape, 0 if ids == "u8" else -20, 240, IDS[ids], cols)
        for scale in (1.0, 0.37):
            got = pkg.embedding(i, t, scale, data_type=KINDS[dst])
            assert got.shape == (*shape, cols) and torch.equal(got, lookup(i, t, scale, KINDS[dst]))


@pytest.mark.parametrize("table", list(KINDS))
@pytest.mark.parametrize("dst", list(KINDS))
def test_lookup_types(pkg, table, dst):
    for cols in (24, 45):
        t, i = values((50, cols), KINDS[table]), indices((77,), 0, 50)
        assert torch.equal(pkg.embedding(i, t, math.sqrt(cols), data_type=KINDS[dst]), lookup(i, t, math.sqrt(cols), KINDS[dst]))
    assert pkg.embedding(i, t).dtype == KINDS[table]


def test_lookup_far_and_wrong_indices(pkg):
    t = values((10, 8), torch.float32)
    i = torch.tensor([0, 9, 10, -1, 2 ** 31 - 1, 2 ** 31, 2 ** 32, 2 ** 32 + 3, -2 ** 31, 2 ** 62, -2 ** 63, 5], device="cuda")
    assert torch.equal(pkg.embedding(i, t), lookup(i, t, 1.0, torch.float32))
    assert not bool(pkg.embedding(i[:3] * 0, t[:0]).any())


def test_rows_beyond_four_gigabytes(pkg):
    store = torch.empty(5 << 28, dtype=torch.float32, device="cuda")  # 5 GiB: three rows 2.4e9 bytes apart
    t = store.as_strided((3, 8), (600_000_000, 1))
    t.copy_(values((3, 8), torch.float32))
    i = torch.tensor([2, 1, 0, 2], device="cuda")
    assert torch.equal(pkg.embedding(i, t), t[i])
    g = values((4, 8), torch.float32, 1)
    want = pkg.embedding_backward(g, i, 3)
    pkg.embedding_backward_into(t, g, i)
    assert torch.equal(t, want)
    x = store.as_strided((3, 40), (600_000_000, 1))
    x.copy_(values((3, 40), torch.float32, 2))
    y, m, r = pkg.layernorm(x.contiguous(), stats=True)
    assert torch.equal(pkg.layernorm(x), y)
    assert torch.equal(pkg.layernorm_backward(x, x, m, r)[0], pkg.layernorm_backward(x.contiguous(), x.contiguous(), m, r)[0])


@pytest.mark.parametrize("cols", [3, 8, 40, 500])
def test_lookup_strides(pkg, cols):
    t = values((60, cols + 5), torch.float16, 1)[::2, 3:3 + cols]
    i = indices((6, 9, 8), 0, 30)[:, ::2].permute(2, 0, 1)
    guard = torch.full((8, 6, 5, cols + 7), 77.0, device="cuda")
    out = guard[..., 1:1 + cols]
    pkg.embedding_into(out, i, t, 3.0)
    assert torch.equal(out, lookup(i, t, 3.0, torch.float32))
    assert bool((guard[..., :1] == 77.0).all()) and bool((guard[..., 1 + cols:] == 77.0).all())
    # a table of one row for all indices, as a broadcast view
    assert torch.equal(pkg.embedding(i, t[:1].expand(30, cols)), lookup(i * 0, t, 1.0, torch.float16))


@pytest.mark.parametrize("cols", range(1, 9))
@pytest.mark.parametrize("ids", list(IDS))
@pytest.mark.parametrize("dst", list(KINDS))
def test_short_rows(pkg, cols, ids, dst):
    """Tables that fit on the SM and those that do not, indices inside and outside, packed and strided, whole and ragged ends."""
    for rows, count in ((1, 40), (7, 2048 * 3), (255, 5000), (256, 300), (2000, 9001), (9000, 100)):
        t = values((rows, cols + 1), torch.float32, cols)[:, 1:]
        i = indices((count + 8,), 0 if ids == "u8" else -3, min(rows + 9, 256) if ids == "u8" else rows + 9, IDS[ids], rows)
        for view in (i[:count], i[8:], i[3:3 + count], i[::2]):
            assert torch.equal(pkg.embedding(view, t, 0.3, data_type=KINDS[dst]), lookup(view, t, 0.3, KINDS[dst])), (rows, count)


def test_palette_of_a_label_map(pkg):
    labels = indices((2, 120, 161), 0, 256, torch.uint8)
    palette = values((256, 3), torch.float32)
    assert torch.equal(pkg.embedding(labels, palette, 0.5, data_type=torch.float16), lookup(labels, palette, 0.5, torch.float16))


@pytest.mark.parametrize("cols", COLS)
@pytest.mark.parametrize("grad,dst,ids", [("f32", "f32", "i32"), ("bf16", "f32", "i64"), ("f16", "f16", "u8"), ("f32", "bf16", "i64")])
def test_gradient(pkg, cols, grad, dst, ids):
    for count, rows in ((1, 1), (1, 5), (3, 200), (33, 7), (700, 211), (2049, 100)):
        g = values((count, cols), KINDS[grad], cols)
        i = indices((count,), 0 if ids == "u8" else -3, rows + 3, IDS[ids], cols)
        got = pkg.embedding_backward(g, i, rows, 0.7, data_type=KINDS[dst])
        assert got.shape == (rows, cols) and got.dtype == KINDS[dst]
        check_grad(got, g, i, 0.7, what=f"{count} of {rows}")


# more indices than one kernel takes at once
@pytest.mark.parametrize("cols", [c for c in COLS if c <= 1024])
@pytest.mark.parametrize("grad,dst", [("f32", "f32"), ("bf16", "f32"), ("f16", "f16")])
def test_gradient_of_many_indices(pkg, cols, grad, dst):
    for count, rows in ((16384, 9000), (16385, 9000), (20011, 70)):
        g, i = values((count, cols), KINDS[grad], cols), indices((count,), -3, rows + 3, torch.int64, cols)
        check_grad(pkg.embedding_backward(g, i, rows, 0.7, data_type=KINDS[dst]), g, i, 0.7, what=f"{count} of {rows}")


# runs around the lengths that groups of lanes, warps and whole blocks take; column counts of every vector width; indices in order
# and in the opposite one
@pytest.mark.parametrize("cols", [1, 2, 7, 12, 64, 65, 200])
@pytest.mark.parametrize("grad", list(KINDS))
def test_gradient_runs_of_every_length(pkg, cols, grad):
    i = torch.repeat_interleave(torch.arange(12), torch.tensor([1, 2, 8, 9, 31, 32, 33, 511, 0, 512, 513, 2000])).cuda()
    g = values((len(i), cols), KINDS[grad], cols)
    shuffled = i[torch.randperm(len(i), generator=torch.Generator().manual_seed(cols)).cuda()]
    for j in (i, 11 - i, shuffled, i * 2048, i * 2047, shuffled * 148 + 3):
        check_grad(pkg.embedding_backward(g, j, 30000, 1.5), g, j, 1.5)
        into = torch.ones((30000, cols), dtype=torch.float32, device="cuda")
        pkg.embedding_backward_into(into, g, j, 1.5, accumulate=True)
        check_grad(into, g, j, 1.5, before=torch.ones_like(into))


# tables around the rows that a block keeps track of, and those left to the kernels for many indices (a wide table of many rows)
@pytest.mark.parametrize("rows,cols", [(2047, 5000), (2048, 5000), (2049, 5000), (4096, 9480), (4097, 9480), (2097152, 33), (300000, 1000),
                                       (1, 70000), (149, 8)])
def test_gradient_of_tables_of_many_rows(pkg, rows, cols):
    g, i = values((37, cols), torch.bfloat16, 1), indices((37,), 0, rows, torch.int64, rows)
    i[5:9] = rows - 1
    got = pkg.embedding_backward(g, i, rows, data_type=torch.bfloat16)
    named = torch.zeros(rows, dtype=torch.bool, device="cuda")
    named[i] = True
    assert not bool(got[~named].any())
    at, inverse = torch.unique(i, return_inverse=True)
    check_grad(got[at], g, inverse, 1.0)


@pytest.mark.parametrize("rows", [1, 2, 255, 256, 1023, 1024, 1025, 40000, 1 << 20, (1 << 20) + 1])
@pytest.mark.parametrize("count", [31, 1024, 8193, 70001])
def test_gradient_of_every_number_of_digits(pkg, rows, count):
    g = values((count, 3), torch.float32, rows)
    i = indices((count,), 0, rows, torch.int64, rows)
    n = check_grad(pkg.embedding_backward(g, i, rows), g, i, 1.0)
    assert int(n.sum()) == count


@pytest.mark.parametrize("cols", [8, 264, 1000])
def test_gradient_of_one_index_for_all_and_of_long_runs(pkg, cols):
    g = values((5000, cols), torch.bfloat16, cols)
    for i in (torch.full((5000,), 3), torch.arange(5000) // 1500, torch.arange(5000).flip(0) // 33, torch.arange(5000) % 2 * 6,
              torch.where(torch.arange(5000) % 3 == 0, 1, torch.arange(5000) % 7)):
        i = i.cuda()
        rows = int(i.max()) + 1
        check_grad(pkg.embedding_backward(g, i, rows), g, i, 1.0)


def test_padding_and_indices_of_other_parts(pkg):
    g = values((400, 72), torch.float32)
    i = indices((20, 20), -10, 30)
    g3 = g.reshape(20, 20, 72)
    for padding in (None, 0, 7, 19, 20, -1, -5):
        got = pkg.embedding_backward(g3, i, 20, 2.0, padding_index=padding)
        check_grad(got, g, i, 2.0, padding if padding is not None and 0 <= padding < 20 else None)
    assert not bool(pkg.embedding_backward(g3, i * 0 + 4, 20, padding_index=4).any())
    assert not bool(pkg.embedding_backward(g3, i * 0 - 4, 20).any())
    nan = torch.where((i == 7).unsqueeze(-1), float("nan"), g3)  # left out means not read into any sum
    assert torch.equal(pkg.embedding_backward(nan, i, 20, padding_index=7), pkg.embedding_backward(g3, i, 20, padding_index=7))


@pytest.mark.parametrize("dst", list(KINDS))
@pytest.mark.parametrize("cols", [6, 256])
def test_accumulate(pkg, dst, cols):
    g, i = values((900, cols), torch.float32, 1), indices((900,), -5, 60)
    before = values((100, cols), KINDS[dst], 2)
    before[80] = float("nan")  # named by no index: stays as it is
    into = before.clone()
    pkg.embedding_backward_into(into, g, i, 0.5, accumulate=True)
    untouched = torch.ones(100, dtype=torch.bool, device="cuda")
    untouched[i[(i >= 0)].long()] = False
    assert torch.equal(into[untouched].view(torch.uint8), before[untouched].view(torch.uint8))
    check_grad(into[:60], g, i, 0.5, before=before[:60])


@pytest.mark.parametrize("cols", [9, 128])
def test_gradient_strides(pkg, cols):
    g = values((6, 7, 40, cols + 3), torch.float16, 1)[:, ::2, :9, 2:2 + cols].permute(1, 0, 2, 3)
    i = indices((6, 4, 40), 0, 30, torch.int64)[:, :, :9].permute(1, 0, 2)
    guard = torch.full((60, cols + 6), 77.0, device="cuda")
    out = guard[::2, 4:4 + cols]
    pkg.embedding_backward_into(out, g, i, 1.5)
    check_grad(out, g, i, 1.5)
    assert bool((guard[1::2] == 77.0).all()) and bool((guard[:, :4] == 77.0).all()) and bool((guard[:, 4 + cols:] == 77.0).all())


def test_empty(pkg):
    t = values((5, 8), torch.float32)
    none = torch.empty((0, 3), dtype=torch.int32, device="cuda")
    assert pkg.embedding(none, t).shape == (0, 3, 8)
    got = pkg.embedding_backward(torch.empty((0, 3, 8), device="cuda"), none, 5)
    assert got.shape == (5, 8) and not bool(got.any())
    keep = t.clone()
    pkg.embedding_backward_into(keep, torch.empty((0, 3, 8), device="cuda"), none, accumulate=True)
    assert torch.equal(keep, t)
    assert pkg.embedding_backward(values((4, 8), torch.float32), indices((4,), 0, 5), 0).shape == (0, 8)


def test_gradient_against_differences(pkg):
    t, i, c = values((12, 20), torch.float32, 1), indices((50,), -2, 12), values((50, 20), torch.float32, 2)
    dt = pkg.embedding_backward(c, i, 12, 3.0)
    for k in range(3):
        e = values((12, 20), torch.float32, 20 + k)
        # the lookup is linear: its difference along e is the lookup of e
        diff = (lookup(i, e, 3.0, torch.float32).double() * c.double()).sum()
        scale = float((dt.double() * e.double()).abs().sum())
        assert abs(float((dt.double() * e.double()).sum() - diff)) <= 64 * U * scale + 1e-6 * abs(float(diff))


def test_equal_calls_give_equal_bits_on_any_stream(pkg):
    g, i = values((20000, 130), torch.bfloat16, 1), (values((20000,), torch.float32, 2).abs() * 900).int()
    t = values((4000, 130), torch.bfloat16, 3)
    first = [pkg.embedding_backward(g, i, 4000), pkg.embedding(i, t)]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for stream in (None, side, side.cuda_stream, None):
        again = [pkg.embedding_backward(g, i, 4000, stream=stream), pkg.embedding(i, t, stream=stream)]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(first, again))


@pytest.mark.parametrize("count", [50, 8000])
def test_equal_calls_of_few_indices_and_replays(pkg, count):
    """Runs of every length, whose positions are put in order after an unordered step; a replay with other indices in place."""
    i = (values((count,), torch.float32, 2) ** 4 * 3).long().clamp_(max=699)
    g = values((count, 130), torch.bfloat16, 1)
    first = pkg.embedding_backward(g, i, 700)
    check_grad(first, g, i, 1.0)
    for _ in range(5):
        assert torch.equal(first, pkg.embedding_backward(g, i, 700))
    ids, into = i.clone(), torch.zeros(700, 130, device="cuda")
    pkg.embedding_backward_into(into, g, ids)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        pkg.embedding_backward_into(into, g, ids)
    for shift in (0, 1, 350):
        ids.copy_((i + shift) % 700)
        into.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(into, torch.roll(first, shift, 0))


def test_python_refusals(pkg):
    t, i = values((5, 8), torch.float32), indices((4,), 0, 5)
    g = values((4, 8), torch.float32)
    for call in (lambda: pkg.embedding(i.cpu(), t), lambda: pkg.embedding(i, t.cpu()), lambda: pkg.embedding(i.float(), t),
                 lambda: pkg.embedding(i.short(), t), lambda: pkg.embedding(i, t.double()), lambda: pkg.embedding(i, t[0]),
                 lambda: pkg.embedding(i, t.t()), lambda: pkg.embedding(i, t, data_type=torch.uint8),
                 lambda: pkg.embedding_into(g[:3], i, t), lambda: pkg.embedding_into(g[:, :7], i, t),
                 lambda: pkg.embedding_into(g[:1].expand(4, 8), i, t),
                 lambda: pkg.embedding_backward(g, i[:3], 5), lambda: pkg.embedding_backward(g.double(), i, 5),
                 lambda: pkg.embedding_backward(g, i.float(), 5), lambda: pkg.embedding_backward(g, i, 5, data_type=torch.int32),
                 lambda: pkg.embedding_backward_into(t[:, :7], g, i), lambda: pkg.embedding_backward_into(t[:1].expand(5, 8), g, i)):
        with pytest.raises(pkg.ops.Error):
            call()
