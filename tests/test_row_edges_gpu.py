"""The row operators where they could go wrong: clusters, infinite rows, long sums, wide tables, the sorted gradient."""
import pytest
import torch

from row_bounds import U, check, layernorm64, layernorm_backward64

pytestmark = pytest.mark.gpu

KINDS = {"u8": torch.uint8, "f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def values(shape, kind, seed=0):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    if kind == torch.uint8:
        return torch.randint(0, 256, shape, generator=gen, device="cuda", dtype=torch.uint8)
    return torch.randn(shape, generator=gen, device="cuda").to(kind)


# clusters of two, four and eight CTAs, with one row each, which is exchanged first thing, and with more
@pytest.mark.parametrize("cols", [8193, 12288, 16385, 20000, 32769, 40003, 65536])
@pytest.mark.parametrize("src,grad", [("f16", "f16"), ("f32", "f32"), ("u8", "bf16")])
def test_backward_of_rows_split_over_clusters(pkg, cols, src, grad):
    w = values((cols,), torch.float32, 1)
    for rows in (1, 2, 19, 160):
        x, g = values((rows, cols), KINDS[src], cols), values((rows, cols), KINDS[grad], 3)
        (_, m, r), _ = layernorm64(x, None, None, 1e-5)
        m, r = m.float(), r.float()
        first = pkg.layernorm_backward(g, x, m, r, w)
        want, bound = layernorm_backward64(g, x, m, r, w)
        for got, y, e, what in zip(first, want, bound, ("dsrc", "dweight", "dbias")):
            check(got, y, e, what)
        # launched back to back: CTAs of a cluster start while those of the launch before end
        again = [pkg.layernorm_backward(g, x, m, r, w) for _ in range(20)]
        alone = [pkg.layernorm_backward(g, x, m, r, w, weight_grad=False, bias_grad=False)[0] for _ in range(20)]
        assert all(torch.equal(a, f) for call in again for a, f in zip(call, first)) and all(torch.equal(a, first[0]) for a in alone)


@pytest.mark.parametrize("accumulate", [False, True])
def test_gradient_of_a_table_of_many_columns(pkg, accumulate):
    cols = 16_780_000
    ids = torch.full((70,), 1, device="cuda")
    ids[50:60] = 0
    g = (torch.arange(70 * 256, device="cuda") % 251).reshape(70, 256).half().repeat(1, cols // 256 + 1)[:, :cols]
    into = torch.ones((3, cols), device="cuda")
    pkg.embedding_backward_into(into, g, ids, accumulate=accumulate)
    for row in range(3):
        want = g[:, :256].float()[ids == row].sum(0) + accumulate  # whole numbers: exact
        assert torch.equal(into[row], want.repeat(cols // 256 + 1)[:cols])


# every kernel of the forward pass: groups of lanes, a CTA per row, few rows, chunks, rows that start anywhere
@pytest.mark.parametrize("src", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("rows,cols", [(40, 1), (40, 24), (300, 768), (300, 77), (9, 1000), (300, 2048), (300, 2051), (9, 20000), (9, 20003)])
def test_statistics_of_rows_with_infinities(pkg, src, rows, cols):
    """The mean of a row that holds infinities of one sign is that infinity, of both NaN; the other rows do not notice."""
    x = torch.randn((rows, cols), device="cuda").to(KINDS[src])
    clean = pkg.layernorm(x, stats=True)
    bad = x.clone()
    inf = float("inf")
    bad[1, cols - 1], bad[3, cols // 2], bad[4, :], bad[5, 0], bad[6, 0] = inf, -inf, inf, float("nan"), inf
    bad[6, cols - 1] = -inf
    _, mean, rstd = got = pkg.layernorm(bad, stats=True)
    want = bad.double().mean(1)
    hit = [1, 3, 4, 5, 6]
    same = (mean[hit].double() == want[hit]) | (mean[hit].isnan() & want[hit].isnan())
    assert bool(same.all()), (mean[hit], want[hit])
    assert bool(rstd[hit].isnan().all()) and bool(got[0][hit].isnan().any(1).all())
    keep = torch.ones(rows, dtype=torch.bool, device="cuda")
    keep[hit] = False
    assert all(torch.equal(a[keep], b[keep]) for a, b in zip(got, clean))


# clusters of eight and of four CTAs, and rows too long for those; broadcast rows, so that only their number is large
@pytest.mark.parametrize("cols,big", [(40_000, 18), (20_000, 37), (65_537, 8)])
def test_sums_over_many_long_rows(pkg, cols, big):
    """No float32 sum over the rows is deeper than 48 + rows / 64 + 1300 additions (row_bounds.py): 1 is half a step of 2^24, so a
    chain that begins with that loses every addend."""
    rows = 300_000
    one = torch.ones((1, cols), device="cuda").expand(rows, cols)
    m, r = torch.zeros(rows, device="cuda"), torch.ones(rows, device="cuda")
    r[:big] = 2.0 ** 24  # h = (1 - 0) r
    _, dw, db = pkg.layernorm_backward(one, one, m, r, src_grad=False)
    k = 48 + rows / 64 + 1300
    want = torch.full((cols,), float(r.double().sum()), dtype=torch.float64, device="cuda")
    check(dw, want, U * (k + 4) * want, "dweight")
    check(db, torch.full_like(want, rows), torch.full_like(want, U * (k + 2) * rows), "dbias")


def test_arguments_out_of_range(pkg):
    g, i = torch.ones((4, 8), device="cuda"), torch.arange(4, device="cuda")
    want = pkg.embedding_backward(g, i, 5)
    for padding in (5, -1, 2 ** 63, -2 ** 70, 2 ** 32):  # values outside the table: none
        assert torch.equal(pkg.embedding_backward(g, i, 5, padding_index=padding), want)
    Error = pkg.ops.Error
    for call in (lambda: pkg.embedding_backward(g, i, -1), lambda: pkg.embedding_backward(g, i, 5, 1e39),
                 lambda: pkg.embedding(i, g, 1e39), lambda: pkg.embedding_into(want[:4], i, g, -1e39), lambda: pkg.layernorm(g, epsilon=1e39),
                 lambda: pkg.layernorm(g, epsilon=None), lambda: pkg.embedding(i, g, "2")):
        with pytest.raises(Error):
            call()


def test_more_elements_than_32_bits_count(pkg):
    n = 2 ** 31 - 5
    ids = torch.empty(n, dtype=torch.uint8, device="cuda").random_(0, 256)
    table = values((256, 2), torch.float16)
    out = pkg.embedding(ids, table)
    for a in (0, n // 2 - 1000, n - 100_003):
        assert torch.equal(out[a:a + 100_003], table[ids[a:a + 100_003].long()])
    del out, ids
    rows = 310_000_003
    x = torch.empty((rows, 7), dtype=torch.float16, device="cuda").normal_()
    y, m, r = pkg.layernorm(x, stats=True)
    dx = pkg.layernorm_backward(y, x, m, r, weight_grad=False, bias_grad=False)[0]
    for a in (0, 2 ** 28 - 50, rows - 1000):
        b = a + 1000
        (y64, m64, r64), (dy, dm, dr) = layernorm64(x[a:b], None, None, 1e-5)
        for got, want, bound in ((y, y64, dy), (m, m64, dm), (r, r64, dr)):
            check(got[a:b], want, bound)
        (dx64, _, _), (ex, _, _) = layernorm_backward64(y[a:b], x[a:b], m[a:b], r[a:b], None)
        check(dx[a:b], dx64, ex)


@pytest.mark.parametrize("cols", [40, 77, 1000, 2051, 9001])
def test_one_row_broadcast_to_many(pkg, cols):
    """Inputs whose rows are one and the same in memory."""
    x, g = (values((1, 1, cols), torch.float32, k).expand(30, 20, cols) for k in (1, 2))
    y, m, r = pkg.layernorm(x, stats=True)
    # (packed rows start elsewhere, which deals the values out differently: other bits, the same bounds)
    for a, b, e in zip((y.reshape(600, cols), m.flatten(), r.flatten()), *layernorm64(x.reshape(600, cols), None, None, 1e-5)):
        check(a, b, e)
    got = pkg.layernorm_backward(g, x, m, r)
    want, bound = layernorm_backward64(g.reshape(600, cols), x.reshape(600, cols), m, r, None)
    for a, b, e in zip(got, want, bound):
        check(a.reshape(b.shape), b, e)
