"""LayerNorm and its gradient against a plain 64-bit implementation, with the error bounds of row_bounds.py."""
import pytest
import torch

from row_bounds import check, layernorm64, layernorm_backward64

pytestmark = pytest.mark.gpu

KINDS = {"u8": torch.uint8, "f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
EPS = 1e-5


def values(shape, kind, seed=0, scale=1.0, offset=0.0):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    if kind == torch.uint8:
        return torch.randint(0, 256, shape, generator=gen, device="cuda", dtype=torch.uint8)
    return (torch.randn(shape, generator=gen, device="cuda") * scale + offset).to(kind)


def verify(pkg, x, w, b, out_kind, eps=EPS, axes=1):
    y, m, r = pkg.layernorm(x, w, b, eps, axes=axes, data_type=out_kind, stats=True)
    assert y.shape == x.shape and y.dtype == out_kind and m.dtype == r.dtype == torch.float32
    cols = 1
    for k in x.shape[x.dim() - axes:]:
        cols *= k
    flat = x.reshape(-1, cols)
    (y64, m64, r64), (dy, dm, dr) = layernorm64(flat, *(None if v is None else v.flatten() for v in (w, b)), eps)
    check(m.flatten(), m64, dm, "mean")
    check(r.flatten(), r64, dr, "rstd")
    check(y.reshape(-1, cols), y64, dy, "result")
    return y, m, r


def verify_backward(pkg, g, x, m, r, w, axes=1, **more):
    dx, dw, db = pkg.layernorm_backward(g, x, m, r, w, axes=axes, **more)
    cols = 1
    for k in x.shape[x.dim() - axes:]:
        cols *= k
    want, bound = layernorm_backward64(g.reshape(-1, cols), x.reshape(-1, cols), m, r, None if w is None else w.flatten())
    if dx is not None:
        check(dx.reshape(-1, cols), want[0], bound[0], "dsrc")
    if dw is not None:
        check(dw.flatten(), want[1], bound[1], "dweight")
    if db is not None:
        check(db.flatten(), want[2], bound[2], "dbias")
    return dx, dw, db


# row lengths around every boundary of the kernels: lanes, vectors, warps, blocks, clusters, the split of long rows
LENGTHS = [1, 2, 3, 7, 8, 9, 31, 32, 33, 64, 96, 127, 128, 130, 255, 256, 257, 512, 588, 768, 1000, 1023, 1024, 1025, 1536, 2047, 2048,
           2051, 4096, 4104, 5000, 8191, 8192, 8200, 16384, 16387, 32768, 32776, 50001]


@pytest.mark.parametrize("cols", LENGTHS)
@pytest.mark.parametrize("src,dst", [("f16", "f16"), ("bf16", "f32"), ("f32", "bf16"), ("u8", "f32")])
def test_row_lengths(pkg, cols, src, dst):
    for rows in (1, 5, 67):
        x = values((rows, cols), KINDS[src], cols + rows)
        w = values((cols,), torch.float32, 1, 0.3, 1.0)
        b = values((cols,), torch.float32, 2, 0.3)
        verify(pkg, x, w, b, KINDS[dst])


@pytest.mark.parametrize("cols", LENGTHS)
@pytest.mark.parametrize("src,grad", [("f16", "f16"), ("bf16", "f32"), ("f32", "f32"), ("u8", "bf16")])
def test_backward_row_lengths(pkg, cols, src, grad):
    for rows in (1, 67, 301):
        x = values((rows, cols), KINDS[src], cols + rows)
        g = values((rows, cols), KINDS[grad], 3)
        w = values((cols,), torch.float32, 1, 0.3, 1.0)
        _, m, r = pkg.layernorm(x, stats=True)
        verify_backward(pkg, g, x, m, r, w)


# the forward pass of the same, long rows in chunks too
@pytest.mark.parametrize("cols", [17, 33, 77, 257, 385, 767, 1001, 1021, 2051, 5001, 8189, 8193, 16369, 24553, 50003])
@pytest.mark.parametrize("src,dst", [("f16", "f16"), ("bf16", "f32"), ("f32", "f32"), ("u8", "bf16")])
def test_rows_that_start_anywhere(pkg, cols, src, dst):
    for rows in (1, 7, 150, 1203) if cols < 10000 else (1, 7, 40):
        x = values((rows, cols), KINDS[src], cols, 1.0, 3.0)
        w, b = values((cols,), torch.float32, 1, 0.3, 1.0), values((cols,), torch.bfloat16, 2, 0.3)
        for wb in ((w, b), (None, None)):
            verify(pkg, x, *wb, KINDS[dst])
        (want, _, _), (bound, _, _) = layernorm64(x, w, b, EPS)
        for width, starts in ((cols + 5, (3, 3)), (cols + 8, (1, 9)), (cols + 16, (8, 8)), (cols + 5, (0, 3))):
            wide = [torch.full((rows, width + 9), 255 if k == torch.uint8 else float("nan"), device="cuda").to(k) for k in (KINDS[src], KINDS[dst])]
            xs, ys = (t[:, s:s + cols] for t, s in zip(wide, starts))
            xs.copy_(x)
            pkg.layernorm_into(ys, xs, w, b, EPS)
            check(ys, want, bound, "result")
            ys.fill_(float("nan"))
            assert bool(wide[1].isnan().all())
            if src == dst:
                pkg.layernorm_into(xs, xs, w, b, EPS)
                check(xs, want, bound, "result in place")
                xs.fill_(float("nan"))
                assert bool(wide[0].isnan().all())


# rows that are no whole vectors: all tensors packed; slices whose rows start alike, with other values around them; slices whose rows
# do not; what lies around the rows is neither used nor written
@pytest.mark.parametrize("cols", [17, 33, 77, 257, 385, 767, 1001, 2051, 4099, 5001, 9999])
@pytest.mark.parametrize("src,grad", [("f16", "f16"), ("bf16", "f32"), ("f32", "f32"), ("u8", "bf16")])
def test_backward_of_rows_that_start_anywhere(pkg, cols, src, grad):
    out = KINDS[grad]
    for rows in (1, 7, 150, 1203):
        x, g = values((rows, cols), KINDS[src], cols), values((rows, cols), KINDS[grad], 3)
        w = values((cols,), torch.float32, 1, 0.3, 1.0)
        _, m, r = pkg.layernorm(x, stats=True)
        verify_backward(pkg, g, x, m, r, w)
        for width, starts in ((cols + 5, (3, 3, 3)), (cols + 8, (1, 9, 1)), (cols + 16, (8, 8, 8)), (cols + 5, (0, 3, 5))):
            wide = [torch.full((rows, width + 9), 255 if k == torch.uint8 else float("nan"), device="cuda").to(k)
                    for k in (KINDS[src], KINDS[grad], out)]
            xs, gs, ds = (t[:, s:s + cols] for t, s in zip(wide, starts))
            xs.copy_(x)
            gs.copy_(g)
            dw, db = torch.empty(cols, device="cuda"), torch.empty(cols, device="cuda")
            pkg.layernorm_backward_into(ds, dw, db, gs, xs, m, r, w)
            want, bound = layernorm_backward64(g, x, m, r, w)
            for got, y, e, what in zip((ds, dw, db), want, bound, ("dsrc", "dweight", "dbias")):
                check(got, y, e, what)
            ds.fill_(float("nan"))
            assert bool(wide[2].isnan().all())
            pkg.layernorm_backward_into(gs, None, None, gs, xs, m, r, w)  # in place
            check(gs, want[0], bound[0], "dsrc in place")


# gradients of another type than the rows, above the row length one kernel holds too
@pytest.mark.parametrize("cols", [20, 130, 760, 1030, 4096, 10001, 65536, 65537, 70001])
@pytest.mark.parametrize("src,grad", [("f32", "f16"), ("f32", "bf16"), ("u8", "f16"), ("u8", "f32"), ("f16", "f32"), ("f16", "bf16"),
                                      ("bf16", "f16"), ("bf16", "bf16")])
def test_backward_of_mixed_types(pkg, cols, src, grad):
    x, g = values((301, cols), KINDS[src], cols), values((301, cols), KINDS[grad], 3)
    w = values((cols,), torch.float32, 1, 0.3, 1.0)
    _, m, r = pkg.layernorm(x, stats=True)
    verify_backward(pkg, g, x, m, r, w)


# around the rows and columns that go in one launch
@pytest.mark.parametrize("cols", [1, 31, 33, 255, 257, 2049, 4095, 4096, 4097])
@pytest.mark.parametrize("src,grad", [("f32", "f32"), ("u8", "f16"), ("bf16", "bf16")])
def test_backward_of_few_rows(pkg, cols, src, grad):
    for rows in (1, 2, 8, 9, 64, 65, 255, 256, 257):
        x, g = values((rows, cols), KINDS[src], cols), values((rows, cols), KINDS[grad], 3)
        w = values((cols,), torch.bfloat16, 1, 0.3, 1.0)
        _, m, r = pkg.layernorm(x, stats=True)
        verify_backward(pkg, g, x, m, r, None)
        full = verify_backward(pkg, g, x, m, r, w)
        for want in ((1, 0, 0), (0, 1, 0), (0, 0, 1), (0, 1, 1)):
            out = pkg.layernorm_backward(g, x, m, r, w, src_grad=bool(want[0]), weight_grad=bool(want[1]), bias_grad=bool(want[2]))
            assert all(o is None or torch.equal(o, f) for o, f in zip(out, full)) and [o is not None for o in out] == [bool(k) for k in want]
        into, dw, db = g.clone(), torch.empty_like(w), torch.empty_like(w)
        pkg.layernorm_backward_into(into, dw, db, into, x, m, r, w)
        want, bound = layernorm_backward64(g, x, m, r, w)
        for got, y, e, what in zip((into, dw, db), want, bound, ("dsrc", "dweight", "dbias")):
            check(got, y, e, what + " in place")


@pytest.mark.parametrize("src", list(KINDS))
@pytest.mark.parametrize("dst", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("wk,bk", [(None, None), ("f32", None), (None, "bf16"), ("f16", "f32"), ("bf16", "bf16")])
def test_types(pkg, src, dst, wk, bk):
    for cols in (48, 77, 1200, 9000):
        x = values((9, cols), KINDS[src], 5)
        w = values((cols,), KINDS[wk], 1, 0.3, 1.0) if wk else None
        b = values((cols,), KINDS[bk], 2, 0.3) if bk else None
        _, m, r = verify(pkg, x, w, b, KINDS[dst])
        verify_backward(pkg, values((9, cols), KINDS[dst], 6), x, m, r, w)
        verify_backward(pkg, values((9, cols), KINDS[dst], 7), x, m, r, w, data_type=torch.float32)


@pytest.mark.parametrize("rows", [2, 31, 149, 1000, 4099, 30011])
@pytest.mark.parametrize("cols", [12, 96, 333, 768])
def test_many_rows(pkg, rows, cols):
    x = values((rows, cols), torch.bfloat16, rows, 2.0, 1.0)
    w = values((cols,), torch.float32, 1, 0.3, 1.0)
    _, m, r = verify(pkg, x, w, None, torch.bfloat16)
    verify_backward(pkg, values((rows, cols), torch.bfloat16, 4), x, m, r, w)


@pytest.mark.parametrize("want", [(1, 0, 0), (0, 1, 0), (0, 0, 1), (0, 1, 1), (1, 0, 1), (1, 1, 0)])
@pytest.mark.parametrize("cols", [100, 1024, 2500, 40000])
def test_only_the_gradients_asked_for(pkg, want, cols):
    x, g = values((307, cols), torch.float16, 1), values((307, cols), torch.float16, 2)
    w = values((cols,), torch.float16, 3, 0.3, 1.0)
    _, m, r = pkg.layernorm(x, w, stats=True)
    out = verify_backward(pkg, g, x, m, r, w, src_grad=bool(want[0]), weight_grad=bool(want[1]), bias_grad=bool(want[2]))
    assert tuple(o is not None for o in out) == tuple(bool(v) for v in want)
    full = pkg.layernorm_backward(g, x, m, r, w)
    for a, b in zip(out, full):
        assert a is None or torch.equal(a, b)


@pytest.mark.parametrize("src", ["f32", "u8", "f16"])
def test_whole_images_are_rows(pkg, src):
    for shape in ((3, 29, 31, 3), (2, 224, 224, 3), (1, 480, 641, 4)):
        x = values(shape, KINDS[src], 9)
        verify(pkg, x, None, None, torch.float32, axes=3)
    x = values((2, 32, 40, 3), KINDS[src], 9)
    w = values((32, 40, 3), torch.float32, 1, 0.3, 1.0)
    _, m, r = verify(pkg, x, w, w * 0.5, torch.float16, axes=3)
    assert m.shape == (2,)
    dx, dw, db = verify_backward(pkg, values(x.shape, torch.float32, 3), x, m, r, w, axes=3)
    assert dw.shape == db.shape == (32, 40, 3)


def test_large_offsets_and_flat_rows(pkg):
    x = values((16, 1024), torch.float32, 1, 1.0, 4000.0)
    x[3] = 7.25
    x[4] = 0.0
    x[5, 1:] = 0.0
    w, b = values((1024,), torch.float32, 2), values((1024,), torch.float32, 3)
    y, m, r = verify(pkg, x, w, b, torch.float32)
    assert torch.equal(y[3], b) and torch.equal(y[4], b)


def test_zero_epsilon_and_infinities_stay_in_their_rows(pkg):
    x = values((40, 768), torch.float32, 1)
    clean = pkg.layernorm(x, epsilon=0.0)
    bad = x.clone()
    bad[7, 3], bad[8, 0], bad[21, 767], bad[30] = float("inf"), float("nan"), float("-inf"), 5.0
    y = pkg.layernorm(bad, epsilon=0.0)
    keep = torch.ones(40, dtype=torch.bool, device="cuda")
    keep[[7, 8, 21, 30]] = False
    assert torch.equal(y[keep], clean[keep])
    assert bool(y[[7, 8, 21]].isnan().any(1).all()) and bool(y[30].isnan().all())  # 0 * (1 / 0)


@pytest.mark.parametrize("kind", ["f32", "bf16", "u8"])
@pytest.mark.parametrize("cols", [5, 64, 250, 2000])
def test_strided_rows(pkg, kind, cols):
    """Rows of a wider tensor, every second one, transposed, and with other strides on every side."""
    wide = values((12, 20, 4, cols + 11), KINDS[kind], 1)
    x = wide[:, ::2, :3, 5:5 + cols].permute(1, 0, 2, 3)
    w = values((cols + 3,), torch.float32, 2)[3:]  # off the vector boundary
    want = pkg.layernorm(x.contiguous(), w.clone(), data_type=torch.float32)
    guard = torch.full((10, 12, 3, cols + 9), 77.0, device="cuda")
    out = guard[..., 2:2 + cols]
    m, r = (torch.full((10 * 12 * 3 + 2,), 5.0, device="cuda") for _ in range(2))
    pkg.layernorm_into(out, x, w, mean=m[1:-1].reshape(10, 12, 3), rstd=r[1:-1].reshape(10, 12, 3))
    (y64, m64, r64), (dy, dm, dr) = layernorm64(x.reshape(-1, cols), w, None, EPS)
    check(out.reshape(-1, cols), y64, dy, "result")
    check(m[1:-1], m64, dm, "mean")
    assert float(m[0]) == float(m[-1]) == float(r[0]) == float(r[-1]) == 5.0
    assert bool((guard[..., :2] == 77.0).all()) and bool((guard[..., 2 + cols:] == 77.0).all())
    check(want.reshape(-1, cols), y64, dy, "packed")
    m, r = m[1:-1].reshape(10, 12, 3).clone(), r[1:-1].reshape(10, 12, 3).clone()
    g = values((10, 12, 3, cols * 2), torch.float32, 4)[..., 1:1 + cols]
    guard = torch.full((10, 12, 3, cols + 9), 77.0, device="cuda")
    dx = guard[..., 3:3 + cols]
    params = torch.full((2 * cols + 6,), 5.0, device="cuda")
    dw, db = params[1:1 + cols], params[cols + 5:2 * cols + 5]
    pkg.layernorm_backward_into(dx, dw, db, g, x, m, r, w)
    want, bound = layernorm_backward64(g.reshape(-1, cols), x.reshape(-1, cols), m, r, w)
    for got, a, b in zip((dx.reshape(-1, cols), dw, db), want, bound):
        check(got, a, b)
    assert bool((guard[..., :3] == 77.0).all()) and bool((guard[..., 3 + cols:] == 77.0).all())
    assert float(params[0]) == 5.0 and bool((params[1 + cols:cols + 5] == 5.0).all()) and float(params[-1]) == 5.0


@pytest.mark.parametrize("cols", [64, 333, 1024, 5000, 40000, 150528])
def test_in_place(pkg, cols):
    x, g = values((11, cols), torch.float16, 1), values((11, cols), torch.float16, 2)
    w = values((cols,), torch.float32, 3, 0.3, 1.0)
    y, m, r = pkg.layernorm(x, w, stats=True)
    z = x.clone()
    pkg.layernorm_into(z, z, w)
    assert torch.equal(z, y)
    full = pkg.layernorm_backward(g, x, m, r, w)
    for into in ("grad", "src"):
        gg, xx = g.clone(), x.clone()
        dw, db = torch.empty_like(w), torch.empty_like(w)
        dx = gg if into == "grad" else xx
        pkg.layernorm_backward_into(dx, dw, db, gg, xx, m, r, w)
        assert all(torch.equal(a, b) for a, b in zip((dx, dw, db), full)), into


def test_empty(pkg):
    x = torch.empty((0, 7, 16), device="cuda")
    y, m, r = pkg.layernorm(x, stats=True)
    assert y.shape == x.shape and m.shape == (0, 7)
    dx, dw, db = pkg.layernorm_backward(y, x, m, r)
    torch.cuda.synchronize()
    assert dx.shape == x.shape and dw.shape == (16,) and not bool(dw.any()) and not bool(db.any())
    with pytest.raises(pkg.ops.Error):
        pkg.layernorm(torch.empty((3, 0), device="cuda"))


def test_gradient_against_differences(pkg):
    """d(sum(y c)) along random directions, from 64-bit differences of the formula."""
    x, w, b = values((6, 200), torch.float32, 1), values((200,), torch.float32, 2, 0.3, 1.0), values((200,), torch.float32, 3)
    c = values((6, 200), torch.float32, 4)
    _, m, r = pkg.layernorm(x, w, b, stats=True)
    dx, dw, db = pkg.layernorm_backward(c, x, m, r, w)

    def loss(xx, ww, bb):
        return (layernorm64(xx, ww, bb, EPS)[0][0] * c.double()).sum()

    for k in range(4):
        ex, ew, eb = (values(t.shape, torch.float32, 10 + k + 5 * i).double() for i, t in enumerate((x, w, b)))
        h = 1e-5
        diff = (loss(x.double() + h * ex, w.double() + h * ew, b.double() + h * eb)
                - loss(x.double() - h * ex, w.double() - h * ew, b.double() - h * eb)) / (2 * h)
        got = (dx.double() * ex).sum() + (dw.double() * ew).sum() + (db.double() * eb).sum()
        # 1e-10 h^2 of the differences, and 2400 products with gradients each off by at most about 30 float32 steps
        scale = (dx.double() * ex).abs().sum() + (dw.double() * ew).abs().sum() + (db.double() * eb).abs().sum()
        assert abs(float(diff - got)) <= 64 * 2.0 ** -24 * float(scale) + 1e-6 * abs(float(diff))


def test_equal_calls_give_equal_bits_on_any_stream(pkg):
    x, g = values((3000, 520), torch.bfloat16, 1), values((3000, 520), torch.bfloat16, 2)
    w = values((520,), torch.float32, 3)
    first = [*pkg.layernorm(x, w, stats=True)]
    first += pkg.layernorm_backward(g, x, first[1], first[2], w)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for stream in (None, side, side.cuda_stream):
        again = [*pkg.layernorm(x, w, stats=True, stream=stream)]
        again += pkg.layernorm_backward(g, x, again[1], again[2], w, stream=stream)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_python_refusals(pkg):
    x = values((4, 8), torch.float32)
    m = torch.zeros(4, device="cuda")
    Error = pkg.ops.Error
    for call in (lambda: pkg.layernorm(x.cpu()), lambda: pkg.layernorm(x.double()), lambda: pkg.layernorm(x, axes=0),
                 lambda: pkg.layernorm(x, axes=3), lambda: pkg.layernorm(x.t()), lambda: pkg.layernorm(x, x[0, :7]),
                 lambda: pkg.layernorm(x, x[:, 0]), lambda: pkg.layernorm(x, None, x[0].double()), lambda: pkg.layernorm(x, epsilon=-1.0),
                 lambda: pkg.layernorm(x, data_type=torch.uint8), lambda: pkg.layernorm_into(x[:3], x),
                 lambda: pkg.layernorm_into(x[:1].expand(4, 8), x), lambda: pkg.layernorm_into(x.clone(), x, mean=m[:3]),
                 lambda: pkg.layernorm_into(x.clone(), x, mean=m.half()),
                 lambda: pkg.layernorm_backward(x[:3], x, m, m), lambda: pkg.layernorm_backward(x, x, m[:2], m),
                 lambda: pkg.layernorm_backward(x, x, m, m, x[0, :5]),
                 lambda: pkg.layernorm_backward(x, x, m, m, src_grad=False, weight_grad=False, bias_grad=False),
                 lambda: pkg.layernorm_backward_into(x[:1].expand(4, 8), None, None, x, x, m, m)):
        with pytest.raises(Error):
            call()
