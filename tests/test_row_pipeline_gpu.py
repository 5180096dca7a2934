"""The row operators as they are used together: a batch of images through the pre-processing operators, its patches and a
sequence of tokens into a model's first activations, and a training step's gradients back to every parameter."""
import math

import numpy as np
import pytest
import torch

from gpu_util import to_dev
from row_bounds import U, check

pytestmark = pytest.mark.gpu

N, P, T, V, D = 3, 16, 21, 500, 192  # images, patch edge, tokens per text, vocabulary, width


def _patches(x):
    n, c, h, w = x.shape
    return x.reshape(n, c, h // P, P, w // P, P).permute(0, 2, 4, 3, 5, 1).reshape(n, (h // P) * (w // P), P * P * c)


def _setup():
    rng = np.random.default_rng(5)
    images = to_dev(rng.integers(0, 256, (N, 90, 120, 3), dtype=np.uint8))
    gen = torch.Generator(device="cuda")
    gen.manual_seed(3)
    rand = lambda *s: torch.randn(s, generator=gen, device="cuda")  # noqa: E731
    p = {"pw": 1 + 0.1 * rand(P * P * 3), "pb": 0.1 * rand(P * P * 3), "proj": 0.05 * rand(P * P * 3, D), "table": rand(V, D),
         "pos": rand(64, D), "w": 1 + 0.1 * rand(D), "b": 0.1 * rand(D)}
    ids = torch.randint(0, V, (N, T), generator=gen, device="cuda", dtype=torch.int32)
    ids[1, 15:] = 0  # padding
    c = rand(N, 12 + T, D)
    return images, p, ids, c


def _step(pkg, images, p, ids, c):
    """Forward and backward, gradients written out; the plain products are torch's."""
    batch = torch.empty((N, 3, 48, 64), device="cuda")
    pkg.fused_preprocess_into(batch, images, resize_dim=(64, 48), interp=1, layout="NCHW", base=(123.0, 117.0, 104.0),
                              mul=(0.017, 0.0175, 0.0174), srcCast=False)
    patches = _patches(batch)
    h, pm, pr = pkg.layernorm(patches, p["pw"], p["pb"], stats=True)
    seen = h @ p["proj"]
    where = torch.arange(12 + T, device="cuda").expand(N, 12 + T)
    words = pkg.embedding(ids, p["table"], math.sqrt(D))
    x = torch.cat([seen, words], 1) + pkg.embedding(where, p["pos"])
    y, m, r = pkg.layernorm(x, p["w"], p["b"], stats=True)
    dx, dw, db = pkg.layernorm_backward(c, x, m, r, p["w"])
    grads = {"w": dw, "b": db, "pos": pkg.embedding_backward(dx, where, 64),
             "table": pkg.embedding_backward(dx[:, 12:], ids, V, math.sqrt(D), padding_index=0)}
    dseen = dx[:, :12]
    grads["proj"] = h.flatten(0, 1).t() @ dseen.flatten(0, 1)
    _, grads["pw"], grads["pb"] = pkg.layernorm_backward(dseen @ p["proj"].t(), patches, pm, pr, p["pw"], src_grad=False)
    return batch, y, grads


def _plain(batch, p, ids, c):
    p = {k: v.double().requires_grad_() for k, v in p.items()}

    def norm(x, w, b):
        z = x - x.mean(-1, keepdim=True)
        return z / torch.sqrt((z * z).mean(-1, keepdim=True) + 1e-5) * w + b

    table = torch.cat([p["table"][:1].detach(), p["table"][1:]])
    seen = norm(_patches(batch.double()), p["pw"], p["pb"]) @ p["proj"]
    y = norm(torch.cat([seen, table[ids.long()] * math.sqrt(D)], 1) + p["pos"][:12 + T], p["w"], p["b"])
    (y * c.double()).sum().backward()
    return y.detach(), {k: v.grad for k, v in p.items()}


@pytest.fixture()
def full_precision_products():
    old = torch.backends.cuda.matmul.allow_tf32
    torch.backends.cuda.matmul.allow_tf32 = False
    yield
    torch.backends.cuda.matmul.allow_tf32 = old


def test_a_training_step(pkg, full_precision_products):
    images, p, ids, c = _setup()
    batch, y, grads = _step(pkg, images, p, ids, c)
    y64, want = _plain(batch, p, ids, c)
    # about 800 float32 additions lie between a parameter and the result at most; each is off by 2^-24 of magnitudes that do not
    # exceed sixteen times the largest value
    tol = 800 * 16 * U
    check(y, y64, torch.full_like(y64, tol * float(y64.abs().max())), "result")
    for k, g in want.items():
        check(grads[k], g, torch.full_like(g, tol * float(g.abs().max())), k)


def test_a_captured_step_replays_with_new_inputs(pkg, full_precision_products):
    images, p, ids, c = _setup()
    _step(pkg, images, p, ids, c)  # the first call on a device is not capturable
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _, y, grads = _step(pkg, images, p, ids, c)
    other = torch.randint(0, V, ids.shape, device="cuda", dtype=torch.int32)
    for tokens in (ids.clone(), other):
        ids.copy_(tokens)
        graph.replay()
        torch.cuda.synchronize()
        _, y2, grads2 = _step(pkg, images, p, ids, c)
        torch.cuda.synchronize()
        assert torch.equal(y, y2) and all(torch.equal(grads[k], grads2[k]) for k in grads)


def test_two_captured_graphs_keep_their_workspaces_apart(pkg):
    g = [torch.randn((3000, 72), device="cuda") for _ in range(2)]
    ids = [torch.randint(0, 300, (3000,), device="cuda") for _ in range(2)]
    want = [pkg.embedding_backward(g[k], ids[k], 300) for k in range(2)]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for k in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[k]):
            outs.append(pkg.embedding_backward(g[k], ids[k], 300))
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(20):
        for k in range(2):
            with torch.cuda.stream(streams[k]):
                graphs[k].replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_objects_with_layouts(pkg):
    cv = pkg.cvcuda
    images = cv.as_tensor(torch.randint(0, 256, (2, 40, 48, 3), device="cuda", dtype=torch.uint8), "NHWC")
    y, m, r = cv.layernorm(images, axes="HWC", stats=True)
    assert (y.layout, y.dtype, m.layout, m.shape) == ("NHWC", np.float32, "N", (2,))
    assert torch.equal(y.cuda(), pkg.layernorm(images.cuda(), axes=3))
    w = torch.ones(3, device="cuda")
    z, m, r = cv.layernorm(images, w, axes="C", dtype=cv.Type.BF16, stats=True)
    assert z.dtype == torch.bfloat16 and m.layout == "NHW"
    dx, dw, db = cv.layernorm_backward(z, images, m, r, w, axes="C", dtype=cv.Type.F32)
    assert dx.layout == "NHWC" and dx.dtype == np.float32 and dw.layout == "C"
    with pytest.raises(pkg.ops.Error):
        cv.layernorm(images, axes="WH")
    out = cv.Tensor((2, 40, 48, 3), cv.Type.F32, "NHWC")
    assert cv.layernorm_into(out, images, axes="HWC") is out and torch.equal(out.cuda(), y.cuda())
    labels = cv.as_tensor(torch.randint(0, 256, (2, 40, 48), device="cuda", dtype=torch.uint8), "NHW")
    palette = cv.as_tensor(torch.rand((256, 3), device="cuda"), "NC")
    colours = cv.embedding(labels, palette, 255.0, dtype=cv.Type.F16)
    assert (colours.layout, colours.shape, colours.dtype) == ("NHWC", (2, 40, 48, 3), np.float16)
    grad = cv.embedding_backward(colours, labels, 256)
    into = cv.Tensor((256, 3), cv.Type.F32, "NC")
    cv.embedding_backward_into(into, colours, labels, accumulate=True)
    assert torch.equal(grad.cuda(), into.cuda())
    assert torch.equal(cv.embedding_into(out, labels, palette).cuda(), pkg.embedding(labels.cuda(), palette.cuda()))


def test_page_locked_host_memory(pkg):
    x = torch.randn(9, 300).pin_memory()
    y = pkg.layernorm(x)
    table, ids = torch.randn(20, 64).pin_memory(), torch.arange(20).flip(0).pin_memory()
    e = pkg.embedding(ids, table)
    torch.cuda.synchronize()
    assert torch.equal(y, pkg.layernorm(x.cuda())) and torch.equal(e.cpu(), table.flip(0))
