"""The embedding lookup's gradient with more indices than one kernel takes: sort, clearing, sums of runs and join, with everything that
test_embedding_gpu.py tries on few indices."""
import pytest
import torch

from test_embedding_gpu import IDS, KINDS, check_grad, indices, values

pytestmark = pytest.mark.gpu

COUNT = 9000  # one kernel takes 8192


def sorted_path(pkg, g, rows):
    """Whether the call has a workspace, which only these kernels have."""
    n, c = g.shape[-1], g.numel() // g.shape[-1]
    return pkg.rows._embedding_workspace_size(pkg.rows._TYPES[g.dtype], n, c, 6, rows) > 0


@pytest.mark.parametrize("dst", list(KINDS))
@pytest.mark.parametrize("cols", [6, 256, 1001])
@pytest.mark.parametrize("ids", list(IDS))
def test_accumulate(pkg, dst, cols, ids):
    g, i = values((COUNT, cols), torch.float32, 1), indices((COUNT,), 0 if ids == "u8" else -5, 60, IDS[ids])
    i[5000:7000] = 17  # a run of several blocks among the others
    assert sorted_path(pkg, g, 100)
    before = values((100, cols), KINDS[dst], 2)
    before[80] = float("nan")  # named by no index: stays as it is
    into = before.clone()
    pkg.embedding_backward_into(into, g, i, 0.5, accumulate=True)
    untouched = torch.ones(100, dtype=torch.bool, device="cuda")
    untouched[i[i >= 0].long()] = False
    assert torch.equal(into[untouched].view(torch.uint8), before[untouched].view(torch.uint8))
    check_grad(into[:60], g, i, 0.5, before=before[:60])


@pytest.mark.parametrize("ids", ["i32", "i64"])
@pytest.mark.parametrize("cols", [5, 72])
def test_padding_and_indices_of_other_parts(pkg, ids, cols):
    g = values((COUNT, cols), torch.float32)
    i = indices((100, 90), -10, 30, IDS[ids])
    g3 = g.reshape(100, 90, cols)
    assert sorted_path(pkg, g3, 20)
    for padding in (None, 0, 7, 19, 20, -1, -5):
        got = pkg.embedding_backward(g3, i, 20, 2.0, padding_index=padding)
        check_grad(got, g, i, 2.0, padding if padding is not None and 0 <= padding < 20 else None)
    assert not bool(pkg.embedding_backward(g3, i * 0 + 4, 20, padding_index=4).any())
    assert not bool(pkg.embedding_backward(g3, i * 0 - 4, 20).any())
    nan = torch.where((i == 7).unsqueeze(-1), float("nan"), g3)  # left out means not read into any sum
    assert torch.equal(pkg.embedding_backward(nan, i, 20, padding_index=7), pkg.embedding_backward(g3, i, 20, padding_index=7))
    # indices of other parts that only 64 bits tell apart
    if ids == "i64":
        far = torch.where(i < 5, i + (1 << 32), torch.where(i > 25, i - (1 << 40), i))
        check_grad(pkg.embedding_backward(g3, far, 20), g, far, 1.0)


@pytest.mark.parametrize("cols", [9, 128, 300])
@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("accumulate", [False, True])
def test_strides(pkg, cols, kind, accumulate):
    g = values((60, 7, 240, cols + 3), KINDS[kind], 1)[:, ::2, :40, 2:2 + cols].permute(1, 0, 2, 3)
    i = indices((60, 4, 100), 0, 30, torch.int64)[:, :, 1:81:2].permute(1, 0, 2)
    assert g.shape[:-1] == i.shape and sorted_path(pkg, g, 30)
    guard = torch.full((60, cols + 6), 77.0, device="cuda")
    out = guard[::2, 4:4 + cols]
    pkg.embedding_backward_into(out, g, i, 1.5, accumulate=accumulate)
    check_grad(out, g, i, 1.5, before=torch.full_like(out, 77.0) if accumulate else None)
    assert bool((guard[1::2] == 77.0).all()) and bool((guard[:, :4] == 77.0).all()) and bool((guard[:, 4 + cols:] == 77.0).all())
    # one row of the gradient for all positions, as a broadcast view; rows of the table from the last to the first
    one = g[:1, :1, :1].expand(4, 60, 40, cols)
    check_grad(pkg.embedding_backward(one, i, 30), one.contiguous(), i, 1.0)


# runs around the lengths that a warp, a group of 32 positions, the warps and the whole block of the join take, behind a run that
# shifts them against the groups; indices in order, in the opposite one and shuffled
@pytest.mark.parametrize("cols", [1, 8, 65, 257, 1000])
@pytest.mark.parametrize("grad,ids", [("f32", "i64"), ("bf16", "i32"), ("f16", "i64"), ("f32", "u8")])
def test_runs_of_every_length(pkg, cols, grad, ids):
    lengths = torch.tensor([0, 1, 2, 7, 8, 9, 31, 32, 33, 63, 64, 65, 511, 0, 512, 513, 544, 545, 2000, 4200, 40, 100])
    shuffle = torch.randperm(int(lengths.sum()) + 31, generator=torch.Generator().manual_seed(cols)).cuda()
    for shift in (0, 1, 8, 17, 31):
        lengths[0] = shift
        i = torch.repeat_interleave(torch.arange(len(lengths)), lengths).cuda()
        g = values((len(i), cols), KINDS[grad], cols + shift)
        assert sorted_path(pkg, g, 200)
        for j in (i, len(lengths) - 1 - i, i[shuffle[shuffle < len(i)]], i * 9 + 3):
            j = j.to(IDS[ids])
            check_grad(pkg.embedding_backward(g, j, 200, 1.5), g, j, 1.5)
            into = torch.ones((200, cols), dtype=torch.float32, device="cuda")
            pkg.embedding_backward_into(into, g, j, 1.5, accumulate=True)
            check_grad(into, g, j, 1.5, before=torch.ones_like(into))


@pytest.mark.parametrize("cols", [8, 257, 1000])
def test_one_index_for_all(pkg, cols):
    for count in (8193, 20000):
        g = values((count, cols), torch.bfloat16, cols)
        for i in (torch.full((count,), 3), torch.arange(count) // 1500, torch.arange(count).flip(0) // 33, torch.arange(count) % 2 * 6):
            i = i.cuda()
            rows = int(i.max()) + 1
            check_grad(pkg.embedding_backward(g, i, rows), g, i, 1.0)


def test_equal_calls_and_replays(pkg):
    """A replay with other indices in place gives the bits of a call with them. (Not those of the first call, moved: where the sorted runs
    lie against the groups of 32 positions settles the order of their sums.)"""
    i = (values((COUNT,), torch.float32, 2) ** 4 * 3).long().clamp_(max=699)
    g = values((COUNT, 130), torch.bfloat16, 1)
    assert sorted_path(pkg, g, 700)
    first = pkg.embedding_backward(g, i, 700)
    check_grad(first, g, i, 1.0)
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
        assert torch.equal(into, pkg.embedding_backward(g, ids, 700))
        check_grad(into, g, ids, 1.0)
