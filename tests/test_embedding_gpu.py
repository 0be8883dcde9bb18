"""embedding and its gradient on the GPU: ids that repeat from once to always,
runs across parts, tables of every size of key, widths of every alignment."""

import pytest
import torch

import routed_reference as ref
from layer_reference import assert_within
from test_grouped_gpu import lib  # noqa: F401

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
SPMM_DEV_BAD_COLUMN = 1


def normal(*shape, dtype=F32, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def ids_of(n, rows, seed=0, power=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.rand(n, generator=g, dtype=torch.float64) ** power * rows).long().clamp(max=rows - 1).cuda()


def check(lib, ids, rows, width, dtype, scale=1.0, padding=None, seed=0):  # noqa: F811
    table, dy = normal(rows, width, dtype=dtype, seed=seed), normal(*ids.shape, width, dtype=dtype, seed=seed + 1)
    tl = table.clone().requires_grad_(True)
    y = lib.embedding(ids, tl, scale, padding)
    assert torch.equal(y.detach(), (table.float()[ids.long()] * scale).to(dtype))
    (d,) = torch.autograd.grad(y, tl, dy)
    assert_within(d, *ref.embedding_grad_reference(ids, dy, rows, scale, padding), "dtable")
    assert torch.equal(lib.embedding_grad(ids, dy, rows, scale, padding), d)
    return d


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("width", [1, 2, 3, 4, 7, 8, 31, 64, 100, 257, 512, 1001, 1024, 1026, 4096, 5000])
def test_widths(lib, width, dtype):  # noqa: F811
    check(lib, ids_of(150, 40, seed=width), 40, width, dtype, scale=3.0, seed=width)


@pytest.mark.parametrize("n", [1, 2, 31, 32, 33, 64, 65, 1000, 4096, 4097, 20011])
@pytest.mark.parametrize("rows", [1, 2, 1000, 1024, 1025, 70000, 1 << 20, (1 << 20) + 1])
def test_numbers_of_ids_and_rows(lib, n, rows):  # noqa: F811
    check(lib, ids_of(n, rows, seed=n), rows, 16, F32, scale=0.5)


@pytest.mark.parametrize("n", [2048, 2049, 8191, 8192, 8193, 131072, 131073])
@pytest.mark.parametrize("rows", [200, 1025, (1 << 20) + 1])
def test_where_the_sort_s_blocks_change(lib, n, rows):  # noqa: F811
    check(lib, ids_of(n, rows, seed=n, power=3.0), rows, 8, F32)


@pytest.mark.parametrize("power", [1.0, 4.0, 40.0])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_repeated_ids(lib, power, dtype):  # noqa: F811
    """Runs of one id within a part, across two, over hundreds."""
    check(lib, ids_of(9001, 3001, seed=2, power=power), 3001, 48, dtype, scale=2.0)
    check(lib, torch.full((9001,), 17, device="cuda"), 3001, 48, dtype)
    for run in (31, 32, 33, 63, 64, 65, 96, 160):   # every place of a run's end within a part
        check(lib, torch.arange(3000, device="cuda") // run, 101, 8, dtype)


def test_shapes_types_and_order(lib):  # noqa: F811
    ids = ids_of(24, 50, seed=1)
    for shaped in (ids.view(2, 3, 4), ids.int(), ids.view(6, 4).T, torch.tensor(7, device="cuda")):
        check(lib, shaped, 50, 24, F16)
    table = normal(50, 24)
    assert lib.embedding(torch.empty(0, 3, dtype=torch.int64, device="cuda"), table).shape == (0, 3, 24)
    d = lib.embedding_grad(torch.empty(0, dtype=torch.int32, device="cuda"), torch.empty(0, 24, device="cuda"), 50)
    assert d.shape == (50, 24) and bool((d == 0).all())
    strided = normal(50, 96, dtype=F16)[:, 5:29]
    assert torch.equal(lib.embedding(ids, strided), lib.embedding(ids, strided.contiguous()))


def test_padding_id_gets_no_gradient(lib):  # noqa: F811
    ids = ids_of(500, 20, seed=3)
    d = check(lib, ids, 20, 32, F32, padding=int(ids[0]))
    assert bool((d[int(ids[0])] == 0).all())


@pytest.mark.parametrize("n", [40, 6000])
def test_ids_outside_the_table(lib, n):  # noqa: F811
    """Zeros, no gradient, the device status; all other rows as ever."""
    ids = ids_of(n, 30, seed=4)
    bad = ids.clone()
    bad[3], bad[11], bad[12] = 30, -1, 1 << 40
    table, dy = normal(30, 40), normal(n, 40, seed=1)
    y = lib.embedding(bad, table)
    assert lib.device_status(True)[0] == SPMM_DEV_BAD_COLUMN
    outside = (bad < 0) | (bad >= 30)
    assert torch.equal(y, torch.where(outside[:, None], torch.zeros_like(y), table[bad.clamp(0, 29)]))
    d = lib.embedding_grad(bad, dy, 30)
    assert lib.device_status(True)[0] == SPMM_DEV_BAD_COLUMN
    assert_within(d, *ref.embedding_grad_reference(bad, dy, 30, 1.0))


def test_the_same_bits_every_time(lib):  # noqa: F811
    ids, dy = ids_of(30000, 5000, power=5.0), normal(30000, 64, dtype=BF16)
    first = lib.embedding_grad(ids, dy, 5000)
    for _ in range(5):
        assert torch.equal(lib.embedding_grad(ids, dy, 5000), first)


def test_values_that_are_not_finite(lib):  # noqa: F811
    """They reach their own id's row and column alone."""
    ids, dy = ids_of(3000, 100, seed=5), normal(3000, 16)
    dy[1234, 3] = float("nan")
    d = lib.embedding_grad(ids, dy, 100)
    bad = ~torch.isfinite(d)
    assert int(bad.sum()) == 1 and bool(bad[int(ids[1234]), 3])


def test_gradient_against_differences(lib):  # noqa: F811
    """embedding is linear in the table: <dtable, v> = <dy, embedding(v)>."""
    ids, dy, v = ids_of(700, 60, seed=6), normal(700, 24), normal(60, 24, seed=1)
    d = check(lib, ids, 60, 24, F32, scale=1.5)
    d = lib.embedding_grad(ids, dy, 60, 1.5)
    want = (lib.embedding(ids, v, 1.5).double() * dy.double()).sum()
    slack = (ref.embedding_grad_reference(ids, dy, 60, 1.5)[1] * v.double().abs()).sum() + 1e-5 * float(want.abs()) + 2e-3
    assert abs(float((d.double() * v.double()).sum() - want)) < float(slack)


def test_the_graph_of_the_gradient(lib):  # noqa: F811
    """Kept, used twice, freed, of a table that is no leaf; ids that were changed in between are refused."""
    ids, table, dy = ids_of(300, 60), normal(60, 24).requires_grad_(True), normal(300, 24)
    want = lib.embedding_grad(ids, dy, 60, 3.0)
    y = lib.embedding(ids, table * 2, 1.5)
    (first,) = torch.autograd.grad(y, table, dy, retain_graph=True)
    (second,) = torch.autograd.grad(y, table, dy)
    assert torch.equal(first, want) and torch.equal(second, want)   # twice is exact
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(y, table, dy)
    y = lib.embedding(ids, table)
    ids[0] = 0
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    with torch.no_grad():
        assert not lib.embedding(ids, table).requires_grad
    with torch.inference_mode():
        assert not lib.embedding(ids, table).requires_grad
    y = lib.embedding(ids, table)
    y.add_(1).sum().backward()   # the result may be changed in place
    assert torch.equal(table.grad, lib.embedding_grad(ids, torch.ones(300, 24, device="cuda"), 60))


def test_captured_and_replayed(lib):  # noqa: F811
    ids, table, dy = ids_of(5000, 2000), normal(2000, 40, dtype=F16), normal(5000, 40, dtype=F16)
    lib.embedding_grad(ids, dy, 2000)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, d = lib.embedding(ids, table), lib.embedding_grad(ids, dy, 2000)
    for seed in (1, 2, 3):
        ids.copy_(ids_of(5000, 2000, seed=seed, power=seed))
        dy.copy_(normal(5000, 40, dtype=F16, seed=seed))
        graph.replay()
        assert torch.equal(y, lib.embedding(ids, table)) and torch.equal(d, lib.embedding_grad(ids, dy, 2000))


def test_refusals(lib):  # noqa: F811
    ids, table = ids_of(10, 5), normal(5, 8)
    for call, text in ((lambda: lib.embedding(ids.float(), table), "int32 or int64"),
                       (lambda: lib.embedding(ids.cpu(), table), "must be CUDA tensor"),
                       (lambda: lib.embedding(ids, table.double()), "supports only FP16, BF16 and FP32"),
                       (lambda: lib.embedding(ids, table[0]), "two-dimensional"),
                       (lambda: lib.embedding(ids, table[:, :0]), "feature width"),
                       (lambda: lib.embedding(ids, table, float("inf")), "scale must be finite"),
                       (lambda: lib.embedding(ids, table, 1.0, 5), "padding_id"),
                       (lambda: lib.embedding(ids, table, 1.0, -1), "padding_id"),
                       (lambda: lib.embedding_grad(ids, normal(9, 8), 5), "shape of ids"),
                       (lambda: lib.embedding_grad(ids, normal(10, 8), -1), "must not be negative")):
        with pytest.raises(RuntimeError, match=text):
            call()
    tl = table.clone().requires_grad_(True)
    (d,) = torch.autograd.grad(lib.embedding(ids, tl).sum(), tl, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        d.sum().backward()


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("run", [31, 32, 33, 256, 257, 1024 * 32 - 1, 1024 * 32, 1024 * 32 + 1, 100000])
@pytest.mark.parametrize("width", [16, 33])
def test_long_runs_to_the_last_row(lib, run, width, dtype):  # noqa: F811
    """Whole numbers, whose fp32 sums are exact in any order: a lost, doubled or misplaced row shows."""
    g = torch.Generator(device="cuda").manual_seed(run)
    runs = [5, run, 1, run + 40, 3]      # of the ids 2, 9, 3, 0, 7, in shuffled order
    ids = torch.cat([torch.full((n,), i, device="cuda") for n, i in zip(runs, (2, 9, 3, 0, 7))])
    ids = ids[torch.randperm(len(ids), generator=g, device="cuda")]
    dy = torch.randint(-8, 9, (len(ids), width), generator=g, device="cuda")
    want = torch.zeros(11, width, dtype=torch.int64, device="cuda").index_add_(0, ids, dy)
    assert int(want.abs().max()) < 1 << 16 and 8 * len(ids) < 1 << 24
    d = lib.embedding_grad(ids, dy.to(dtype), 11)
    assert torch.equal(d, want.float().to(dtype))
    d = lib.embedding_grad(ids, dy.to(dtype), 11, 0.25, 9)
    want[9] = 0
    assert torch.equal(d, (want.float() * 0.25).to(dtype))
