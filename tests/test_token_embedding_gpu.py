"""token_embedding against its formula: the rows exactly (one rounding where scaled), the table's gradient against fp64
sums within n fp32 additions (n 2^-24 of the sum of magnitudes) and the result's rounding."""

import pytest
import torch

from _gpu_util import DEV, log
from cdssm_hip import token_embedding
from cdssm_hip.train import token_embedding_bwd, token_embedding_fwd

pytestmark = pytest.mark.gpu

U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


def tokens(T, V, kind, seed=0):
    g = torch.Generator().manual_seed(seed)
    if kind == "uniform":
        return torch.randint(0, V, (T,), generator=g)
    if kind == "one":
        return torch.full((T,), V // 2)
    return (torch.exp(torch.rand(T, generator=g, dtype=torch.float64) * torch.log(torch.tensor(V + 1.0))) - 1).long().clamp(0, V - 1)


def check(ids, w, gy, scale=1.0, padding_idx=None):
    dtype, (V, C) = w.dtype, w.shape
    w = w.detach().requires_grad_()
    y = token_embedding(ids, w, scale=scale, padding_idx=padding_idx)
    (dw,) = torch.autograd.grad(y, w, gy)
    assert y.dtype == dtype and y.shape == (*ids.shape, C) and dw.dtype == dtype and dw.shape == w.shape
    flat = ids.reshape(-1).long()
    rows = w.detach().double()[flat]
    want = rows * torch.tensor(scale, dtype=torch.float32).double()
    assert torch.equal(y.reshape(-1, C), want.float().to(dtype) if dtype == torch.float32 else (w.detach()[flat].float() * scale).to(dtype))
    keep = torch.ones_like(flat, dtype=torch.bool) if padding_idx is None else flat != padding_idx % V
    g64 = gy.reshape(-1, C).double()[keep] * scale
    total = torch.zeros(V, C, dtype=torch.float64, device=DEV).index_add_(0, flat[keep], g64)
    size = torch.zeros(V, C, dtype=torch.float64, device=DEV).index_add_(0, flat[keep], g64.abs())
    n = torch.bincount(flat, minlength=V).double()[:, None]
    bound = (n + 4) * 2.0 ** -24 * size
    bound = bound + U[dtype] * (total.abs() + bound)
    off = (dw.double() - total).abs()
    log(f"  dW: {float((off / (bound + 1e-300)).max()):.3f} of its bound")
    assert bool((off <= bound).all())
    return y, dw


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("kind", ["uniform", "zipf", "one"])
@pytest.mark.parametrize("T,V,C", [(1, 1, 1), (1, 97, 64), (31, 97, 128), (32, 5, 100), (200, 97, 7), (333, 50257, 36),
                                   (1025, 300, 130), (5000, 70000, 64), (4096, 1000, 1024)])
def test_rows_and_gradient(T, V, C, kind, dtype):
    log(f"[embedding] T{T} V{V} C{C} {kind} {dtype}")
    g = torch.Generator().manual_seed(T)
    w = torch.randn(V, C, generator=g).to(dtype).to(DEV)
    gy = torch.randn(T, C, generator=g).to(dtype).to(DEV)
    ids = tokens(T, V, kind, T).to(DEV)
    a = check(ids, w, gy)
    b = check(ids.to(torch.int32), w, gy)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    check(ids, w, gy, scale=C ** 0.5, padding_idx=-1 if V > 1 else None)


def test_more_rows_than_a_launch_has_threads():
    """2^26 rows of one column, a wave each: more threads than one dimension of a launch holds."""
    n = (1 << 26) + 261
    w = torch.arange(n, device=DEV, dtype=torch.int32).remainder_(251).to(torch.bfloat16).view(n, 1)
    ids = torch.tensor([n - 1, 0, (1 << 24) + 3, n - 1, 1 << 26], device=DEV)
    gy = torch.tensor([[1.0], [2.0], [4.0], [8.0], [16.0]], dtype=torch.bfloat16, device=DEV)
    assert torch.equal(token_embedding_fwd(ids, w), w[ids])
    dw = token_embedding_bwd(gy, ids, n)
    assert dw.count_nonzero() == 4
    assert dw[[n - 1, 0, (1 << 24) + 3, 1 << 26], 0].tolist() == [9.0, 2.0, 4.0, 16.0]
    many = torch.arange(n, device=DEV, dtype=torch.int32).remainder_(7)
    y = token_embedding_fwd(many, w)
    assert torch.equal(y.view(-1), w[:7, 0][many])


@pytest.mark.parametrize("kind", ["uniform", "zipf", "one"])
@pytest.mark.parametrize("T,V,C", [(16384, 300, 8), (16385, 70000, 24), (40001, 700, 40), (70000, 1, 2)])
def test_long_lists_of_tokens(T, V, C, kind):
    """More tokens than the sort keeps between its passes; the forward's order and the backward's own give the same bits, once
    more from a graph that is kept."""
    g = torch.Generator().manual_seed(T)
    w = torch.randn(V, C, generator=g).to(torch.bfloat16).to(DEV)
    gy = torch.randn(T, C, generator=g).to(torch.bfloat16).to(DEV)
    ids = tokens(T, V, kind, T).to(DEV)
    ids[::97] = V  # no such row
    ids[5::89] = 0
    _, dw = check(ids.clamp(max=V - 1), w, gy)
    ws = w.detach().requires_grad_()
    y = token_embedding(ids, ws, padding_idx=0 if V > 1 else None)
    first, = torch.autograd.grad(y, ws, gy, retain_graph=True)
    again, = torch.autograd.grad(y, ws, gy)
    direct = token_embedding_bwd(gy, ids, V, padding_idx=0 if V > 1 else None)
    assert torch.equal(first, again) and torch.equal(first, direct)
    keep = (ids < V) & (ids > 0) if V > 1 else ids < V
    want = token_embedding_bwd(gy[keep], ids[keep], V)
    assert torch.equal(first, want)


@pytest.mark.parametrize("kind", ["uniform", "zipf", "one"])
@pytest.mark.parametrize("T,V,C", [(140000, 70000, 3), (16385, (1 << 20) + 3, 8), (5001, 1 << 22, 2), (70001, 20000001, 1)])
def test_many_tokens_of_many_rows(T, V, C, kind):
    """Sorts in two levels, of buckets with one and with more workgroups each."""
    g = torch.Generator().manual_seed(T)
    w = torch.randn(V, C, generator=g).to(DEV)
    gy = torch.randn(T, C, generator=g).to(DEV)
    ids = tokens(T, V, kind, T).to(DEV)
    # the sums by differences of running ones in fp64 (2^-53 of the whole at a step): atomic additions to one row take minutes
    pad = None if kind == "one" else 3
    gk = gy.double() if pad is None else gy.double() * (ids != pad)[:, None]
    at = torch.argsort(ids, stable=True)
    ends = torch.searchsorted(ids[at], torch.arange(V, device=DEV), right=True)

    def sums(v):
        run = torch.cat([torch.zeros(1, C, dtype=torch.float64, device=DEV), v[at].cumsum(0)])[ends]
        return torch.diff(run, dim=0, prepend=run.new_zeros(1, C))

    n = torch.diff(ends, prepend=ends.new_zeros(1)).double()[:, None]
    total, size = sums(gk), sums(gk.abs())
    bound = (n + 4) * 2.0 ** -24 * size + T * 2.0 ** -52 * gk.abs().sum(0) * (n > 0)
    bound = bound + U[torch.float32] * (total.abs() + bound)
    ws = w.detach().requires_grad_()
    y = token_embedding(ids, ws, padding_idx=pad)
    (dw,) = torch.autograd.grad(y, ws, gy)
    assert torch.equal(y, w[ids]) and bool(((dw.double() - total).abs() <= bound).all())
    del total, size, bound, n, ends
    ids[::97] = V  # no such row
    ids[5::89] = V - 1
    keep = ids < V
    a = token_embedding_bwd(gy, ids, V)
    assert torch.equal(a, token_embedding_bwd(gy[keep], ids[keep].to(torch.int32), V))
    ws = w.detach().requires_grad_()
    (b,) = torch.autograd.grad(token_embedding(ids, ws), ws, gy)
    assert torch.equal(a, b)


def test_the_sort_takes_tokens_plus_rows():
    """Four million tokens of a table of 2^26 rows, with the forward's order and the backward's own: by one workgroup for 256 rows that
    reads every token's id this would be 10^12 reads, seconds; it is some 10 ms, held to a second."""
    T, V = 1 << 22, 1 << 26
    ids = torch.randint(0, V, (T,), device=DEV)
    w = torch.ones(V, 1, dtype=torch.bfloat16, device=DEV, requires_grad=True)
    gy = torch.ones(T, 1, dtype=torch.bfloat16, device=DEV)
    begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    begin.record()
    (a,) = torch.autograd.grad(token_embedding(ids, w), w, gy)
    b = token_embedding_bwd(gy, ids, V)
    end.record()
    end.synchronize()
    log(f"  {begin.elapsed_time(end):.1f} ms")
    want = torch.bincount(ids, minlength=V).to(torch.bfloat16)
    assert torch.equal(a.view(-1), want) and torch.equal(b.view(-1), want)
    assert begin.elapsed_time(end) < 1000


def test_a_sort_in_two_levels_captured():
    T, V, C = 20000, 1 << 20, 4
    w = torch.randn(V, C, device=DEV)
    ids = tokens(T, V, "zipf", 4).to(DEV)
    gy = torch.randn(T, C, device=DEV)
    token_embedding_bwd(gy, ids, V)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        dw = token_embedding_bwd(gy, ids, V)
    for k in range(3):
        ids.copy_(tokens(T, V, "zipf" if k % 2 else "uniform", 5 + k).to(DEV))
        gy.normal_()
        graph.replay()
        want = token_embedding_bwd(gy, ids, V)
        torch.cuda.synchronize()
        assert torch.equal(dw, want)


def test_batched_ids_strides_and_expanded_gradients():
    g = torch.Generator().manual_seed(1)
    table = torch.randn(50, 80, generator=g).to(torch.bfloat16).to(DEV)
    ids = torch.randint(0, 50, (6, 40), generator=g).to(DEV)
    wide = torch.randn(6, 40, 72, generator=g).to(torch.bfloat16).to(DEV)
    check(ids, table[:, 3:67], wide[..., 5:69], scale=2.0)
    check(ids.t(), table[::2, :64][:25].contiguous().repeat(2, 1), wide.transpose(0, 1)[..., :64])
    w = table.clone().requires_grad_()
    token_embedding(ids, w).sum().backward()
    n = torch.bincount(ids.reshape(-1), minlength=50)
    assert torch.equal(w.grad, n[:, None].to(torch.bfloat16).expand(50, 80))


def test_ids_out_of_range_and_no_tokens():
    w = torch.randn(20, 64, device=DEV).requires_grad_()
    ids = torch.tensor([3, -1, 20, 3, 1 << 40, -(1 << 40), 19], device=DEV)
    y = token_embedding(ids, w)
    bad = torch.tensor([False, True, True, False, True, True, False], device=DEV)
    assert torch.isnan(y[bad]).all() and torch.equal(y[~bad], w.detach()[ids[~bad]])
    (dw,) = torch.autograd.grad(y, w, torch.ones_like(y))
    want = torch.zeros_like(w)
    want[3], want[19] = 2, 1
    assert torch.equal(dw, want)
    y = token_embedding(ids[:0], w)
    assert y.shape == (0, 64)
    (dw,) = torch.autograd.grad(y, w, torch.ones_like(y))
    assert torch.equal(dw, torch.zeros_like(w))


def test_the_padding_row_takes_no_gradient_whatever_it_gets():
    w = torch.randn(20, 64, device=DEV).to(torch.bfloat16).requires_grad_()
    ids = torch.randint(0, 20, (500,), device=DEV)
    gy = torch.randn(500, 64, device=DEV).to(torch.bfloat16)
    gy[ids == 7] = float("nan")
    (dw,) = torch.autograd.grad(token_embedding(ids, w, padding_idx=7), w, gy)
    assert torch.isfinite(dw).all() and torch.equal(dw[7], torch.zeros_like(dw[7]))


def test_gradient_against_differences_and_the_same_bits_again():
    """The map is linear: its difference along a direction is the gradient's product with it, up to fp32 sums."""
    g = torch.Generator().manual_seed(2)
    w = torch.randn(300, 96, generator=g).to(DEV)
    u = torch.randn(300, 96, generator=g).to(DEV)
    ids = tokens(3000, 300, "zipf", 3).to(DEV)
    gy = torch.randn(3000, 96, generator=g).to(DEV)
    dw = token_embedding_bwd(gy, ids, 300, 1.5)
    diff = (token_embedding_fwd(ids, w + u, 1.5).double() - token_embedding_fwd(ids, w - u, 1.5).double()) / 2
    got, want = (dw.double() * u).sum(), (diff * gy).sum()
    assert abs(float(got - want)) <= 2.0 ** -20 * float((diff * gy).abs().sum())
    for _ in range(3):
        assert torch.equal(dw, token_embedding_bwd(gy, ids, 300, 1.5))


def test_on_another_stream_and_captured():
    w = torch.randn(500, 128, device=DEV).to(torch.bfloat16)
    ids = tokens(700, 500, "zipf", 4).to(DEV)
    gy = torch.randn(700, 128, device=DEV).to(torch.bfloat16)
    want = token_embedding_fwd(ids, w), token_embedding_bwd(gy, ids, 500)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = token_embedding_fwd(ids, w), token_embedding_bwd(gy, ids, 500)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, dw = token_embedding_fwd(ids, w), token_embedding_bwd(gy, ids, 500)
    for k in range(4):
        ids.copy_(tokens(700, 500, "zipf" if k % 2 else "one", 5 + k).to(DEV))
        gy.normal_()
        graph.replay()
        want = token_embedding_fwd(ids, w), token_embedding_bwd(gy, ids, 500)
        torch.cuda.synchronize()
        assert torch.equal(y, want[0]) and torch.equal(dw, want[1])


def test_second_derivatives_raise_and_changed_ids_too():
    w = torch.randn(20, 8, device=DEV, requires_grad=True)
    ids = torch.tensor([1, 2, 1], device=DEV)
    (dw,) = torch.autograd.grad((token_embedding(ids, w) ** 2).sum(), w, create_graph=True)
    with pytest.raises(RuntimeError, match="second derivative"):
        dw.sum().backward()
    y = token_embedding(ids, w)
    ids.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    with torch.no_grad():
        assert not token_embedding(ids, w).requires_grad


def test_refusals():
    w = torch.randn(20, 64, device=DEV)
    ids = torch.zeros(4, dtype=torch.long, device=DEV)
    with pytest.raises(TypeError, match="float32 or bfloat16"):
        token_embedding(ids, w.half())
    with pytest.raises(TypeError, match="int64 or int32"):
        token_embedding(ids.float(), w)
    with pytest.raises(ValueError, match="padding_idx"):
        token_embedding(ids, w, padding_idx=20)
    with pytest.raises(ValueError, match="padding_idx"):
        token_embedding_bwd(torch.zeros(4, 64, device=DEV), ids, 20, padding_idx=-21)
    with pytest.raises(ValueError, match="grad must be"):
        token_embedding_bwd(torch.zeros(5, 64, device=DEV), ids, 20)
    with pytest.raises(ValueError, match=r"\(V, C\)"):
        token_embedding(ids, w[0])
    with pytest.raises(RuntimeError, match="GPU only"):
        token_embedding(ids.cpu(), w.cpu())
    with pytest.raises(RuntimeError, match="ids is on"):
        token_embedding(ids.cpu(), w)
