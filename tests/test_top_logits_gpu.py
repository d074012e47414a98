"""top_logits against a stable sort of whole numbers that order (value, id) on the CPU: equal bits, equal ids."""

import pytest
import torch

from _gpu_util import DEV, log

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp32": torch.float32}


def oracle(x, k):
    """values, ids: the k largest by (value, then lower id); -0 equals 0, NaN above all."""
    x = x.cpu()
    bits = (x.float() + 0.0).view(torch.int32).long()
    order = torch.where(bits < 0, -2 ** 31 - bits, bits)
    order = torch.where(torch.isnan(x), 2 ** 40, order)
    ids = torch.sort(order, dim=-1, descending=True, stable=True).indices[..., :k]
    return x.gather(-1, ids), ids


def same_bits(a, b):
    kind = torch.int16 if a.dtype == torch.bfloat16 else torch.int32
    return torch.equal(a.cpu().contiguous().view(kind), b.cpu().contiguous().view(kind))


def check(x, k):
    from cdssm_hip import top_logits
    v, i = top_logits(x, k)
    torch.cuda.synchronize()
    wv, wi = oracle(x, k)
    assert v.dtype == x.dtype and i.dtype == torch.int64 and v.shape == i.shape == wi.shape
    assert torch.equal(i.cpu(), wi) and same_bits(v, wv)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("T,V,k", [
    (1, 1, 1), (3, 2, 2), (1, 63, 63), (5, 64, 64), (2, 65, 65), (4, 129, 128), (1, 1000, 1), (7, 1001, 50),
    (64, 32000, 50), (300, 777, 100), (511, 4099, 33), (512, 4099, 64), (700, 3001, 65), (2047, 520, 5), (2048, 521, 5),
    (2100, 1025, 128), (9, 50257, 128), (1, 262144, 64), (3, 131071, 127)])
def test_top_logits_of_normal_rows(T, V, k, dtype):
    log(f"[top] T{T} V{V} k{k} {dtype}")
    g = torch.Generator().manual_seed(T * V + k)
    check(torch.randn(T, V, generator=g).mul_(3).to(DT[dtype]).to(DEV), k)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("T", [2, 600, 2100])
@pytest.mark.parametrize("kind", ["constant", "ties", "rising", "falling", "masked", "all_masked", "nan", "zeros", "infinite"])
def test_rows_of_every_order(kind, T, dtype):
    log(f"[top] {kind} T{T} {dtype}")
    V = 3001
    g = torch.Generator().manual_seed(T)
    x = torch.randn(T, V, generator=g)
    if kind == "constant":
        x = torch.full((T, V), -2.5)
    elif kind == "ties":
        x = torch.randint(-3, 4, (T, V), generator=g).float()
    elif kind == "rising":
        x = (torch.arange(V) // 5).float().expand(T, V).clone()
    elif kind == "falling":
        x = -(torch.arange(V) // 5).float().expand(T, V).clone()
    elif kind == "masked":  # fewer words than k are left in most rows, and masks of the lowest value
        x[torch.rand(T, V, generator=g) < 0.99] = -float("inf")
        x[::2][x[::2] == -float("inf")] = torch.finfo(DT[dtype]).min
    elif kind == "all_masked":
        x = torch.full((T, V), -float("inf"))
    elif kind == "nan":
        x[torch.rand(T, V, generator=g) < 0.02] = float("nan")
        x[0] = -torch.tensor(float("nan"))
    elif kind == "zeros":
        x = torch.where(torch.rand(T, V, generator=g) < 0.5, 0.0, -0.0)
        x[:, 100] = 1e-41  # a subnormal number lies above them
        x[:, 200] = -1e-41
    elif kind == "infinite":
        x[torch.rand(T, V, generator=g) < 0.005] = float("inf")
        x[torch.rand(T, V, generator=g) < 0.005] = -float("inf")
    for k in (1, 40, 64, 90, 128):
        check(x.to(DT[dtype]).to(DEV), k)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("T,V,lead,pad", [(5, 500, 1, 3), (600, 501, 3, 0), (2100, 333, 5, 8), (1, 97, 7, 1)])
def test_rows_that_start_anywhere(T, V, lead, pad, dtype):
    """A slice of wider rows, whose ends would be the largest if they were read."""
    g = torch.Generator().manual_seed(V)
    wide = torch.full((T, lead + V + pad), float("inf"))
    wide[:, lead:lead + V] = torch.randn(T, V, generator=g)
    check(wide.to(DT[dtype]).to(DEV)[:, lead:lead + V], 20)


def test_leading_dimensions_and_views():
    from cdssm_hip import top_logits
    x = torch.randn(2, 3, 100, device=DEV)
    check(x, 7)
    check(x.transpose(0, 1), 7)
    check(x.transpose(1, 2), 3)                       # no dense rows: copied
    check(x[0, 0], 5)
    check(x[:1, :1].expand(4, 3, 100), 9)
    v, i = top_logits(torch.empty(0, 100, device=DEV), 7)
    assert v.shape == i.shape == (0, 7)


def test_captured_and_replayed_on_new_logits():
    from cdssm_hip import top_logits
    x = torch.randn(64, 5000, device=DEV)
    top_logits(x, 50)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        v, i = top_logits(x, 50)
    for seed in range(4):
        x.copy_(torch.randn(64, 5000, generator=torch.Generator().manual_seed(seed)))
        graph.replay()
        wv, wi = top_logits(x, 50)
        torch.cuda.synchronize()
        assert torch.equal(v, wv) and torch.equal(i, wi)
        assert torch.equal(i.cpu(), oracle(x, 50)[1])


def test_two_streams_at_once():
    from cdssm_hip import top_logits
    xs = [torch.randn(700, 4001, device=DEV) for _ in range(2)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    out = []
    for _ in range(3):
        for s, x in zip(streams, xs):
            with torch.cuda.stream(s):
                out.append((x, top_logits(x, 40)))
    torch.cuda.synchronize()
    for x, (v, i) in out:
        assert torch.equal(i.cpu(), oracle(x, 40)[1])


def test_a_gradient_is_refused():
    from cdssm_hip import top_logits
    x = torch.randn(4, 50, device=DEV, requires_grad=True)
    with pytest.raises(NotImplementedError, match="no gradient"):
        top_logits(x, 3)
    with torch.no_grad():
        check(x, 3)


def test_more_elements_than_32_bits_hold():
    from cdssm_hip import top_logits
    T, V = 68000, 32000  # 2.2e9 logits
    x = torch.empty(T, V, dtype=torch.bfloat16, device=DEV).normal_(generator=torch.Generator(device=DEV).manual_seed(0))
    v, i = top_logits(x, 7)
    for rows in (slice(0, 3), slice(67100, 67110), slice(T - 3, T)):  # either side of 2^31 elements
        wv, wi = oracle(x[rows], 7)
        assert torch.equal(i[rows].cpu(), wi) and same_bits(v[rows], wv)
