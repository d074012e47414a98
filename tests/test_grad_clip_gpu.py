"""global_grad_norm, clip_grads and clip_grad_norm_ against fp64: the norm within one fp32 rounding (2^-24) and 2^-40 for
the fp64 sums, a scaled value within the roundings of the factor, the product and the result's type."""

import math

import pytest
import torch

from _gpu_util import DEV, log
from cdssm_hip import clip_grad_norm_, clip_grads, global_grad_norm

pytestmark = pytest.mark.gpu

HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


def tensors(sizes, dtypes, seed=0, mag=1.0):
    g = torch.Generator().manual_seed(seed)
    return [(mag * (1 + i % 3) * torch.randn(*s, generator=g)).to(dt).to(DEV)
            for i, (s, dt) in enumerate(zip(sizes, dtypes * len(sizes)))]


def exact_norm(ts):
    return math.sqrt(math.fsum(float(t.double().square().sum()) for t in ts if t.numel()))


def check(ts, max_norm, out=None):
    before = [t.clone() for t in ts]
    want = exact_norm(before)
    norm = global_grad_norm(ts)
    assert abs(float(norm) - want) <= (2.0 ** -24 + 2.0 ** -40) * want
    got = clip_grads(ts, max_norm, out=out)
    assert got.dtype == torch.float32 and got.shape == () and torch.equal(got, norm)
    c = min(1.0, max_norm / (want + 1e-6))
    for t, b, o in zip(ts, before, ts if out is None else out):
        if out is not None:
            assert torch.equal(t, b)
        exact = b.double() * c
        off = (o.double() - exact).abs()
        assert bool((off <= exact.abs() * (HALF[o.dtype] + 2.5 * 2.0 ** -24) + 2.0 ** -134).all())
    return norm


@pytest.mark.parametrize("dtypes", [[torch.float32], [torch.bfloat16], [torch.float32, torch.bfloat16]])
@pytest.mark.parametrize("sizes", [
    [(1,)], [(7,), (3, 5), (1, 1, 1)], [(16384,), (16385,), (16383,)], [(128, 3000), (97,), (0,), (5000, 129)],
    [(64, i + 1) for i in range(300)],
], ids=["one", "small", "chunks", "mixed", "many"])
def test_norm_and_clipping(sizes, dtypes):
    for max_norm in (0.5, 0.0, 1e6):
        check(tensors(sizes, dtypes), max_norm)
    ts = tensors(sizes, dtypes, seed=1)
    check(ts, 0.7, out=[torch.full_like(t, float("nan"), dtype=torch.float32) for t in ts])
    ts = tensors(sizes, dtypes, seed=2)
    check(ts, 0.7, out=[torch.full_like(t, float("nan"), dtype=torch.bfloat16) for t in ts])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_views_of_a_bucket_at_any_offset(dtype):
    sizes = [1, 3, 1000, 17, 40000, 5, 8, 1]
    flat = torch.randn(sum(sizes) + 2, device=DEV).to(dtype)
    edge = flat[0].clone(), flat[-1].clone()
    check(list(flat[1:-1].split(sizes)), 0.3)
    assert torch.equal(flat[0], edge[0]) and torch.equal(flat[-1], edge[1])
    out = torch.full((sum(sizes) + 2,), 5.0, device=DEV)
    check(list(flat[1:-1].split(sizes)), 0.3, out=list(out[1:-1].split(sizes)))
    assert float(out[0]) == 5.0 and float(out[-1]) == 5.0
    out = torch.full((sum(sizes) + 3,), 5.0, device=DEV)  # the two sides never reach a 16-byte boundary together
    check(list(flat[1:-1].split(sizes)), 0.3, out=list(out[2:-1].split(sizes)))


def test_neighbours_in_memory():
    """Runs of neighbours of one type, interrupted by another type, a gap, another order, or outputs that lie elsewhere."""
    sizes = [5, 40000, 0, 129, 33000, 7, 64, 100000, 1, 1, 9000]
    for outs in (None, "together", "apart", "halves"):
        flat = tensors([(sum(sizes) + 50,)], [torch.bfloat16], seed=3)[0]
        own = tensors([(70,), (33001,)], [torch.float32, torch.float32], seed=4)
        ts, at = [], 3
        for i, n in enumerate(sizes):
            ts.append(flat[at:at + n])
            at += n + (8 if i == 3 else 0)
        ts = ts[:2] + own[:1] + ts[2:6] + own[1:] + [ts[8], ts[7]] + ts[9:] + [ts[6]]
        rest, out = flat.clone(), None
        if outs == "apart":
            out = [torch.empty_like(t, dtype=torch.float32) for t in ts]
        elif outs:
            into = torch.full((sum(t.numel() for t in ts) + 1,), float("nan"), device=DEV,
                              dtype=torch.float32 if outs == "together" else torch.bfloat16)
            out = list(into[:-1].split([t.numel() for t in ts]))
        check(ts, 0.7, out=out)
        covered = torch.zeros_like(flat, dtype=torch.bool)
        for t in ts:
            if t.dtype == torch.bfloat16 and t.numel():
                covered[t.storage_offset():t.storage_offset() + t.numel()] = True
        assert torch.equal(flat[~covered], rest[~covered])
        if outs in ("together", "halves"):
            assert torch.isnan(into[-1]) and torch.isfinite(into[:-1]).all()


def test_no_clipping_changes_no_bit():
    ts = tensors([(100, 100), (33,)], [torch.bfloat16, torch.float32])
    before = [t.clone() for t in ts]
    clip_grads(ts, 1e6)
    assert all(torch.equal(a, b) for a, b in zip(ts, before))


def test_zero_infinite_and_nan_norms_as_torch_scales_them():
    for special in (0.0, float("inf"), float("nan")):
        ts = tensors([(1000,), (37,)], [torch.float32])
        if special == 0.0:
            [t.zero_() for t in ts]
        else:
            ts[1][5] = special
        ps = [torch.nn.Parameter(torch.zeros_like(t)) for t in ts]
        for p, t in zip(ps, ts):
            p.grad = t.clone()
        want = torch.nn.utils.clip_grad_norm_(ps, 1.0)
        got = clip_grads(ts, 1.0)
        assert torch.equal(got.isnan(), want.isnan()) and (bool(got.isnan()) or float(got) == float(want))
        for p, t in zip(ps, ts):
            assert torch.equal(torch.nan_to_num(p.grad, nan=123.0), torch.nan_to_num(t, nan=123.0))


def test_squares_beyond_fp32():
    ts = [torch.full((4,), 1e25, device=DEV), torch.full((4,), 1e-30, device=DEV)]
    assert float(global_grad_norm(ts)) == pytest.approx(2e25, rel=1e-6)
    check(ts, 1.0)
    tiny = [torch.full((4,), 1e-30, device=DEV)]
    assert float(global_grad_norm(tiny)) == pytest.approx(2e-30, rel=1e-6)


def test_dense_layouts_one_tensor_and_none():
    t = torch.randn(30, 40, device=DEV).t()
    check([t], 0.5)
    c = torch.randn(2, 6, 5, 7, device=DEV).to(memory_format=torch.channels_last)
    check([c], 0.5, out=[torch.empty_like(c)])
    one = torch.randn(100, device=DEV)
    before = one.clone()
    n = clip_grads(one, 0.1)
    assert float(n) == pytest.approx(float(before.norm()), rel=1e-6)
    assert float(global_grad_norm([])) == 0.0 and float(clip_grads([], 1.0)) == 0.0
    assert float(global_grad_norm(torch.empty(0, device=DEV))) == 0.0
    assert float(clip_grads([torch.empty(0, device=DEV)], 1.0)) == 0.0


def test_parameters_with_and_without_gradients():
    ps = [torch.nn.Parameter(torch.randn(50, 20, device=DEV)) for _ in range(3)]
    ps[0].grad, ps[2].grad = torch.randn(50, 20, device=DEV), torch.randn(50, 20, device=DEV)
    want = exact_norm([ps[0].grad, ps[2].grad])
    assert float(clip_grad_norm_(ps, 1.0)) == pytest.approx(want, rel=1e-6)
    assert exact_norm([ps[0].grad, ps[2].grad]) == pytest.approx(1.0, rel=1e-5) and ps[1].grad is None
    assert float(clip_grad_norm_(iter(ps), 10.0)) == pytest.approx(1.0, rel=1e-5)


def test_on_another_stream_and_captured():
    ts = tensors([(300, 70), (129,), (5000,)], [torch.bfloat16, torch.float32])
    outs = [torch.empty_like(t, dtype=torch.float32) for t in ts]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a = clip_grads(ts, 0.5, out=outs)
    torch.cuda.current_stream().wait_stream(side)
    want = [o.clone() for o in outs]
    b = clip_grads(ts, 0.5, out=outs)
    assert torch.equal(a, b) and all(torch.equal(o, w) for o, w in zip(outs, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        n = clip_grads(ts, 0.5, out=outs)
    for k in range(4):
        for t, v in zip(ts, tensors([(300, 70), (129,), (5000,)], [torch.bfloat16, torch.float32], seed=k, mag=k + 0.1)):
            t.copy_(v)
        graph.replay()
        got, gn = [o.clone() for o in outs], n.clone()
        e = [torch.empty_like(o) for o in outs]
        en = clip_grads(ts, 0.5, out=e)
        torch.cuda.synchronize()
        assert torch.equal(gn, en) and all(torch.equal(x, y) for x, y in zip(got, e))


def test_refusals():
    a, b = torch.randn(10, device=DEV), torch.randn(10, device=DEV)
    with pytest.raises(ValueError, match="given twice"):
        clip_grads([a, b, a], 1.0)
    with pytest.raises(ValueError, match="gaps or overlaps"):
        clip_grads([torch.randn(10, 4, device=DEV)[:, :3]], 1.0)
    with pytest.raises(ValueError, match="gaps or overlaps"):
        global_grad_norm([torch.randn(1, 4, device=DEV).expand(3, 4)])
    with pytest.raises(TypeError, match="float32 or bfloat16"):
        clip_grads([a.half()], 1.0)
    with pytest.raises(ValueError, match="max_norm"):
        clip_grads([a], -1.0)
    with pytest.raises(ValueError, match="max_norm"):
        clip_grads([a], float("nan"))
    with pytest.raises(ValueError, match="1 gradients, 2 outputs"):
        clip_grads([a], 1.0, out=[a, b])
    with pytest.raises(ValueError, match="size, layout and device"):
        clip_grads([a], 1.0, out=[b[:9]])
    with pytest.raises(ValueError, match="another gradient's"):
        clip_grads([a, b], 1.0, out=[b, a])
    with pytest.raises(RuntimeError, match="GPU only"):
        global_grad_norm([a.cpu()])
    c = torch.randn(20, device=DEV)
    with pytest.raises(ValueError, match="shares memory"):  # in place, in part the same
        clip_grads([c[:11], c[10:]], 1.0)
    with pytest.raises(ValueError, match="shares memory"):  # an output in part another gradient, and in part its own
        clip_grads([c[:10], c[10:]], 1.0, out=[b, c[5:15]])
    with pytest.raises(ValueError, match="shares memory"):
        clip_grads([c[:10]], 1.0, out=[c[1:11]])
    with pytest.raises(ValueError, match="shares memory"):  # the same place as another type
        clip_grads([c[:10]], 1.0, out=[c.view(torch.bfloat16)[:10]])
    with pytest.raises(TypeError):
        clip_grads([a, None], 1.0)
    clip_grads([c[:10], c[10:]], 1.0)
    assert float(global_grad_norm([c[:11], c[10:]])) > 0.0  # reading twice is no harm


def test_a_graph_that_saved_a_gradient_notices_its_clipping():
    a = torch.randn(50, device=DEV, requires_grad=True)
    (h,) = torch.autograd.grad((a ** 3).sum(), a)
    z = (a * h).sum()  # saves h
    clip_grads([h], 0.1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        z.backward()
    v = torch.ones(5, device=DEV)
    before = v._version
    clip_grads([torch.ones(5, device=DEV)], 0.1, out=[v])
    assert v._version > before


def test_an_output_may_be_its_own_gradient():
    ts = tensors([(100,), (33,)], [torch.bfloat16, torch.float32])
    want = [t.clone() for t in ts]
    clip_grads(want, 0.5)
    other = torch.empty_like(ts[1])
    clip_grads(ts, 0.5, out=[ts[0], other])
    assert torch.equal(ts[0], want[0]) and torch.equal(other, want[1])
