"""distillation_loss and its gradient against the definition in 64 bits on the CPU.

Tolerances, before any run: with A the largest |x - max| / tau of a row (teacher's list included), every exponential is off by at
most 2^-24 (3 A + 4) relative (two roundings of the argument, the rounded 1 / tau, the function's own 2 ulp), and a lane's sum
of n = V / 64 + 16 terms by n 2^-24 more; log q and log p are off by the same, absolutely, and their own rounding 2^-24 A.  So with
e = 2^-24 (4 A + n + K + 16): a token's loss by 2 tau^2 e (1 + |log ratio|), its gradient by |s| tau e (q + p), and by half a step
of its type.  Losses are added in 64 bits."""

import pytest
import torch

from _gpu_util import DEV, log

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp32": torch.float32}
INF = float("inf")


def definition(x, z, ids, tau, weight):
    """(each token's loss, gradient, error bounds of both) in 64 bits; weight: the upstream gradient of each token."""
    x, z, ids, weight = x.detach().cpu().double(), z.cpu().double(), ids.cpu().long(), weight.cpu().double()
    T, V = x.shape
    K = z.shape[1]
    each, grad = torch.zeros(T, dtype=torch.float64), torch.zeros(T, V, dtype=torch.float64)
    e_each, e_grad = torch.zeros_like(each), torch.zeros_like(grad)
    for t in range(T):
        part = z[t] != -INF
        if not part.any():
            continue
        zt, it = z[t][part] / tau, ids[t][part]
        if not ((it >= 0) & (it < V)).all():
            each[t] = float("nan")
            grad[t] = float("nan")
            continue
        logp = zt - torch.logsumexp(zt, 0)
        xs = (x[t] - x[t].max()) / tau  # (the maximum first: in 64 bits too a logit of -3e38 leaves log V no place)
        logq = xs - torch.logsumexp(xs, 0)
        p = logp.exp()
        counts = p > 2.0 ** -149
        each[t] = tau ** 2 * (p * (logp - logq[it]))[counts].sum()
        full = torch.zeros(V, dtype=torch.float64).index_add_(0, it, p)
        grad[t] = weight[t] * tau * (logq.exp() - full)
        finite = x[t][torch.isfinite(x[t])]
        A = max(float(finite.max() - finite.min()) / tau if finite.numel() else 0.0, float(zt.max() - zt.min()))
        e = 2.0 ** -24 * (4 * A + V / 64 + 16 + K + 16)
        ratio = float((logp - logq[it]).abs().max())
        e_each[t] = 2 * tau ** 2 * e * (1 + (ratio if ratio < 1e30 else 0.0))
        e_grad[t] = weight[t].abs() * tau * e * (logq.exp() + full)
    return each, grad, e_each, e_grad


def inputs(T, V, K, dtype, tdtype, seed, ids="any", empty=0.2, short=0.2):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(T, V, generator=g).mul_(3)
    z = torch.randn(T, K, generator=g).mul_(4)
    if ids == "distinct":
        i = torch.stack([torch.randperm(V, generator=g)[:K] for _ in range(T)])
    else:
        i = torch.randint(0, V, (T, K), generator=g)  # some twice
    short_rows = torch.rand(T, generator=g) < short
    z[short_rows, K // 2:] = -INF
    z[torch.rand(T, generator=g) < empty] = -INF
    return x.to(DT[dtype]).to(DEV), z.to(DT[tdtype]).to(DEV), i.to(DEV)


def check(x, z, ids, tau, reduction, up=None):
    from cdssm_hip import distillation_loss
    x = x.detach().requires_grad_(True)
    loss = distillation_loss(x, z, ids, temperature=tau, reduction=reduction)
    assert loss.dtype == torch.float32 and loss.shape == (x.shape[:-1] if reduction == "none" else ())
    g, = torch.autograd.grad(loss, x, up)
    torch.cuda.synchronize()
    rows = x.reshape(-1, x.shape[-1])
    T = rows.shape[0]
    z2, i2 = z.reshape(T, -1), ids.reshape(T, -1)
    has = (z2 != -INF).any(1).cpu()
    count = int(has.sum())
    w = torch.ones(T) if up is None else up.reshape(-1).cpu() if reduction == "none" else up.cpu().expand(T)
    w = w.double() / (max(1, count) if reduction == "mean" else 1)
    each, grad, e_each, e_grad = definition(rows, z2, i2, tau, w)
    if reduction == "none":
        want, tol = each, e_each + 2.0 ** -24 * each.abs()
    elif reduction == "sum":
        want, tol = each.sum(), e_each.sum() + 2.0 ** -24 * each.sum().abs()
    else:
        want = each.sum() / count if count else torch.tensor(float("nan"), dtype=torch.float64)
        tol = e_each.sum() / max(1, count) + 2.0 ** -24 * want.abs()
    close(loss.detach().cpu().double().reshape(want.shape), want, tol)
    assert g.dtype == x.dtype and g.shape == x.shape
    got = g.cpu().double().reshape(grad.shape)
    close(got, grad, e_grad + torch.finfo(x.dtype).eps / 2 * grad.abs() + torch.finfo(x.dtype).smallest_normal)
    assert (got[~has] == 0).all()


def close(got, want, tol):
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    odd = ~torch.isfinite(want)
    assert torch.equal(got[odd & ~torch.isnan(want)], want[odd & ~torch.isnan(want)])
    diff = (got - want).abs()[~odd]
    off = torch.where(diff == 0, 0.0, diff / tol[~odd] if tol.dim() else diff / tol)
    if off.numel():
        log(f"  worst {float(off.max()):.3f} of the bound")
        assert float(off.max()) <= 1.0


@pytest.mark.parametrize("dtype,tdtype", [("bf16", "bf16"), ("fp32", "fp32"), ("bf16", "fp32"), ("fp32", "bf16")])
@pytest.mark.parametrize("T,V,K,tau,reduction", [
    (1, 1, 1, 1.0, "mean"), (2, 3, 5, 1.0, "sum"), (5, 17, 8, 2.0, "none"), (200, 97, 8, 1.0, "mean"), (33, 1000, 64, 0.7, "sum"),
    (70, 1001, 65, 4.0, "none"), (40, 513, 256, 1.0, "mean"), (4, 50257, 128, 1.0, "none"), (600, 301, 16, 2.0, "mean"),
    (511, 130, 3, 1.0, "none"), (4100, 61, 4, 1.0, "mean")])
def test_loss_and_gradient(T, V, K, tau, reduction, dtype, tdtype):
    log(f"[distill] T{T} V{V} K{K} tau {tau} {reduction} {dtype} {tdtype}")
    x, z, ids = inputs(T, V, K, dtype, tdtype, seed=T + V + K)
    up = torch.randn(T, generator=torch.Generator().manual_seed(1)).to(DEV) if reduction == "none" else None
    check(x, z, ids, tau, reduction, up)


def test_upstream_gradients_of_one_number():
    x, z, ids = inputs(20, 50, 6, "fp32", "fp32", 3)
    check(x, z, ids, 1.5, "mean", torch.tensor(-0.37, device=DEV))
    check(x, z, ids, 1.5, "sum", torch.tensor(2.5, device=DEV))


def test_ids_of_four_bytes_and_leading_dimensions():
    x, z, ids = inputs(12, 40, 5, "bf16", "fp32", 4)
    check(x.view(3, 4, 40), z.view(3, 4, 5), ids.int().view(3, 4, 5), 1.0, "mean")
    check(x[0], z[0], ids[0].int(), 1.0, "sum")
    up = torch.randn(3, 1, device=DEV).expand(3, 4)
    check(x.view(3, 4, 40), z.view(3, 4, 5), ids.view(3, 4, 5), 1.0, "none", up)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("T,V,lead,pad", [(5, 96, 0, 32), (5, 97, 0, 31), (5, 97, 1, 2), (600, 333, 3, 4), (4100, 41, 0, 7),
                                          (3, 97, 0, 3000)])
def test_slices_of_wider_rows(T, V, lead, pad, dtype):
    """Logits as a slice of padded rows: nothing outside it is read, the gradient is dense or strided, its values the same."""
    x, z, ids = inputs(T, V, 6, dtype, dtype, 5)
    wide = torch.full((T, lead + V + pad), float("nan"), dtype=x.dtype, device=DEV)
    wide[:, lead:lead + V] = x
    check(wide[:, lead:lead + V], z, ids, 1.0, "mean")


def test_no_dense_rows_and_broadcast_rows():
    x, z, ids = inputs(20, 64, 6, "fp32", "fp32", 6)
    check(x.t().contiguous().t(), z, ids, 1.0, "mean")
    check(x[:1].expand(20, 64), z, ids, 1.0, "mean")
    check(x, z[:1].expand(20, 6), ids[:1].expand(20, 6), 1.0, "mean")
    base = x[:1].clone().requires_grad_(True)
    from cdssm_hip import distillation_loss
    g, = torch.autograd.grad(distillation_loss(base.expand(20, 64), z, ids, reduction="sum"), base)
    _, grad, _, e = definition(base.expand(20, 64), z, ids, 1.0, torch.ones(20))
    want = grad.sum(0)
    assert ((g.cpu().double()[0] - want).abs() <= e.sum(0) + 2.0 ** -24 * 40 * grad.abs().sum(0)).all()


def test_words_listed_twice_and_lists_longer_than_the_vocabulary():
    x, z, ids = inputs(30, 4, 12, "fp32", "fp32", 7)
    check(x, z, ids, 1.0, "mean")
    check(x, z, torch.full_like(ids, 2), 1.0, "sum")


@pytest.mark.parametrize("T", [4, 600, 4100])
def test_infinities_nan_and_masks(T):
    x, z, ids = inputs(T, 50, 6, "fp32", "fp32", 8, empty=0.0, short=0.0, ids="distinct")
    z[0] = -INF                                   # no teacher: whatever the logits hold
    x[0] = float("nan")
    x[1, ::2] = -INF                              # half of the words masked
    z[1] = torch.where(ids[1] % 2 == 0, -INF, z[1])
    x[2, ids[2, 0]] = -INF                        # the teacher's word masked: an infinite loss
    x[3, :] = torch.finfo(torch.float32).min      # equal logits of the lowest value
    check(x, z, ids, 1.0, "none", torch.ones(T, device=DEV))


@pytest.mark.parametrize("bad", ["nan", "inf", "all -inf", "teacher nan", "teacher inf"])
def test_a_token_without_a_distribution_is_nan_and_alone(bad):
    from cdssm_hip import distillation_loss
    x, z, ids = inputs(6, 50, 6, "fp32", "fp32", 9, empty=0.0)
    clean = distillation_loss(x, z, ids, reduction="none")
    if bad == "all -inf":
        x[2] = -INF
    elif bad.startswith("teacher"):
        z[2, 1] = float(bad.split()[1])
    else:
        x[2, 7] = float(bad)
    x.requires_grad_(True)
    loss = distillation_loss(x, z, ids, reduction="none")
    g, = torch.autograd.grad(loss, x, torch.ones(6, device=DEV))
    assert torch.isnan(loss[2]) and torch.isnan(g[2]).all()
    keep = [0, 1, 3, 4, 5]
    assert torch.equal(loss[keep], clean[keep]) and torch.isfinite(g[keep]).all()


@pytest.mark.parametrize("bad", [-1, 50, 2 ** 31, -2 ** 40])
def test_an_id_out_of_range_is_nan_unless_it_takes_no_part(bad):
    x, z, ids = inputs(6, 50, 6, "fp32", "fp32", 10, empty=0.0)
    ids[2, 3] = bad
    z[2, 3] = 1.0
    ids[4, 2] = bad
    z[4, 2] = -INF
    check(x, z, ids, 1.0, "none", torch.ones(6, device=DEV))


def test_large_logits_and_temperatures():
    x, z, ids = inputs(8, 200, 6, "fp32", "fp32", 11, empty=0.0)
    check(x + 3e8, z, ids, 1.0, "mean")
    check(x * 100, z * 100, ids, 100.0, "mean")
    check(x * 0.01, z * 0.01, ids, 0.01, "mean")


def test_no_tokens():
    from cdssm_hip import distillation_loss
    x = torch.empty(0, 50, device=DEV, requires_grad=True)
    z, ids = torch.empty(0, 4, device=DEV), torch.empty(0, 4, device=DEV, dtype=torch.long)
    for reduction in ("mean", "sum", "none"):
        loss = distillation_loss(x, z, ids, reduction=reduction)
        assert torch.isnan(loss) if reduction == "mean" else float(loss.detach().sum()) == 0
        g, = torch.autograd.grad(loss.sum(), x)
        assert g.shape == x.shape
    x = torch.randn(3, 50, device=DEV, requires_grad=True)
    loss = distillation_loss(x, torch.full((3, 4), -INF, device=DEV), torch.zeros(3, 4, device=DEV, dtype=torch.long))
    g, = torch.autograd.grad(loss, x)
    assert torch.isnan(loss) and (g == 0).all()


def test_the_gradient_against_differences():
    """Steps of 2^-10 along single logits in the definition, in 64 bits, give the gradient to the step's square."""
    from cdssm_hip import distillation_loss
    x, z, ids = inputs(3, 30, 5, "fp32", "fp32", 12, empty=0.0)
    x.requires_grad_(True)
    g, = torch.autograd.grad(distillation_loss(x, z, ids, 1.3, "sum"), x)
    h = 2.0 ** -10
    one = torch.ones(3)
    for t, v in [(0, 3), (1, int(ids[1, 0])), (2, int(ids[2, 4])), (2, 29)]:
        d = torch.zeros(3, 30, dtype=torch.float64)
        d[t, v] = h
        up, down = (definition(x.detach().cpu().double() + s * d, z, ids, 1.3, one)[0].sum() for s in (1, -1))
        # third derivatives of the loss are at most tau^-1 in size
        assert abs(float(g[t, v]) - float(up - down) / (2 * h)) <= h * h + 2e-6


def test_the_same_bits_every_time_and_on_another_stream():
    from cdssm_hip import distillation_loss
    x, z, ids = inputs(700, 1003, 16, "bf16", "bf16", 13)
    x.requires_grad_(True)

    def run():
        loss = distillation_loss(x, z, ids)
        return loss.detach(), torch.autograd.grad(loss, x)[0]
    a = run()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        b = run()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_captured_forward_and_backward():
    from cdssm_hip import distillation_loss
    x, z, ids = inputs(300, 501, 16, "fp32", "fp32", 14)
    x.requires_grad_(True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(distillation_loss(x, z, ids), x)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss = distillation_loss(x, z, ids)
        g, = torch.autograd.grad(loss, x)
    for seed in range(4):
        nx, nz, nids = inputs(300, 501, 16, "fp32", "fp32", 20 + seed)
        with torch.no_grad():
            x.copy_(nx)
        z.copy_(nz)
        ids.copy_(nids)
        graph.replay()
        torch.cuda.synchronize()
        y = nx.requires_grad_(True)
        want = distillation_loss(y, nz, nids)
        wg, = torch.autograd.grad(want, y)
        torch.cuda.synchronize()
        assert torch.equal(loss, want) and torch.equal(g, wg)


def test_logits_that_changed_since_are_noticed():
    from cdssm_hip import distillation_loss
    x, z, ids = inputs(5, 20, 3, "fp32", "fp32", 15)
    x.requires_grad_(True)
    y = x * 1.0
    loss = distillation_loss(y, z, ids)
    y.mul_(2.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_the_calls_without_autograd_give_the_same_bits(reduction):
    from cdssm_hip import distillation_loss
    from cdssm_hip.distill import distillation_loss_bwd, distillation_loss_fwd
    x, z, ids = inputs(50, 201, 9, "bf16", "fp32", 17)
    up = torch.randn(50, device=DEV) if reduction == "none" else torch.tensor(0.7, device=DEV)
    loss, ws = distillation_loss_fwd(x, z, ids, 2.0, reduction)
    g = distillation_loss_bwd(up, x, z, ids, ws, 2.0, reduction)
    y = x.clone().requires_grad_(True)
    want = distillation_loss(y, z, ids, 2.0, reduction)
    assert torch.equal(loss, want.detach()) and torch.equal(g, torch.autograd.grad(want, y, up)[0])
    for bad in (None, ws[:-1], ws.cpu()):
        with pytest.raises(ValueError, match="not the workspace"):
            distillation_loss_bwd(up, x, z, ids, bad, 2.0, reduction)
    with pytest.raises(ValueError, match="the gradient of logits"):
        distillation_loss_bwd(torch.ones(7, device=DEV), x, z, ids, ws, 2.0, reduction)
    e, ws = distillation_loss_fwd(x[:0], z[:0], ids[:0], 1.0, reduction)
    assert ws is None
    up = torch.empty(0, device=DEV) if reduction == "none" else up
    assert distillation_loss_bwd(up, x[:0], z[:0], ids[:0], None, 1.0, reduction).shape == (0, 201)


def test_refusals_that_need_tensors_on_the_gpu():
    from cdssm_hip import distillation_loss, top_logits
    x, z, ids = inputs(6, 20, 3, "fp32", "fp32", 18)
    for call, error, msg in (
            (lambda: distillation_loss(x.double(), z, ids), TypeError, "logits must be"),
            (lambda: distillation_loss(x, z.half(), ids), TypeError, "teacher_logits must be"),
            (lambda: distillation_loss(x, z, ids.short()), TypeError, "teacher_ids must be"),
            (lambda: distillation_loss(x, z.cpu(), ids), RuntimeError, "teacher_logits on cpu"),
            (lambda: distillation_loss(x, z, ids.cpu()), RuntimeError, "teacher_ids on"),
            (lambda: distillation_loss(x, z[:5], ids[:5]), ValueError, "K of 1 .. 256"),
            (lambda: distillation_loss(x, z[:, :2], ids), ValueError, "K of 1 .. 256"),
            (lambda: distillation_loss(x, z[:, :0], ids[:, :0]), ValueError, "K of 1 .. 256"),
            (lambda: distillation_loss(x, z.repeat(1, 100), ids.repeat(1, 100)), ValueError, "K of 1 .. 256"),
            (lambda: distillation_loss(x, z, ids, temperature=0.0), ValueError, "temperature"),
            (lambda: distillation_loss(x, z, ids, temperature=float("nan")), ValueError, "temperature"),
            (lambda: distillation_loss(x, z, ids, reduction="batchmean"), ValueError, "reduction"),
            (lambda: top_logits(x.half(), 3), TypeError, "logits must be"),
            (lambda: top_logits(x, 0), ValueError, "k must be"),
            (lambda: top_logits(x, 21), ValueError, "k must be"),
            (lambda: top_logits(x.repeat(1, 10), 129), ValueError, "k must be"),
            (lambda: top_logits(x[:, :0], 1), ValueError, "V >= 1")):
        with pytest.raises(error, match=msg):
            call()


def test_derivatives_that_are_not_there_raise():
    from cdssm_hip import distillation_loss
    x, z, ids = inputs(5, 20, 3, "fp32", "fp32", 16, empty=0.0)
    x.requires_grad_(True)
    g, = torch.autograd.grad(distillation_loss(x, z, ids), x, create_graph=True)
    with pytest.raises(RuntimeError, match="no second derivative"):
        torch.autograd.grad(g.square().sum(), x)
    with pytest.raises(NotImplementedError, match="no gradient to teacher_logits"):
        distillation_loss(x, z.clone().requires_grad_(True), ids)


def test_more_logits_than_32_bits_hold():
    """Rows on either side of 2^31 elements have the bits of the same rows alone (in runs of the same launch shape)."""
    from cdssm_hip.distill import distillation_loss_bwd, distillation_loss_fwd
    T, V, K = 68000, 32000, 4
    g = torch.Generator(device=DEV).manual_seed(0)
    x = torch.empty(T, V, dtype=torch.bfloat16, device=DEV).normal_(generator=g)
    z = torch.randn(T, K, device=DEV, generator=g)
    ids = torch.randint(0, V, (T, K), device=DEV, generator=g)
    up = torch.randn(T, device=DEV, generator=g)
    loss, ws = distillation_loss_fwd(x, z, ids, 1.0, "none")
    grad = distillation_loss_bwd(up, x, z, ids, ws, 1.0, "none")
    for lo in (0, 65000):
        rows = slice(lo, lo + 3000)
        want, ws = distillation_loss_fwd(x[rows], z[rows], ids[rows], 1.0, "none")
        assert torch.equal(loss[rows], want)
        assert torch.equal(grad[rows], distillation_loss_bwd(up[rows], x[rows], z[rows], ids[rows], ws, 1.0, "none"))


@pytest.mark.parametrize("ld,V", [(128, 97), (104, 97), (99, 97), (131, 130)])
def test_what_lies_between_the_gradient_s_rows_stays(ld, V):
    from cdssm_hip import _lib
    x, z, ids = inputs(5, V, 4, "fp32", "fp32", 19)
    wide = torch.full((5, ld), -7.0, device=DEV)
    lib, stream = _lib.load(), _lib.stream_of(DEV)
    loss = torch.empty((), device=DEV)
    ws = torch.empty(lib.cdssm_distillation_workspace_bytes(5), dtype=torch.uint8, device=DEV)
    up = torch.ones((), device=DEV)
    args = (0, 0, 8, x.data_ptr(), V, z.data_ptr(), ids.data_ptr(), 1.0, 2)
    _lib.check(lib.cdssm_distillation_fwd(*args, loss.data_ptr(), ws.data_ptr(), 5, V, 4, stream), "fwd")
    _lib.check(lib.cdssm_distillation_bwd(*args, up.data_ptr(), ws.data_ptr(), wide.data_ptr(), ld, 5, V, 4, stream), "bwd")
    y = x.clone().requires_grad_(True)
    from cdssm_hip import distillation_loss
    want, = torch.autograd.grad(distillation_loss(y, z, ids, reduction="sum"), y)
    torch.cuda.synchronize()
    assert torch.equal(wide[:, :V], want) and (wide[:, V:] == -7.0).all()


@pytest.mark.parametrize("reduction", ["none", "mean"])
@pytest.mark.parametrize("low,tau", [(-1e9, 1.0), (float(torch.finfo(torch.float32).min), 1.0), (-20.0, 0.05), (-20.0, 1.0)])
@pytest.mark.parametrize("bad", [-1, 50])
def test_an_id_out_of_range_is_nan_at_any_probability(bad, low, tau, reduction):
    """A list padded with an id that no word has and a low, finite logit: probabilities that fp32 holds as 0, and one that it does
    not.  Loss and gradient follow the same rule."""
    x, z, ids = inputs(6, 50, 6, "fp32", "fp32", 21, empty=0.0, short=0.0)
    ids[2, 3:] = bad
    z[2, 3:] = low
    check(x, z, ids, tau, reduction, torch.ones(6, device=DEV) if reduction == "none" else None)


def test_teacher_probabilities_below_the_normal_numbers():
    """e^-95 = 2^-137 is a probability that fp32 holds, if only as a subnormal number: a word of it that the student rules out
    makes the loss infinite.  e^-110 = 2^-159 is none."""
    x, z, ids = inputs(3, 50, 2, "fp32", "fp32", 22, empty=0.0, short=0.0, ids="distinct")
    z[:, 0], z[:, 1] = 0.0, torch.tensor([-95.0, -110.0, -80.0], device=DEV)
    x[torch.arange(3), ids[:, 1]] = -INF
    check(x, z, ids, 1.0, "none", torch.ones(3, device=DEV))


@pytest.mark.parametrize("T", [16384, 16385, 50021])
def test_losses_of_many_tokens_as_one(T):
    """The sum goes through 16384 tokens a round; the last round is a whole one, one token, and any number of them.  It is formed in 64
    bits and rounded once, from the tokens' own losses.  A gradient is r (q - p) with r q and r p rounded apart: six roundings lie
    between that of the sum and count times that of the mean (the upstream gradient over the count, its product with 1 / sum, both sides'
    products with the exponential and their last ones), each of at most 2^-24 (q + p), where q + p = 2 q - (q - p)."""
    from cdssm_hip import distillation_loss
    x, z, ids = inputs(T, 9, 3, "fp32", "fp32", 23)
    x.requires_grad_(True)
    each = distillation_loss(x, z, ids, reduction="none").detach().double().cpu()
    count = int((z != -INF).any(1).sum())
    g, = torch.autograd.grad(distillation_loss(x, z, ids, reduction="sum"), x)
    q = torch.softmax(x.detach().double(), 1)
    for reduction, by in (("sum", 1), ("mean", count)):
        loss = distillation_loss(x, z, ids, reduction=reduction)
        assert abs(float(loss.detach()) - float(each.sum()) / by) <= 2.0 ** -23 * float(each.sum()) / by
        got, = torch.autograd.grad(loss, x)
        assert ((got.double() * by - g.double()).abs() <= 6 * 2.0 ** -24 * (2 * q - g.double())).all()
        assert (got[(z == -INF).all(1)] == 0).all()


def test_a_single_row_of_any_stride():
    """No second row is reached by a single row's stride, so it may have any."""
    from cdssm_hip import top_logits
    x, z, ids = inputs(1, 50, 6, "fp32", "fp32", 24, empty=0.0)
    far = x.as_strided((1, 50), (2 ** 33, 1))
    check(far, z, ids, 1.0, "mean")
    assert all(torch.equal(a, b) for a, b in zip(top_logits(far, 5), top_logits(x, 5)))
