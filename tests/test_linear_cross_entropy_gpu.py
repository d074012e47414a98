"""linear_cross_entropy against its formula in fp64 on the same inputs.

Bounds, elementwise, from the arithmetic (u = 2^-24, half a step of fp32; b = 2^-8, half a step of bf16):
  logits   d products summed in fp32: e_l = (d + 16) u sum_k |x_k w_k| (fp32 operands enter as three bf16 planes, six
           plane products kept: the dropped ones add at most 4 u of the same sum, and the sum has 6 d terms)
  loss     two logits' errors and a few fp32 roundings of numbers up to |lse|: 2 e_l + 16 u (1 + |lse|)
  g        relative error of p: that of 2^(..): e_p = 2 e_l + 16 u (1 + |lse|) (arguments below 1: e^x - 1 <= 2 x), and
           its rounding: b |g| in bf16; as three planes in fp32: 2 u |g|.  fp32 holds no normal number below 2^-126,
           so a probability below it (a logit 88 under the maximum) is 0: at most 2^-126 off, whatever its relative
           error, and so are products and sums that fall below it
  dx, dW   sums of n terms: (n + 16) u sum |g| |w|, the errors of g, and the result's rounding
"""

import pytest
import torch

from _gpu_util import DEV, log
from cdssm_hip import linear_cross_entropy
from cdssm_hip.train import linear_cross_entropy_bwd, linear_cross_entropy_fwd

pytestmark = pytest.mark.gpu

U, B16 = 2.0 ** -24, 2.0 ** -8
TINY = 2.0 ** -126
IGNORE = -100


def make(T, V, d, dtype, seed=0, ignored=0.0, spread=1.0, shape=None):
    g = torch.Generator().manual_seed(seed)
    w = torch.randn(V, d, generator=g) / d ** 0.5
    y = torch.randint(0, V, (T,), generator=g)
    x = spread * torch.randn(T, d, generator=g) + 6 * torch.rand(T, 1, generator=g) * w[y]
    y[torch.rand(T, generator=g) < ignored] = IGNORE
    return x.to(dtype).to(DEV), w.to(dtype).to(DEV), y.to(DEV), torch.randn(T, generator=g).to(DEV)


def reference(x, w, y, up, reduction, ignore=IGNORE):
    """loss, dx, dW and their bounds, fp64."""
    half = x.dtype == torch.bfloat16
    keep = y != ignore
    x, w, up = x.double()[keep], w.double(), up.double()[keep]
    at = y[keep].long()
    n, d = x.shape
    terms = d if half else 6 * d
    l = x @ w.t()
    e_l = (terms + 16) * U * (x.abs() @ w.abs().t()).amax(1)
    lse = torch.logsumexp(l, 1)
    each = lse - l.gather(1, at[:, None])[:, 0]
    e_loss = 2 * e_l + 16 * U * (1 + lse.abs())
    p = torch.exp(l - lse[:, None])
    g = p.clone()
    g.scatter_add_(1, at[:, None], -torch.ones_like(g[:, :1]))
    s = up if reduction == "none" else torch.full_like(each, 1.0 / max(n, 1)) if reduction == "mean" else torch.ones_like(each)
    if reduction != "none":
        s = s * up_scalar(up)
    g = g * s[:, None]
    e_g = p * s.abs()[:, None] * 2 * e_loss[:, None] + g.abs() * (B16 + 4 * U if half else 6 * U) + TINY * (1 + s.abs()[:, None])
    out = B16 if half else U
    dx, dw = g @ w, g.t() @ x
    k = 1 if half else 6
    e_dx = e_g @ w.abs() + (k * w.shape[0] + 16) * U * (g.abs() @ w.abs())
    e_dw = e_g.t() @ x.abs() + (k * n + 16) * U * (g.abs().t() @ x.abs())
    e_dx, e_dw = e_dx + TINY * w.shape[0], e_dw + TINY * max(n, 1)
    e_dx, e_dw = e_dx + out * (dx.abs() + e_dx), e_dw + out * (dw.abs() + e_dw)
    full = lambda v: torch.zeros(keep.shape[0], *v.shape[1:], dtype=v.dtype, device=v.device).index_put((keep,), v)  # noqa: E731
    if reduction == "none":
        loss, e = full(each), full(e_loss + U * each.abs())
    else:
        loss, e = each.sum(), e_loss.sum()
        if reduction == "mean":
            loss, e = loss / n, e / max(n, 1)
        e = e + U * loss.abs()
    return loss, e, full(dx), full(e_dx), dw, e_dw


def up_scalar(up):
    return 0.75


def within(name, got, want, bound):
    got = got.detach().double()
    assert torch.isfinite(got).all(), f"{name}: not finite"
    off = (got - want).abs()
    worst = float((off / (bound + 1e-300)).max()) if off.numel() else 0.0
    log(f"  {name}: {worst:.3f} of its bound")
    assert bool((off <= bound).all()), f"{name}: {worst:.3f} of its bound"


def check(x, w, y, up, reduction, **kw):
    x, w = x.detach().requires_grad_(), w.detach().requires_grad_()
    loss = linear_cross_entropy(x, w, y, reduction=reduction, **kw)
    grad = up.reshape(loss.shape) if reduction == "none" else torch.tensor(up_scalar(up), device=DEV)
    dx, dw = torch.autograd.grad(loss, (x, w), grad)
    assert loss.dtype == torch.float32 and dx.dtype == x.dtype and dw.dtype == w.dtype
    assert dx.shape == x.shape and dw.shape == w.shape
    d = x.shape[-1]
    want = reference(x.detach().reshape(-1, d), w.detach(), y.reshape(-1), up, reduction, kw.get("ignore_index", IGNORE))
    within("loss", loss.reshape(want[0].shape), want[0], want[1])
    within("dx", dx.reshape(-1, d), want[2], want[3])
    within("dW", dw, want[4], want[5])
    return loss, dx, dw


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,V,d,reduction,ignored", [
    (1, 1, 1, "mean", 0.0), (1, 97, 64, "sum", 0.0), (3, 5, 7, "none", 0.0), (200, 97, 128, "mean", 0.1),
    (257, 300, 72, "none", 0.3), (256, 256, 256, "sum", 0.0), (300, 1000, 200, "mean", 0.5), (513, 777, 320, "none", 0.1),
    (64, 5000, 1000, "mean", 0.0), (1031, 257, 33, "sum", 0.9), (2048, 64, 512, "mean", 0.0),
])
def test_loss_and_gradients(T, V, d, reduction, ignored, dtype):
    log(f"[lce] T{T} V{V} d{d} {reduction} {dtype}")
    check(*make(T, V, d, dtype, seed=T + V, ignored=ignored), reduction)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_strided_operands_int32_labels_and_another_ignore_index(dtype):
    x, w, y, up = make(6 * 50, 130, 96, dtype, seed=3)
    wide = torch.randn(6, 50, 107, device=DEV).to(dtype)
    wide[:, :, 5:101] = x.view(6, 50, 96)
    table = torch.randn(130, 104, device=DEV).to(dtype)
    table[:, 8:] = w
    y = y.view(6, 50).to(torch.int32)
    y[2, 7:] = 11
    check(wide[:, :, 5:101], table[:, 8:], y, up, "none", ignore_index=11)
    check(wide.transpose(0, 1)[:, :, 5:101], table[:, 8:], y.t(), up, "mean", ignore_index=11)
    check(x[::3], w[::2], torch.where(y.reshape(-1)[::3] < 65, y.reshape(-1)[::3], 11), up[::3], "sum", ignore_index=11)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_ignored_rows_enter_nothing_whatever_they_hold(dtype):
    x, w, y, up = make(700, 300, 128, dtype, seed=4, ignored=0.4)
    clean = check(x, w, y, up, "mean")
    bad = x.clone()
    bad[y == IGNORE] = float("nan")
    bad[(y == IGNORE).nonzero()[0]] = float("inf")
    got = check(bad, w, y, up, "mean")
    for a, b in zip(clean, got):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_no_valid_label_and_no_token(reduction, dtype):
    x, w, y, _ = make(70, 40, 64, dtype, seed=5, ignored=2.0)
    for n in (70, 0):
        xs, ws = x[:n].detach().requires_grad_(), w.detach().requires_grad_()
        loss = linear_cross_entropy(xs, ws, y[:n], reduction=reduction)
        dx, dw = torch.autograd.grad(loss, (xs, ws), torch.ones_like(loss))
        if reduction == "mean":
            assert torch.isnan(loss)
        else:
            assert torch.equal(loss, torch.zeros_like(loss)) and loss.shape == ((n,) if reduction == "none" else ())
        assert torch.equal(dx, torch.zeros_like(dx)) and torch.equal(dw, torch.zeros_like(dw))


def test_a_label_out_of_range_gives_nan():
    x, w, y, _ = make(300, 100, 64, torch.bfloat16, seed=6)
    y[17], y[30] = 100, -3
    loss = linear_cross_entropy(x, w, y, reduction="none")
    assert torch.isnan(loss[[17, 30]]).all() and torch.isfinite(loss).sum() == 298
    assert torch.isnan(linear_cross_entropy(x, w, y))
    xs, ws = x.requires_grad_(), w.requires_grad_()
    dx, _ = torch.autograd.grad(linear_cross_entropy(xs, ws, y, reduction="none").nansum(), (xs, ws))
    assert torch.isnan(dx[17]).all() and torch.isfinite(dx[18:30]).all()


def test_nan_rows_stay_in_their_rows_forward():
    x, w, y, _ = make(300, 100, 64, torch.bfloat16, seed=7)
    x[40, 3] = float("nan")
    loss = linear_cross_entropy(x, w, y, reduction="none")
    assert torch.isnan(loss[40]) and torch.isfinite(loss).sum() == 299


def test_logits_of_minus_infinity():
    """Words whose logit is -inf have probability zero; whole tiles of them too."""
    x, w, y, _ = make(40, 900, 64, torch.bfloat16, seed=8)
    x = x.abs() + 0.1
    w[300:] = float("-inf")
    y = y % 300
    loss = linear_cross_entropy(x, w, y, reduction="none")
    want = linear_cross_entropy(x, w[:300], y, reduction="none")
    assert torch.isfinite(loss).all() and torch.equal(loss, want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_large_logits(dtype):
    """Logits of hundreds, of both signs: the maximum is taken out before the exponentials."""
    x, w, y, up = make(300, 700, 64, dtype, seed=9, spread=60.0)
    check(x, w, y, up, "mean")
    x, w, y, up = make(100, 600, 64, dtype, seed=10)
    x = x + 40 * torch.ones_like(x)
    w = w - 0.5  # every logit far below zero
    check(x, w.to(dtype), y, up, "sum")


def test_logits_beyond_1e30():
    """Logits of -1e32 (and no larger one) and of 1e32: the loss is a difference of two of them, off by the errors of both
    (64 terms: 80 u |l| each) and 16 u |l| as bounded above; the gradients are made of probabilities, finite."""
    for sign in (-1.0, 1.0):
        x = torch.full((40, 64), 1e16, dtype=torch.bfloat16, device=DEV)
        w = torch.full((300, 64), sign * 1e14, dtype=torch.bfloat16, device=DEV)
        y = torch.arange(40, device=DEV)
        l = float(x[0].double() @ w[0].double())
        loss = linear_cross_entropy(x, w, y, reduction="none")
        assert bool((loss.double().abs() <= 2 * 80 * U * abs(l) + 16 * U * abs(l)).all())
        xs = x.detach().requires_grad_()
        (dx,) = torch.autograd.grad(linear_cross_entropy(xs, w, y), xs)
        assert torch.isfinite(dx).all()  # 300 g of at most 1, of 40 rows, times 1e14


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("size", [1e3, 1e4, 1e5, 1e6, 1e7, 1e9, 1e30])
def test_a_dominating_word_at_its_label_has_no_gradient(size, dtype):
    """One word's logit is far above the others, which are 0: its p is 1 and theirs e^-1000 = 0, so where it is the label the gradients are 0,
    and where another word is, g is 1 and -1.  Each logit is one product, whatever it is rounded to the same on both sides."""
    T, V, d = 70, 300, 64
    x = torch.zeros(T, d, dtype=dtype, device=DEV)
    x[:, 0] = size ** 0.5 * (1 + torch.rand(T, generator=torch.Generator().manual_seed(26))).to(dtype).to(DEV)
    w = torch.zeros(V, d, dtype=dtype, device=DEV)
    w[7, 0] = size ** 0.5 * 1.37
    y = torch.full((T,), 7, device=DEV)
    for reduction in ("sum", "none"):
        loss, ws = linear_cross_entropy_fwd(x, w, y, reduction=reduction)
        dx, dw = linear_cross_entropy_bwd(torch.ones_like(loss), w, ws, x.shape, reduction)
        assert loss.count_nonzero() == 0 and dx.count_nonzero() == 0 and dw.count_nonzero() == 0
    y[3] = 200
    loss, ws = linear_cross_entropy_fwd(x, w, y, reduction="none")
    dx, dw = linear_cross_entropy_bwd(torch.ones(T, device=DEV), w, ws, x.shape, "none")
    want = torch.zeros_like(dx)
    want[3] = w[7]
    assert torch.equal(dx, want)
    want = torch.zeros_like(dw)
    want[7], want[200] = x[3], -x[3]
    assert torch.equal(dw, want)


@pytest.mark.parametrize("size", [100, 1001, 12345, 654321, 9876543])
def test_neighbouring_large_logits_have_their_probabilities(size):
    """Two words at logits that are whole numbers 1 apart, exact in fp32, the others at 0: p = 1 / (1 + e^-1) and its rest, within the
    few roundings of numbers near 1 (an argument below 2, its exponential, log2 of the sum, the three planes of g: 16 u)."""
    V, d = 300, 64
    x = torch.zeros(3, d, device=DEV)
    x[:, 0], x[:, 1], x[:, 2:] = size, 1.0, 0.0
    x[:, 40] = 0.75
    w = torch.zeros(V, d, device=DEV)
    w[11, 0], w[290, 0], w[290, 1] = 1.0, 1.0, -1.0
    y = torch.tensor([11, 290, 150], device=DEV)
    loss, ws = linear_cross_entropy_fwd(x, w, y, reduction="none")
    dx, dw = linear_cross_entropy_bwd(torch.tensor([1.0, 0.0, 0.0], device=DEV), w, ws, x.shape, "none")
    p = 1 / (1 + torch.exp(torch.tensor(-1.0, dtype=torch.float64)))
    assert abs(float(dw[290, 40]) - 0.75 * float(1 - p)) <= 16 * U * 0.75
    assert abs(float(dw[11, 40]) + 0.75 * float(1 - p)) <= 16 * U * 0.75
    assert abs(float(dx[0, 1]) + float(1 - p)) <= 16 * U
    dx, dw = linear_cross_entropy_bwd(torch.tensor([0.0, 0.0, 1.0], device=DEV), w, ws, x.shape, "none")
    assert abs(float(dw[11, 40]) - 0.75 * float(p)) <= 16 * U * 0.75
    assert float(dw[150, 40]) == -0.75 and dw[[0, 299]].count_nonzero() == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("sign", [-1.0, 1.0])
def test_equal_logits_share_the_probability_at_any_size(sign, dtype):
    """300 words with the logit of 1e32 or -1e32 each: p is 1 / 300, within half a step of the result's type and of g's in bf16."""
    V, d = 300, 64
    x = torch.full((2, d), 1e16, device=DEV).to(dtype)
    w = torch.full((V, d), sign * 1e14, device=DEV).to(dtype)
    y = torch.tensor([5, 299], device=DEV)
    _, ws = linear_cross_entropy_fwd(x, w, y, reduction="none")
    dx, dw = linear_cross_entropy_bwd(torch.tensor([1.0, 0.0], device=DEV), w, ws, x.shape, "none")
    want = torch.full((V, 1), 1 / 300, dtype=torch.float64, device=DEV)
    want[5] -= 1
    off = (dw.double() / x[0, 0].double() - want).abs()
    assert bool((off <= want.abs() * (2 * B16 if dtype == torch.bfloat16 else 2 * U) + 16 * U * want.abs()).all())


@pytest.mark.parametrize("d", [1, 64])
def test_fp32_products_are_those_of_whole_numbers(d):
    """fp32 logits of one product each: three planes of both operands leave out at most 2^-24 + 2^-34 of it, the sum of the six products
    kept is rounded (2 u if cut off; the smaller ones' sums are below 2^-8 of it), and where the other word's logit is 0 and this one
    above 100 the loss of the other is the logit.  Significands with long runs of ones leave most in the second and third plane."""
    g = torch.Generator().manual_seed(27)
    one = 1 + 2.0 ** -7 - 2.0 ** -23
    x = torch.cat([torch.tensor([one, 1 + 2.0 ** -8 - 2.0 ** -23, 1 + 2.0 ** -8 + 2.0 ** -17, 1.5 - 2.0 ** -23, 2 - 2.0 ** -23]),
                   1 + torch.rand(2000, generator=g)])
    for other in (one, 1 + 2.0 ** -8 + 2.0 ** -17, 1.25, 1.984375 - 2.0 ** -22):
        xs = torch.zeros(x.numel(), d, device=DEV)
        xs[:, d // 2] = 128 * x.to(DEV)
        w = torch.zeros(2, d, device=DEV)
        w[0, d // 2] = other
        y = torch.ones(x.numel(), dtype=torch.long, device=DEV)
        want = xs[:, d // 2].double() * w[0, d // 2].double()
        off = (linear_cross_entropy(xs, w, y, reduction="none").double() - want) / want
        log(f"  {float(off.min()) / U:.2f} .. {float(off.max()) / U:.2f} u, mean {float(off.mean()) / U:.2f}")
        assert float(off.abs().max()) <= 3.01 * U


def test_fp32_at_the_ends_of_its_range():
    """Operands whose first plane would round to infinity, and subnormal ones: finite logits and gradients.  bf16 has no number
    between 0 and 2^-133, and may take those below 2^-126 as 0: each of an operand's second and third plane is off by at most 2^-126,
    a logit by 2^-125 (sum |x| + sum |w|) more than the bound above, a loss by twice that (8 and 16 in the rows of 2^128, whose gradients
    are bounded by |g| <= 1, 2^-100 in the others)."""
    top = torch.finfo(torch.float32).max
    x = torch.zeros(4, 64, device=DEV)
    x[0, 0], x[1, 0], x[2, 0], x[3, 0] = top, -top, 2.0 ** -140, 1.0
    w = torch.zeros(3, 64, device=DEV)
    w[0, 0], w[1, 0] = 2.0 ** -127 * 1.999, 2.0 ** -126
    y = torch.tensor([0, 1, 2, 2], device=DEV)
    up = torch.ones(4, device=DEV)
    for _ in range(2):
        want = reference(x, w, y, up, "none")
        lost = 2.0 ** -125 * (x.double().abs().sum(1) + w.double().abs().sum(1).amax())
        loss, ws = linear_cross_entropy_fwd(x, w, y, reduction="none")
        within("loss", loss, want[0], want[1] + 2 * lost)
        dx, dw = linear_cross_entropy_bwd(up, w, ws, x.shape, "none")
        within("dx", dx[2:], want[2][2:], want[3][2:] + 8 * lost[2:, None] * w.double().abs().sum(0))
        assert torch.isfinite(dx).all() and bool((dx.abs() <= 2 * w.abs().amax(0)).all())
        assert not torch.isnan(dw).any()
        w[0, 1] = top
        x[:, 1] = 2.0 ** -126


def test_many_tokens_and_few_words():
    """More tokens than the packing has workgroups for; ignored rows in long runs, and in all of the first workgroups."""
    T, V, d = 70001, 90, 40
    x, w, y, up = make(T, V, d, torch.bfloat16, seed=21, ignored=0.3)
    y[:5000] = IGNORE
    y[33000:34111] = IGNORE
    check(x, w, y, up, "mean")
    loss = linear_cross_entropy(x, w, y, reduction="none")
    want = reference(x, w, y, up, "none")
    within("loss", loss, want[0], want[1])


@pytest.mark.parametrize("T,V,d,reduction,ignored", [
    (2600, 2500, 64, "mean", 0.0), (3000, 2300, 200, "none", 0.3), (700, 9000, 129, "sum", 0.1), (25100, 97, 40, "mean", 0.5),
    (65, 25000, 320, "none", 0.0), (2561, 2305, 576, "mean", 0.02), (5000, 4800, 31, "mean", 0.999)])
def test_enough_tiles_for_the_large_ones(T, V, d, reduction, ignored):
    """Logits of 96 tiles of 256 x 256 or more."""
    check(*make(T, V, d, torch.bfloat16, seed=T, ignored=ignored), reduction)


@pytest.mark.parametrize("gap", [8, 3])
def test_strided_rows_in_large_tiles(gap):
    T, V, d = 2400, 2700, 192
    x, w, y, up = make(T, V, d, torch.bfloat16, seed=23, ignored=0.2)
    xs = torch.full((T, d + gap), float("nan"), dtype=torch.bfloat16, device=DEV)
    ws = torch.full((V, d + gap), float("nan"), dtype=torch.bfloat16, device=DEV)
    xs[:, :d], ws[:, :d] = x, w
    a = check(xs[:, :d], ws[:, :d], y.to(torch.int32), up, "mean")
    b = check(x, w, y, up, "mean")
    assert all(torch.equal(p, q) for p, q in zip(a, b))


@pytest.mark.parametrize("T,V,d,reduction", [(38, 10000, 200, "none"), (300, 2000, 128, "mean"), (60, 97, 64, "sum"),
                                             (2000, 9000, 192, "none"), (5, 50000, 64, "mean")])
def test_the_rounding_at_the_label_is_made_up_for(T, V, d, reduction):
    """Labels that differ: g at the label, most of its row, is as good as in fp32 for both gradients; of the bound above only
    the roundings of the other words' g stay (b |g| each) and that of the result."""
    x, w, _, up = make(T, V, d, torch.bfloat16, seed=24, spread=0.5)
    y = torch.randperm(V, generator=torch.Generator().manual_seed(25))[:T].to(DEV)
    xs, ws = x.detach().requires_grad_(), w.detach().requires_grad_()
    loss = linear_cross_entropy(xs, ws, y, reduction=reduction)
    grad = up if reduction == "none" else torch.tensor(0.75, device=DEV)
    dx, dw = torch.autograd.grad(loss, (xs, ws), grad)
    x, w = x.double(), w.double()
    l = x @ w.t()
    lse = torch.logsumexp(l, 1, keepdim=True)
    e_p = 2 * (2 * (d + 16) * U * (x.abs() @ w.abs().t()).amax(1, keepdim=True) + 16 * U * (1 + lse.abs()))
    p = torch.exp(l - lse)
    s = (up.double() if reduction == "none" else torch.full((T,), 0.75 / (T if reduction == "mean" else 1), device=DEV).double())[:, None]
    g = p.clone()
    g[torch.arange(T, device=DEV), y] -= 1
    others = p.clone()
    others[torch.arange(T, device=DEV), y] = 0
    e_g = (p * e_p + others * (B16 + 4 * U) + g.abs() * 4 * U) * s.abs() + TINY * (1 + s.abs())
    g = g * s
    for name, got, want, bound, terms in (("dx", dx, g @ w, e_g @ w.abs() + TINY * V, V), ("dW", dw, g.t() @ x, e_g.t() @ x.abs() + TINY * T, T)):
        size = g.abs() @ w.abs() if name == "dx" else g.abs().t() @ x.abs()
        bound = bound + (terms + 18) * U * size
        within(name, got, want, bound + B16 * (want.abs() + bound))


def made_up(x, w, y, s):
    """dx, dW and their bounds for factors s (T) where g at the label is as good as in fp32: of the bound above only the
    roundings of the other words' g stay (b |g| each) and that of the result."""
    T, V = x.shape[0], w.shape[0]
    x, w, s = x.double(), w.double(), s.double()[:, None]
    l = x @ w.t()
    lse = torch.logsumexp(l, 1, keepdim=True)
    e_p = 2 * (2 * (x.shape[1] + 16) * U * (x.abs() @ w.abs().t()).amax(1, keepdim=True) + 16 * U * (1 + lse.abs()))
    p = torch.exp(l - lse)
    rows = torch.arange(T, device=DEV)
    g, others = p.clone(), p.clone()
    g[rows, y] -= 1
    others[rows, y] = 0
    e_g = (p * e_p + others * (B16 + 4 * U) + g.abs() * 4 * U) * s.abs() + TINY * (1 + s.abs())
    g = g * s
    dx, dw = g @ w, g.t() @ x
    e_dx = e_g @ w.abs() + TINY * V + (V + 18) * U * (g.abs() @ w.abs())
    e_dw = e_g.t() @ x.abs() + TINY * T + (T + 18) * U * (g.abs().t() @ x.abs())
    return dx, e_dx + B16 * (dx.abs() + e_dx), dw, e_dw + B16 * (dw.abs() + e_dw)


@pytest.mark.parametrize("T,V,d,words", [(33, 300, 64, 1), (2000, 3000, 64, 20), (700, 9000, 129, 3), (3000, 5000, 1100, 40),
                                         (40001, 600, 72, 7)])
def test_the_rounding_at_repeated_labels_is_made_up_for(T, V, d, words):
    """Few words are the labels of all tokens, and the factors' signs alternate: a word's row of dW is a sum that nearly cancels,
    of terms whose roundings do not."""
    g = torch.Generator().manual_seed(T)
    w = (torch.randn(V, d, generator=g) / d ** 0.5).to(torch.bfloat16)
    y = torch.randint(0, words, (T,), generator=g) * (V // words)
    x = (torch.ones(T, d) + 0.1 * torch.randn(T, d, generator=g) + 14 * torch.rand(T, 1, generator=g) * w[y].float()).to(torch.bfloat16)
    up = torch.where(torch.arange(T) % 2 == 0, 1.0, -1.0)
    x, w, y, up = x.to(DEV), w.to(DEV), y.to(DEV), up.to(DEV)
    xs, ws = x.detach().requires_grad_(), w.detach().requires_grad_()
    dx, dw = torch.autograd.grad(linear_cross_entropy(xs, ws, y, reduction="none"), (xs, ws), up)
    want = made_up(x, w, y, up)
    within("dx", dx, want[0], want[1])
    within("dW", dw, want[2], want[3])
    (alone,) = torch.autograd.grad(linear_cross_entropy(x, ws, y, reduction="none"), ws, up)
    within("dW alone", alone, want[2], want[3])


@pytest.mark.parametrize("n", [1, 17, 40, 300, 20000])
def test_probabilities_lost_from_one_side(n):
    """p - 1 of a p below 2^-9 rounds to -1 in bf16, always in the same direction.  One word is the label of n tokens of p = 1 / 568
    with factor 1 and of n of p = 10^-9 with factor -1: its row of dW is n times the difference, made of what the rounding loses.
    Where x is 1 the products' own sums are whole numbers, without error: p's relative error e_p and the 2 n additions of p stay."""
    V, d = 568, 64
    w = torch.zeros(V, d, dtype=torch.bfloat16, device=DEV)
    w[5, 0] = -14.0
    x = torch.zeros(2 * n, d, dtype=torch.bfloat16, device=DEV)
    x[:, 32:] = 1.0
    x[n:, 0] = 1.0
    y = torch.full((2 * n,), 5, device=DEV)
    up = torch.ones(2 * n, device=DEV)
    up[n:] = -1.0
    _, ws = linear_cross_entropy_fwd(x, w, y, reduction="none")
    dx, dw = linear_cross_entropy_bwd(up, w, ws, x.shape, "none")
    p = torch.softmax(x.double() @ w.double().t(), 1)[:, 5]
    want = (p * up.double()).sum()
    e = ((2 * 16 * U * (1 + 6.4) + (2 * n + 18) * U) * p.sum()).expand(32)
    within("dW", dw[5, 32:], want.expand(32), e + B16 * (want + e))
    if n <= 300:
        want = made_up(x, w, y, up)
        within("dx", dx, want[0], want[1])
        within("dW", dw, want[2], want[3])


def test_one_gradient_alone_and_the_same_bits_again():
    """The same call gives the same bits.  A gradient asked for alone is cut into other shares (its sums may be split
    at other places), so it is held to its bound, not to the bits of the two together."""
    x, w, y, _ = make(1500, 700, 192, torch.bfloat16, seed=11, ignored=0.2)
    up = torch.tensor(0.75, device=DEV)
    loss, ws = linear_cross_entropy_fwd(x, w, y)
    dx, dw = linear_cross_entropy_bwd(up, w, ws, x.shape)
    dx1, none = linear_cross_entropy_bwd(up, w, ws, x.shape, need_weight=False)
    none2, dw1 = linear_cross_entropy_bwd(up, w, ws, x.shape, need_x=False)
    assert none is None and none2 is None
    want = reference(x, w, y, torch.zeros(1500, device=DEV), "mean")
    within("dx alone", dx1, want[2], want[3])
    within("dW alone", dw1, want[4], want[5])
    loss2, ws2 = linear_cross_entropy_fwd(x, w, y)
    dx2, dw2 = linear_cross_entropy_bwd(up, w, ws2, x.shape)
    assert torch.equal(loss, loss2) and torch.equal(dx, dx2) and torch.equal(dw, dw2)
    xs = x.detach().requires_grad_()
    (dx3,) = torch.autograd.grad(linear_cross_entropy(xs, w, y), xs, up)
    assert torch.equal(dx1, dx3)


@pytest.mark.parametrize("dtype,T,V,d", [(torch.bfloat16, 4100, 40000, 72), (torch.float32, 2050, 30000, 40)])
def test_several_pieces_of_the_vocabulary(dtype, T, V, d):
    """More softmax gradient than is kept at a time."""
    check(*make(T, V, d, dtype, seed=12, ignored=0.05), "mean")


def test_gradient_against_differences():
    """Central differences of the fp64 formula, along random directions: the formula's own second-order error at
    h = 1e-4 is below 1e-7 of the slope, the gradients' fp32 errors below 1e-5."""
    x, w, y, _ = make(60, 90, 48, torch.float32, seed=13, ignored=0.2)
    xs, ws = x.requires_grad_(), w.requires_grad_()
    dx, dw = torch.autograd.grad(linear_cross_entropy(xs, ws, y), (xs, ws))

    def f(a, b):
        return torch.nn.functional.cross_entropy(a @ b.t(), y, ignore_index=IGNORE)

    g = torch.Generator().manual_seed(14)
    for _ in range(4):
        u = torch.randn(x.shape, generator=g).double().to(DEV)
        v = torch.randn(w.shape, generator=g).double().to(DEV)
        h, X, W = 1e-4, x.detach().double(), w.detach().double()
        slope = (f(X + h * u, W + h * v) - f(X - h * u, W - h * v)) / (2 * h)
        got = (dx.double() * u).sum() + (dw.double() * v).sum()
        size = (dx.double() * u).abs().sum() + (dw.double() * v).abs().sum()
        assert abs(float(got - slope)) <= 1e-5 * float(size)


def test_on_another_stream_and_captured():
    """A captured forward and backward, replayed on new inputs among eager calls, gives the eager bits."""
    x, w, y, _ = make(400, 500, 128, torch.bfloat16, seed=15, ignored=0.1)
    up = torch.ones((), device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        loss, ws = linear_cross_entropy_fwd(x, w, y)
        dx, dw = linear_cross_entropy_bwd(up, w, ws, x.shape)
    torch.cuda.current_stream().wait_stream(side)
    eager = linear_cross_entropy_fwd(x, w, y)
    assert torch.equal(loss, eager[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        gl, gws = linear_cross_entropy_fwd(x, w, y)
        gdx, gdw = linear_cross_entropy_bwd(up, w, gws, x.shape)
    for k in range(4):
        nx, nw, ny, _ = make(400, 500, 128, torch.bfloat16, seed=20 + k, ignored=0.1 * k)
        x.copy_(nx), w.copy_(nw), y.copy_(ny)
        graph.replay()
        el, ews = linear_cross_entropy_fwd(nx, nw, ny)
        edx, edw = linear_cross_entropy_bwd(up, nw, ews, nx.shape)
        torch.cuda.synchronize()
        assert torch.equal(gl, el) and torch.equal(gdx, edx) and torch.equal(gdw, edw)


def test_one_row_of_any_shape():
    x, w, y, _ = make(1, 50, 64, torch.bfloat16, seed=16)
    a = linear_cross_entropy(x[0], w, y[0], reduction="none")
    b = linear_cross_entropy(x.view(1, 1, 64), w, y.view(1, 1), reduction="none")
    assert a.shape == () and b.shape == (1, 1) and torch.equal(a, b[0, 0])


def test_frozen_operands_and_a_changed_weight():
    x, w, y, up = make(100, 60, 64, torch.bfloat16, seed=17)
    xs, ws = x.detach().requires_grad_(), w.detach().requires_grad_()
    (dw,) = torch.autograd.grad(linear_cross_entropy(x, ws, y), ws)
    (dx,) = torch.autograd.grad(linear_cross_entropy(xs, w, y), xs)
    want = reference(x, w, y, torch.zeros(100, device=DEV), "mean")
    within("dx", dx, want[2] / 0.75, want[3] / 0.75)
    within("dW", dw, want[4] / 0.75, want[5] / 0.75)
    loss = linear_cross_entropy(xs, ws, y)
    with torch.no_grad():
        xs.zero_()  # the forward keeps its own copy of the rows
    (again,) = torch.autograd.grad(loss, xs)
    assert torch.equal(again, dx) or bool(((again.double() - want[2] / 0.75).abs() <= want[3] / 0.75).all())
    loss = linear_cross_entropy(x, ws, y)
    with torch.no_grad():
        ws.zero_()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_second_derivatives_raise_and_a_graph_kept_gives_the_same_again():
    x, w, y, _ = make(60, 50, 64, torch.float32, seed=22)
    xs, ws = x.requires_grad_(), w.requires_grad_()
    loss = linear_cross_entropy(xs, ws, y)
    first = torch.autograd.grad(loss, (xs, ws), retain_graph=True)
    dx, dw = torch.autograd.grad(loss, (xs, ws), create_graph=True)
    assert torch.equal(dx, first[0]) and torch.equal(dw, first[1])
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(dx.sum(), ws)
    (dx,) = torch.autograd.grad(linear_cross_entropy(xs, w.detach(), y), xs, create_graph=True)
    with pytest.raises(RuntimeError, match="second derivative"):
        dx.sum().backward()
    with torch.inference_mode():
        assert torch.equal(linear_cross_entropy(x, w, y), loss)
    with torch.no_grad():
        assert not linear_cross_entropy(xs, ws, y).requires_grad


def test_refusals():
    x, w, y, _ = make(10, 20, 64, torch.bfloat16)
    with pytest.raises(TypeError, match="float32 or bfloat16"):
        linear_cross_entropy(x.half(), w.half(), y)
    with pytest.raises(TypeError, match="share dtype"):
        linear_cross_entropy(x.float(), w, y)
    with pytest.raises(TypeError, match="int64 or int32"):
        linear_cross_entropy(x, w, y.float())
    with pytest.raises(ValueError, match="labels must be"):
        linear_cross_entropy(x, w, y[:5])
    with pytest.raises(ValueError, match=r"weight \(V, d\)"):
        linear_cross_entropy(x, w[:, :32], y)
    with pytest.raises(ValueError, match="reduction"):
        linear_cross_entropy(x, w, y, reduction="batchmean")
    loss, ws = linear_cross_entropy_fwd(x, w, y)
    with pytest.raises(ValueError, match="the gradient of a none"):
        linear_cross_entropy_bwd(torch.ones((), device=DEV), w, ws, x.shape, "none")
    with pytest.raises(ValueError, match="the gradient of a mean"):
        linear_cross_entropy_bwd(torch.ones(10, device=DEV), w, ws, x.shape)
    with pytest.raises(ValueError, match="not the workspace"):
        linear_cross_entropy_bwd(torch.ones((), device=DEV), w, ws[:64], x.shape)
    with pytest.raises(ValueError, match="not the workspace"):  # that of a longer forward
        linear_cross_entropy_bwd(torch.ones((), device=DEV), w, torch.cat([ws, ws]), x.shape)
    with pytest.raises(ValueError, match="not the workspace"):  # that of one token more
        linear_cross_entropy_bwd(torch.ones(9, device=DEV), w, ws, x[:9].shape, "none")
    with pytest.raises(ValueError, match="not the workspace"):
        linear_cross_entropy_bwd(torch.ones((), device=DEV), w, None, x.shape)
    with pytest.raises(TypeError, match="float32 or bfloat16"):
        linear_cross_entropy_bwd(torch.ones((), device=DEV), w.half(), ws, x.shape)
    with pytest.raises(ValueError, match="reduction"):
        linear_cross_entropy_bwd(torch.ones((), device=DEV), w, ws, x.shape, "batchmean")
    with pytest.raises(RuntimeError, match="GPU only"):
        linear_cross_entropy(x.cpu(), w.cpu(), y.cpu())
    with pytest.raises(RuntimeError, match="labels is on"):
        linear_cross_entropy(x, w, y.cpu())


def test_a_backward_with_another_weight_is_refused():
    """Sizes that the workspace rounds up to the same: fewer words, more words, fewer columns."""
    x, w, y, _ = make(300, 100, 128, torch.bfloat16, seed=28)
    up = torch.ones((), device=DEV)
    _, ws = linear_cross_entropy_fwd(x, w, y)
    for n in (90, 97, 99, 101, 120, 128):
        with pytest.raises(ValueError, match="not the workspace"):
            linear_cross_entropy_bwd(up, torch.zeros(n, 128, dtype=torch.bfloat16, device=DEV), ws, x.shape)
    for dtype in (torch.float32, torch.bfloat16):
        a, b = x[:, :100].to(dtype), w[:, :100].to(dtype)
        _, ws = linear_cross_entropy_fwd(a, b, y)
        for d in (96, 99, 101, 128):
            with pytest.raises(ValueError, match="not the workspace"):
                linear_cross_entropy_bwd(up, torch.zeros(100, d, dtype=dtype, device=DEV), ws, (300, d))
        linear_cross_entropy_bwd(up, b, ws, a.shape)


@pytest.mark.parametrize("T,V,d", [(300, 40, 1000), (512, 64, 600), (513, 64, 72), (320, 40, 64), (321, 40, 64), (544, 700, 520), (40, 2, 64)])
def test_labels_around_the_sizes_where_their_sums_take_another_form(T, V, d):
    """Few rows by one launch, up to 512 and eight to a word; chunks of 32 sorted rows behind that."""
    for seed, ignored in ((T, 0.0), (T + 1, 0.4)):
        x, w, y, up = make(T, V, d, torch.bfloat16, seed=seed, ignored=ignored)
        _, _, dw = check(x, w, y, up, "none")
        keep = y != IGNORE
        want = made_up(x[keep], w, y[keep], up[keep])
        within("dW", dw, want[2], want[3])


def test_more_rows_captured_and_a_workspace_used_again():
    """A captured step with sorted labels gives the eager bits on new inputs; a kept workspace those of its other factors, on two streams at
    once too."""
    T, V, d = 2000, 300, 128
    x, w, y, up = make(T, V, d, torch.bfloat16, seed=30, ignored=0.1)
    linear_cross_entropy_bwd(up, w, linear_cross_entropy_fwd(x, w, y, reduction="none")[1], x.shape, "none")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _, gws = linear_cross_entropy_fwd(x, w, y, reduction="none")
        gdx, gdw = linear_cross_entropy_bwd(up, w, gws, x.shape, "none")
    for k in range(3):
        nx, nw, ny, nu = make(T, V, d, torch.bfloat16, seed=31 + k, ignored=0.3 * k)
        x.copy_(nx), w.copy_(nw), y.copy_(ny), up.copy_(nu)
        graph.replay()
        _, ws = linear_cross_entropy_fwd(nx, nw, ny, reduction="none")
        dx, dw = linear_cross_entropy_bwd(nu, nw, ws, nx.shape, "none")
        torch.cuda.synchronize()
        assert torch.equal(gdx, dx) and torch.equal(gdw, dw)
    first = [linear_cross_entropy_bwd(u, nw, ws, nx.shape, "none") for u in (nu, -2 * nu)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    both = []
    for s, u in zip(streams, (nu, -2 * nu)):
        with torch.cuda.stream(s):
            both.append(linear_cross_entropy_bwd(u, nw, ws, nx.shape, "none"))
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for a, b in zip(first, both) for p, q in zip(a, b))
    assert torch.equal(first[0][1], dw)
