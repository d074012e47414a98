"""int4_linear and its weights against plain products in 64 bits on the CPU.

Exact cases: x whole numbers up to 8, scales powers of two. Every sum is then a whole number below 136 * 8 * K * 2 < 2^24 of the
smallest scale, which fp32 holds, so the result is the exact one rounded once, bit for bit.

Other cases: besides half a step of bf16 (2^-8 relative) for the result, a group's sum of g products of up to 144 |x| is rounded
at most 2 g times, the groups' sums once each; roundings of no common direction add up to less than 8 times their root mean
square: 8 sqrt(2 g + K / g) 2^-24 144 sum |x| s over a group's mean share.  With a norm weight x' itself is off by 2^-17."""

import math

import pytest
import torch

from _gpu_util import DEV, log

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


def weight_of(N, K, group, seed, powers=False):
    g = torch.Generator().manual_seed(seed)
    codes = torch.randint(-8, 8, (N, K), generator=g, dtype=torch.int8)
    G = -(-K // group)
    if powers:
        scales = torch.exp2(torch.randint(-1, 1, (N, G), generator=g).float())
    else:
        scales = (0.5 + torch.rand(N, G, generator=g)) / math.sqrt(K)
    return codes, scales.to(BF)


def wide(codes, scales, group):
    return codes.double() * scales.double().repeat_interleave(group, 1)[:, :codes.shape[1]]


def packed(codes, scales, group):
    from cdssm_hip import pack_int4
    return pack_int4(codes.to(DEV), scales.to(DEV), group)


SIZES = [(1, 1, 1), (1, 16, 128), (2, 17, 129), (3, 33, 100), (5, 100, 7), (7, 50, 255), (16, 64, 256), (17, 65, 1024), (32, 48, 384),
         (33, 31, 640), (64, 128, 512), (64, 200, 1000), (1, 3104, 1024), (40, 4992, 768), (9, 16, 4104), (64, 9000, 136)]


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("M,N,K", SIZES)
def test_whole_numbers_come_out_exactly(M, N, K, group):
    from cdssm_hip import int4_linear
    log(f"[int4] exact M{M} N{N} K{K} g{group}")
    codes, scales = weight_of(N, K, group, M + N + K, powers=True)
    x = torch.randint(-8, 9, (M, K), generator=torch.Generator().manual_seed(K)).to(BF)
    y = int4_linear(x.to(DEV), packed(codes, scales, group))
    want = (x.double() @ wide(codes, scales, group).t()).float().to(BF)
    assert y.dtype == BF and torch.equal(y.cpu(), want)


def bound(x, codes, scales, group, y, norm=False):
    K = x.shape[1]
    P = 144 * (x.abs() @ scales.double().repeat_interleave(group, 1)[:, :K].t())
    groups = -(-K // group)
    e = 8 * math.sqrt(2 * min(group, K) + groups) * 2.0 ** -24 * P / math.sqrt(groups)
    if norm:  # x' to 2^-17, the row's scale to a few steps
        e = e + 2.0 ** -17 * (x.abs() @ wide(codes, scales, group).abs().t()) + 2.0 ** -20 * y.abs()
    return e + 2.0 ** -8 * y.abs()


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("extra", ["", "bias", "residual", "norm", "all"])
@pytest.mark.parametrize("M,N,K", [(1, 1024, 1024), (5, 300, 768), (16, 100, 2000), (33, 77, 1100), (64, 1136, 1024), (2, 40, 28672),
                                   (6, 33, 45), (20, 12300, 2050)])
def test_against_64_bits(M, N, K, extra, group):
    from cdssm_hip import int4_linear
    log(f"[int4] M{M} N{N} K{K} g{group} {extra}")
    codes, scales = weight_of(N, K, group, M + N + K)
    g = torch.Generator().manual_seed(M * K)
    x = torch.randn(M, K, generator=g).mul_(2).to(BF)
    bias = torch.randn(N, generator=g).to(BF) if extra in ("bias", "all") else None
    res = torch.randn(M, N, generator=g).to(BF) if extra in ("residual", "all") else None
    nw = (1 + 0.2 * torch.randn(K, generator=g)).to(BF) if extra in ("norm", "all") else None
    on = lambda t: None if t is None else t.to(DEV)  # noqa: E731
    y = int4_linear(on(x), packed(codes, scales, group), bias=on(bias), residual=on(res), norm_weight=on(nw), eps=1e-5)
    xd = x.double()
    if nw is not None:
        xd = xd * torch.rsqrt(xd.pow(2).mean(1, keepdim=True) + 1e-5) * nw.double()
    want = xd @ wide(codes, scales, group).t()
    if bias is not None:
        want = want + bias.double()
    if res is not None:
        want = want + res.double()
    off = ((y.cpu().double() - want).abs() / bound(xd, codes, scales, group, want, nw is not None)).max()
    log(f"  worst {float(off):.3f} of the bound")
    assert float(off) <= 1.0


@pytest.mark.parametrize("dtype", [BF, torch.float32])
@pytest.mark.parametrize("N,K,group", [(1, 1, 32), (3, 31, 32), (16, 128, 64), (50, 1000, 128), (33, 100, 64)])
def test_quantize_is_its_definition(N, K, group, dtype):
    """Scales and codes are the ones that the same steps give in torch (every step is one rounding), and half a code off at most."""
    from cdssm_hip import quantize_int4
    w = torch.randn(N, K, generator=torch.Generator().manual_seed(N * K)).to(dtype)
    w[0, 0] = 0.0
    q = quantize_int4(w.to(DEV), group)
    codes, scales = (t.cpu() for t in q.unpack())
    G = -(-K // group)
    padded = torch.zeros(N, G * group).index_copy_(1, torch.arange(K), w.float()).view(N, G, group)
    want_s = (padded.abs().amax(2) / 7.0).to(BF)
    by = torch.where(want_s == 0, 1.0, want_s.float())[..., None]
    want_c = torch.round(padded / by).clamp(-8, 7).view(N, G * group)[:, :K].to(torch.int8)
    assert torch.equal(scales, want_s) and torch.equal(codes, want_c)
    err = (q.dequantize().cpu().double() - w.double()).abs()
    # (the largest magnitude is 7 codes, and the scale's own rounding, 2^-8 of 7 codes, adds to the half)
    assert (err <= (0.5 + 7 * 2.0 ** -8) * scales.double().repeat_interleave(group, 1)[:, :K]).all()


def test_groups_of_zeros_of_tiny_and_of_infinite_weights():
    from cdssm_hip import quantize_int4
    w = torch.randn(4, 96)
    w[0] = 0.0
    w[1, :32] = 2.0 ** -125
    w[2, 40] = float("inf")
    w[3, 70] = float("nan")
    d = quantize_int4(w.to(DEV), 32).dequantize().cpu()
    assert (d[0] == 0).all() and (d[1, :32] == 0).all()
    assert torch.isnan(d[2, 32:64]).all() and torch.isnan(d[3, 64:]).all()
    assert torch.isfinite(d[2, :32]).all() and torch.isfinite(d[3, :64]).all()


@pytest.mark.parametrize("N,K,group", [(1, 1, 32), (17, 300, 32), (40, 129, 64), (100, 1000, 128)])
def test_pack_and_unpack(N, K, group):
    codes, scales = weight_of(N, K, group, N + K)
    q = packed(codes, scales, group)
    c, s = q.unpack()
    assert torch.equal(c.cpu(), codes) and torch.equal(s.cpu(), scales)
    assert torch.equal(q.dequantize(torch.float64).cpu(), wide(codes, scales, group).float().double())


def test_strides_alignment_and_leading_dimensions():
    from cdssm_hip import int4_linear
    codes, scales = weight_of(50, 136, 64, 0, powers=True)
    w, ref = packed(codes, scales, 64), wide(codes, scales, 64)
    big = torch.randint(-8, 9, (12, 3 * 136 + 5), generator=torch.Generator().manual_seed(1)).to(BF).to(DEV)
    for x in (big[:, :136], big[:, 1:137], big[:, 8:144], big[::2, 5:141], big[:1, 3:139].expand(12, 136),
              big[:, :136].t().contiguous().t()):
        assert torch.equal(int4_linear(x, w).cpu(), (x.cpu().double() @ ref.t()).float().to(BF))
    x = big[:, :136].reshape(3, 4, 136)
    res = torch.randint(-8, 9, (3, 4, 60)).to(BF).to(DEV)[..., :50]
    y = int4_linear(x, w, residual=res)
    assert y.shape == (3, 4, 50)
    assert torch.equal(y.cpu(), (x.cpu().double() @ ref.t() + res.cpu().double()).float().to(BF))
    assert torch.equal(int4_linear(x[0, 0], w).cpu(), (x[0, 0].cpu().double() @ ref.t()).float().to(BF))
    assert int4_linear(x[:0], w).shape == (0, 4, 50)
    nw = torch.ones(137, dtype=BF, device=DEV)
    a, b = (int4_linear(x, w, norm_weight=n, eps=1e-6) for n in (nw[:136].clone(), nw[1:]))  # either side of the alignment
    assert torch.equal(a, b)


def test_rows_do_not_depend_on_their_neighbours():
    """A row's bits are the same alone as in a batch, whatever the other rows hold."""
    from cdssm_hip import int4_linear
    codes, scales = weight_of(300, 1000, 128, 2)
    w = packed(codes, scales, 128)
    x = torch.randn(64, 1000, generator=torch.Generator().manual_seed(3)).to(BF).to(DEV)
    y = int4_linear(x, w)
    bad = x.clone()
    bad[1::2] = float("nan")
    assert torch.equal(int4_linear(bad, w)[::2], y[::2])
    assert torch.isnan(int4_linear(bad, w)[1::2]).all()
    for m in (1, 3, 16, 20, 40):
        assert torch.equal(int4_linear(x[:m], w), y[:m])


def test_captured_replayed_and_on_two_streams():
    from cdssm_hip import int4_linear
    codes, scales = weight_of(1136, 1024, 64, 4)
    w = packed(codes, scales, 64)
    x = torch.randn(8, 1024, device=DEV).to(BF)
    int4_linear(x, w)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = int4_linear(x, w)
    for seed in range(4):
        x.copy_(torch.randn(8, 1024, generator=torch.Generator().manual_seed(seed)))
        graph.replay()
        want = int4_linear(x, w)
        torch.cuda.synchronize()
        assert torch.equal(y, want)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    out = []
    for _ in range(3):
        for s in streams:
            with torch.cuda.stream(s):
                out.append(int4_linear(x, w))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in out)


def test_refusals_that_need_tensors_on_the_gpu():
    from cdssm_hip import Int4Weight, int4_linear, pack_int4
    codes, scales = weight_of(50, 136, 64, 0)
    w = packed(codes, scales, 64)
    x = torch.randn(4, 136, device=DEV).to(BF)
    with pytest.raises(TypeError, match="bfloat16"):
        int4_linear(x.float(), w)
    with pytest.raises(ValueError, match=r"\(\.\.\., 136\)"):
        int4_linear(x[:, :135], w)
    with pytest.raises(ValueError, match="at most 64 rows"):
        int4_linear(x[:1].expand(65, 136), w)
    with pytest.raises(ValueError, match="bias must be"):
        int4_linear(x, w, bias=torch.zeros(49, device=DEV))
    with pytest.raises(ValueError, match="residual must be"):
        int4_linear(x, w, residual=torch.zeros(4, 49, device=DEV))
    with pytest.raises(ValueError, match="norm_weight must be"):
        int4_linear(x, w, norm_weight=torch.zeros(50, device=DEV))
    with pytest.raises(RuntimeError, match="bias is on cpu"):
        int4_linear(x, w, bias=torch.zeros(50))
    with pytest.raises(NotImplementedError, match="no gradient to x"):
        int4_linear(x.clone().requires_grad_(True), w)
    for name, shape in (("bias", (50,)), ("residual", (4, 50)), ("norm_weight", (136,))):
        with pytest.raises(NotImplementedError, match=f"no gradient to {name}"):
            int4_linear(x, w, **{name: torch.zeros(shape, device=DEV, requires_grad=True)})
    with torch.no_grad():
        int4_linear(x.clone().requires_grad_(True), w, bias=torch.zeros(50, device=DEV, requires_grad=True))
    with pytest.raises(ValueError, match="not a 4-bit weight"):  # a handle whose sizes are not its tensors'
        int4_linear(x, Int4Weight(w.words, w.scales, 500, 136, 64))
    with pytest.raises(ValueError, match="not a 4-bit weight"):
        int4_linear(x, Int4Weight(w.words, w.scales, 50, 136, 32))
    with pytest.raises(ValueError, match="within -8 .. 7"):
        pack_int4(torch.full((4, 32), 8, dtype=torch.int8, device=DEV), torch.ones(4, 1, dtype=BF, device=DEV), 32)


@pytest.mark.parametrize("N,K", [(40, 300), (40, 1024), (3000, 1024), (200, 1200), (5000, 1300), (33, 8200), (1, 20000), (17, 28672),
                                 (12300, 2048)])
def test_the_order_of_a_sum_does_not_depend_on_the_batch(N, K):
    """Few and many columns, short and long rows (the kernel that keeps x, the other one, and rows split over workgroups)."""
    from cdssm_hip import int4_linear
    codes, scales = weight_of(N, K, 64, N + K)
    w = packed(codes, scales, 64)
    x = torch.randn(64, K, generator=torch.Generator().manual_seed(5)).to(BF).to(DEV)
    nw = (1 + 0.1 * torch.randn(K, generator=torch.Generator().manual_seed(6))).to(BF).to(DEV)
    for kw in ({}, {"norm_weight": nw, "eps": 1e-6}):
        y = int4_linear(x, w, **kw)
        for m in (1, 5, 17, 33, 50):
            assert torch.equal(int4_linear(x[:m], w, **kw), y[:m])


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("M,N,K", [(1, 1, 8200), (3, 50, 10000), (20, 600, 8199), (64, 2040, 8192), (33, 100, 28672), (2, 16, 65536)])
def test_long_rows_of_few_columns(M, N, K, group):
    """Whole numbers again, of at most 2: 15 * 2 * K < 2^24 of the smallest scale."""
    from cdssm_hip import int4_linear
    codes, scales = weight_of(N, K, group, M + N, powers=True)
    g = torch.Generator().manual_seed(K)
    x = torch.randint(-1, 2, (M, K), generator=g).to(BF)
    bias, res = torch.randint(-8, 9, (N,), generator=g).to(BF), torch.randint(-8, 9, (M, N), generator=g).to(BF)
    y = int4_linear(x.to(DEV), packed(codes, scales, group), bias=bias.to(DEV), residual=res.to(DEV))
    want = x.double() @ wide(codes, scales, group).t() + bias.double() + res.double()
    assert torch.equal(y.cpu(), want.float().to(BF))


@pytest.mark.parametrize("M,N,K,col,C,taps,group", [(1, 3104, 1024, 1024, 1024, 4, 64), (64, 3104, 1024, 1024, 1024, 4, 128),
                                                    (5, 100, 768, 7, 50, 1, 32), (33, 77, 100, 0, 77, 8, 64), (20, 300, 250, 290, 10, 2, 32),
                                                    (17, 4992, 1000, 1536, 1536, 4, 128), (3, 200, 2048, 50, 100, 4, 64),
                                                    (40, 12416, 2048, 4096, 4096, 4, 64)])
def test_a_product_with_the_conv_step_is_the_two_calls(M, N, K, col, C, taps, group):
    from cdssm_hip import int4_linear, int4_linear_conv_step
    from cdssm_hip.lm import conv1d_silu_step
    log(f"[int4 conv] M{M} N{N} K{K} col {col} C{C} taps {taps}")
    codes, scales = weight_of(N, K, group, M + N)
    w = packed(codes, scales, group)
    g = torch.Generator().manual_seed(K)
    r = lambda *s: torch.randn(*s, generator=g).to(BF).to(DEV)  # noqa: E731
    x, bias, nw, win, cw, cb = r(M, K), r(N), 1 + 0.1 * r(K), r(M, taps - 1, C), r(C, 1, taps), r(C)
    win2 = win.clone()
    for _ in range(2):  # the second step reads what the first left in the window
        y, z = int4_linear_conv_step(x, w, bias, nw, 1e-6, col, win, cw, cb)
        want = int4_linear(x, w, bias=bias, norm_weight=nw, eps=1e-6)
        wz = conv1d_silu_step(want[:, col:col + C], win2, cw, cb)
        assert torch.equal(y, want) and torch.equal(z, wz) and torch.equal(win, win2)


def test_a_missing_workspace_is_refused():
    from cdssm_hip import _lib
    lib = _lib.load()
    for N, K, norm in ((16, 1 << 15, 0), (12416, 2048, 1)):
        assert lib.cdssm_int4_linear_workspace_bytes(4, N, K, norm) > 0
        assert lib.cdssm_int4_linear(1, 16, K, 16, 16, 64, None, None, 0, 16 if norm else None, 0.0, 16, N, None, 4, N, K, None) == -1
        assert "workspace" in _lib.last_error()


def test_refusals_of_the_conv_step():
    from cdssm_hip import int4_linear_conv_step
    codes, scales = weight_of(50, 136, 64, 0)
    w = packed(codes, scales, 64)
    z = lambda *s: torch.zeros(*s, dtype=BF, device=DEV)  # noqa: E731
    args = [z(4, 136), w, z(50), z(136), 1e-6, 10, z(4, 3, 20), z(20, 4), z(20)]

    def call(i, v):
        return int4_linear_conv_step(*args[:i], v, *args[i + 1:])
    for i, v, error, msg in ((5, 31, RuntimeError, "inside the product"), (5, -1, RuntimeError, "inside the product"),
                             (6, z(4, 2, 20), ValueError, "window must be"), (6, z(4, 3, 20).float(), ValueError, "window must be"),
                             (6, z(4, 20, 3).transpose(1, 2), ValueError, "window must be"), (7, z(19, 4), ValueError, "conv_weight"),
                             (0, z(136), ValueError, "x must be"), (8, torch.zeros(20, dtype=BF), RuntimeError, "must be on"),
                             (7, z(20, 4).requires_grad_(True), NotImplementedError, "no gradient")):
        with pytest.raises(error, match=msg):
            call(i, v)
    with pytest.raises(RuntimeError, match="kernel_size <= 8"):
        int4_linear_conv_step(*args[:6], z(4, 8, 20), z(20, 9), z(20))


def test_more_codes_than_32_bits_hold():
    from cdssm_hip import int4_linear, pack_int4
    N, K, group = 140000, 32768, 128  # 4.6e9 codes, 2.3 GB packed
    g = torch.Generator(device=DEV).manual_seed(0)
    codes = torch.randint(-8, 8, (N, K), dtype=torch.int8, device=DEV, generator=g)
    scales = torch.exp2(torch.randint(-1, 1, (N, K // group), device=DEV, generator=g).float()).to(BF)
    w = pack_int4(codes, scales, group)
    x = torch.randint(-1, 2, (3, K), device=DEV, generator=g).to(BF)
    y = int4_linear(x, w)
    for cols in (slice(0, 5), slice(131070, 131075), slice(N - 5, N)):  # either side of 2^32 codes
        want = (x.cpu().double() @ wide(codes[cols].cpu(), scales[cols].cpu(), group).t()).float().to(BF)
        assert torch.equal(y[:, cols].cpu(), want)
    c, s = w.unpack()
    assert torch.equal(c[-7:], codes[-7:]) and torch.equal(s[-7:], scales[-7:])


def test_what_lies_between_the_result_s_rows_stays():
    from cdssm_hip import _lib, int4_linear
    codes, scales = weight_of(50, 136, 64, 0)
    w = packed(codes, scales, 64)
    x = torch.randn(20, 136, device=DEV).to(BF)
    wide_y = torch.full((22, 61), -7.0, dtype=BF, device=DEV)
    st = _lib.load().cdssm_int4_linear(1, x.data_ptr(), 136, w.words.data_ptr(), w.scales.data_ptr(), 64, None, None, 0, None, 0.0,
                                       wide_y[1:].data_ptr(), 61, None, 20, 50, 136, _lib.stream_of(DEV))
    _lib.check(st, "cdssm_int4_linear")
    want = int4_linear(x, w)
    torch.cuda.synchronize()
    assert torch.equal(wide_y[1:21, :50], want)
    wide_y[1:21, :50] = -7.0
    assert (wide_y == -7.0).all()


def step_bound(xd, codes, scales, group, y):
    """Products of codes and x are exact in fp32, and what is added has no other parts: every one of a group's g sums is off by at most
    2^-24 of the magnitudes added so far, and so are the groups' sums, the product with a scale and the waves' joining."""
    K = xd.shape[1]
    return 2.0 ** -24 * (min(group, K) + 2 * -(-K // group) + 24) * (xd.abs() @ wide(codes, scales, group).abs().t()) + 2.0 ** -8 * y.abs()


@pytest.mark.parametrize("large", [2.0 ** 14, 2.0 ** 20, 2.0 ** 60])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("M,N,K,group", [(1, 48, 128, 128), (3, 100, 1024, 64), (64, 200, 1000, 32), (20, 4000, 1024, 128),
                                         (5, 300, 2000, 128), (33, 9000, 2048, 64), (2, 40, 9000, 128)])
def test_a_large_element_costs_the_columns_that_leave_it_out_nothing(M, N, K, group, norm, large):
    from cdssm_hip import int4_linear
    log(f"[int4] M{M} N{N} K{K} g{group} norm {norm} large {large:.0e}")
    codes, scales = weight_of(N, K, group, M + N + K)
    g = torch.Generator().manual_seed(K)
    x = torch.randn(M, K, generator=g).to(BF)
    for m, at in enumerate(torch.randint(0, K, (M,), generator=g).tolist()):
        x[m, at] = large * (-1) ** m
        codes[:, at] = 0
    xd = x.double()
    kw = {}
    if norm:
        nw = (1 + 0.2 * torch.randn(K, generator=g)).to(BF)
        xd = xd * torch.rsqrt(xd.pow(2).mean(1, keepdim=True) + 1e-5) * nw.double()
        kw = dict(norm_weight=nw.to(DEV), eps=1e-5)
    y = int4_linear(x.to(DEV), packed(codes, scales, group), **kw)
    want = xd @ wide(codes, scales, group).t()
    e = step_bound(xd, codes, scales, group, want)
    if norm:  # x' to 2^-17, the row's scale to a few steps
        e = e + 2.0 ** -17 * (xd.abs() @ wide(codes, scales, group).abs().t()) + 2.0 ** -20 * want.abs()
    off = ((y.cpu().double() - want).abs() / e).max()
    log(f"  worst {float(off):.3f} of the bound")
    assert float(off) <= 1.0


@pytest.mark.parametrize("M,N,K", [(2, 48, 128), (20, 300, 1000), (5, 300, 2000)])
def test_factors_of_two_come_out_of_a_product(M, N, K):
    """Without a norm nothing but the exponents changes, up to sums of 8 |x| over a group below 2^128."""
    from cdssm_hip import int4_linear
    codes, scales = weight_of(N, K, 128, M + N + K)
    w = packed(codes, scales, 128)
    x = torch.randn(M, K, generator=torch.Generator().manual_seed(K)).to(BF).to(DEV)
    y = int4_linear(x, w).double()
    for e in (-60, 60, 100, 116):
        assert torch.equal(int4_linear(x * 2.0 ** e, w).double(), y * 2.0 ** e)


def test_infinities_and_nan_in_x():
    """Not finite in any column, as the formula has it: infinite where the weight is not 0, NaN where it is and where infinities meet."""
    from cdssm_hip import int4_linear
    codes, scales = weight_of(100, 256, 64, 7)
    codes[:50, 9], codes[50:, 9] = 0, 3
    w = packed(codes, scales, 64)
    x = torch.randn(4, 256, generator=torch.Generator().manual_seed(1)).to(BF)
    clean = int4_linear(x.to(DEV), w)
    x[0, 9], x[1, 9], x[2, 9] = float("inf"), -float("inf"), float("nan")
    y = int4_linear(x.to(DEV), w)
    assert torch.isnan(y[:3, :50]).all() and (y[0, 50:] == float("inf")).all() and (y[1, 50:] == -float("inf")).all()
    assert torch.isnan(y[2]).all() and torch.equal(y[3], clean[3])
    assert torch.isnan(int4_linear(x.to(DEV), w, norm_weight=torch.ones(256, dtype=BF, device=DEV))[:3]).all()


@pytest.mark.parametrize("M,N,K", [(4, 48, 128), (20, 300, 1000), (5, 300, 2000), (4, 12416, 2048), (3, 40, 9000)])
def test_rows_whose_squares_pass_fp32_are_nan_and_alone(M, N, K):
    from cdssm_hip import int4_linear
    codes, scales = weight_of(N, K, 128, M + N + K)
    w = packed(codes, scales, 128)
    x = torch.randn(M, K, generator=torch.Generator().manual_seed(K)).to(BF).to(DEV)
    nw, bias = torch.ones(K, dtype=BF, device=DEV), torch.ones(N, dtype=BF, device=DEV)
    clean = int4_linear(x, w, bias=bias, norm_weight=nw, eps=1e-6)
    x[1, K // 2] = 2.0 ** 64
    x[2] *= 2.0 ** 60 / 64  # (below: the same row but for eps)
    y = int4_linear(x, w, bias=bias, norm_weight=nw, eps=1e-6)
    assert torch.isnan(y[1]).all()
    assert torch.equal(y[3:], clean[3:]) and torch.equal(y[0], clean[0])
    want = x[2].cpu().double() @ wide(codes, scales, 128).t() * torch.rsqrt(x[2].cpu().double().pow(2).mean()) + 1
    assert torch.isfinite(y[2]).all() and ((y[2].cpu().double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -8).all()


def fingerprint_of(w):
    """The definition in whole numbers modulo 2^64."""
    bits = w.contiguous().view(torch.int16 if w.dtype == BF else torch.int32).tolist()
    size = 2 if w.dtype == BF else 4
    per, total = -(-len(bits[0]) * size // 16), 0
    for n, row in enumerate(bits):
        raw = b"".join((v % 2 ** (8 * size)).to_bytes(size, "little") for v in row).ljust(16 * per, b"\0")
        for c in range(per):
            h = (n * per + c + 1) * 0x9e3779b97f4a7c15 % 2 ** 64
            for i in range(4):
                h = (h ^ int.from_bytes(raw[16 * c + 4 * i:16 * c + 4 * i + 4], "little")) * 0x6a09e667f3bcc909 % 2 ** 64
                h ^= h >> 32
            total += h
    total %= 2 ** 64
    return total - 2 ** 64 if total >= 2 ** 63 else total


@pytest.mark.parametrize("dtype", [BF, torch.float32])
@pytest.mark.parametrize("N,K", [(1, 1), (3, 7), (5, 8), (9, 129), (2, 1200)])
def test_fingerprints_are_their_definition(N, K, dtype):
    """Of a weight as it lies, by columns, off 16 bytes, and in rows of a wider tensor whose other elements are none of it."""
    from cdssm_hip.int4 import fingerprints
    w = torch.randn(N, K, generator=torch.Generator().manual_seed(N * K)).to(dtype).to(DEV)
    off, on = (torch.full((N, K + 16), float("nan"), dtype=dtype, device=DEV) for _ in range(2))
    off[:, 3:3 + K], on[:, 8:8 + K] = w, w
    assert fingerprints([w, w.t().contiguous().t(), off[:, 3:3 + K], on[:, 8:8 + K]]) == [fingerprint_of(w.cpu())] * 4


def test_fingerprints_of_many_rows_and_any_change():
    from cdssm_hip.int4 import fingerprints
    w = torch.randn(10007, 130, device=DEV).to(BF)
    first = fingerprints([w])[0]
    assert fingerprints([w, w.clone()]) == [first, first]
    for n, k in ((0, 0), (10006, 129), (8192, 64)):
        other = w.clone()
        other.view(torch.int16)[n, k] ^= 1
        assert fingerprints([other])[0] != first
    assert fingerprints([w.flip(0)])[0] != first and fingerprints([w[:, 1:]])[0] != fingerprints([w[:, :-1]])[0]
    sizes = [(1 + i % 5, 1 + 3 * i) for i in range(150)]  # more than a launch takes, of both types
    ws = [torch.randn(*s, device=DEV).to((BF, torch.float32)[i % 2]) for i, s in enumerate(sizes)]
    assert fingerprints(ws) == [fingerprint_of(w.cpu()) for w in ws]
    for bad, error in ((w.half(), TypeError), (w[0], ValueError), (w.cpu(), RuntimeError), (w[:0], ValueError)):
        with pytest.raises((error, RuntimeError)):
            fingerprints([w, bad])
