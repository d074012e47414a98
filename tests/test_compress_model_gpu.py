"""A smaller model from a larger one through the public entry points: a teacher's top logits, the student's loss against them and
its gradients, the student's weights in 4 bits, its decode steps.

Gradients in fp32: as in the training step's test, both sides compute the same products in different orders around the same
blocks: 2e-5 of the largest value.  Decode steps: against the same steps with the 4-bit products in 64 bits, both sides round to
bf16 after every product, and a rounding that falls the other way (2^-8) goes on through the following layers: 2e-2 of the
largest logit, as for the other bf16 steps."""

import pytest
import torch

from _gpu_util import DEV, log, rel
from cdssm_hip import clip_grad_norm_, lm
from cdssm_hip.lm import CDSSMConfig, CDSSMLMHeadModel

pytestmark = pytest.mark.gpu


def model(dtype, d_model=128, n_layers=2, vocab=97, seed=0):
    torch.manual_seed(seed)
    cfg = CDSSMConfig(d_model=d_model, n_layers=n_layers, context_length=256, vocab_size=vocab, state_dim=2, d_inner=d_model)
    m = CDSSMLMHeadModel(cfg)
    with torch.no_grad():  # paths that are zero at the start
        for blk in m.blocks:
            blk.v_residual_gate.normal_(std=1.0)
            blk.shortcut_scale.fill_(0.3)
            blk.D.normal_(std=0.1)
    return m.to(DEV, dtype)


def tokens(seed, B=2, L=60, vocab=97):
    return torch.randint(0, vocab, (B, L), generator=torch.Generator().manual_seed(seed)).to(DEV)


def kl(logits, z, ids, tau):
    """The definition in torch, mean over the tokens that take part."""
    part = z != -float("inf")
    has = part.any(-1)
    logp = torch.log_softmax(torch.where(has[..., None], z, 0.0).float() / tau, -1)
    p = torch.where(part & has[..., None], logp.exp(), 0.0)
    logq = torch.log_softmax(logits.float() / tau, -1).gather(-1, ids)
    each = torch.where(p > 0, p * (logp - logq), 0.0).sum(-1) * tau ** 2
    return each.sum() / has.sum()


@pytest.mark.parametrize("vocab", [97, 2100])  # 2100: the head's product is computed with padded words, logits strided
def test_a_student_s_gradients_against_torch_around_the_same_blocks(vocab):
    ids = tokens(1, vocab=vocab)
    teacher = model(torch.float32, d_model=192, seed=5, vocab=vocab)
    z, at = teacher.top_logits(ids, 8)
    assert z.shape == at.shape == (2, 60, 8) and not z.requires_grad
    with torch.no_grad():
        top = teacher(ids)
        assert torch.equal(z, top.gather(-1, at)) and torch.equal(z[..., 0], top.amax(-1))
    z[:, 50:] = -float("inf")  # padding
    a, b = (model(torch.float32, vocab=vocab) for _ in range(2))
    la = a.distill_loss(ids, z, at, temperature=2.0)
    lb = kl(b(ids), z, at, 2.0)
    assert abs(la.item() - lb.item()) <= 2e-6 * (1 + lb.item())
    la.backward()
    lb.backward()
    for (name, p), q in zip(a.named_parameters(), b.parameters()):
        if q.grad is None:
            assert p.grad is None
            continue
        e = rel(p.grad, q.grad)
        log(f"  {name}: {e:.2e}")
        assert e <= 2e-5, name
    with torch.no_grad():
        assert abs(float(a.distill_loss(ids, z, at, temperature=2.0)) - la.item()) <= 1e-6 * la.item()


def plain_int4_linear(x, weight, bias=None, residual=None, norm_weight=None, eps=0.0):
    y = x.double()
    if norm_weight is not None:
        y = y * torch.rsqrt(y.pow(2).mean(-1, keepdim=True) + eps) * norm_weight.double()
    y = y @ weight.dequantize(torch.float64).t()
    for t in (bias, residual):
        if t is not None:
            y = y + t.double()
    return y.to(x.dtype)


def steps(m, ids, n=5):
    with torch.no_grad():
        logits, caches = m.prefill(ids)
        out = [logits]
        for _ in range(n):
            out.append(m.decode_step(out[-1].argmax(-1), caches))
    return torch.stack(out)


@pytest.mark.parametrize("B,d,group,fused", [(1, 1024, 64, True), (3, 256, 32, True), (64, 128, 128, True), (2, 192, 64, True),
                                             (2, 128, 64, False)])
def test_decode_steps_with_4_bit_weights(B, d, group, fused, monkeypatch):
    log(f"[int4 decode] B{B} d{d} group {group}")
    m = model(torch.bfloat16, d_model=d).eval()
    for blk in m.blocks:
        blk.fused_step = fused
    m.quantize_int4_(group)
    ids = tokens(2, B=B, L=37)
    got = steps(m, ids)
    with monkeypatch.context() as mp:
        mp.setattr(lm, "int4_linear", plain_int4_linear)
        with torch.no_grad():
            logits, caches = m.prefill(ids)
            for k in range(5):
                want = m.decode_step(got[k].argmax(-1), caches)  # the same tokens
                e = rel(got[k + 1], want)
                log(f"  step {k}: {e:.2e}")
                assert e <= 2e-2


def test_going_back_gives_the_bf16_steps_and_the_head_may_stay():
    m = model(torch.bfloat16).eval()
    ids = tokens(3)
    before = steps(m, ids)
    m.quantize_int4_(32)
    assert not torch.equal(steps(m, ids)[1:], before[1:])
    assert torch.equal(steps(m, ids)[0], before[0])  # prefill keeps the bf16 weights
    m.quantize_int4_(32, head=False)
    with torch.no_grad():
        _, caches = m.prefill(ids)
    assert "int4" in caches[0] and "int4_head" not in caches[-1]
    m.quantize_int4_(None)
    assert torch.equal(steps(m, ids), before)


def test_captured_steps_equal_eager_ones():
    m = model(torch.bfloat16, d_model=256).eval()
    m.quantize_int4_(64)
    ids = tokens(4, B=4)
    with torch.no_grad():
        logits, eager = m.prefill(ids)
        _, caches = m.prefill(ids)
        graph = m.decode_graph(caches)
        new = logits.argmax(-1)
        for _ in range(5):
            a = graph(new).clone()
            b = m.decode_step(new, eager)
            torch.cuda.synchronize()
            assert torch.equal(a, b)
            new = b.argmax(-1)


def test_refusals():
    with pytest.raises(TypeError, match="bfloat16 model"):
        model(torch.float32).quantize_int4_()
    m = model(torch.bfloat16).eval()
    with pytest.raises(ValueError, match="group_size"):
        m.quantize_int4_(48)
    m.quantize_int4_()
    with torch.no_grad():
        with pytest.raises(ValueError, match="at most 64 rows"):
            m.prefill(tokens(5, B=65, L=3))
        m.blocks[1].out_proj.weight.mul_(2.0)
        with pytest.raises(RuntimeError, match="changed since quantize_int4_"):
            m.prefill(tokens(5))
        m.quantize_int4_()
        _, caches = m.prefill(tokens(5))
        m.embedding.weight.mul_(0.5)
        with pytest.raises(RuntimeError, match="changed since quantize_int4_"):
            m.prefill(tokens(5))
    m.quantize_int4_()
    with torch.no_grad():
        _, caches = m.prefill(tokens(5))
    with pytest.raises(NotImplementedError, match="no gradient"):
        m.decode_step(tokens(5)[:, 0], caches)  # with gradients enabled


def test_the_whole_way_from_a_teacher_to_a_served_student():
    teacher, student = model(torch.bfloat16, d_model=256, seed=1), model(torch.bfloat16, seed=2)
    opt = torch.optim.SGD(student.parameters(), lr=0.1)
    for k in range(3):
        ids = tokens(20 + k)
        z, at = teacher.top_logits(ids, 16)
        opt.zero_grad()
        loss = student.distill_loss(ids, z, at, temperature=2.0)
        loss.backward()
        norm = clip_grad_norm_(student.parameters(), 1.0)
        opt.step()
        assert torch.isfinite(loss) and torch.isfinite(norm)
        assert all(torch.isfinite(p.grad).all() for p in student.parameters() if p.grad is not None)
    student.eval().quantize_int4_(64)
    with torch.no_grad():
        logits, caches = student.prefill(ids)
        graph = student.decode_graph(caches)
        for _ in range(4):
            values, words = lm.top_logits(logits, 5)
            assert torch.equal(values[:, 0], logits.amax(-1))
            logits = graph(words[:, 0]).clone()
            assert torch.isfinite(logits).all()


def test_weights_are_quantized_as_they_are_now():
    """Also after bf16 steps and a write through .data: no copy of an earlier state of them is taken."""
    m, fresh = (model(torch.bfloat16, d_model=256, seed=s).eval() for s in (0, 7))
    ids = tokens(7)
    m.quantize_int4_(64)
    steps(m, ids)
    for p, q in zip((w for b in m.blocks for w in (b.gate_proj.weight, b.gate_proj.bias, b.Q_proj.weight)),
                    (w for b in fresh.blocks for w in (b.gate_proj.weight, b.gate_proj.bias, b.Q_proj.weight))):
        q.data.normal_(std=0.1)
        p.data.copy_(q.data)
    m.quantize_int4_(64)
    fresh.load_state_dict(m.state_dict())
    fresh.quantize_int4_(64)
    assert torch.equal(steps(m, ids), steps(fresh, ids))


def sources(m):
    blk = m.blocks[1]
    return {"in_proj": blk.in_proj.weight, "gate_proj": blk.gate_proj.weight, "Q_proj": blk.Q_proj.weight,
            "out_proj": blk.out_proj.weight, "head": m.lm_head.weight}


@pytest.mark.parametrize("how", ["scaled", "one element", "rows exchanged", "one row turned round"])
@pytest.mark.parametrize("name", ["in_proj", "gate_proj", "Q_proj", "out_proj", "head"])
def test_weights_changed_through_data_are_noticed(name, how):
    """A write through .data moves neither the address nor the version counter of a parameter."""
    m = model(torch.bfloat16, d_model=256).eval()
    ids = tokens(6)
    before = steps(m, ids)
    m.quantize_int4_(64)
    steps(m, ids)
    w = sources(m)[name]
    version = w._version
    old = w.data.clone()
    if how == "scaled":
        w.data.mul_(2.0)
    elif how == "one element":
        w.data[-1, -1] += 1.0
    elif how == "rows exchanged":
        w.data[:2] = w.data[:2].flip(0)
    else:
        w.data[0] = w.data[0].flip(0)
    assert w._version == version and not torch.equal(w, old)
    with torch.no_grad(), pytest.raises(RuntimeError, match="changed since quantize_int4_"):
        m.prefill(ids)
    w.data.copy_(old)
    steps(m, ids)  # as they were
    m.quantize_int4_(None)
    assert torch.equal(steps(m, ids), before)


def test_copies_of_a_model_keep_their_4_bit_weights():
    import copy
    m = model(torch.bfloat16, d_model=256).eval()
    m.quantize_int4_(64)
    ids = tokens(8)
    want = steps(m, ids)
    other = copy.deepcopy(m)
    assert torch.equal(steps(other, ids), want)
    with torch.no_grad():
        other.blocks[0].in_proj.weight.mul_(2.0)
        with pytest.raises(RuntimeError, match="changed since quantize_int4_"):
            other.prefill(ids)
    assert torch.equal(steps(m, ids), want)


def test_weights_that_are_no_dense_tensors_are_watched_too():
    """A weight of strided rows, off 16 bytes, and one of dense columns."""
    m = model(torch.bfloat16, d_model=256).eval()
    ids = tokens(9)
    blk = m.blocks[0]
    wide = torch.zeros(blk.out_proj.weight.shape[0], 300, dtype=torch.bfloat16, device=DEV)
    blk.out_proj.weight = torch.nn.Parameter(wide[:, 3:259].copy_(blk.out_proj.weight.detach()))
    blk.Q_proj.weight = torch.nn.Parameter(blk.Q_proj.weight.detach().t().contiguous().t())
    m.quantize_int4_(64)
    want = steps(m, ids)
    wide[:, :3] = 1.0  # not the weight's
    assert torch.equal(steps(m, ids), want)
    for w in (blk.out_proj.weight, blk.Q_proj.weight):
        m.quantize_int4_(64)
        w.data[5, 200] += 1.0
        with torch.no_grad(), pytest.raises(RuntimeError, match="changed since quantize_int4_"):
            m.prefill(ids)


def test_a_block_s_own_cache_is_checked_every_time():
    """A block called by itself checks its weights too, also where its cache is that of an earlier prompt, and leaves nothing of it."""
    m = model(torch.bfloat16, d_model=256).eval()
    m.quantize_int4_(64)
    blk, x, cache = m.blocks[1], torch.randn(2, 20, 256, device=DEV).to(torch.bfloat16), {}
    with torch.no_grad():
        for _ in range(2):
            blk(x, cache=cache)
            assert "int4" in cache
        with pytest.raises(ValueError, match="at most 64 rows"):
            blk(x[:1].expand(65, 20, 256), cache=cache)
        blk.Q_proj.weight.data[0, 0] += 1.0
        with pytest.raises(RuntimeError, match="changed since quantize_int4_"):
            blk(x, cache=cache)
        m.quantize_int4_(None)
        blk(x, cache=cache)
        assert "int4" not in cache and "w_gq" in cache
        blk.step(x[:, 0], None, cache)


def plain_conv_step(u, window, weight, bias):
    """silu of the taps' sum over the window and the new row, the window moved on by one."""
    full = torch.cat([window, u.unsqueeze(1)], 1)
    y = (full.double() * weight.double().reshape(weight.shape[0], -1).t()).sum(1) + bias.double()
    window.copy_(full[:, 1:])
    return (y * torch.sigmoid(y)).to(u.dtype)


@pytest.mark.parametrize("B,d,group,fused", [(1, 1024, 64, True), (3, 256, 32, True), (64, 128, 128, True), (2, 192, 64, True),
                                             (2, 128, 64, False)])
def test_decode_steps_against_plain_products_and_a_plain_conv(B, d, group, fused, monkeypatch):
    """As above with in_proj and the conv by their definitions too: their columns, norm, biases and window are the block's."""
    log(f"[int4 decode] B{B} d{d} group {group}")
    m = model(torch.bfloat16, d_model=d).eval()
    with torch.no_grad():
        for blk in m.blocks:
            blk.fused_step = fused
            blk.norm.weight.normal_(1.0, 0.2)
            blk.in_proj.bias.normal_(std=0.2)
            blk.conv.bias.normal_(std=0.2)
        m.final_norm.weight.normal_(1.0, 0.2)
    m.quantize_int4_(group)
    ids = tokens(2, B=B, L=37)
    got = steps(m, ids)
    calls = []

    def plain_linear(*args, **kw):
        calls.append("linear")
        return plain_int4_linear(*args, **kw)

    def plain_linear_conv_step(x, weight, bias, norm_weight, eps, col, window, conv_weight, conv_bias):
        calls.append("conv step")
        y = plain_int4_linear(x, weight, bias, norm_weight=norm_weight, eps=eps)
        return y, plain_conv_step(y[:, col:col + conv_bias.shape[0]], window, conv_weight, conv_bias)
    monkeypatch.setattr(lm, "int4_linear", plain_linear)
    monkeypatch.setattr(lm, "int4_linear_conv_step", plain_linear_conv_step)
    with torch.no_grad():
        _, caches = m.prefill(ids)
        for k in range(5):
            want = m.decode_step(got[k].argmax(-1), caches)
            e = rel(got[k + 1], want)
            log(f"  step {k}: {e:.2e}")
            assert e <= 2e-2
    assert calls.count("conv step") == 5 * 2 and calls.count("linear") == 5 * (2 * 2 + 1)
