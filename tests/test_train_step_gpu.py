"""A training step through the public entry points: CDSSMLMHeadModel.loss (embedding, blocks, head loss), its backward and
clip_grad_norm_, against the same model with torch's embedding, logits, cross_entropy and clip_grad_norm_.

In fp32 both sides compute the same products in fp32 in different orders; the blocks between them are the same
kernels on inputs that are equal (the embedding copies rows).  The tolerance 2e-5 of the largest value is 2^-24 times
the about 100 terms' magnitudes that meet in a value here (d 64, vocabulary 97, 200 tokens), twice."""

import pytest
import torch

from _gpu_util import DEV, log, rel
from cdssm_hip import clip_grad_norm_, clip_grads, global_grad_norm, linear_cross_entropy, token_embedding
from cdssm_hip.lm import CDSSMConfig, CDSSMLMHeadModel

pytestmark = pytest.mark.gpu


def model(dtype, state_dim=2, seed=0):
    torch.manual_seed(seed)
    cfg = CDSSMConfig(d_model=64, n_layers=2, context_length=256, vocab_size=97, state_dim=state_dim, d_inner=128)
    return CDSSMLMHeadModel(cfg).to(DEV, dtype)


def batch(seed, B=2, L=100, ignored=0.2):
    g = torch.Generator().manual_seed(seed)
    ids = torch.randint(0, 97, (B, L), generator=g)
    labels = torch.randint(0, 97, (B, L), generator=g)
    labels[torch.rand(B, L, generator=g) < ignored] = -100
    return ids.to(DEV), labels.to(DEV)


@pytest.mark.parametrize("state_dim", [2, 16])
def test_a_step_against_torch_around_the_same_blocks(state_dim):
    ids, labels = batch(1)
    a, b = model(torch.float32, state_dim), model(torch.float32, state_dim)
    la = a.loss(ids, labels)
    lb = torch.nn.functional.cross_entropy(b(ids).flatten(0, 1), labels.flatten())
    assert abs(la.item() - lb.item()) <= 1e-6 * lb.item()
    la.backward()
    lb.backward()
    na, nb = clip_grad_norm_(a.parameters(), 0.5), torch.nn.utils.clip_grad_norm_(b.parameters(), 0.5)
    assert abs(float(na) - float(nb)) <= 1e-5 * float(nb) and float(nb) > 0.5
    for (name, p), q in zip(a.named_parameters(), b.parameters()):
        if q.grad is None:  # the first block's value gate, which nothing uses
            assert p.grad is None
            continue
        e = rel(p.grad, q.grad)
        log(f"  {name}: {e:.2e}")
        assert e <= 2e-5, name


def test_bf16_loss_without_gradients_and_the_same_bits_again():
    """The loss of the bf16 model is that of its logits before their rounding to bf16: within 2^-8 of the largest logit
    (each logit's rounding, and the label's) of the loss of the rounded ones."""
    ids, labels = batch(2)
    m = model(torch.bfloat16)
    with torch.no_grad():
        loss = m.loss(ids, labels)
        logits = m(ids).float()
        want = torch.nn.functional.cross_entropy(logits.flatten(0, 1), labels.flatten())
        assert abs(float(loss) - float(want)) <= 2 * 2.0 ** -8 * float(logits.abs().max())
        each = m.loss(ids, labels, reduction="none")
        assert each.shape == labels.shape and torch.equal(each == 0, labels == -100)
        assert torch.equal(loss, m.loss(ids, labels))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_steps_of_an_optimizer_run(dtype):
    m = model(dtype)
    opt = torch.optim.AdamW(m.parameters(), lr=1e-3)
    for k in range(3):
        opt.zero_grad()
        loss = m.loss(*batch(10 + k))
        loss.backward()
        norm = clip_grad_norm_(m.parameters(), 1.0)
        opt.step()
        assert torch.isfinite(loss) and torch.isfinite(norm)
        assert all(torch.isfinite(p.grad).all() for p in m.parameters() if p.grad is not None)


def test_a_captured_step_replayed_among_eager_work():
    """loss, backward and clipping captured in one graph (warmed up on a side stream, as torch asks for), replayed on new
    batches with eager steps of a second model between: every replay gives the eager model's bits."""
    a, b = model(torch.bfloat16), model(torch.bfloat16)
    ids, labels = batch(30)

    def step(m, ids, labels):
        grads = torch.autograd.grad(m.loss(ids, labels), list(m.parameters()), allow_unused=True)
        grads = [g for g in grads if g is not None]
        return clip_grads(grads, 0.1), grads

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step(a, ids, labels)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm, grads = step(a, ids, labels)
    for k in range(3):
        ni, nl = batch(40 + k, ignored=0.1 * k)
        ids.copy_(ni), labels.copy_(nl)
        graph.replay()
        want, wgrads = step(b, ni, nl)
        torch.cuda.synchronize()
        assert torch.equal(norm, want) and len(grads) == len(wgrads)
        assert all(torch.equal(x, y) for x, y in zip(grads, wgrads))


def test_forward_mode_derivatives_raise():
    """Neither a plain operand's tangent nor that of one with a gradient is dropped in silence."""
    w, x = torch.randn(30, 64, device=DEV), torch.randn(10, 64, device=DEV)
    ids = torch.arange(10, device=DEV)
    ad = torch.autograd.forward_ad
    with ad.dual_level():
        for requires_grad in (False, True):
            dw = ad.make_dual(w.clone().requires_grad_(requires_grad), torch.ones_like(w))
            dx = ad.make_dual(x.clone().requires_grad_(requires_grad), torch.ones_like(x))
            with pytest.raises(NotImplementedError, match="token_embedding has no forward-mode"):
                token_embedding(ids, dw)
            for a, b in ((dx, w), (x, dw)):
                with pytest.raises(NotImplementedError, match="linear_cross_entropy has no forward-mode"):
                    linear_cross_entropy(a, b, ids)
        with pytest.raises(NotImplementedError, match="global_grad_norm has no forward-mode"):
            global_grad_norm([x, ad.make_dual(w, torch.ones_like(w))])
        before = w.clone()
        with pytest.raises(NotImplementedError, match="clip_grads has no forward-mode"):
            clip_grads([ad.make_dual(w, torch.ones_like(w))], 0.1)
        with pytest.raises(NotImplementedError, match="clip_grads has no forward-mode"):
            clip_grads([x], 0.1, out=[ad.make_dual(torch.empty_like(x), torch.ones_like(x))])
        assert torch.equal(w, before)
        assert torch.equal(token_embedding(ids, w), w[ids])
