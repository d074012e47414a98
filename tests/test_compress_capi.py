"""Argument checks of top logits, distillation and 4-bit weights: refused calls launch nothing, so they run without a GPU."""

import ctypes
import sys

import pytest
import torch

from cdssm_hip import _lib

TOP = dict(dtype=1, logits=16, ld=100, values=16, ids=16, T=4, V=100, k=8, stream=None)
FWD = dict(dtype=1, teacher_dtype=1, id_bytes=8, logits=16, ld=100, z=16, ids=16, tau=1.0, reduction=1, loss=16, ws=256, T=4, V=100,
           K=8, stream=None)
BWD = dict(dtype=1, teacher_dtype=1, id_bytes=8, logits=16, ld=100, z=16, ids=16, tau=1.0, reduction=1, gloss=16, ws=256, grad=16,
           ldg=100, T=4, V=100, K=8, stream=None)
PACK = dict(codes=16, scales=16, words=16, word_scales=16, N=16, K=128, group=64, stream=None)
QUANT = dict(dtype=1, W=16, ldw=128, codes=16, scales=16, N=16, K=128, group=64, stream=None)
LIN = dict(dtype=1, X=16, ldx=128, words=16, word_scales=16, group=64, bias=None, R=None, ldr=0, wnorm=None, eps=0.0, Y=16, ldy=16,
           ws=None, M=4, N=16, K=128, stream=None)
CONV = dict(dtype=1, X=16, ldx=128, words=16, word_scales=16, group=64, bias=None, wnorm=16, eps=0.0, Y=16, ldy=16, ws=None, M=4,
            N=16, K=128, col=4, window=16, w=16, b=16, y=16, C=8, taps=4, stream=None)


@pytest.mark.parametrize("name,args,over,msg", [
    ("cdssm_top_logits", TOP, dict(dtype=2), "dtype"),
    ("cdssm_top_logits", TOP, dict(logits=None), "null"),
    ("cdssm_top_logits", TOP, dict(ids=None), "null"),
    ("cdssm_top_logits", TOP, dict(k=0), "1 <= k"),
    ("cdssm_top_logits", TOP, dict(k=101), "1 <= k"),
    ("cdssm_top_logits", TOP, dict(V=1000, ld=1000, k=129), "1 <= k"),
    ("cdssm_top_logits", TOP, dict(T=0), "1 <= T"),
    ("cdssm_top_logits", TOP, dict(V=(1 << 24) + 1, ld=1 << 25), "2^24"),
    ("cdssm_top_logits", TOP, dict(ld=99), "row stride"),
    ("cdssm_top_logits", TOP, dict(logits=17), "aligned"),
    ("cdssm_top_logits", TOP, dict(ids=20), "aligned"),
    ("cdssm_distillation_fwd", FWD, dict(dtype=3), "dtypes"),
    ("cdssm_distillation_fwd", FWD, dict(teacher_dtype=-1), "dtypes"),
    ("cdssm_distillation_fwd", FWD, dict(id_bytes=2), "4 or 8 bytes"),
    ("cdssm_distillation_fwd", FWD, dict(reduction=3), "reduction"),
    ("cdssm_distillation_fwd", FWD, dict(tau=0.0), "temperature"),
    ("cdssm_distillation_fwd", FWD, dict(tau=float("nan")), "temperature"),
    ("cdssm_distillation_fwd", FWD, dict(K=257), "K <= 256"),
    ("cdssm_distillation_fwd", FWD, dict(K=0), "1 <= K"),
    ("cdssm_distillation_fwd", FWD, dict(T=0), "1 <= T"),
    ("cdssm_distillation_fwd", FWD, dict(ld=99), "row strides"),
    ("cdssm_distillation_fwd", FWD, dict(z=None), "null"),
    ("cdssm_distillation_fwd", FWD, dict(ws=None), "null"),
    ("cdssm_distillation_fwd", FWD, dict(ws=260), "workspace"),
    ("cdssm_distillation_fwd", FWD, dict(loss=None), "loss"),
    ("cdssm_distillation_bwd", BWD, dict(grad=None), "grad"),
    ("cdssm_distillation_bwd", BWD, dict(gloss=None), "gloss"),
    ("cdssm_distillation_bwd", BWD, dict(ldg=99), "row stride"),
    ("cdssm_distillation_bwd", BWD, dict(ids=20), "aligned"),
    ("cdssm_int4_pack", PACK, dict(words=None), "null"),
    ("cdssm_int4_pack", PACK, dict(words=24), "aligned"),
    ("cdssm_int4_pack", PACK, dict(group=16), "groups of 32, 64 or 128"),
    ("cdssm_int4_pack", PACK, dict(N=1 << 24, K=1 << 24), "2^34"),
    ("cdssm_int4_unpack", PACK, dict(codes=None), "null"),
    ("cdssm_int4_quantize", QUANT, dict(dtype=2), "dtype"),
    ("cdssm_int4_quantize", QUANT, dict(ldw=127), "row stride"),
    ("cdssm_int4_quantize", QUANT, dict(K=0), "1 <= N, K"),
    ("cdssm_int4_linear", LIN, dict(dtype=0), "bf16 only"),
    ("cdssm_int4_linear", LIN, dict(M=0), "M <= 64"),
    ("cdssm_int4_linear", LIN, dict(M=65), "M <= 64"),
    ("cdssm_int4_linear", LIN, dict(X=None), "null"),
    ("cdssm_int4_linear", LIN, dict(ldx=120), "cover K"),
    ("cdssm_int4_linear", LIN, dict(ldx=132), "16-byte aligned"),
    ("cdssm_int4_linear", LIN, dict(K=127, ldx=127), "16-byte aligned"),
    ("cdssm_int4_linear", LIN, dict(X=24), "16-byte aligned"),
    ("cdssm_int4_linear", LIN, dict(wnorm=24), "16-byte aligned"),
    ("cdssm_int4_linear", LIN, dict(ldy=1 << 25), "row strides"),
    ("cdssm_int4_linear", LIN, dict(ldy=15), "row strides"),
    ("cdssm_int4_linear", LIN, dict(R=16, ldr=15), "row strides"),
    ("cdssm_int4_linear", LIN, dict(words=8), "aligned"),
    ("cdssm_int4_linear", LIN, dict(Y=17), "aligned"),
    ("cdssm_int4_linear", LIN, dict(N=12416, ldy=12416, K=2048, ldx=2048, wnorm=16), "workspace"),
    ("cdssm_int4_linear_conv_step", CONV, dict(window=None), "null"),
    ("cdssm_int4_linear_conv_step", CONV, dict(y=None), "null"),
    ("cdssm_int4_linear_conv_step", CONV, dict(col=9), "inside the product"),
    ("cdssm_int4_linear_conv_step", CONV, dict(taps=9), "kernel_size <= 8"),
    ("cdssm_int4_linear_conv_step", CONV, dict(w=17), "aligned"),
    ("cdssm_int4_linear_conv_step", CONV, dict(M=65), "M <= 64"),
])
def test_invalid_arguments_are_refused(name, args, over, msg):
    assert getattr(_lib.load(), name)(*{**args, **over}.values()) == -1
    assert msg in _lib.last_error()


def test_sizes():
    lib = _lib.load()
    assert lib.cdssm_distillation_workspace_bytes(100) == 256 + 1200
    assert lib.cdssm_distillation_workspace_bytes(0) == -1
    # 16 columns and 128 k take 1 KB of codes, and 16 scales for every group of the 128
    assert lib.cdssm_int4_code_bytes(17, 129) == 4 * 1024
    assert [lib.cdssm_int4_scale_bytes(17, 129, g) for g in (32, 64, 128)] == [4 * 128, 4 * 64, 4 * 32]
    assert lib.cdssm_int4_code_bytes(0, 4) == -1 and lib.cdssm_int4_scale_bytes(4, 4, 48) == -1


def test_workspaces_of_a_product_are_sized_without_a_device():
    n = _lib.load().cdssm_int4_linear_workspace_bytes
    assert n(0, 16, 128, 0) == -1 and n(65, 16, 128, 0) == -1 and n(4, 0, 128, 0) == -1
    assert n(64, 32000, 1024, 0) == n(64, 32000, 1024, 1) == 0            # x is kept: nothing besides
    assert n(64, 32000, 4096, 0) == 0
    # a norm of long rows and many columns: two planes of 4 row tiles x 32 blocks, and the squares of 2 shares
    assert n(64, 32000, 4096, 1) == 2 * 2 * 64 * 4096 + 2 * 64 * 4


def test_python_checks_off_the_gpu():
    from cdssm_hip import Int4Weight, distillation_loss, int4_linear, pack_int4, quantize_int4, top_logits
    x, z, ids = torch.randn(4, 8), torch.randn(4, 3), torch.zeros(4, 3, dtype=torch.long)
    for call in (lambda: top_logits(x, 2), lambda: distillation_loss(x, z, ids), lambda: quantize_int4(x, 32),
                 lambda: pack_int4(torch.zeros(4, 8, dtype=torch.int8), torch.ones(4, 1).bfloat16(), 32)):
        with pytest.raises(RuntimeError, match="GPU only"):
            call()
    with pytest.raises(ValueError, match="group_size"):
        quantize_int4(x, 16)
    with pytest.raises(ValueError, match="not a 4-bit weight"):
        int4_linear(x, Int4Weight(torch.zeros(1024, dtype=torch.uint8), torch.zeros(32, dtype=torch.bfloat16), 4, 8, 64))


def test_missing_nodes_are_named(monkeypatch):
    import cdssm_hip
    from cdssm_hip import distill
    monkeypatch.setattr(distill, "_nodes", None)
    monkeypatch.setitem(sys.modules, "cdssm_hip._compress_nodes", None)
    monkeypatch.delattr(cdssm_hip, "_compress_nodes", raising=False)
    with pytest.raises(RuntimeError, match="_compress_nodes.so not found or not loadable"):
        distill._native()


@pytest.mark.parametrize("over,msg", [(dict(count=0), "at least one"), (dict(dtype=2), "dtypes"), (dict(W=None), "null"),
                                      (dict(sums=None), "null"), (dict(N=0), "1 <= N, K"), (dict(ldw=127), "row strides"),
                                      (dict(W=17), "aligned"), (dict(sums=20), "aligned"), (dict(N=1 << 24, K=1 << 24, ldw=1 << 24), "2^34")])
def test_invalid_arguments_of_fingerprints_are_refused(over, msg):
    """The second of two weights is wrong: nothing is launched for the first either."""
    a = {**dict(count=2, dtype=1, W=16, ldw=128, N=16, K=128, sums=16), **over}
    i64 = ctypes.c_int64 * 2
    args = ((ctypes.c_int * 2)(1, a["dtype"]), (ctypes.c_void_p * 2)(16, a["W"]), i64(128, a["ldw"]), i64(16, a["N"]), i64(128, a["K"]))
    assert _lib.load().cdssm_int4_fingerprints(a["count"], *args, a["sums"], None) == -1
    assert msg in _lib.last_error()
