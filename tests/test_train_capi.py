"""Argument checks of the training-step entry points (embedding, head loss, gradient clipping): refused calls launch
nothing, so they run without a GPU."""

import ctypes

import pytest

from _gpu_util import log  # noqa: F401
from cdssm_hip import _lib


def _call(name, args, over):
    args = dict(args)
    args.update(over)
    return getattr(_lib.load(), name)(*args.values())


FWD = dict(dtype=1, label_bytes=8, x=16, ldx=64, W=16, ldw=64, labels=16, ignore=-100, reduction=1, loss=16, ws=256, T=4, V=8,
           d=64, stream=None)
BWD = dict(dtype=1, W=16, ldw=64, reduction=1, gloss=16, fwd=256, dx=16, lddx=64, dW=16, lddw=64, ws=256, T=4, V=8, d=64,
           stream=None)
EMB = dict(dtype=1, id_bytes=8, ids=16, W=16, ldw=64, scale=1.0, padding=-1, y=16, order=None, T=4, V=8, C=64, stream=None)
EMBB = dict(dtype=1, id_bytes=8, ids=16, dy=16, lddy=64, scale=1.0, padding=-1, order=None, dW=16, ws=256, T=4, V=8, C=64, stream=None)


@pytest.mark.parametrize("name,args,over,msg", [
    ("cdssm_linear_cross_entropy_fwd", FWD, dict(dtype=2), "dtype"),
    ("cdssm_linear_cross_entropy_fwd", FWD, dict(label_bytes=2), "4 or 8 bytes"),
    ("cdssm_linear_cross_entropy_fwd", FWD, dict(reduction=3), "reduction"),
    ("cdssm_linear_cross_entropy_fwd", FWD, dict(T=0), "1 <= T"),
    ("cdssm_linear_cross_entropy_fwd", FWD, dict(V=(1 << 24) + 1), "2^24"),
    ("cdssm_linear_cross_entropy_fwd", FWD, dict(ldx=63), "row strides"),
    ("cdssm_linear_cross_entropy_fwd", FWD, dict(ldw=63), "row strides"),
    ("cdssm_linear_cross_entropy_fwd", FWD, dict(labels=None), "null"),
    ("cdssm_linear_cross_entropy_fwd", FWD, dict(ws=None), "null"),
    ("cdssm_linear_cross_entropy_bwd", BWD, dict(dx=None, dW=None), "dx or dW"),
    ("cdssm_linear_cross_entropy_bwd", BWD, dict(lddw=60), "row strides"),
    ("cdssm_linear_cross_entropy_bwd", BWD, dict(gloss=None), "null"),
    ("cdssm_linear_cross_entropy_bwd", BWD, dict(fwd=None), "null"),
    ("cdssm_token_embedding_fwd", EMB, dict(dtype=3), "dtype"),
    ("cdssm_token_embedding_fwd", EMB, dict(id_bytes=1), "4 or 8 bytes"),
    ("cdssm_token_embedding_fwd", EMB, dict(ldw=10), "row stride"),
    ("cdssm_token_embedding_fwd", EMB, dict(C=0, ldw=0), "C >= 1"),
    ("cdssm_token_embedding_fwd", EMB, dict(y=None), "null"),
    ("cdssm_token_embedding_bwd", EMBB, dict(T=1 << 29), "2^28"),
    ("cdssm_token_embedding_bwd", EMBB, dict(lddy=1), "row stride"),
    ("cdssm_token_embedding_bwd", EMBB, dict(ws=None), "null"),
])
def test_invalid_arguments_are_refused(name, args, over, msg):
    assert _call(name, args, over) == -1
    assert msg in _lib.last_error()


def _clip(over):
    P, I, N = ctypes.c_void_p * 2, ctypes.c_int * 2, ctypes.c_int64 * 2
    args = dict(count=2, ins=P(16, 32), di=I(0, 1), outs=P(16, 32), do=I(0, 1), n=N(4, 4), max_norm=1.0, norm=16, ws=256,
                stream=None)
    args.update({k: (P if k in ("ins", "outs") else I if k in ("di", "do") else N)(*v) if isinstance(v, tuple) else v
                 for k, v in over.items()})
    return _lib.load().cdssm_clip_grads(*args.values())


@pytest.mark.parametrize("over,msg", [
    (dict(count=-1), "negative count"),
    (dict(ins=(16, None)), "null pointer"),
    (dict(outs=(None, 32)), "null pointer"),
    (dict(n=(4, -1)), "size out of range"),
    (dict(n=(4, (1 << 38) + 1)), "size out of range"),
    (dict(di=(0, 5)), "dtype"),
    (dict(do=(2, 1)), "dtype"),
    (dict(ins=(18, 32)), "aligned"),
    (dict(ins=(16, 33)), "aligned"),
    (dict(max_norm=-1.0), "max_norm"),
    (dict(max_norm=float("nan")), "max_norm"),
    (dict(norm=None), "null"),
    (dict(ws=None), "null"),
    (dict(outs=None), "null"),
])
def test_clip_grads_refuses_invalid_arguments(over, msg):
    assert _clip(over) == -1
    assert msg in _lib.last_error()


def test_workspace_sizes():
    lib = _lib.load()
    assert lib.cdssm_linear_cross_entropy_workspace_bytes(1, 16, 64, 0, 8, 64) == -1
    assert lib.cdssm_linear_cross_entropy_bwd_workspace_bytes(2, 16, 64, 4, 8, 64) == -1
    assert lib.cdssm_token_embedding_bwd_workspace_bytes(4, 0, 8) == -1
    assert lib.cdssm_grad_norm_workspace_bytes(-1) == -1
    assert lib.cdssm_token_embedding_order_bytes(0, 8) == -1
    assert lib.cdssm_token_embedding_order_bytes(1000, 100) == 4096 + 1024
    assert lib.cdssm_token_embedding_bwd_workspace_bytes(1000, 100, 64) == 4096 + 1024 + 4 * 31 * 64
    # a weight that the kernels cannot read in place (fp32, or rows that are no whole 128 bytes) is packed
    n = lib.cdssm_linear_cross_entropy_workspace_bytes
    base = n(1, 256, 1024, 512, 32000, 1024)
    assert n(1, 258, 1024, 512, 32000, 1024) - base == 2 * 32000 * 1024
    # (fp32: three planes of x and W, statistics of tiles of 128 words instead of 256, and no list of the words' first rows)
    assert n(0, 256, 1024, 512, 32000, 1024) - base == 2 * (3 * 32000 + 2 * 512) * 1024 + 8 * 125 * 512 - 4 * 32000
    # the backward keeps at most 256 MB of softmax gradient, whatever the vocabulary
    b = lib.cdssm_linear_cross_entropy_bwd_workspace_bytes
    assert b(1, 256, 64, 16384, 1 << 20, 64) <= (256 << 20) + (256 << 20)


def test_the_loss_keeps_its_checks_off_the_gpu():
    import torch
    from cdssm_hip import clip_grads, global_grad_norm, linear_cross_entropy, token_embedding
    from cdssm_hip.train import linear_cross_entropy_bwd
    x, w, y = torch.randn(4, 8), torch.randn(5, 8), torch.zeros(4, dtype=torch.long)
    with pytest.raises(RuntimeError, match="GPU only"):
        linear_cross_entropy(x, w, y)
    with pytest.raises(RuntimeError, match="GPU only"):
        token_embedding(y, w)
    with pytest.raises(RuntimeError, match="GPU only"):
        clip_grads([x], 1.0)
    with pytest.raises(RuntimeError, match="GPU only"):
        linear_cross_entropy_bwd(torch.ones(()), w, None, x.shape)
    assert float(global_grad_norm([])) == 0.0


def test_missing_nodes_are_named(monkeypatch):
    import sys
    import torch
    import cdssm_hip
    from cdssm_hip import global_grad_norm, train
    monkeypatch.setattr(train, "_nodes", None)
    monkeypatch.setitem(sys.modules, "cdssm_hip._train_nodes", None)
    monkeypatch.delattr(cdssm_hip, "_train_nodes", raising=False)
    with pytest.raises(RuntimeError, match="_train_nodes.so not found or not loadable"):
        global_grad_norm([torch.zeros(3)])


def test_room_for_a_sort_in_two_levels():
    """Where one workgroup for 256 ids would read more than 2^26 ids in all, the tokens are sorted into at most 2^16 buckets first."""
    lib = _lib.load()
    n = lib.cdssm_token_embedding_order_bytes
    assert n(16384, 1 << 20) == 4 * 16384 + 8 * (1 << 20)
    assert n(32768, 1 << 20) == 2 * 4 * 32768 + 8 * (1 << 20) + 8 * 4096
    assert n(65536, 1 << 28) == 2 * 4 * 65536 + 8 * (1 << 28) + 8 * 65536
    assert lib.cdssm_token_embedding_bwd_workspace_bytes(32768, 1 << 20, 64) == n(32768, 1 << 20) + 4 * 1024 * 64


def test_clip_grads_without_the_outputs_types():
    assert _clip(dict(do=None)) == -1
    assert "null" in _lib.last_error()


def test_clip_grads_returns_when_memory_runs_out():
    """Two million tensors that lie apart take 60 MB of host memory for the launches' arguments; without it the call returns an error."""
    import subprocess
    import sys
    import torch
    if torch.cuda.is_available():
        pytest.skip("made-up addresses: where a GPU could be given them the call is not made")
    child = """
import ctypes, resource, sys
sys.path[:0] = %r
from cdssm_hip import _lib
lib, N = _lib.load(), 2000000
ins, di, n = (ctypes.c_void_p * N)(*[16] * N), (ctypes.c_int * N)(), (ctypes.c_int64 * N)(*[1] * N)
used = int(open('/proc/self/statm').read().split()[0]) * resource.getpagesize()
resource.setrlimit(resource.RLIMIT_AS, (used + (8 << 20), used + (8 << 20)))
for st in (lib.cdssm_grad_norm(N, ins, di, n, 16, 256, None),
           lib.cdssm_clip_grads(N, ins, di, ins, di, n, 1.0, 16, 256, None)):
    print(st, _lib.last_error())
""" % (sys.path,)
    r = subprocess.run([sys.executable, "-c", child], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, (r.returncode, r.stderr[-300:])
    lines = r.stdout.splitlines()
    assert len(lines) == 2 and all(k.startswith("-") and "host memory" in k for k in lines), r.stdout
