"""CPU: what the operators of a training step refuse, before anything touches a GPU: at the C ABI (status and message, nothing
enqueued) and in the Python functions."""
import ctypes

import pytest
import torch

from deepsignal_plant_amd import _native as nat
from deepsignal_plant_amd import train_ops as ops

P = 4096   # an address that no refused call follows


def refused(rc, message):
    assert rc == nat.DSP_EINVAL and message in nat.last_error(), (rc, nat.last_error())


def test_embedding_refusals_at_the_abi():
    L = nat.lib()
    fwd = lambda n=8, tokens=P, tt=nat.DT_U8, w=P, vocab=16, dim=4, ft=nat.FT_F32, out=P: L.dsp_embedding_forward(None, n, tokens, tt, w, vocab, dim, ft, 1.0, out)
    refused(fwd(n=-1), "number of tokens")
    refused(fwd(n=2 ** 31), "number of tokens")
    refused(fwd(vocab=0), "1 .. 2^31 - 2 rows")
    refused(fwd(vocab=2 ** 31 - 1), "1 .. 2^31 - 2 rows")
    refused(fwd(dim=0), "1 .. 65,536 values")
    refused(fwd(dim=65537), "1 .. 65,536 values")
    refused(fwd(tt=9), "token type")
    refused(fwd(ft=3), "element type")
    refused(fwd(tokens=None), "NULL")
    refused(fwd(w=None), "NULL")
    refused(fwd(out=None), "NULL")
    refused(fwd(out=P + 2), "not aligned")
    assert fwd(n=0, tokens=None, out=None) == 0
    size = L.dsp_embedding_workspace(8, 1600, 4)
    bwd = lambda pad=-1, g=P, out=P, ws=P, size=size: L.dsp_embedding_backward(None, 8, P, nat.DT_U8, g, 1600, 4, nat.FT_F32, pad, 1.0, out, ws, size)
    assert size > 0 and L.dsp_embedding_workspace(8, 16, 4) == 0
    refused(bwd(pad=1600), "padding_idx")
    refused(bwd(pad=-2), "padding_idx")
    refused(bwd(g=None), "NULL")
    refused(bwd(out=None), "NULL")
    refused(bwd(ws=None), "NULL")
    refused(bwd(size=size - 1), "workspace too small")
    refused(bwd(ws=P + 16), "256 bytes")
    refused(bwd(g=P + 1), "not aligned")
    refused(L.dsp_embedding_workspace(-1, 16, 4), "number of tokens")


def test_lstm_refusals_at_the_abi():
    L = nat.lib()

    def layer(batch=4, steps=3, inputs=5, hidden=6, directions=2, missing=None):
        l = nat.LstmLayer(batch, steps, inputs, hidden, directions)
        for k in ("w_ih", "w_hh", "b_ih", "b_hh"):
            for d in range(2):
                getattr(l, k)[d] = None if missing == (k, d) else P
        return l
    fwd = lambda l, x=P, y=P: L.dsp_lstm_forward(None, None if l is None else ctypes.byref(l), x, None, None, y, P, P, P, P, 1)
    refused(fwd(None), "NULL layer")
    refused(fwd(layer(directions=3)), "one direction or two")
    refused(fwd(layer(directions=0)), "one direction or two")
    for bad in (dict(steps=0), dict(inputs=0), dict(hidden=0), dict(batch=-1)):
        refused(fwd(layer(**bad)), "positive")
    refused(fwd(layer(hidden=8193)), "8,192 units")
    refused(fwd(layer(inputs=16385)), "16,384 inputs")
    refused(fwd(layer(batch=2 ** 22 + 1)), "2^22 sequences")
    refused(fwd(layer(batch=2 ** 15, steps=2 ** 15)), "2^30 of both")
    refused(fwd(layer(missing=("b_hh", 1))), "NULL weight")
    refused(fwd(layer(batch=2 ** 20, steps=2 ** 9, hidden=2 ** 10)), "would not fit")
    refused(fwd(layer(batch=2 ** 20, steps=1, hidden=2 ** 11)), "2^31 - 1 values in a state")
    refused(fwd(layer(), x=None), "NULL pointer")
    refused(fwd(layer(), y=None), "NULL pointer")
    assert fwd(layer(batch=0), x=None, y=None) == 0
    l = layer()
    size, g = L.dsp_lstm_workspace(ctypes.byref(l)), nat.LstmGrads()
    bwd = lambda g, dc0=P, ws=P, size=size, l=l: L.dsp_lstm_backward(None, ctypes.byref(l), P, None, P, P, None, None, None, None, None, dc0,
                                                                  None if g is None else ctypes.byref(g), ws, size)
    refused(bwd(None), "NULL layer")
    refused(bwd(g), "NULL weight or gradient")
    for k in ("w_ih", "w_hh", "b_ih", "b_hh"):
        getattr(g, k)[0] = getattr(g, k)[1] = P
    refused(bwd(g, dc0=None), "NULL pointer")
    refused(bwd(g, size=size - 1), "workspace too small")
    refused(bwd(g, ws=P + 64), "256 bytes")
    refused(bwd(g, l=layer(missing=("w_hh", 0))), "NULL weight")


def test_linear_refusals_at_the_abi():
    L = nat.lib()
    size = L.dsp_linear_workspace(8, 4, 2)
    fwd = lambda m=8, k=4, n=2, x=P, w=P, y=P: L.dsp_linear_forward(None, m, k, n, x, w, None, y)
    bwd = lambda w=P, gy=P, dw=P, ws=P, size=size: L.dsp_linear_backward(None, 8, 4, 2, P, w, gy, None, dw, None, ws, size)
    refused(fwd(m=-1), "number of rows")
    refused(fwd(m=2 ** 30), "number of rows")
    for bad in (dict(k=0), dict(n=0), dict(k=16385), dict(n=16385)):
        refused(fwd(**bad), "1 .. 16,384")
    for k in ("x", "w", "y"):
        refused(fwd(**{k: None}), "NULL")
    assert fwd(m=0, x=None, y=None) == 0 and size > 0
    for k in ("w", "gy", "dw"):
        refused(bwd(**{k: None}), "NULL")
    refused(bwd(ws=None), "workspace too small")
    refused(bwd(size=size - 1), "workspace too small")
    refused(bwd(ws=P + 16), "256 bytes")
    refused(L.dsp_linear_workspace(1, 0, 1), "1 .. 16,384")


def test_loss_refusals_at_the_abi():
    L = nat.lib()
    size = L.dsp_cross_entropy_workspace(8)

    def fwd(n=8, c=4, x=P, ft=nat.FT_F32, stride=4, y=P, lt=nat.DT_I64, red=0, loss=P, stat=P, total=P, ws=P, size=size):
        return L.dsp_cross_entropy_forward(None, n, c, x, ft, stride, y, lt, None, -100, red, loss, stat, total, None, ws, size)
    refused(fwd(n=-1), "number of rows")
    refused(fwd(c=0), "number of classes")
    refused(fwd(stride=3), "rows overlap")
    refused(fwd(ft=7), "element type")
    refused(fwd(lt=nat.DT_F32), "labels")
    refused(fwd(red=3), "reduction")
    for k in ("x", "y", "loss", "stat", "total"):
        refused(fwd(**{k: None}), "NULL")
    refused(fwd(ws=None), "workspace")
    refused(fwd(size=size - 1), "workspace too small")
    refused(L.dsp_cross_entropy_workspace(-1), "negative")
    refused(L.dsp_cross_entropy_backward(None, 8, 4, P, 0, 4, P, nat.DT_I64, None, -100, 0, P, P, None, 0, P), "NULL")
    assert L.dsp_cross_entropy_backward(None, 0, 4, None, 0, 4, None, nat.DT_I64, None, -100, 0, None, None, None, 0, None) == 0


def test_clip_refusals_at_the_abi():
    L = nat.lib()

    def clip(n=1, size=10, ptr=P, out=P, ft=nat.FT_F32, oft=nat.FT_F32, max_norm=1.0, norm=P, ws=P, bytes_=1 << 20):
        return L.dsp_clip_grad_norm(None, n, (ctypes.c_void_p * 1)(ptr), (ctypes.c_int64 * 1)(size), (ctypes.c_int32 * 1)(ft),
                                    (ctypes.c_void_p * 1)(out), (ctypes.c_int32 * 1)(oft), max_norm, norm, ws, bytes_)
    refused(clip(n=-1), "negative count")
    refused(clip(norm=None), "NULL")
    refused(clip(ws=None), "NULL")
    refused(clip(ws=P + 8), "256 bytes")
    refused(clip(size=-1), "negative size")
    refused(clip(ptr=None), "NULL tensor")
    refused(clip(out=None), "NULL tensor")
    refused(clip(ft=5), "element type")
    refused(clip(oft=nat.FT_BF16), "type or float32")
    refused(clip(ft=nat.FT_BF16, oft=nat.FT_F16), "type or float32")
    refused(clip(ptr=P + 2), "not aligned")
    refused(clip(max_norm=-1.0), "max_norm")
    refused(clip(max_norm=float("nan")), "max_norm")
    refused(clip(bytes_=100), "workspace too small")


def test_python_refusals():
    t, w = torch.zeros(4, dtype=torch.int64), torch.zeros(16, 4)
    with pytest.raises(RuntimeError, match="no CPU path"):
        ops.embedding(t, w)
    with pytest.raises(RuntimeError, match="no CPU path"):
        ops.cross_entropy(torch.zeros(4, 2), t)
    with pytest.raises(RuntimeError, match="no CPU path"):
        ops.lstm(torch.zeros(1, 1, 4), [torch.zeros(8, 4), torch.zeros(8, 2), torch.zeros(8), torch.zeros(8)])
    with pytest.raises(RuntimeError, match="no CPU path"):
        ops.clip_grad_norm([w], 1.0)
    with pytest.raises(RuntimeError, match="no CPU path"):
        ops.grad_norm([w])
    with pytest.raises(ValueError, match="4 weights"):
        ops.lstm(torch.zeros(1, 1, 4), [w] * 5)
    with pytest.raises(ValueError, match="max_norm"):
        ops.clip_grad_norm([w], -1.0)
    with pytest.raises(ValueError, match="no tensors"):
        ops.clip_grad_norm([], 1.0)
    with pytest.raises(ValueError, match="norm_type"):
        ops.clip_grad_norm_([], 1.0, norm_type=1.0)
    with pytest.raises(ValueError, match="float32, bfloat16"):
        ops.grad_norm([torch.zeros(3, dtype=torch.float64)])
    with pytest.raises(ValueError, match="dense"):
        ops.grad_norm([torch.eye(3).to_sparse()])
    with pytest.raises(ValueError, match="expected a tensor"):
        ops.embedding([1, 2], w)
    assert float(ops.clip_grad_norm_([], 1.0)) == 0.0 and float(ops.clip_grad_norm_([torch.nn.Parameter(w)], 1.0)) == 0.0


def test_overlaps_are_found_behind_a_tensor_inside_another():
    """an output that overlaps a long gradient which a shorter one, also a view of it, comes after"""
    from deepsignal_plant_amd.train_ops import _Pieces
    base = torch.zeros(200)
    ins = _Pieces([base[:100], base[10:20]])
    with pytest.raises(ValueError, match="overlaps a gradient"):
        _Pieces([base[50:60]]).check_apart_from("clip_grad_norm", ins)
    _Pieces([base[100:110]]).check_apart_from("clip_grad_norm", ins)
    _Pieces([base[100:110]]).check_apart_from("clip_grad_norm", _Pieces([base[110:120]]))


def _calls():
    """name -> (a call of an operator, the tensors of it that can carry a derivative)"""
    w, x = torch.zeros(16, 4), torch.zeros(3, 4)
    lstm = [torch.zeros(1, 2, 4), torch.zeros(8, 4), torch.zeros(8, 2), torch.zeros(8), torch.zeros(8), torch.zeros(1, 1, 2), torch.zeros(1, 1, 2)]
    return {"embedding": (lambda w: ops.embedding(torch.zeros(4, dtype=torch.int64), w), [w]),
            "lstm": (lambda *t: ops.lstm(t[0], t[1:5], *t[5:]), lstm),
            "linear": (ops.linear, [x, w, torch.zeros(16)]),
            "cross_entropy": (lambda x, w: ops.cross_entropy(x, torch.zeros(3, dtype=torch.int64), weight=w), [x, torch.ones(4)]),
            "grad_norm": (lambda *g: ops.grad_norm(g), [x, w]),
            "clip_grad_norm": (lambda a, b, c: ops.clip_grad_norm([a, b], 1.0, out=[c, b]), [x, w, torch.zeros(3, 4)])}


@pytest.mark.parametrize("name", sorted(_calls()))
def test_forward_mode_derivatives_and_traces_are_refused(name):
    """a dual tensor's requires_grad is False, and its derivative would be lost; a trace would keep the empty output"""
    from torch.autograd import forward_ad
    call, tensors = _calls()[name]
    for k, t in enumerate(tensors):
        with forward_ad.dual_level():
            args = list(tensors)
            args[k] = forward_ad.make_dual(t, torch.ones_like(t))
            with pytest.raises(RuntimeError, match="forward-mode"):
                call(*args)
            with pytest.raises(RuntimeError, match="no CPU path"):   # no derivative in sight
                call(*tensors)
    with pytest.raises(RuntimeError, match="torch.jit.trace"):
        torch.jit.trace(call, tuple(tensors))


def test_clipping_in_place_refuses_a_dual_gradient():
    from torch.autograd import forward_ad
    p = torch.nn.Parameter(torch.zeros(3))
    with forward_ad.dual_level():
        p.grad = forward_ad.make_dual(torch.ones(3), torch.ones(3))
        with pytest.raises(RuntimeError, match="forward-mode"):
            ops.clip_grad_norm_([p], 1.0)


@pytest.mark.parametrize("name", sorted(_calls()))
def test_what_is_not_there_or_no_tensor_is_refused(name):
    """None and a list in every required place: ValueError, with the operator's name"""
    call, tensors = _calls()[name]
    optional = {"lstm": (5, 6), "linear": (2,), "cross_entropy": (1,)}.get(name, ())
    for k in range(len(tensors)):
        for wrong in ([None] if k not in optional else []) + [[1.0, 2.0]]:
            args = list(tensors)
            args[k] = wrong
            # every other tensor is on the host: whichever is met first is refused, and none as if it had an attribute that it lacks
            with pytest.raises((ValueError, RuntimeError), match=name):
                call(*args)
    for wrong in (None, [1.0]):
        with pytest.raises(ValueError, match=name):
            call(*[wrong] * len(tensors))
