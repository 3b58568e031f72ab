"""The operators of a training step over the gfx950 kernels: what the reference's `train` (train.py:75-119) takes from torch
around ModelBiLSTM.

  embedding        lookup with scaling, gradient by sorted tokens             (nn.Embedding, models.py:186)
  lstm             one layer, one or both directions                          (nn.LSTM, models.py:137-157)
  linear           a fully connected layer                                    (nn.Linear, models.py:147-161)
  cross_entropy    softmax cross entropy with class weights                   (nn.CrossEntropyLoss)
  clip_grad_norm_  clipping by the norm over many gradients, in place         (nn.utils.clip_grad_norm_)
  clip_grad_norm   the same into other tensors;  grad_norm: the norm alone

The first four are differentiable once by torch's autograd.  Everything runs on the tensors' GPU and its current stream,
enqueues kernels only (no copy, no synchronisation; workspaces come from torch's allocator, so a captured call's belong to its
graph) and gives the same bits for the same inputs and sizes.  There is no CPU path.  ValueError for shapes, types and values;
RuntimeError for tensors that are not on one GPU, that carry a forward-mode derivative, and inside torch.jit.trace."""
from __future__ import annotations

import ctypes
import math
from array import array
from operator import attrgetter

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable
from torch.autograd.graph import increment_version

from . import _native as nat

_FLOAT = {torch.float32: nat.FT_F32, torch.bfloat16: nat.FT_BF16, torch.float16: nat.FT_F16}
_TOKEN = {torch.float32: nat.DT_F32, torch.uint8: nat.DT_U8, torch.uint16: nat.DT_U16, torch.int32: nat.DT_I32, torch.int64: nat.DT_I64}
TOKEN_TYPES = frozenset(_TOKEN)   # of embedding
_LABEL = {torch.uint8: nat.DT_U8, torch.int32: nat.DT_I32, torch.int64: nat.DT_I64}
_REDUCE = {"mean": 0, "sum": 1, "none": 2}


# lists of tensors go through map(): a loop in Python costs as much as the kernels of a small call
_dtype, _layout, _shape, _requires_grad = map(attrgetter, ("dtype", "layout", "shape", "requires_grad"))


_is_tracing = getattr(torch._C, "_is_tracing", torch.jit.is_tracing)   # the public call tests for scripts first, 0.3 us


def _refuse_unseen(who, tensors):
    """What would see an operator's output and not the operator: a trace records the empty output, and a dual tensor's derivative, which
    requires_grad says nothing of, would be left out, as if it were zero"""
    if _is_tracing():
        raise RuntimeError("%s: torch.jit.trace cannot record the library's operators" % who)
    if getattr(forward_ad, "_current_level", 0) >= 0:   # inside a dual level
        for t in tensors:
            if isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None:
                raise RuntimeError("%s: no forward-mode derivative is computed" % who)


def _one_gpu(who, *tensors):
    """the index of the tensors' GPU"""
    _refuse_unseen(who, tensors)
    dev = -1
    for t in tensors:
        if not isinstance(t, torch.Tensor):
            raise ValueError("%s: expected a tensor, got %s" % (who, type(t).__name__))
    for t in tensors:
        at = t.get_device()
        if at != dev or dev < 0:
            if at < 0:
                raise RuntimeError("%s: tensors must live on a GPU (no CPU path)" % who)
            if dev >= 0:
                raise RuntimeError("%s: tensors on cuda:%d and cuda:%d" % (who, dev, at))
            dev = at
    return dev


# the stream handle alone; the Stream object that the public call makes costs 2 us of a call of 10
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda dev: torch.cuda.current_stream(dev).cuda_stream)


def _call(dev, fn, *args):
    """one call of the library on GPU `dev` and its current stream"""
    if torch.cuda.current_device() == dev:
        rc = fn(_raw_stream(dev), *args)
    else:
        with torch.cuda.device(dev):
            rc = fn(_raw_stream(dev), *args)
    if rc:
        nat.check(rc)


def _capture(dev):
    """the number of the capture that the current stream of GPU `dev` is part of; 0: none"""
    if torch.cuda.current_device() == dev and not torch.cuda.is_current_stream_capturing():
        return 0
    return nat.lib().dsp_stream_capture_id(_raw_stream(dev))


def _ptr(t):
    return None if t is None else t.data_ptr()


def _plain(grad):
    """a gradient as its values lie in memory: complex arithmetic behind an operator hands back views that stand for their negative"""
    grad = grad.contiguous()
    return grad.resolve_neg() if grad.is_neg() else grad


def _workspace(like, size):
    return like.new_empty(nat.check(size), dtype=torch.uint8)


def _differentiable_once(backward):
    """autograd.function.once_differentiable, whose wrapping is skipped where no graph of the backward pass is asked for (it costs
    several microseconds)"""
    with_graph = once_differentiable(backward)

    def run(ctx, *grads):
        return with_graph(ctx, *grads) if torch.is_grad_enabled() else backward(ctx, *grads)
    return staticmethod(run)


# ---- embedding ----------------------------------------------------------------------------------------------------------------
def _embedding_forward(tokens, weight, scale):
    rows, dim = weight.shape
    out = weight.new_empty((*tokens.shape, dim))
    _call(weight.get_device(), nat.lib().dsp_embedding_forward, tokens.numel(), tokens.data_ptr(), _TOKEN[tokens.dtype], weight.data_ptr(), rows, dim,
          _FLOAT[weight.dtype], scale, out.data_ptr())
    return out


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, tokens, weight, scale, padding_idx):
        ctx.save_for_backward(tokens)
        ctx.how = *weight.shape, scale, padding_idx
        return _embedding_forward(tokens, weight, scale)

    @_differentiable_once
    def backward(ctx, grad):
        tokens, = ctx.saved_tensors
        rows, dim, scale, padding_idx = ctx.how
        n, L = tokens.numel(), nat.lib()
        grad = _plain(grad)
        out = grad.new_empty((rows, dim))
        size = L.dsp_embedding_workspace(n, rows, dim)
        ws = _workspace(grad, size) if size else None
        _call(grad.get_device(), L.dsp_embedding_backward, n, tokens.data_ptr(), _TOKEN[tokens.dtype], grad.data_ptr(), rows, dim, _FLOAT[grad.dtype],
              padding_idx, scale, out.data_ptr(), _ptr(ws), size)
        return None, out, None, None


def embedding(tokens, weight, scale=1.0, padding_idx=None):
    """scale * weight[tokens]: [..., dim] for tokens of any shape and weight [rows, dim] (float32, bfloat16 or float16).

    tokens: uint8, uint16, int32, int64, or float32 as the reference feeds k-mer codes (cut towards zero).  A token outside the
    table gives a row of NaN and no gradient.  padding_idx: that row of the table gets no gradient (negative: from the end).
    Products and the gradient's sums are held in 32 bits and rounded once."""
    _one_gpu("embedding", tokens, weight)
    if tokens.dtype not in _TOKEN:
        raise ValueError("embedding: tokens must be uint8, uint16, int32, int64 or float32, got %s" % tokens.dtype)
    if weight.dtype not in _FLOAT or weight.dim() != 2:
        raise ValueError("embedding: weight must be [rows, dim] in float32, bfloat16 or float16, got %s %s" % (list(weight.shape), weight.dtype))
    scale = ctypes.c_float(float(scale)).value   # as the kernels get it
    if not math.isfinite(scale):
        raise ValueError("embedding: scale must be finite in float32")
    pad = -1   # none
    if padding_idx is not None:
        pad = int(padding_idx)
        if not -weight.shape[0] <= pad < weight.shape[0]:
            raise ValueError("embedding: padding_idx %d is not a row of the table" % pad)
        pad %= weight.shape[0]
    tokens = tokens.contiguous()
    if tokens.requires_grad:
        tokens = tokens.detach()
    if weight.requires_grad and torch.is_grad_enabled():
        return _Embedding.apply(tokens, weight.contiguous(), scale, pad)
    return _embedding_forward(tokens, weight.contiguous(), scale)


# ---- lstm -----------------------------------------------------------------------------------------------------------------------
def _layer(x, weights):
    p, two = list(map(torch.Tensor.data_ptr, weights)), ctypes.c_void_p * 2
    if len(p) == 4:
        p += [None] * 4
    return nat.LstmLayer(*x.shape, weights[1].shape[1], len(weights) // 4, two(p[0], p[4]), two(p[1], p[5]), two(p[2], p[6]), two(p[3], p[7]))


def _lstm_forward(x, h0, c0, weights, save):
    l, new = _layer(x, weights), x.new_empty
    B, T, H, D = l.batch, l.steps, l.hidden, l.directions
    y, hn, cn = new((B, T, D * H)), new((D, B, H)), new((D, B, H))
    gates = cells = None
    if save or T > 1:
        gates, cells = new((D, B, T, 4 * H)), new((2, D, B, T if save else 1, H))
    _call(x.get_device(), nat.lib().dsp_lstm_forward, ctypes.byref(l), x.data_ptr(), _ptr(h0), _ptr(c0), y.data_ptr(), hn.data_ptr(), cn.data_ptr(), _ptr(gates),
          _ptr(cells), int(save))
    return y, hn, cn, gates, cells


class _Lstm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, h0, c0, *weights):
        y, hn, cn, gates, cells = _lstm_forward(x, h0, c0, weights, True)
        ctx.save_for_backward(x, c0, gates, cells, *weights)
        ctx.set_materialize_grads(False)
        return y, hn, cn

    @_differentiable_once
    def backward(ctx, gy, ghn, gcn):
        x, c0, gates, cells, *weights = ctx.saved_tensors
        l, L = _layer(x, weights), nat.lib()
        gy, ghn, gcn = (None if g is None else _plain(g) for g in (gy, ghn, gcn))
        dx = torch.empty_like(x) if ctx.needs_input_grad[0] else None
        states = (l.directions, l.batch, l.hidden)
        dh0 = x.new_empty(states) if ctx.needs_input_grad[1] else None
        dc0 = x.new_empty(states)
        dws = [torch.empty_like(w) for w in weights]
        g = nat.LstmGrads()
        for d in range(l.directions):
            g.w_ih[d], g.w_hh[d], g.b_ih[d], g.b_hh[d] = (w.data_ptr() for w in dws[4 * d:4 * d + 4])
        ws = _workspace(x, L.dsp_lstm_workspace(ctypes.byref(l)))
        _call(x.get_device(), L.dsp_lstm_backward, ctypes.byref(l), x.data_ptr(), _ptr(c0), gates.data_ptr(), cells.data_ptr(), _ptr(gy), _ptr(ghn),
              _ptr(gcn), _ptr(dx), _ptr(dh0), dc0.data_ptr(), ctypes.byref(g), ws.data_ptr(), ws.numel())
        return (dx, dh0, dc0 if ctx.needs_input_grad[2] else None, *dws)


def lstm(x, weights, h0=None, c0=None):
    """One LSTM layer: (y [batch, steps, directions * hidden], hn, cn [directions, batch, hidden]) of x [batch, steps, input], as
    torch.nn.LSTM(batch_first=True).  float32 only.

    weights: weight_ih [4 * hidden, input], weight_hh [4 * hidden, hidden], bias_ih, bias_hh [4 * hidden], and the same four of the
    reverse direction for a bidirectional layer (the order of the state_dict; gates i, f, g, o).  h0, c0 [directions, batch,
    hidden]: zeros where not given.  One step with the states handed on is the form for running sequences.  The gradient costs
    memory of 6 * hidden values a step, sequence and direction from the forward to the backward pass; under torch.no_grad none."""
    weights = list(weights)
    if len(weights) not in (4, 8):
        raise ValueError("lstm: expected the 4 weights of one direction or the 8 of two, got %d" % len(weights))
    given = [x, *weights, *(t for t in (h0, c0) if t is not None)]
    _one_gpu("lstm", *given)
    if set(map(_dtype, given)) != {torch.float32}:
        raise ValueError("lstm: tensors must be float32")
    if x.dim() != 3 or weights[1].dim() != 2:
        raise ValueError("lstm: x must be [batch, steps, input] and weight_hh [4 * hidden, hidden]")
    hidden, dirs = weights[1].shape[1], len(weights) // 4
    want = [(4 * hidden, x.shape[2]), (4 * hidden, hidden), (4 * hidden,), (4 * hidden,)] * dirs
    if list(map(_shape, weights)) != want:
        raise ValueError("lstm: the weights have shapes %s, expected %s" % ([tuple(w.shape) for w in weights], want))
    for name, t in (("h0", h0), ("c0", c0)):
        if t is not None and t.shape != (dirs, x.shape[0], hidden):
            raise ValueError("lstm: %s has shape %s, expected %s" % (name, tuple(t.shape), (dirs, x.shape[0], hidden)))
    if not all(map(torch.Tensor.is_contiguous, given)):
        x, h0, c0 = (None if t is None else t.contiguous() for t in (x, h0, c0))
        weights = [w.contiguous() for w in weights]
    if torch.is_grad_enabled() and any(map(_requires_grad, given)):
        return _Lstm.apply(x, h0, c0, *weights)
    return _lstm_forward(x, h0, c0, weights, False)[:3]


# ---- linear ------------------------------------------------------------------------------------------------------------------
def _linear_forward(x, weight, bias):
    outputs, inputs = weight.shape
    y = x.new_empty((*x.shape[:-1], outputs))
    _call(x.get_device(), nat.lib().dsp_linear_forward, x.numel() // inputs, inputs, outputs, x.data_ptr(), weight.data_ptr(), _ptr(bias), y.data_ptr())
    return y


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias):
        ctx.save_for_backward(x, weight)
        ctx.has_bias = bias is not None
        return _linear_forward(x, weight, bias)

    @_differentiable_once
    def backward(ctx, grad):
        x, weight = ctx.saved_tensors
        (outputs, inputs), L = weight.shape, nat.lib()
        rows, grad = x.numel() // inputs, _plain(grad)
        dx = torch.empty_like(x) if ctx.needs_input_grad[0] else None
        dw, db = torch.empty_like(weight), weight.new_empty(outputs) if ctx.has_bias else None
        ws = _workspace(x, L.dsp_linear_workspace(rows, inputs, outputs))
        _call(x.get_device(), L.dsp_linear_backward, rows, inputs, outputs, x.data_ptr(), weight.data_ptr(), grad.data_ptr(), _ptr(dx), dw.data_ptr(), _ptr(db),
              ws.data_ptr(), ws.numel())
        return dx, dw, db


def linear(x, weight, bias=None):
    """x weight^T + bias: [..., outputs] for x [..., inputs], weight [outputs, inputs], bias [outputs]; float32, at most 16,384 inputs
    and outputs.  (torch's own bias gradient is a sum that clears flags by a memset: captured into a graph, its replays went wrong here.)"""
    given = (x, weight) if bias is None else (x, weight, bias)
    _one_gpu("linear", *given)
    for t in given:
        if t.dtype != torch.float32:
            raise ValueError("linear: tensors must be float32, got %s" % t.dtype)
    if weight.dim() != 2 or x.dim() < 1 or x.shape[-1] != weight.shape[1] or 0 in weight.shape:
        raise ValueError("linear: x must be [..., inputs] and weight [outputs, inputs], got %s and %s" % (list(x.shape), list(weight.shape)))
    if bias is not None and tuple(bias.shape) != (weight.shape[0],):
        raise ValueError("linear: bias must be [%d], got %s" % (weight.shape[0], list(bias.shape)))
    x, weight, bias = x.contiguous(), weight.contiguous(), None if bias is None else bias.contiguous()
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias)):
        return _Linear.apply(x, weight, bias)
    return _linear_forward(x, weight, bias)


# ---- cross entropy ---------------------------------------------------------------------------------------------------------------
def _loss_args(logits, labels, weight, ignore_index, reduction):
    return (logits.shape[0], logits.shape[1], logits.data_ptr(), _FLOAT[logits.dtype], logits.stride(0), labels.data_ptr(), _LABEL[labels.dtype], _ptr(weight),
            ignore_index, reduction)


def _loss_forward(logits, labels, weight, ignore_index, reduction, want_grad):
    n, L = logits.shape[0], nat.lib()
    loss = logits.new_empty((n,) if reduction == 2 else (), dtype=torch.float32)
    keep = logits.new_empty(1 + n, dtype=torch.float64)   # the sum of the weights, and two float32 of each row
    grad = logits.new_empty(logits.shape) if want_grad and reduction != 2 else None
    ws = _workspace(logits, L.dsp_cross_entropy_workspace(n))
    at = keep.data_ptr()
    _call(logits.get_device(), L.dsp_cross_entropy_forward, *_loss_args(logits, labels, weight, ignore_index, reduction), loss.data_ptr(), at + 8, at,
          _ptr(grad), ws.data_ptr(), ws.numel())
    return loss, keep, grad


class _CrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, labels, weight, ignore_index, reduction):
        loss, keep, ctx.unit_grad = _loss_forward(logits, labels, weight, ignore_index, reduction, True)
        ctx.capture = _capture(logits.get_device())
        ctx.save_for_backward(logits, labels, weight, keep)
        ctx.how = ignore_index, reduction
        return loss

    @_differentiable_once
    def backward(ctx, upstream):
        logits, labels, weight, keep = ctx.saved_tensors
        # the gradient that the forward pass left is handed out once; a second pass over a retained graph computes its own, and so does
        # one that is captured apart from the forward pass: each of its replays would find what the one before it wrote
        grad, ctx.unit_grad = ctx.unit_grad, None
        unit = grad is not None and ctx.capture == _capture(logits.get_device())
        if not unit:
            grad = logits.new_empty(logits.shape)
        upstream, at = _plain(upstream), keep.data_ptr()
        _call(logits.get_device(), nat.lib().dsp_cross_entropy_backward, *_loss_args(logits, labels, weight, *ctx.how), at + 8, at, upstream.data_ptr(), int(unit),
              grad.data_ptr())
        return grad, None, None, None, None


def cross_entropy(logits, labels, weight=None, ignore_index=-100, reduction="mean"):
    """Softmax cross entropy of logits [n, classes] (float32, bfloat16, float16) against labels [n] (int64, int32, uint8), as
    torch.nn.functional.cross_entropy with class indices; the loss is float32.

    weight [classes] float32: weight of each class.  Rows labelled ignore_index count for nothing, whatever they hold, and get a
    gradient of zeros; reduction "mean" divides by the sum of the other labels' weights (NaN where there are none).  A label that
    is no class makes its row's loss and gradient NaN.  Where the logits require a gradient it is computed with the loss, for
    an upstream gradient of 1; another one makes the backward pass compute it again from the logits."""
    _one_gpu("cross_entropy", logits, labels, *(() if weight is None else (weight,)))
    if logits.dim() != 2 or logits.dtype not in _FLOAT or logits.shape[1] < 1:
        raise ValueError("cross_entropy: logits must be [n, classes] in float32, bfloat16 or float16, got %s %s" % (list(logits.shape), logits.dtype))
    if tuple(labels.shape) != (logits.shape[0],) or labels.dtype not in _LABEL:
        raise ValueError("cross_entropy: labels must be [%d] in int64, int32 or uint8, got %s %s" % (logits.shape[0], list(labels.shape), labels.dtype))
    if weight is not None and (tuple(weight.shape) != (logits.shape[1],) or weight.dtype != torch.float32):
        raise ValueError("cross_entropy: weight must be [%d] in float32, got %s %s" % (logits.shape[1], list(weight.shape), weight.dtype))
    if weight is not None and weight.requires_grad and torch.is_grad_enabled():
        raise ValueError("cross_entropy: no gradient is computed for the class weights")
    if reduction not in _REDUCE:
        raise ValueError("cross_entropy: reduction must be 'mean', 'sum' or 'none'")
    n, c = logits.shape
    if (c > 1 and logits.stride(1) != 1) or (n > 1 and logits.stride(0) < c):
        logits = logits.contiguous()
    labels, weight, how = labels.contiguous(), None if weight is None else weight.detach().contiguous(), _REDUCE[reduction]
    if logits.requires_grad and torch.is_grad_enabled():
        return _CrossEntropy.apply(logits, labels, weight, int(ignore_index), how)
    return _loss_forward(logits, labels, weight, int(ignore_index), how, False)[0]


# ---- the norm of many gradients -----------------------------------------------------------------------------------------------
def _is_dense(t):
    """whether the values fill one piece of memory, in whatever order"""
    if t.is_contiguous():
        return True
    size = 1
    for stride, n in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n != 1):
        if stride != size:
            return False
        size *= n
    return True


def _check_grads(who, grads):
    """the index of their GPU"""
    _refuse_unseen(who, grads)
    for g in grads:
        if not isinstance(g, torch.Tensor):
            raise ValueError("%s: gradients must be dense tensors" % who)
    if set(map(_layout, grads)) != {torch.strided}:
        raise ValueError("%s: gradients must be dense tensors" % who)
    for dtype in set(map(_dtype, grads)):
        if dtype not in _FLOAT:
            raise ValueError("%s: gradients must be float32, bfloat16 or float16, got %s" % (who, dtype))
    return _one_gpu(who, *grads) if len(set(map(torch.Tensor.get_device, grads))) > 1 else _one_gpu(who, grads[0])


class _Pieces(object):
    """where tensors lie: addresses, numbers of values, types, and (start, end) of those that are not empty in order"""

    def __init__(self, tensors, like=None):   # like: another's numbers of values
        self.ptrs = array("q", map(torch.Tensor.data_ptr, tensors))
        self.numels = array("q", map(torch.Tensor.numel, tensors)) if like is None else like.numels
        self.types = array("i", map(_FLOAT.__getitem__, map(_dtype, tensors)))
        self.spans = sorted([(p, p + n * (2 if t else 4)) for p, n, t in zip(self.ptrs, self.numels, self.types) if n])

    def check_apart(self, who):
        end = 0
        for start, stop in self.spans:
            if start < end:
                raise ValueError("%s: tensors that are written overlap in memory" % who)
            end = stop

    def check_apart_from(self, who, others):
        if not self.spans or not others.spans or others.spans[0][0] >= self.spans[-1][1] or self.spans[0][0] >= max(end for _, end in others.spans):
            return
        other = iter(others.spans)
        at = next(other, None)
        for start, end in self.spans:
            while at and at[1] <= start:
                at = next(other, None)
            if at and at[0] < end:
                raise ValueError("%s: an output overlaps a gradient (clip_grad_norm_ works in place)" % who)


class _Reaches(object):
    """the memory from a strided tensor's first value to its last"""

    def __init__(self, tensors):
        self.spans = sorted((t.data_ptr(), t.data_ptr() + t.element_size() * (1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride())))) for t in tensors if t.numel())


def _run_clip(dev, like, grads, outs, max_norm):
    n, L, numels = len(grads.ptrs), nat.lib(), grads.numels.buffer_info()[0]
    norm = like.new_empty((), dtype=torch.float32)
    ws = _workspace(like, L.dsp_clip_workspace(n, numels))
    at = lambda pieces, name: None if pieces is None else getattr(pieces, name).buffer_info()[0]
    _call(dev, L.dsp_clip_grad_norm, n, at(grads, "ptrs"), numels, at(grads, "types"), at(outs, "ptrs"), at(outs, "types"), max_norm, norm.data_ptr(),
          ws.data_ptr(), ws.numel())
    return norm


def _max_norm(who, max_norm):
    max_norm = float(max_norm)
    if not max_norm >= 0:
        raise ValueError("%s: max_norm must not be negative" % who)
    return max_norm


@torch.no_grad()
def grad_norm(grads):
    """The 2-norm over all values of a list of tensors, as a float32 scalar on their GPU; squares and sums are held in 64 bits."""
    grads = list(grads)
    if not grads:
        raise ValueError("grad_norm: no tensors")
    dev = _check_grads("grad_norm", grads)
    grads = [g if _is_dense(g) else g.contiguous() for g in grads]   # (a view that stands for its negative has the same norm)
    return _run_clip(dev, grads[0], _Pieces(grads), None, 0.0)


@torch.no_grad()
def clip_grad_norm(grads, max_norm, out=None):
    """(norm, clipped): min(1, max_norm / (norm + 1e-6)) times every gradient, written into other tensors.

    out: one contiguous tensor for each gradient, of its shape, in its type or in float32 (the gradients an optimizer with
    32-bit weights takes); new ones where it is not given.  The gradients are left as they are: no output may lie in the memory
    that one of them spans."""
    who, grads = "clip_grad_norm", list(grads)
    max_norm = _max_norm(who, max_norm)
    if not grads:
        raise ValueError("clip_grad_norm: no tensors")
    if out is not None:
        out = list(out)
        _refuse_unseen(who, out)
    dev = _check_grads(who, grads)
    if out is None:
        out = [g.new_empty(g.shape) for g in grads]
    if len(out) != len(grads):
        raise ValueError("clip_grad_norm: %d outputs for %d gradients" % (len(out), len(grads)))
    for o in out:
        if not isinstance(o, torch.Tensor):
            raise ValueError("clip_grad_norm: expected a tensor, got %s" % type(o).__name__)
    if set(map(torch.Tensor.get_device, out)) != {dev}:
        _one_gpu(who, grads[0], *out)
    if list(map(_shape, grads)) != list(map(_shape, out)) or not all(map(torch.Tensor.is_contiguous, out)):
        raise ValueError("clip_grad_norm: an output must be contiguous and of its gradient's shape")
    for g, o in set(zip(map(_dtype, grads), map(_dtype, out))):
        if o is not g and o is not torch.float32:
            raise ValueError("clip_grad_norm: an output must be of its gradient's type or float32")
    strided = []
    if not all(map(torch.Tensor.is_contiguous, grads)) or any(map(torch.Tensor.is_neg, grads)):
        strided = [g for g in grads if not g.is_contiguous()]
        grads = list(map(_plain, grads))
    ins = _Pieces(grads)
    outs = _Pieces(out, ins)
    outs.check_apart(who)
    outs.check_apart_from(who, ins)
    if strided:
        outs.check_apart_from(who, _Reaches(strided))
    norm = _run_clip(dev, grads[0], ins, outs, max_norm)
    increment_version(out)   # as torch's own writes do: a graph that saved one of them notices
    return norm, out


@torch.no_grad()
def clip_grad_norm_(parameters, max_norm, norm_type=2.0, error_if_nonfinite=False):
    """Scale the gradients of `parameters` (a tensor or an iterable of them) in place so that their 2-norm over all values is at
    most max_norm, as torch.nn.utils.clip_grad_norm_; returns the norm before, a float32 scalar on their GPU.

    The gradients may be of different types and sizes, all on one GPU.  A gradient that two parameters share counts once.  Where
    there is nothing to clip they are read but not written.  error_if_nonfinite waits for the norm and raises RuntimeError
    before anything is changed."""
    who = "clip_grad_norm_"
    if float(norm_type) != 2.0:
        raise ValueError("clip_grad_norm_: norm_type must be 2")
    max_norm = _max_norm(who, max_norm)
    grads = [p.grad for p in ((parameters,) if isinstance(parameters, torch.Tensor) else parameters) if p.grad is not None]
    if not grads:
        return torch.zeros(())
    dev = _check_grads(who, grads)
    grads = list({(g.data_ptr(), g.shape, g.stride(), g.dtype): g for g in grads}.values())
    use = [g if _is_dense(g) else g.contiguous() for g in grads]
    for g, u in zip(grads, use):
        if u is not g and any(s == 0 and n > 1 for s, n in zip(g.stride(), g.shape)):
            raise ValueError("clip_grad_norm_: an expanded gradient cannot be scaled in place")
    pieces = _Pieces(use)
    pieces.check_apart(who)
    if error_if_nonfinite:
        norm = _run_clip(dev, use[0], pieces, None, 0.0)
        if not math.isfinite(norm.item()):
            raise RuntimeError("clip_grad_norm_: the norm of the gradients is not finite, so they cannot be clipped")
    norm = _run_clip(dev, use[0], pieces, pieces, max_norm)
    increment_version(use)
    for g, u in zip(grads, use):
        if u is not g:
            g.copy_(u)
    return norm
