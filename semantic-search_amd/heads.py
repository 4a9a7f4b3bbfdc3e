"""Head operators: a model's last layer and how likely the given labels are under it.

    scores = log_probs(logits, ids, top=3, temperature=3.2)       # next to MapEngine.stage1
    g_logits = log_probs_grad(logits, ids, scores, grad_log_prob=g, temperature=3.2)
    logits = linear(features, weight, bias, planes=True, out_dtype=torch.float32)
    g = linear_grad(g_logits, features, weight, planes=True)      # g.x, g.weight, g.bias

Each is one call of the C ABI on the current stream: it allocates its answers and a workspace with torch,
enqueues its kernels and returns.  Nothing is kept between calls, so a call can be captured into a graph.
The backward passes are functions of their own, not recorded by autograd: tensors that require a gradient
are refused while autograd records, tensors with a tangent (forward mode) always.  There is no CPU fallback.

The gradient of a log probability with respect to the temperature T needs no pass over the logits: it is
-(log_prob + entropy) / T, which is what calibrating T on labelled frames descends along.
"""
from __future__ import annotations

import ctypes as C
from typing import NamedTuple, Optional

import torch
from torch.autograd import forward_ad

from . import _capi

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
ACTIVATIONS = {None: 0, "relu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4}
MAX_TOP = 32


class LogProbs(NamedTuple):
    """Answers of `log_probs`, float32 except the ids (int32).  row_max is the largest logit, log_sum the
    logarithm of sum exp((logit - row_max) / temperature)."""
    log_prob: torch.Tensor
    entropy: torch.Tensor
    top_ids: torch.Tensor
    top_log_prob: torch.Tensor
    row_max: torch.Tensor
    log_sum: torch.Tensor


class LinearGrads(NamedTuple):
    x: Optional[torch.Tensor]
    weight: Optional[torch.Tensor]
    bias: Optional[torch.Tensor]


def _tangent(t):
    """Whether forward-mode differentiation follows t (no_grad does not stop it)."""
    return forward_ad._current_level >= 0 and forward_ad.unpack_dual(t).tangent is not None


def _gpu(device, **tensors):
    """Every tensor lies on `device`, a GPU, and neither mode of autograd would record it."""
    if device.type != "cuda":
        raise ValueError(f"expected tensors on a GPU, got {device}: the head operators have no CPU fallback")
    grad = torch.is_grad_enabled()
    for name, t in tensors.items():
        if t is None:
            continue
        if t.device != device:
            raise ValueError(f"{name}: expected a tensor on {device}, got {t.device}")
        if grad and t.requires_grad:
            raise RuntimeError(f"{name} requires a gradient, which autograd does not record here: call under "
                               "torch.no_grad() and use log_probs_grad / linear_grad for the backward pass")
        if _tangent(t):
            raise RuntimeError(f"{name} carries a tangent, which forward-mode differentiation does not get through here: "
                               "pass its primal and use log_probs_grad / linear_grad")
        if t.is_neg():   # a lazy view, as of a conjugate's imaginary part: memory holds the opposite values
            raise ValueError(f"{name} is a view that negates when it is read; pass {name}.resolve_neg()")


def _shape(name, t, dtype, shape):
    if t.dtype != dtype or t.shape != shape:
        raise ValueError(f"{name}: expected {dtype} {tuple(shape)}, got {t.dtype} {tuple(t.shape)}")


def _dtype(name, t):
    if t.dtype not in _DTYPES:
        raise ValueError(f"{name}: expected float32, bfloat16 or float16, got {t.dtype}")
    return _DTYPES[t.dtype]


def _merge(sizes, *strides):
    """Dimensions that every stride list walks as one are merged.  Returns (sizes, strides...) as lists."""
    if 0 in sizes:
        return ([0],) + tuple([0] for _ in strides)
    n, out = [], [[] for _ in strides]
    for i, size in enumerate(sizes):
        if size == 1:
            continue
        if n and all(o[-1] == s[i] * size for o, s in zip(out, strides)):
            n[-1] *= size
            for o, s in zip(out, strides):
                o[-1] = s[i]
        else:
            n.append(size)
            for o, s in zip(out, strides):
                o.append(s[i])
    return (n,) + tuple(out)


def _one(name, sizes, strides, dense=False):
    """(size, stride) of dimensions that must merge into one (of stride 1 where `dense`)."""
    n, s = _merge(sizes, strides)
    if not n:
        return 1, 1
    if len(n) > 1 or (dense and s[0] != 1 and n[0] != 0):
        raise ValueError(f"{name}: strides {tuple(strides)} of sizes {tuple(sizes)} are not those of one "
                         f"{'dense ' if dense else ''}dimension; pass a contiguous tensor")
    return n[0], s[0]


def _two(name, sizes, *strides):
    """((batch, rows), [(batch stride, row stride) of each]) of dimensions that must merge into two."""
    merged = _merge(sizes, *strides)
    n = merged[0]
    if len(n) > 2:
        raise ValueError(f"{name}: the leading dimensions {tuple(sizes)} do not merge into two; pass contiguous tensors")
    pad = 2 - len(n)
    return tuple([1] * pad + n), [tuple([0] * pad + s) for s in merged[1:]]


def _call(device, entry, args, workspace=None):
    """One C call with `device` current; the workspace, if any, is torch's, on the current stream."""
    if torch.cuda.current_device() != device.index:
        with torch.cuda.device(device):
            return _call(device, entry, args, workspace)
    if workspace is not None:
        need = workspace(C.byref(args))
        if need < 0:
            _capi.check(1)
        if need:
            ws = torch.empty(need, dtype=torch.uint8, device=device)
            args.workspace, args.workspace_bytes = ws.data_ptr(), need
    _capi.check(entry(C.byref(args), torch._C._cuda_getCurrentRawStream(device.index)))


def _score_layout(logits, ids, dim):
    """The (layout, batch, rows, classes, strides) that the C ABI wants for logits with their classes
    along `dim`: "rows" where no dimension follows it, "planes" otherwise."""
    nd = logits.dim()
    if not -nd <= dim < nd:
        raise ValueError(f"dim {dim} is out of range for logits of {nd} dimensions")
    d = dim % nd
    sizes, st = list(logits.shape), list(logits.stride())
    want = sizes[:d] + sizes[d + 1:]
    if ids.dtype not in (torch.int32, torch.int64) or list(ids.shape) != want:
        raise ValueError(f"ids: expected int32 or int64 {tuple(want)}, got {ids.dtype} {tuple(ids.shape)}")
    V, ist = sizes[d], list(ids.stride())
    if V < 1:
        raise ValueError("logits have no classes")
    if d == nd - 1:
        if st[d] != 1 and V > 1:
            raise ValueError(f"logits: the classes (dimension {d}) have stride {st[d]}, 1 is needed; pass a contiguous tensor")
        if len(_merge(sizes[:d], st[:d], ist)[0]) > 2:
            ist = list(torch.empty(want, device="meta").stride())
            ids = ids.contiguous()
        (batch, rows), (ls, is_) = _two("logits", sizes[:d], st[:d], ist)
        return 0, batch, rows, V, ls[0], ls[1], ids, is_[0], is_[1]
    rows, _ = _one("logits (dimensions after the classes)", sizes[d + 1:], st[d + 1:], dense=True)
    batch, bs = _one("logits (dimensions before the classes)", sizes[:d], st[:d])
    try:
        _, i_row = _one("ids", sizes[d + 1:], ist[d:])
        _, i_batch = _one("ids", sizes[:d], ist[:d])
    except ValueError:
        ids = ids.contiguous()
        i_row, i_batch = 1, rows
    return 1, batch, rows, V, bs, st[d], ids, i_batch, i_row


def log_probs(logits: torch.Tensor, ids: torch.Tensor, *, dim: int = -1, temperature: float = 1.0, top: int = 0,
              ignore_id: int = -100) -> LogProbs:
    """Log probability of `ids` under softmax(logits / temperature) along `dim`, with the entropy (nats) and
    the `top` most probable classes of every position.

    logits: float32, bfloat16 or float16.  [..., classes] (dim the last), a language model's layout; or
    [envs, classes, height, width] (dim 1), a segmentation head's.  Views are read where they lie: rows of
    any stride whose leading dimensions merge into two, planes of any stride.
    ids: int32 or int64, the logits' shape without `dim`.

    Ties go to the lowest class.  An id equal to `ignore_id` has log probability 0, any other id outside
    [0, classes) NaN.  A logit of -inf masks its class; where fewer than `top` classes are left, the other
    alternatives have id -1 and log probability -inf; where none is, log_prob is -inf and the entropy 0.  A
    position that holds a NaN or +inf has NaN for everything but row_max (the largest that is a number) and
    an ignored id's 0, and ids -1.
    """
    dt = _dtype("logits", logits)
    top = int(top)
    layout, batch, rows, V, bs, inner, ids, ib, ir = _score_layout(logits, ids, dim)
    if not 0 <= top <= min(MAX_TOP, V):
        raise ValueError(f"top must be in [0, {min(MAX_TOP, V)}], got {top}")
    _gpu(logits.device, logits=logits, ids=ids)
    shape = ids.shape
    d = dim % logits.dim()
    dev = logits.device
    stats = torch.empty((4,) + tuple(shape), dtype=torch.float32, device=dev)
    log_prob, entropy, row_max, log_sum = stats.unbind(0)
    top_shape = tuple(shape[:d]) + (top,) + tuple(shape[d:])
    top_ids = torch.empty(top_shape, dtype=torch.int32, device=dev)
    top_log_prob = torch.empty(top_shape, dtype=torch.float32, device=dev)
    a = _capi.LogProbsArgs(
        dtype=dt, layout=layout, batch=batch, rows=rows, classes=V, logits=logits.data_ptr(), batch_stride=bs,
        inner_stride=inner, ids=ids.data_ptr(), ids_batch_stride=ib, ids_row_stride=ir, ignore_id=int(ignore_id),
        ids_64=int(ids.dtype == torch.int64), top=top, temperature=float(temperature), log_prob=log_prob.data_ptr(),
        entropy=entropy.data_ptr(), row_max=row_max.data_ptr(), log_sum=log_sum.data_ptr(), top_ids=top_ids.data_ptr(),
        top_log_prob=top_log_prob.data_ptr())
    lib = _capi.load()
    _call(dev, lib.ssmap_log_probs, a, lib.ssmap_log_probs_workspace)
    return LogProbs(log_prob, entropy, top_ids, top_log_prob, row_max, log_sum)


def log_probs_grad(logits: torch.Tensor, ids: torch.Tensor, scores: LogProbs, *, dim: int = -1, temperature: float = 1.0,
                   ignore_id: int = -100, grad_log_prob: Optional[torch.Tensor] = None,
                   grad_entropy: Optional[torch.Tensor] = None, grad_top: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The gradient with respect to the logits of a loss whose gradients with respect to `log_prob`,
    `entropy` and `top_log_prob` are given (None counts as 0; float32 of those shapes, expanded views
    welcome).  `scores` is log_probs' answer for the same logits, ids, dim, temperature and ignore_id.
    Returns a dense tensor of the logits' shape and type."""
    dev = logits.device
    dt = _dtype("logits", logits)
    layout, batch, rows, V, bs, inner, ids, ib, ir = _score_layout(logits, ids, dim)
    shape = ids.shape
    d = dim % logits.dim()
    f32, keep = torch.float32, []

    def dense(name, t, shape, dtype=f32):
        if t is None:
            return None
        _shape(name, t, dtype, torch.Size(shape))
        t = t.contiguous()
        keep.append(t)
        return t.data_ptr()

    g_l, g_e = dense("grad_log_prob", grad_log_prob, shape), dense("grad_entropy", grad_entropy, shape)
    g_t, top, top_ids = None, 0, None
    if grad_top is not None:
        top = scores.top_ids.shape[d] if scores.top_ids.dim() == logits.dim() else 0
        top_shape = tuple(shape[:d]) + (top,) + tuple(shape[d:])
        g_t = dense("grad_top", grad_top, top_shape)
        top_ids = dense("scores.top_ids", scores.top_ids, top_shape, torch.int32)
    stats = [dense("scores." + name, getattr(scores, name), shape) for name in ("row_max", "log_sum", "entropy")]
    _gpu(dev, logits=logits, ids=ids, grad_log_prob=grad_log_prob, grad_entropy=grad_entropy, grad_top=grad_top,
         row_max=scores.row_max, log_sum=scores.log_sum, entropy=scores.entropy, top_ids=scores.top_ids)
    grad = torch.empty(logits.shape, dtype=logits.dtype, device=dev)
    a = _capi.LogProbsGradArgs(
        dtype=dt, layout=layout, batch=batch, rows=rows, classes=V, logits=logits.data_ptr(), batch_stride=bs,
        inner_stride=inner, ids=ids.data_ptr(), ids_batch_stride=ib, ids_row_stride=ir, ignore_id=int(ignore_id),
        ids_64=int(ids.dtype == torch.int64), top=top, temperature=float(temperature),
        row_max=stats[0], log_sum=stats[1], entropy=stats[2], top_ids=top_ids, g_log_prob=g_l, g_entropy=g_e, g_top=g_t,
        grad=grad.data_ptr())
    _call(dev, _capi.load().ssmap_log_probs_grad, a)
    return grad


def _activation(name):
    if name not in ACTIVATIONS:
        raise ValueError(f"unknown activation {name!r}: expected one of {', '.join(map(repr, ACTIVATIONS))}")
    return ACTIVATIONS[name]


def _weight(x, weight):
    """(outer, inner, row stride) of a weight [outer, inner] for x [..., inner]."""
    if x.dim() < 1 or weight.dim() != 2 or weight.dtype != x.dtype or weight.shape[1] != x.shape[-1]:
        raise ValueError(f"weight: expected {x.dtype} [outer, {x.shape[-1] if x.dim() else '?'}], got {weight.dtype} {tuple(weight.shape)}")
    outer, inner = weight.shape
    for name, t in (("x", x), ("weight", weight)):
        if t.stride(-1) != 1 and inner > 1:
            raise ValueError(f"{name}: the last dimension has stride {t.stride(-1)}, 1 is needed; pass a contiguous tensor")
    return outer, inner, weight.stride(0)


def _linear_layout(x, y_shape, y, planes, name):
    """(batch, rows, x strides, strides of y or None): y is a tensor of y_shape that a kernel reads."""
    if not planes:
        if y is not None and y.stride(-1) != 1 and y_shape[-1] > 1:
            raise ValueError(f"{name}: the last dimension has stride {y.stride(-1)}, 1 is needed; pass a contiguous tensor")
        lead = list(x.shape[:-1])
        if y is None:
            (batch, rows), (xs,) = _two("x", lead, list(x.stride()[:-1]))
            return batch, rows, xs, (0, 0)
        (batch, rows), (xs, ys) = _two(f"x and {name}", lead, list(x.stride()[:-1]), list(y.stride()[:-1]))
        return batch, rows, xs, ys
    rows, row_stride = _one("x (dimensions between the first and the last)", x.shape[1:-1], x.stride()[1:-1])
    ys = (0, 0)
    if y is not None:
        _one(f"{name} (dimensions after the planes)", y_shape[2:], y.stride()[2:], dense=True)
        ys = (y.stride(0), y.stride(1))
    return x.shape[0], rows, (x.stride(0), row_stride), ys


def _y_shape(x, outer, planes):
    if not planes:
        return tuple(x.shape[:-1]) + (outer,)
    if x.dim() < 3:
        raise ValueError(f"planes: x is [envs, positions..., inner], got {tuple(x.shape)}")
    return (x.shape[0], outer) + tuple(x.shape[1:-1])


def linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, *, activation: Optional[str] = None,
           residual: Optional[torch.Tensor] = None, planes: bool = False, out_dtype: Optional[torch.dtype] = None,
           keep_pre: bool = False):
    """act(x weight^T + bias) + residual, with everything after the product in its epilogue.

    x [..., inner] and weight [outer, inner] in float32, bfloat16 or float16; bias [outer] in their type or
    float32; activation None, "relu", "gelu", "gelu_tanh" or "silu".  Returns [..., outer] in out_dtype
    (x's type or float32; default x's), which is also the residual's type and shape.

    planes=True takes x [envs, positions..., inner] and returns one plane per output,
    [envs, outer, positions...]: with out_dtype=torch.float32 these are the logits of MapEngine.step.

    keep_pre=True returns (y, pre) with pre = x weight^T + bias in x's type, for linear_grad.
    """
    dt, act, dev = _dtype("x", x), _activation(activation), x.device
    out_dtype = x.dtype if out_dtype is None else out_dtype
    if out_dtype != x.dtype and out_dtype != torch.float32:
        raise ValueError(f"out_dtype: expected {x.dtype} or torch.float32, got {out_dtype}")
    outer, inner, w_stride = _weight(x, weight)
    shape = _y_shape(x, outer, planes)
    if bias is not None:
        if tuple(bias.shape) != (outer,) or bias.dtype not in (x.dtype, torch.float32):
            raise ValueError(f"bias: expected {x.dtype} or float32 ({outer},), got {bias.dtype} {tuple(bias.shape)}")
        bias = bias.contiguous()
    if residual is not None:
        _shape("residual", residual, out_dtype, torch.Size(shape))
    batch, rows, xs, rs = _linear_layout(x, shape, residual, planes, "residual")
    _gpu(dev, x=x, weight=weight, bias=bias, residual=residual)
    y = torch.empty(shape, dtype=out_dtype, device=dev)
    pre = torch.empty(shape, dtype=x.dtype, device=dev) if keep_pre else None
    a = _capi.LinearArgs(
        dtype=dt, out_dtype=_DTYPES[out_dtype], activation=act, layout=int(planes), batch=batch, rows=rows, inner=inner,
        outer=outer, x=x.data_ptr(), x_batch_stride=xs[0], x_row_stride=xs[1], w=weight.data_ptr(), w_row_stride=w_stride,
        bias=None if bias is None else bias.data_ptr(), bias_dtype=dt if bias is None else _DTYPES[bias.dtype],
        residual=None if residual is None else residual.data_ptr(), res_batch_stride=rs[0], res_inner_stride=rs[1],
        y=y.data_ptr(), pre=None if pre is None else pre.data_ptr())
    lib = _capi.load()
    _call(dev, lib.ssmap_linear, a, lib.ssmap_linear_workspace)
    return (y, pre) if keep_pre else y


def linear_grad(grad: torch.Tensor, x: torch.Tensor, weight: torch.Tensor, *, activation: Optional[str] = None,
                pre: Optional[torch.Tensor] = None, planes: bool = False, need_x: bool = True, need_weight: bool = True,
                need_bias: bool = True) -> LinearGrads:
    """Gradients of `linear` with respect to x, weight and bias, all in x's type, from `grad` = dL/dy (x's
    type or float32; it is also the residual's gradient).  With an activation, `pre` is what
    linear(..., keep_pre=True) returned.  16-bit x: where grad act'(pre) is no value of x's type, the two
    products sum two parts of it, which hold 16 (bfloat16) or 22 (float16) of its bits and take twice the
    time; float16 values are scaled for it by the power of two that the largest finite |grad| asks for, so
    that only what lies below 2^-38 of that is lost.  An infinite x or weight can make NaN of what the
    formula calls infinite."""
    dt, act, dev = _dtype("x", x), _activation(activation), x.device
    outer, inner, w_stride = _weight(x, weight)
    shape = _y_shape(x, outer, planes)
    if grad.dtype not in (x.dtype, torch.float32) or tuple(grad.shape) != shape:
        raise ValueError(f"grad: expected {x.dtype} or float32 {shape}, got {grad.dtype} {tuple(grad.shape)}")
    if act and pre is None:
        raise ValueError(f"activation {activation!r} needs pre, from linear(..., keep_pre=True)")
    if pre is not None:
        _shape("pre", pre, x.dtype, torch.Size(shape))
        pre = pre.contiguous()
    batch, rows, xs, gs = _linear_layout(x, shape, grad, planes, "grad")
    _gpu(dev, grad=grad, x=x, weight=weight, pre=pre)
    g_x = torch.empty(x.shape, dtype=x.dtype, device=dev) if need_x else None
    g_w = torch.empty(weight.shape, dtype=x.dtype, device=dev) if need_weight else None
    g_b = torch.empty((outer,), dtype=x.dtype, device=dev) if need_bias else None
    ptr = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    a = _capi.LinearGradArgs(
        dtype=dt, grad_dtype=_DTYPES[grad.dtype], activation=act, layout=int(planes), batch=batch, rows=rows, inner=inner,
        outer=outer, g=grad.data_ptr(), g_batch_stride=gs[0], g_inner_stride=gs[1], pre=ptr(pre), x=x.data_ptr(),
        x_batch_stride=xs[0], x_row_stride=xs[1], w=weight.data_ptr(), w_row_stride=w_stride, g_x=ptr(g_x), g_w=ptr(g_w),
        g_bias=ptr(g_b))
    lib = _capi.load()
    _call(dev, lib.ssmap_linear_grad, a, lib.ssmap_linear_grad_workspace)
    return LinearGrads(g_x, g_w, g_b)
