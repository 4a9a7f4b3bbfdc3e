"""Head operators: argument checks and layouts, which answer without a GPU."""
import ctypes

import pytest
import torch

import semantic_search_amd as ssa
from semantic_search_amd import heads


def _scores(shape, top=0, dim=-1):
    f = torch.zeros(shape)
    d = dim % (len(shape) + 1)
    t = list(shape[:d]) + [top] + list(shape[d:])
    return ssa.LogProbs(f, f, torch.zeros(t, dtype=torch.int32), torch.zeros(t), f, f)


def test_merging_dimensions():
    assert heads._merge([4, 5, 6], [30, 6, 1]) == ([120], [1])
    assert heads._merge([4, 5, 6], [60, 6, 1]) == ([4, 30], [60, 1])
    assert heads._merge([4, 1, 6], [6, 99, 1]) == ([24], [1])
    assert heads._merge([4, 5], [5, 1], [10, 1]) == ([4, 5], [5, 1], [10, 1])
    assert heads._merge([4, 5], [0, 0]) == ([20], [0])          # an expanded tensor
    assert heads._merge([4, 0, 5], [1, 1, 1]) == ([0], [0])
    assert heads._merge([], []) == ([], [])


def test_layouts_of_logits():
    x, ids = torch.zeros(3, 6, 11), torch.zeros(3, 6, dtype=torch.int64)
    got = heads._score_layout(x[:, :-1], ids[:, 1:], -1)
    assert got[:6] == (0, 3, 5, 11, 66, 11) and got[7:] == (6, 1)
    got = heads._score_layout(x, ids, 2)
    assert got[:6] == (0, 1, 18, 11, 0, 11) and got[7:] == (0, 1)
    planes = torch.zeros(2, 7, 4, 5)
    got = heads._score_layout(planes[:, 1:6], torch.zeros(2, 4, 5, dtype=torch.int32), 1)
    assert got[:6] == (1, 2, 20, 5, 140, 20) and got[7:] == (20, 1)
    # planes of single pixels, a batch of none
    assert heads._score_layout(torch.zeros(2, 7, 1), torch.zeros(2, 1, dtype=torch.int32), 1)[:4] == (1, 2, 1, 7)
    assert heads._score_layout(torch.zeros(0, 7, 3), torch.zeros(0, 3, dtype=torch.int32), 1)[1:4] == (0, 3, 7)


@pytest.mark.parametrize("make,text", [
    (lambda: ssa.log_probs(torch.zeros(3, 5, dtype=torch.float64), torch.zeros(3, dtype=torch.int64)), "float32, bfloat16 or float16"),
    (lambda: ssa.log_probs(torch.zeros(3, 5), torch.zeros(3)), "ids: expected int32 or int64"),
    (lambda: ssa.log_probs(torch.zeros(3, 5), torch.zeros(4, dtype=torch.int64)), "ids: expected"),
    (lambda: ssa.log_probs(torch.zeros(3, 0), torch.zeros(3, dtype=torch.int64)), "no classes"),
    (lambda: ssa.log_probs(torch.zeros(3, 5), torch.zeros(3, dtype=torch.int64), top=6), r"top must be in \[0, 5\]"),
    (lambda: ssa.log_probs(torch.zeros(3, 50), torch.zeros(3, dtype=torch.int64), top=33), r"top must be in \[0, 32\]"),
    (lambda: ssa.log_probs(torch.zeros(3, 50), torch.zeros(3, dtype=torch.int64), top=-1), "top must be"),
    (lambda: ssa.log_probs(torch.zeros(5, 3).t(), torch.zeros(3, dtype=torch.int64)), "have stride 3"),
    (lambda: ssa.log_probs(torch.zeros(3, 5), torch.zeros(3, dtype=torch.int64), dim=2), "dim 2 is out of range"),
    (lambda: ssa.log_probs(torch.zeros(2, 5, 4, 6)[..., ::2], torch.zeros(2, 4, 3, dtype=torch.int64), dim=1), "dense"),
    (lambda: ssa.log_probs(torch.zeros(9, 9, 9, 5)[::2, ::2, ::2], torch.zeros(5, 5, 5, dtype=torch.int64)), "merge into two"),
    (lambda: ssa.log_probs(torch.zeros(3, 5), torch.zeros(3, dtype=torch.int64)), "no CPU fallback"),
    (lambda: ssa.log_probs_grad(torch.zeros(3, 5), torch.zeros(3, dtype=torch.int64), _scores((3,)), grad_log_prob=torch.zeros(4)), "grad_log_prob: expected"),
    (lambda: ssa.log_probs_grad(torch.zeros(3, 5), torch.zeros(3, dtype=torch.int64), _scores((3,), 2), grad_top=torch.zeros(3, 3)), "grad_top: expected"),
    (lambda: ssa.log_probs_grad(torch.zeros(3, 5), torch.zeros(3, dtype=torch.int64), _scores((4,))), "scores.row_max: expected"),
    (lambda: ssa.log_probs_grad(torch.zeros(3, 5), torch.zeros(3, dtype=torch.int64), _scores((3,))), "no CPU fallback"),
    (lambda: ssa.linear(torch.zeros(3, 5, dtype=torch.int32), torch.zeros(4, 5, dtype=torch.int32)), "x: expected"),
    (lambda: ssa.linear(torch.zeros(3, 5), torch.zeros(4, 6)), "weight: expected"),
    (lambda: ssa.linear(torch.zeros(3, 5), torch.zeros(4, 5, dtype=torch.float16)), "weight: expected"),
    (lambda: ssa.linear(torch.zeros(3, 5), torch.zeros(5, 4).t()), "weight: the last dimension has stride 4"),
    (lambda: ssa.linear(torch.zeros(3, 10)[:, ::2], torch.zeros(4, 5)), "x: the last dimension"),
    (lambda: ssa.linear(torch.zeros(3, 5), torch.zeros(4, 5), torch.zeros(5)), "bias: expected"),
    (lambda: ssa.linear(torch.zeros(3, 5), torch.zeros(4, 5), activation="tanh"), "unknown activation 'tanh'"),
    (lambda: ssa.linear(torch.zeros(3, 5), torch.zeros(4, 5), residual=torch.zeros(4)), "residual: expected"),
    (lambda: ssa.linear(torch.zeros(3, 5), torch.zeros(4, 5), out_dtype=torch.float16), "out_dtype: expected"),
    (lambda: ssa.linear(torch.zeros(3, 5), torch.zeros(4, 5), planes=True), r"planes: x is \[envs"),
    (lambda: ssa.linear(torch.zeros(9, 9, 9, 5)[::2, ::2, ::2], torch.zeros(4, 5)), "merge into two"),
    (lambda: ssa.linear(torch.zeros(3, 5), torch.zeros(4, 5)), "no CPU fallback"),
    (lambda: ssa.linear_grad(torch.zeros(3, 5), torch.zeros(3, 5), torch.zeros(4, 5)), "grad: expected"),
    (lambda: ssa.linear_grad(torch.zeros(3, 4), torch.zeros(3, 5), torch.zeros(4, 5), activation="relu"), "needs pre"),
    (lambda: ssa.linear_grad(torch.zeros(3, 4), torch.zeros(3, 5), torch.zeros(4, 5), activation="relu", pre=torch.zeros(3, 5)), "pre: expected"),
    (lambda: ssa.linear_grad(torch.zeros(3, 4), torch.zeros(3, 5), torch.zeros(4, 5)), "no CPU fallback"),
])
def test_refusals(make, text):
    with pytest.raises(ValueError, match=text):
        make()


def _args(kind, **over):
    p = ctypes.cast(ctypes.create_string_buffer(64), ctypes.c_void_p).value
    c = ssa._capi
    if kind == "log_probs":
        kw = dict(batch=1, rows=2, classes=5, logits=p, ids=p, temperature=1.0, log_prob=p, entropy=p, row_max=p, log_sum=p,
                  top_ids=p, top_log_prob=p)
        cls = c.LogProbsArgs
    elif kind == "log_probs_grad":
        kw = dict(batch=1, rows=2, classes=5, logits=p, ids=p, temperature=1.0, row_max=p, log_sum=p, entropy=p, top_ids=p, grad=p)
        cls = c.LogProbsGradArgs
    elif kind == "linear":
        kw = dict(batch=1, rows=2, inner=3, outer=4, x=p, w=p, y=p)
        cls = c.LinearArgs
    else:
        kw = dict(batch=1, rows=2, inner=3, outer=4, x=p, w=p, g=p, g_x=p, g_w=p, g_bias=p, workspace=p, workspace_bytes=1 << 20)
        cls = c.LinearGradArgs
    kw.update(over)
    return cls(**kw)


@pytest.mark.parametrize("kind,over,text", [
    ("log_probs", dict(dtype=3), "dtype is none"),
    ("log_probs", dict(layout=2), "layout is neither"),
    ("log_probs", dict(classes=0), "1 <= classes"),
    ("log_probs", dict(rows=-1), "batch, rows >= 0"),
    ("log_probs", dict(rows=1 << 39), "fewer than 2\\^40"),
    ("log_probs", dict(top=6), "top must be"),
    ("log_probs", dict(temperature=0.0), "temperature must be"),
    ("log_probs", dict(temperature=float("nan")), "temperature must be"),
    ("log_probs", dict(temperature=float("inf")), "temperature must be"),
    ("log_probs", dict(temperature=-1.0), "temperature must be"),
    ("log_probs", dict(inner_stride=-1), "strides"),
    ("log_probs_grad", dict(ids_row_stride=-1), "strides"),
    ("linear", dict(x_row_stride=-3), "strides"),
    ("linear", dict(res_inner_stride=-3), "strides"),
    ("linear_grad", dict(g_inner_stride=-3), "strides"),
    ("log_probs", dict(rows=2, classes=1 << 20, workspace=1 << 20 | 4, workspace_bytes=1 << 30), "multiple of 16"),
    ("linear_grad", dict(workspace=1 << 20 | 4), "multiple of 16"),
    ("log_probs", dict(logits=None), "null"),
    ("log_probs", dict(entropy=None), "null"),
    ("log_probs", dict(top=1, top_ids=None), "null"),
    ("log_probs_grad", dict(grad=None), "null"),
    ("log_probs_grad", dict(log_sum=None), "null"),
    ("linear", dict(dtype=-1), "dtype is none"),
    ("linear", dict(dtype=1, out_dtype=2), "results' type"),
    ("linear", dict(activation=5), "unknown activation"),
    ("linear", dict(inner=-1), "must not be negative"),
    ("linear", dict(rows=1 << 40), "2\\^40"),
    ("linear", dict(dtype=1, out_dtype=1, bias=8, bias_dtype=2), "bias's type"),
    ("linear", dict(w=None), "null"),
    ("linear", dict(y=None), "null"),
    ("linear_grad", dict(activation=2), "needs pre"),
    ("linear_grad", dict(workspace=None), "workspace"),
    ("linear_grad", dict(workspace_bytes=0), "workspace"),
    ("linear_grad", dict(x=None), "null"),
    ("linear_grad", dict(g=None), "null"),
])
def test_c_entries_refuse_before_touching_the_gpu(kind, over, text):
    lib = ssa._capi.load()
    a = _args(kind, **over)
    assert getattr(lib, "ssmap_" + kind)(ctypes.byref(a), None) == 1
    import re
    assert re.search(text, lib.ssmap_last_error().decode()), lib.ssmap_last_error()
    assert getattr(lib, "ssmap_" + kind)(None, None) == 1


def test_empty_calls_do_nothing():
    lib = ssa._capi.load()
    for kind, over in (("log_probs", dict(rows=0)), ("log_probs", dict(batch=0)), ("log_probs_grad", dict(rows=0)),
                       ("linear", dict(rows=0)), ("linear", dict(outer=0))):
        assert getattr(lib, "ssmap_" + kind)(ctypes.byref(_args(kind, **over)), None) == 0, (kind, over)


def test_struct_sizes():
    c = ssa._capi
    assert [ctypes.sizeof(t) for t in (c.LogProbsArgs, c.LogProbsGradArgs, c.LinearArgs, c.LinearGradArgs)] == [168, 168, 160, 160]


def _grad_workspace(**over):
    p = ctypes.cast(ctypes.create_string_buffer(64), ctypes.c_void_p).value // 16 * 16
    kw = dict(dtype=1, grad_dtype=1, batch=1, x=p, w=p, g=p)
    kw.update(over)
    return ssa._capi.load().ssmap_linear_grad_workspace(ctypes.byref(ssa._capi.LinearGradArgs(**kw)))


def test_the_dense_axis_of_an_operand_is_not_read_from_its_strides():
    """Rows one element apart are dense along both axes; the gradients' products read them along the features, and
    that is what a copy of them lays out: 8191 lines of 512 values, and not 512 of 8191 (filled up to 8192)."""
    rows = dict(layout=0, rows=8191, inner=512, outer=512, g_inner_stride=512, w_row_stride=512, g_w=16)
    assert _grad_workspace(**rows, x_row_stride=1) - _grad_workspace(**rows, x_row_stride=512) == 8191 * 512 * 2
    planes = dict(layout=1, rows=80000, inner=512, outer=41, g_inner_stride=80000, x_row_stride=512, g_x=16)
    assert _grad_workspace(**planes, w_row_stride=1) - _grad_workspace(**planes, w_row_stride=512) == 41 * 512 * 2
    # a line that stands alone has no stride
    one = dict(layout=1, batch=16, rows=307200, inner=256, outer=1, g_batch_stride=307200, g_inner_stride=307200,
               x_batch_stride=307200 * 256, x_row_stride=256, g_x=16)
    assert _grad_workspace(**one, w_row_stride=1) == _grad_workspace(**one, w_row_stride=256) == 0


def test_tangents_are_seen():
    from torch.autograd import forward_ad
    t = torch.ones(3)
    assert not heads._tangent(t)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(t, torch.ones(3))
        assert heads._tangent(dual) and not heads._tangent(t)
        with torch.no_grad():
            assert heads._tangent(dual) and not heads._tangent(forward_ad.unpack_dual(dual).primal)


def test_dz_is_kept_twice_where_16_bits_do_not_hold_it():
    """Parts of dz in the workspace: a float32 gradient and slopes between 0 and 1 round, relu's and none do not."""
    sizes = dict(layout=0, rows=512, inner=64, outer=64, g_inner_stride=64, x_row_stride=64, w_row_stride=64, pre=16)
    one = 512 * 64 * 2
    dz = lambda dtype, g, act: _grad_workspace(**sizes, dtype=dtype, grad_dtype=g, activation=act, g_x=16) - \
        _grad_workspace(**sizes, dtype=dtype, grad_dtype=dtype, activation=0, g_x=16)  # noqa: E731
    for dtype, scale in ((1, 0), (2, 4352)):      # fp16: its scale and the blocks' peaks as well
        assert dz(dtype, dtype, 1) == one
        assert [dz(dtype, dtype, act) for act in (2, 3, 4)] == [2 * one + scale] * 3
        assert [dz(dtype, 0, act) for act in (0, 1, 2)] == [2 * one + scale] * 3
    assert dz(0, 0, 2) == 2 * one                 # float32: once
