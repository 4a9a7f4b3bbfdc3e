"""Head operators against plain 64-bit implementations, at the sizes, strides and masks where they can go
wrong.

Tolerances count roundings.  u = 2^-24 is half a step of float32 relative to the value; h is that of the
result's type (bf16 2^-9 of the next power of two, so at most 2^-8 of the value; fp16 2^-11; fp32 2^-24).
"""
import math

import numpy as np
import pytest
import torch

import semantic_search_amd as ssa

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
SMALLEST = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -25}
TYPES = [torch.float32, torch.bfloat16, torch.float16]
ids_of = lambda v: str(v).replace("torch.", "")  # noqa: E731


def gen(seed):
    return torch.Generator().manual_seed(seed)


# ------------------------------------------------------------------ log probabilities

def plain_scores(x, ids, T, top, ignore=-100):
    """The definition for rows [n, V] on the CPU in 64 bits."""
    z = x.double() / T
    n, V = z.shape
    m = z.max(1).values
    bad = torch.isnan(x.double()).any(1) | (x.double() == math.inf).any(1)
    none = (x.double() == -math.inf).all(1) & ~bad
    ms = torch.where(torch.isfinite(m), m, 0.0)
    e = (z - ms[:, None]).exp()
    s = e.sum(1)
    logp = z - ms[:, None] - s.log()[:, None]
    p = e / s[:, None]
    ent = -torch.where(p > 0, p * logp, 0.0).sum(1)
    nan = torch.tensor(math.nan, dtype=torch.float64)
    ent = torch.where(bad, nan, torch.where(none, 0.0, ent))
    log_sum = torch.where(bad, nan, torch.where(none, -math.inf, s.log()))
    given = torch.empty(n, dtype=torch.float64)
    for i, t in enumerate(ids.tolist()):
        given[i] = (0.0 if t == ignore else math.nan if not 0 <= t < V or bad[i] else -math.inf if none[i] else logp[i, t])
    order = torch.from_numpy(np.lexsort((np.broadcast_to(np.arange(V), (n, V)), -np.nan_to_num(x.double().numpy(), nan=0.0)))[:, :top].copy())
    top_lp = logp.gather(1, order) if top else logp[:, :0]
    gone = (x.double().gather(1, order) == -math.inf) | none[:, None] | bad[:, None]
    top_ids = torch.where(gone, -1, order)
    top_lp = torch.where(gone, -math.inf, top_lp)
    top_lp = torch.where(bad[:, None], nan, top_lp)
    t2 = torch.where(p > 0, p * (z - ms[:, None]) ** 2, 0.0).sum(1)
    return dict(log_prob=given, entropy=ent, log_sum=log_sum, top_ids=top_ids, top_log_prob=top_lp, p=p, logp=logp, t2=t2,
                bad=bad, none=none)


def close(name, got, want, tol):
    got, want = got.double().cpu(), want.double()
    want = torch.where(want.abs() > torch.finfo(torch.float32).max, want.sign() * math.inf, want)    # no float32 holds it
    assert got.shape == want.shape, (name, got.shape, want.shape)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{name}: NaN in other places"
    inf = torch.isinf(want) | torch.isinf(got)
    assert torch.equal(got[inf], want[inf]), f"{name}: infinities"
    ok = ~(torch.isnan(want) | inf)
    off = ((got - want).abs() - torch.as_tensor(tol).expand_as(want))[ok]
    assert off.numel() == 0 or float(off.max()) <= 0, f"{name}: off by {float(off.max())} over the tolerance"


def check_scores(got, want, V):
    """t = (x - m)/T has three roundings, 2^t one and what t's error makes of it (E|t| = entropy - log_sum in
    the sum), a sum over at most V/16 terms in sequence and a tree of at most 12 steps, a logarithm."""
    serial = V / 16 + 32
    ls, H = want["log_sum"].nan_to_num(0, 0, 0), want["entropy"].nan_to_num(0)
    base = U * (serial + 4 * ls.abs() + 4 * H)
    close("log_sum", got.log_sum.reshape(-1), want["log_sum"], base)
    lp = want["log_prob"].nan_to_num(0, 0, 0)
    close("log_prob", got.log_prob.reshape(-1), want["log_prob"], base + 8 * U * lp.abs())
    # W = sum e t: each term 5 roundings relative, e's error through t once more (t^2)
    close("entropy", got.entropy.reshape(-1), want["entropy"], U * (serial * (1 + H) + 8 * H + 4 * want["t2"].nan_to_num(0)) + base)
    assert torch.equal(got.top_ids.long().cpu(), want["top_ids"]), "alternatives"
    tl = want["top_log_prob"].nan_to_num(0, 0, 0)
    close("top_log_prob", got.top_log_prob, want["top_log_prob"], base[:, None] + 8 * U * tl.abs())


def make_rows(n, V, dtype, seed, spread=3.0):
    g = gen(seed)
    x = (torch.randn((n, V), generator=g) * spread).to(dtype)
    ids = torch.randint(0, V, (n,), generator=g)
    ids[::5] = -100
    return x, ids


@pytest.mark.parametrize("dtype", TYPES, ids=ids_of)
@pytest.mark.parametrize("n,V,top", [(1, 1, 1), (3, 2, 2), (5, 3, 0), (4, 7, 7), (33, 8, 3), (130, 40, 5), (7, 64, 32), (9, 65, 32),
                                     (67, 150, 2), (6, 255, 20), (5, 257, 1), (3, 1000, 32), (4, 1025, 5), (3, 2049, 20), (2, 4099, 20),
                                     (3, 9001, 32), (1, 32003, 20), (5, 32003, 0), (2, 70001, 32)])
def test_rows(n, V, top, dtype):
    x, ids = make_rows(n, V, dtype, 11 * n + V)
    got = ssa.log_probs(x.cuda(), ids.cuda(), top=top, temperature=1.7)
    check_scores(got, plain_scores(x, ids, float(np.float32(1.7)), top), V)
    assert got.row_max.cpu().double().equal(x.double().max(1).values)


@pytest.mark.parametrize("dtype", TYPES, ids=ids_of)
def test_many_rows(dtype):
    # more rows than workgroups fit at once, in every kernel's range of sizes
    for n, V, top in ((5000, 40, 2), (1500, 1500, 3), (700, 5000, 2)):
        x, ids = make_rows(n, V, dtype, n)
        got = ssa.log_probs(x.cuda(), ids.cuda(), top=top)
        check_scores(got, plain_scores(x, ids, 1.0, top), V)


@pytest.mark.parametrize("dtype", TYPES, ids=ids_of)
@pytest.mark.parametrize("n", [1, 520])
def test_crowded_alternatives(n, dtype):
    """Rows whose large logits stand a fixed distance apart, so that a few threads of a block read all of
    them and many logits pass for candidates; ascending, descending and equal ones beside them."""
    V, top = 40000, 32
    g = gen(n)
    rows = torch.zeros((7, V))
    for i, (stride, width) in enumerate([(2048, 8 * 31), (1024, 4 * 31), (2048, 8)]):
        at = torch.arange(V) % stride < width
        rows[i, at] = 5 + torch.randn(int(at.sum()), generator=g)
    rows[3] = torch.arange(V) / 1000.0
    rows[4] = -torch.arange(V) / 1000.0
    rows[5] = 1.0
    rows[6, torch.randint(0, V, (3000,), generator=g)] = 7.0
    rows = rows.to(dtype)
    x = torch.zeros((max(n, 7), V), dtype=dtype, device="cuda")
    x[-7:] = rows.cuda()
    ids = torch.arange(x.shape[0]) % 9
    got = ssa.log_probs(x, ids.cuda(), top=top)
    want = plain_scores(rows, ids[-7:], 1.0, top)
    check_scores(ssa.LogProbs(*[t[-7:] for t in got]), want, V)


@pytest.mark.parametrize("dtype", TYPES, ids=ids_of)
@pytest.mark.parametrize("E,V,hw,top", [(1, 1, (1, 1), 1), (2, 3, (1, 5), 3), (3, 8, (7, 9), 2), (2, 40, (16, 33), 3), (1, 150, (13, 21), 5),
                                        (2, 155, (5, 64), 32), (1, 300, (3, 11), 9), (1, 21, (64, 65), 0)])
def test_planes(E, V, hw, top, dtype):
    g = gen(E * V)
    x = (torch.randn((E, V) + hw, generator=g) * 3).to(dtype)
    ids = torch.randint(0, V, (E,) + hw, generator=g, dtype=torch.int32)
    ids[:, ::2, ::3] = -100
    got = ssa.log_probs(x.cuda(), ids.cuda(), dim=1, top=top, temperature=3.2)
    assert got.top_ids.shape == (E, top) + hw and got.top_log_prob.shape == (E, top) + hw
    flat = got._replace(top_ids=got.top_ids.movedim(1, -1).flatten(0, -2), top_log_prob=got.top_log_prob.movedim(1, -1).flatten(0, -2))
    check_scores(flat, plain_scores(x.movedim(1, -1).reshape(-1, V), ids.reshape(-1), float(np.float32(3.2)), top), V)


@pytest.mark.parametrize("dtype", TYPES, ids=ids_of)
@pytest.mark.parametrize("V,top", [(5003, 2), (131072, 0)])
def test_planes_of_many_classes(V, top, dtype):
    """A vocabulary in planes: one thread sums all classes of a position, to no more roundings than few would cost.
    Steps of eight classes are summed (8 roundings) and added with what the additions lose; a rescaling's three roundings
    fade by half with the next; a term has five."""
    g = gen(V)
    at = torch.arange(V).float()
    rows = [torch.randn(V, generator=g) * 2, torch.full((V,), -1.1), at / V, -at / V, at * (200.0 / V), (at % 97) / 97 - 0.3, torch.full((V,), 0.7)]
    rows[1][0] = 0.0
    x = torch.stack(rows).to(dtype)
    ids = torch.tensor([0, 5, V - 1, V // 2, V - 1, 17, V])
    T = 0.9
    got = ssa.log_probs(x.t().contiguous()[None].cuda(), ids[None].cuda(), dim=1, top=top, temperature=T)
    want = plain_scores(x, ids, float(np.float32(T)), top)
    ls, H = want["log_sum"], want["entropy"]
    base = U * (32 + 4 * ls.abs() + 4 * H)
    close("log_sum", got.log_sum[0], ls, base)
    close("log_prob", got.log_prob[0], want["log_prob"], base + 8 * U * want["log_prob"].nan_to_num(0).abs())
    close("entropy", got.entropy[0], H, U * (32 * (1 + H) + 8 * H + 4 * want["t2"]) + base)
    assert torch.equal(got.top_ids[0].t().cpu().long(), want["top_ids"])
    assert got.row_max[0].cpu().double().equal(x.double().max(1).values)


def special_rows(V, dtype, seed):
    """Rows with masks, ties, infinities and the type's extremes, and ids to match."""
    g = gen(seed)
    low, inf = torch.finfo(dtype).min, math.inf
    rows, ids = [], []

    def add(row, i):
        rows.append(row.to(dtype))
        ids.append(i)

    base = torch.randn(V, generator=g) * 2
    add(base, 0)
    add(torch.full((V,), -inf), 1 % V)                                   # a mask that leaves nothing
    add(torch.full((V,), -inf), -100)
    only = torch.full((V,), -inf); only[V // 2] = 0.5
    add(only, V // 2)                                                    # one class left
    add(only, 0)
    half = base.clone(); half[::2] = -inf
    add(half, 0)                                                         # the given class is masked
    add(torch.full((V,), low), V - 1)                                    # nothing but the lowest value
    lows = torch.full((V,), low); lows[V // 3] = base[0]
    add(lows, V // 3)
    add(torch.full((V,), float(torch.finfo(dtype).max)), 0)
    ends = torch.full((V,), low); ends[0] = torch.finfo(dtype).max
    add(ends, 0)
    add(torch.full((V,), 1.25), V - 1)                                   # nothing but ties
    ties = torch.round(base * 2) / 2
    add(ties, 0)
    zeros = torch.zeros(V); zeros[::2] = -0.0
    add(zeros, 0)                                                        # 0 and -0 are equal
    add(torch.arange(V).float().clamp(max=2048) / 64, 0)                 # ascending
    add(-torch.arange(V).float().clamp(max=2048) / 64, 0)
    nan = base.clone(); nan[V // 2] = math.nan
    add(nan, 0)
    add(nan, -100)
    pinf = base.clone(); pinf[V - 1] = inf
    add(pinf, V - 1)
    two = base.clone(); two[0] = inf; two[V - 1] = inf
    add(two, 0)
    gone = torch.full((V,), -inf); gone[V - 1] = math.nan
    add(gone, 0)
    add(base, V)                                                         # ids outside
    add(base, -1)
    add(base, 2 ** 31 - 1)
    return torch.stack(rows), torch.tensor(ids)


@pytest.mark.parametrize("dtype", TYPES, ids=ids_of)
@pytest.mark.parametrize("V", [1, 2, 40, 200, 700, 2500, 40000])
def test_special_rows(V, dtype):
    x, ids = special_rows(V, dtype, V)
    top = min(20, V)
    for i64 in (True, False):
        t = ids if i64 else ids.to(torch.int32)
        got = ssa.log_probs(x.cuda(), t.cuda(), top=top)
        check_scores(got, plain_scores(x, ids, 1.0, top), V)


@pytest.mark.parametrize("dtype", TYPES, ids=ids_of)
def test_special_planes(dtype):
    x, ids = special_rows(40, dtype, 3)
    got = ssa.log_probs(x.t().contiguous()[None].cuda(), ids[None].cuda(), dim=1, top=5)
    flat = got._replace(top_ids=got.top_ids[0].t(), top_log_prob=got.top_log_prob[0].t())
    check_scores(flat, plain_scores(x, ids, 1.0, 5), 40)


@pytest.mark.parametrize("dtype", TYPES, ids=ids_of)
@pytest.mark.parametrize("V,top", [(40, 0), (40, 1), (40, 3), (41, 9), (700, 20), (3, 2), (1, 0)])
def test_special_planes_with_any_number_of_alternatives(V, top, dtype):
    x, ids = special_rows(V, dtype, V + top)
    got = ssa.log_probs(x.t().contiguous()[None].cuda(), ids[None].cuda(), dim=1, top=top)
    flat = got._replace(top_ids=got.top_ids[0].t(), top_log_prob=got.top_log_prob[0].t())
    check_scores(flat, plain_scores(x, ids, 1.0, top), V)
    # an ignored id may be a class
    got = ssa.log_probs(x.t().contiguous()[None].cuda(), ids[None].cuda(), dim=1, top=top, ignore_id=0)
    check_scores(got._replace(top_ids=got.top_ids[0].t(), top_log_prob=got.top_log_prob[0].t()), plain_scores(x, ids, 1.0, top, ignore=0), V)


@pytest.mark.parametrize("dtype", TYPES, ids=ids_of)
@pytest.mark.parametrize("V", [37, 515, 5003])
def test_views(V, dtype):
    """Shifted prompts, a padded vocabulary with NaN behind, an odd start, expanded rows."""
    x, ids = make_rows(3 * 8, V + 3, dtype, V)
    x[:, V:] = math.nan
    whole, idw = x.view(3, 8, V + 3).cuda(), (ids % V).view(3, 8).cuda()
    got = ssa.log_probs(whole[:, :-1, :V], idw[:, 1:], top=3)
    want = plain_scores(x.view(3, 8, -1)[:, :-1, :V].reshape(-1, V), (ids % V).view(3, 8)[:, 1:].reshape(-1), 1.0, 3)
    flat = got._replace(top_ids=got.top_ids.view(-1, 3), top_log_prob=got.top_log_prob.view(-1, 3))
    check_scores(flat, want, V)
    odd = torch.empty(5 * V + 1, dtype=dtype, device="cuda")[1:].view(5, V).copy_(whole[0, :5, :V])
    got = ssa.log_probs(odd, idw[0, :5], top=2)
    check_scores(got, plain_scores(x[:5, :V], ids[:5] % V, 1.0, 2), V)
    row = whole[0, 0, :V].expand(4, V)
    got = ssa.log_probs(row, idw[0, :4], top=2)
    check_scores(got, plain_scores(x[0, :V].expand(4, V), ids[:4] % V, 1.0, 2), V)
    # planes of a wider tensor
    p = x[:, :V].reshape(2, 12, V)[:, :, :35].movedim(-1, 1).contiguous().cuda()
    wide = torch.full((2, 41, 12), math.nan, dtype=dtype, device="cuda")
    wide[:, 3:38] = p
    t = (ids % 35).view(2, 12).cuda()
    got = ssa.log_probs(wide[:, 3:38], t, dim=1, top=2)
    want = ssa.log_probs(p, t, dim=1, top=2)
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_offsets_past_31_bits():
    """The last rows of tensors of more than 2^31 elements, against the same rows by themselves."""
    n, V = 16400, 131072
    x = torch.zeros((n, V), dtype=torch.bfloat16, device="cuda")
    x[-3:] = torch.randn((3, V), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)) * 3
    ids = torch.arange(n, device="cuda") % V
    s = ssa.log_probs(x, ids, top=5)
    want = plain_scores(x[-3:].cpu(), ids[-3:].cpu(), 1.0, 5)
    check_scores(ssa.LogProbs(*[t[-3:] for t in s]), want, V)
    g_l, g_e = torch.ones(n, device="cuda"), torch.full((n,), 0.5, device="cuda")
    g = ssa.log_probs_grad(x, ids, s, grad_log_prob=g_l, grad_entropy=g_e)
    check_grad(g[-3:], x[-3:].cpu(), ids[-3:].cpu(), 1.0, want, g_l[-3:].cpu(), g_e[-3:].cpu(), None)
    del g
    w = torch.randn((16, V), device="cuda", generator=torch.Generator(device="cuda").manual_seed(2)).bfloat16()
    y = ssa.linear(x, w, out_dtype=torch.float32)
    ref = x[-3:].double() @ w.double().t()
    close("y", y[-3:], ref.cpu(), (U * (V + 8) * (x[-3:].double().abs() @ w.double().abs().t())).cpu())
    planes = torch.zeros((1, 8, 270_000_000), dtype=torch.bfloat16, device="cuda")
    planes[0, :, -5:] = torch.randn((8, 5), device="cuda", generator=torch.Generator(device="cuda").manual_seed(3))
    t = torch.full((1, 270_000_000), 3, dtype=torch.int32, device="cuda")
    s = ssa.log_probs(planes, t, dim=1)
    rows = planes[0, :, -5:].t().cpu()
    check_scores(ssa.LogProbs(*[v[0, ..., -5:] if v.numel() else v.view(0).new_zeros((5, 0)) for v in s]),
                 plain_scores(rows, torch.full((5,), 3), 1.0, 0), 8)


def test_empty_and_one_dimensional():
    got = ssa.log_probs(torch.zeros(0, 9, device="cuda"), torch.zeros(0, dtype=torch.int64, device="cuda"), top=2)
    assert got.log_prob.shape == (0,) and got.top_ids.shape == (0, 2)
    x = torch.randn(9, generator=gen(0))
    got = ssa.log_probs(x.cuda(), torch.tensor(4).cuda(), top=2)
    assert got.log_prob.shape == () and got.top_ids.shape == (2,)
    assert abs(float(got.log_prob) - float(x.double().log_softmax(0)[4])) < 40 * U


def plain_scores_grad(x, ids, T, want, g_l, g_e, g_t, ignore=-100):
    """The gradient's formula in 64 bits, and what its roundings scale with."""
    n, V = x.shape
    p, logp = want["p"], torch.where(want["p"] > 0, want["logp"], 0.0)
    g_l = torch.zeros(n, dtype=torch.float64) if g_l is None else torch.where(ids == ignore, 0.0, g_l.double())
    out, size = torch.zeros((n, V), dtype=torch.float64), torch.zeros((n, V), dtype=torch.float64)
    rows = torch.arange(n)
    valid = (ids >= 0) & (ids < V) & (ids != ignore)
    out[rows[valid], ids[valid]] += g_l[valid]
    total, most = g_l.clone(), g_l.abs()
    if g_t is not None:
        ok = want["top_ids"] >= 0
        gt = torch.where(ok, g_t.double(), 0.0)
        out.scatter_add_(1, want["top_ids"].clamp(min=0), gt)
        total, most = total + gt.sum(1), most + gt.abs().sum(1)
    out -= p * total[:, None]
    size += out.abs() + p * most[:, None]
    if g_e is not None:
        h = want["entropy"].nan_to_num(0)
        out -= g_e.double()[:, None] * p * (logp + h[:, None])
        size += (g_e.double().abs()[:, None] * p * (logp.abs() + h[:, None]))
    out[want["none"]] = 0.0
    size[want["none"]] = 0.0
    bad = want["bad"].clone()
    if (g_l != 0).any():
        bad |= ~valid & (ids != ignore)
    out[bad] = math.nan
    size[bad] = 0.0
    return out / T, size / T, logp.abs()


def check_grad(got, x, ids, T, want, g_l, g_e, g_t):
    ref, size, logp = plain_scores_grad(x, ids, T, want, g_l, g_e, g_t)
    # p = 2^t: t has 3 roundings relative to it, the saved log_sum its own error (see check_scores); then at
    # most 40 more operations (32 alternatives are summed one by one)
    serial = x.shape[1] / 16 + 32
    rel = U * (40 + serial + 8 * logp + 8 * want["log_sum"].nan_to_num(0, 0, 0).abs()[:, None] + 4 * want["entropy"].nan_to_num(0)[:, None]
               + 4 * want["t2"].nan_to_num(0)[:, None])
    tol = rel * size + HALF[x.dtype] * ref.nan_to_num(0).abs() * 1.0001 + SMALLEST[x.dtype]
    close("gradient", got, ref, tol)


@pytest.mark.parametrize("dtype", TYPES, ids=ids_of)
@pytest.mark.parametrize("n,V,top", [(1, 1, 1), (3, 2, 2), (4, 7, 3), (33, 40, 5), (5, 64, 32), (21, 150, 2), (5, 257, 1), (3, 1000, 20),
                                     (4, 1025, 5), (2, 4099, 20), (1, 32003, 3), (700, 33, 2)])
def test_grad_rows(n, V, top, dtype):
    x, ids = make_rows(n, V, dtype, 7 * n + V)
    g = gen(n)
    g_l, g_e, g_t = torch.randn(n, generator=g), torch.randn(n, generator=g), torch.randn((n, top), generator=g)
    T = float(np.float32(0.8))
    want = plain_scores(x, ids, T, top)
    dx, dids = x.cuda(), ids.cuda()
    scores = ssa.log_probs(dx, dids, top=top, temperature=0.8)
    for a, b, c in ((g_l, g_e, g_t), (g_l, None, None), (None, g_e, None), (None, None, g_t), (g_l, g_e, None)):
        to = lambda v: None if v is None else v.cuda()  # noqa: E731
        got = ssa.log_probs_grad(dx, dids, scores, temperature=0.8, grad_log_prob=to(a), grad_entropy=to(b), grad_top=to(c))
        assert got.dtype == dtype and got.is_contiguous()
        check_grad(got, x, ids, T, want, a, b, c)


@pytest.mark.parametrize("dtype", TYPES, ids=ids_of)
@pytest.mark.parametrize("V", [2, 40, 700, 5000])
def test_grad_special_rows(V, dtype):
    x, ids = special_rows(V, dtype, V)
    top, n = min(3, V), x.shape[0]
    g = gen(V)
    g_l, g_e, g_t = torch.randn(n, generator=g), torch.randn(n, generator=g), torch.randn((n, top), generator=g)
    want = plain_scores(x, ids, 1.0, top)
    scores = ssa.log_probs(x.cuda(), ids.cuda(), top=top)
    for a, b, c in ((g_l, g_e, g_t), (None, g_e, g_t)):
        to = lambda v: None if v is None else v.cuda()  # noqa: E731
        got = ssa.log_probs_grad(x.cuda(), ids.cuda(), scores, grad_log_prob=to(a), grad_entropy=to(b), grad_top=to(c))
        check_grad(got, x, ids, 1.0, want, a, b, c)


@pytest.mark.parametrize("dtype", TYPES, ids=ids_of)
@pytest.mark.parametrize("E,V,hw,top", [(1, 1, (1, 1), 1), (2, 8, (7, 9), 2), (2, 40, (16, 33), 3), (1, 150, (13, 21), 32), (1, 21, (64, 65), 1)])
def test_grad_planes(E, V, hw, top, dtype):
    g = gen(E * V)
    x = (torch.randn((E, V) + hw, generator=g) * 3).to(dtype)
    ids = torch.randint(0, V, (E,) + hw, generator=g)
    ids[:, ::2, ::3] = -100
    g_l, g_e, g_t = torch.randn((E,) + hw, generator=g), torch.randn((E,) + hw, generator=g), torch.randn((E, top) + hw, generator=g)
    scores = ssa.log_probs(x.cuda(), ids.cuda(), dim=1, top=top, temperature=2.5)
    got = ssa.log_probs_grad(x.cuda(), ids.cuda(), scores, dim=1, temperature=2.5, grad_log_prob=g_l.cuda(), grad_entropy=g_e.cuda(),
                             grad_top=g_t.cuda())
    assert got.shape == x.shape and got.is_contiguous()
    rows = x.movedim(1, -1).reshape(-1, V)
    want = plain_scores(rows, ids.reshape(-1), 2.5, top)
    check_grad(got.movedim(1, -1).reshape(-1, V), rows, ids.reshape(-1), 2.5, want, g_l.reshape(-1), g_e.reshape(-1),
               g_t.movedim(1, -1).reshape(-1, top))


def test_grad_takes_expanded_gradients_and_views():
    x, ids = make_rows(24, 51, torch.float32, 5)
    whole, idw = x.view(3, 8, 51).cuda(), ids.view(3, 8).cuda()
    scores = ssa.log_probs(whole[:, :-1], idw[:, 1:], top=2)
    one = torch.full((1, 1), -0.25, device="cuda")
    got = ssa.log_probs_grad(whole[:, :-1], idw[:, 1:], scores, grad_log_prob=one.expand(3, 7))
    flat, fid = x.view(3, 8, 51)[:, :-1].reshape(-1, 51), ids.view(3, 8)[:, 1:].reshape(-1)
    check_grad(got.view(-1, 51), flat, fid, 1.0, plain_scores(flat, fid, 1.0, 2), torch.full((21,), -0.25), None, None)


def test_grad_leaves_alternatives_outside_alone():
    """Ids of alternatives that no class has give nothing, and nothing is written behind a row."""
    for V, planes in ((700, False), (40, False), (5000, False), (40, True)):
        x, ids = make_rows(4, V, torch.float32, V)
        dx = (x.t()[None].contiguous() if planes else x).cuda()
        t = (ids[None] if planes else ids).cuda()
        d = 1 if planes else -1
        s = ssa.log_probs(dx, t, dim=d, top=3)
        g_t = torch.ones_like(s.top_log_prob)
        bad = s.top_ids.clone()
        bad.select(d, 1).copy_(torch.tensor([V, V + 1, 2 ** 31 - 1, -7])[None] if planes else torch.tensor([V, V + 1, 2 ** 31 - 1, -7]))
        got = ssa.log_probs_grad(dx, t, s._replace(top_ids=bad), dim=d, grad_top=g_t)
        none = s.top_ids.clone()
        none.select(d, 1).fill_(-1)
        assert torch.equal(got, ssa.log_probs_grad(dx, t, s._replace(top_ids=none), dim=d, grad_top=g_t))


def test_grad_against_differences():
    """Central differences of the 64-bit forward formula, step 1e-4: its own error is below 1e-7."""
    x, ids = make_rows(2, 9, torch.float32, 1)
    g = gen(9)
    g_l, g_e, g_t = torch.randn(2, generator=g), torch.randn(2, generator=g), torch.randn((2, 3), generator=g)

    def loss(v):
        w = plain_scores(v, ids, 0.75, 3)
        return (w["log_prob"] * g_l.double() + w["entropy"] * g_e.double() + (w["top_log_prob"] * g_t.double()).sum(1)).sum()

    scores = ssa.log_probs(x.cuda(), ids.cuda(), top=3, temperature=0.75)
    got = ssa.log_probs_grad(x.cuda(), ids.cuda(), scores, temperature=0.75, grad_log_prob=g_l.cuda(), grad_entropy=g_e.cuda(),
                             grad_top=g_t.cuda()).cpu().double()
    for i in range(2):
        for j in range(9):
            up, dn = x.double().clone(), x.double().clone()
            up[i, j] += 1e-4
            dn[i, j] -= 1e-4
            assert abs(float((loss(up) - loss(dn)) / 2e-4) - float(got[i, j])) < 1e-5


def test_temperature_gradient_identity():
    """d log_prob / dT = -(log_prob + entropy) / T, by differences in T."""
    x, ids = make_rows(6, 40, torch.float32, 2)
    T = 1.75
    got = ssa.log_probs(x.cuda(), ids.cuda(), temperature=T, ignore_id=-1000000)
    keep = ids >= 0
    hi, lo = plain_scores(x, ids, T + 1e-4, 0), plain_scores(x, ids, T - 1e-4, 0)
    want = (hi["log_prob"] - lo["log_prob"]) / 2e-4
    have = -(got.log_prob + got.entropy).cpu().double() / T
    assert float((want - have)[keep].abs().max()) < 1e-5


# ------------------------------------------------------------------ the product

def plain_act(z, name):
    if name == "relu":
        return z.clamp(min=0)
    if name == "gelu":
        return z * torch.special.erfc(-z / math.sqrt(2)) / 2
    if name == "gelu_tanh":
        return z * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))
    if name == "silu":
        return z * torch.sigmoid(z)
    return z


def plain_linear(x, w, b, act, r, planes):
    z = x.double() @ w.double().t()
    size = x.double().abs() @ w.double().abs().t()
    if b is not None:
        z, size = z + b.double(), size + b.double().abs()
    y = plain_act(z, act)
    if planes:
        move = lambda v: v.movedim(-1, 1)  # noqa: E731
        z, y, size = move(z), move(y), move(size)
    return (y if r is None else y + r.double()), z, size


ACTS = [None, "relu", "gelu", "gelu_tanh", "silu"]


def make_linear(lead, K, N, dtype, out_dtype, seed, planes=False):
    g = gen(seed)
    x = torch.randn(lead + (K,), generator=g).to(dtype)
    w = (torch.randn((N, K), generator=g) / math.sqrt(max(K, 1))).to(dtype)
    b = torch.randn(N, generator=g)
    shape = (lead[0], N) + lead[1:] if planes else lead + (N,)
    r = torch.randn(shape, generator=g).to(out_dtype)
    return x, w, b, r


def linear_tolerance(ref, y, size, K, out_dtype):
    """K products and sums in float32 (relative to the sum of magnitudes), an activation of slope at most
    1.13 evaluated to about 16 roundings of values up to |y|, a residual, one rounding to the result's type."""
    return 1.13 * U * (K + 8) * size + 16 * U * (y.abs() + 1) + HALF[out_dtype] * ref.abs() * 1.0001 + SMALLEST[out_dtype]


LINEAR_SIZES = [((1,), 1, 1), ((3,), 5, 7), ((1,), 64, 64), ((2, 3), 129, 33), ((16,), 256, 40), ((17,), 255, 130), ((64,), 512, 65),
                ((1,), 1000, 515), ((5,), 4096, 70), ((33, 4), 96, 257), ((130,), 72, 136), ((255,), 1024, 129), ((300,), 33, 300),
                ((513,), 320, 260)]


@pytest.mark.parametrize("dtype", TYPES, ids=ids_of)
@pytest.mark.parametrize("lead,K,N", LINEAR_SIZES)
def test_linear_rows(lead, K, N, dtype):
    for i, (out, act, bias, res) in enumerate([(dtype, None, False, False), (torch.float32, "gelu", True, True), (dtype, "silu", True, False),
                                               (dtype, "relu", False, True), (dtype, "gelu_tanh", True, True)]):
        x, w, b, r = make_linear(lead, K, N, dtype, out, K + N + i)
        b = (b if i % 2 else b.to(dtype)) if bias else None
        r = r if res else None
        ref, z, size = plain_linear(x, w, b, act, r, False)
        cu = lambda t: None if t is None else t.cuda()  # noqa: E731
        got, pre = ssa.linear(x.cuda(), w.cuda(), cu(b), activation=act, residual=cu(r), out_dtype=out, keep_pre=True)
        assert got.dtype == out and pre.dtype == dtype
        close("y", got, ref, linear_tolerance(ref, ref if r is None else ref - r.double(), size, K, out))
        close("pre", pre, z, U * (K + 8) * size + HALF[dtype] * z.abs() * 1.0001 + SMALLEST[dtype])
        again = ssa.linear(x.cuda(), w.cuda(), cu(b), activation=act, residual=cu(r), out_dtype=out)
        assert torch.equal(again, got), "two calls differ"


@pytest.mark.parametrize("dtype", TYPES, ids=ids_of)
@pytest.mark.parametrize("lead,K,N", [((1, 1), 1, 1), ((2, 5), 7, 3), ((1, 9, 13), 33, 8), ((2, 16, 20), 256, 40), ((3, 65), 96, 150),
                                      ((1, 1000), 64, 21), ((2, 300), 130, 155)])
def test_linear_planes(lead, K, N, dtype):
    for i, (out, act, bias, res) in enumerate([(torch.float32, None, True, False), (dtype, "gelu", True, True)]):
        x, w, b, r = make_linear(lead, K, N, dtype, out, K + N + i, planes=True)
        r = r if res else None
        ref, z, size = plain_linear(x, w, b, act, r, True)
        got, pre = ssa.linear(x.cuda(), w.cuda(), b.cuda(), activation=act, residual=None if r is None else r.cuda(), out_dtype=out, planes=True,
                              keep_pre=True)
        close("y", got, ref, linear_tolerance(ref, ref if r is None else ref - r.double(), size, K, out))
        close("pre", pre, z, U * (K + 8) * size + HALF[dtype] * z.abs() * 1.0001 + SMALLEST[dtype])


@pytest.mark.parametrize("dtype", TYPES, ids=ids_of)
@pytest.mark.parametrize("n,K,N", [(8190, 200, 4088), (16400, 64, 2056), (4096, 1000, 8190), (40000, 128, 48), (2000, 2048, 1500), (100, 8200, 600), (2047, 1001, 1037),
                                   (1003, 515, 1501), (700, 1024, 520)])
def test_linear_large(n, K, N, dtype):
    """Sizes that take the largest tiles, split sums and many tiles with partial ones at the ends; forward and
    backward against 64-bit products on the GPU."""
    g = torch.Generator(device="cuda").manual_seed(n + K)
    x = torch.randn((n, K), device="cuda", generator=g).to(dtype)
    w = (torch.randn((N, K), device="cuda", generator=g) / math.sqrt(K)).to(dtype)
    b = torch.randn(N, device="cuda", generator=g)
    xd, wd = x.double(), w.double()

    def check(name, got, want, size, terms, extra=0.0):
        tol = (U * (terms + 8) + extra) * size * 1.0001 + HALF[dtype] * want.abs() * 1.0001 + SMALLEST[dtype]
        off = (got.double() - want).abs() - tol
        assert float(off.max()) <= 0, f"{name}: off by {float(off.max())} over the tolerance"

    size = xd.abs() @ wd.abs().t()
    check("y", ssa.linear(x, w, b), xd @ wd.t() + b.double(), size + b.double().abs(), K)
    dy = torch.randn((n, N), device="cuda", generator=g).to(dtype)
    got = ssa.linear_grad(dy, x, w)
    d = dy.double()
    check("gradient of x", got.x, d @ wd, d.abs() @ wd.abs(), N)
    check("gradient of weight", got.weight, d.t() @ xd, d.abs().t() @ xd.abs(), n)
    check("gradient of bias", got.bias, d.sum(0), d.abs().sum(0), n)


@pytest.mark.parametrize("dtype", TYPES, ids=ids_of)
@pytest.mark.parametrize("K,N", [(8, 1), (24, 17), (72, 40), (256, 40), (512, 64), (2048, 16), (40, 33)])
def test_linear_heads(K, N, dtype):
    """Few classes against many positions, in planes of several frames that start anywhere, and few rows against
    a vocabulary; NaN beside what may be read."""
    B, n = 2, 9001
    g = torch.Generator(device="cuda").manual_seed(K)
    x = torch.full((B, n + 1, K + 3), math.nan, device="cuda", dtype=dtype)[:, :n, 1:K + 1]
    x.copy_(torch.randn((B, n, K), device="cuda", generator=g))
    w = torch.full((N + 1, K + 5), math.nan, device="cuda", dtype=dtype)[:N, 3:K + 3]
    w.copy_(torch.randn((N, K), device="cuda", generator=g) / math.sqrt(K))
    b = torch.randn(N, device="cuda", generator=g)
    r = torch.randn((B, N, n), device="cuda", generator=g)
    ref, _, size = plain_linear(x, w, b, "silu", r, True)
    got = ssa.linear(x, w, b, activation="silu", residual=r, planes=True, out_dtype=torch.float32)
    close("planes", got, ref.cpu(), linear_tolerance(ref, ref - r.double(), size, K, torch.float32).cpu())
    tokens, vocab = w[:min(N, 40)], x[0].reshape(n, K).repeat(2, 1)
    bias = torch.randn(vocab.shape[0], device="cuda", generator=g)
    ref, _, size = plain_linear(tokens, vocab, bias, None, None, False)
    got = ssa.linear(tokens, vocab, bias)
    close("rows", got, ref.cpu(), linear_tolerance(ref, ref, size, K, dtype).cpu())


@pytest.mark.parametrize("dtype", TYPES, ids=ids_of)
@pytest.mark.parametrize("planes", [False, True])
def test_linear_batches_out_of_line(planes, dtype):
    """Batches that do not merge, rows that start anywhere, every size odd: copies of each batch are made."""
    B, n, K, N = 3, 701, 1001, 603
    g = torch.Generator(device="cuda").manual_seed(5)
    x = torch.full((B, n + 2, K + 4), math.nan, device="cuda", dtype=dtype)[:, 1:n + 1, 3:K + 3]
    x.copy_(torch.randn((B, n, K), device="cuda", generator=g))
    w = torch.full((N, K + 1), math.nan, device="cuda", dtype=dtype)[:, :K]
    w.copy_(torch.randn((N, K), device="cuda", generator=g) / math.sqrt(K))
    xd, wd = x.double(), w.double()
    move = (lambda t: t.transpose(1, 2)) if planes else (lambda t: t)
    check = lambda name, got, want, size, terms: close(name, got.double(), want.cpu(), (U * (terms + 8) * size * 1.0001 + HALF[dtype] * want.abs() * 1.0001 + SMALLEST[dtype]).cpu())  # noqa: E731
    check("y", ssa.linear(x, w, planes=planes), move(xd @ wd.t()), move(xd.abs() @ wd.abs().t()), K)
    dy = torch.full((B, N + 1, n + 1) if planes else (B, n + 1, N + 1), math.nan, device="cuda", dtype=dtype)
    dy = dy[:, 1:, :n] if planes else dy[:, 1:, :N]
    dy.copy_(torch.randn(dy.shape, device="cuda", generator=g))
    got = ssa.linear_grad(dy, x, w, planes=planes)
    d = move(dy.double())
    check("gradient of x", got.x, d @ wd, d.abs() @ wd.abs(), N)
    df, xf = d.reshape(-1, N), xd.reshape(-1, K)
    check("gradient of weight", got.weight, df.t() @ xf, df.abs().t() @ xf.abs(), B * n)
    check("gradient of bias", got.bias, df.sum(0), df.abs().sum(0), B * n)


@pytest.mark.parametrize("dtype", TYPES, ids=ids_of)
def test_linear_views(dtype):
    """Rows of wider tensors, odd starts, expanded residuals; NaN beside what may be read."""
    for K, N, n in ((40, 24, 6), (67, 33, 40), (256, 64, 3), (264, 136, 200)):
        x, w, b, _ = make_linear((4, n), K, N, dtype, dtype, K)
        wide_x = torch.full((4, n + 1, K + 3), math.nan, dtype=dtype, device="cuda")
        wide_w = torch.full((N, K + 5), math.nan, dtype=dtype, device="cuda")
        wide_x[:, :n, 1:K + 1] = x.cuda()
        wide_w[:, 2:K + 2] = w.cuda()
        r = torch.randn((1, 1, N), generator=gen(1)).to(dtype)
        got = ssa.linear(wide_x[:, :n, 1:K + 1], wide_w[:, 2:K + 2], b.cuda(), residual=r.cuda().expand(4, n, N), activation="silu")
        ref, _, size = plain_linear(x, w, b, "silu", r, False)
        close("y", got, ref, linear_tolerance(ref, ref - r.double(), size, K, dtype))
        planes = torch.randn((4, N + 2, n), generator=gen(2)).to(dtype).cuda()
        got = ssa.linear(wide_x[:, :n, 1:K + 1], wide_w[:, 2:K + 2], b.cuda(), residual=planes[:, 1:N + 1], planes=True)
        ref, _, size = plain_linear(x, w, b, None, planes[:, 1:N + 1].cpu(), True)
        close("planes", got, ref, linear_tolerance(ref, ref, size, K, dtype) + 8 * U)


def test_linear_of_nothing():
    z = lambda *s: torch.zeros(s, device="cuda")  # noqa: E731
    assert ssa.linear(z(0, 5), z(4, 5)).shape == (0, 4)
    assert ssa.linear(z(3, 5), z(0, 5)).shape == (3, 0)
    b = torch.arange(4.0, device="cuda")
    assert torch.equal(ssa.linear(z(3, 0), z(4, 0), b), b.expand(3, 4))
    g = ssa.linear_grad(z(0, 4), z(0, 5), z(4, 5) + 1)
    assert g.x.shape == (0, 5) and torch.equal(g.weight, z(4, 5)) and torch.equal(g.bias, z(4))
    g = ssa.linear_grad(z(3, 0), z(3, 5), z(0, 5))
    assert torch.equal(g.x, z(3, 5)) and g.weight.shape == (0, 5) and g.bias.shape == (0,)


def test_linear_lets_infinities_and_nan_through():
    for dtype in TYPES:
        x, w, b, _ = make_linear((70,), 65, 66, dtype, dtype, 3)
        w = w.abs() + 0.01
        x[3, 5], x[4, 64] = math.inf, math.nan
        got = ssa.linear(x.to(dtype).cuda(), w.to(dtype).cuda()).cpu().double()
        assert (got[3] == math.inf).all() and torch.isnan(got[4]).all()
        keep = [i for i in range(70) if i not in (3, 4)]
        assert torch.isfinite(got[keep]).all()


@pytest.mark.parametrize("dtype,far", [(torch.bfloat16, 12.5), (torch.float16, 5.25)], ids=ids_of)
def test_gelu_tail_of_16_bit_results(dtype, far):
    """gelu and its slope relative to their own size, every value of the type between -far and far.  The formula is off
    by 7.7e-7 (13 U), the exponential by three roundings of z^2 / 2, sixteen operations around them; the slope's dz holds
    2^-16 of it.  The slope is a sum of two terms of opposite sign: its errors go by their sizes."""
    bits = torch.arange(-32768, 32768, dtype=torch.int32).to(torch.int16).view(dtype)
    z = bits[(bits.float().abs() <= far) & (bits.float().abs() >= 2.0 ** -10)].reshape(-1, 1)
    one = torch.ones((1, 1), dtype=dtype, device="cuda")
    zd = z.double()
    phi, bell = torch.special.erfc(-zd / math.sqrt(2)) / 2, zd * torch.exp(-zd * zd / 2) / math.sqrt(2 * math.pi)
    rel = U * (32 + 2 * zd * zd)
    want = zd * phi
    close("gelu", ssa.linear(z.cuda(), one, activation="gelu"), want, (rel + HALF[dtype] * 1.0001) * want.abs() + SMALLEST[dtype])
    got = ssa.linear_grad(torch.ones_like(z).cuda(), z.cuda(), one, activation="gelu", pre=z.cuda(), need_weight=False, need_bias=False)
    want = phi + bell
    close("slope", got.x, want, (rel + 2.0 ** -16) * (phi + bell.abs()) + HALF[dtype] * want.abs() * 1.0001 + SMALLEST[dtype])


def plain_linear_grad(g, x, w, act, pre, planes):
    dz = g.double()
    slope = torch.ones_like(dz)
    if act:
        z = pre.double().requires_grad_(True)
        slope = torch.autograd.grad(plain_act(z, act).sum(), z)[0]
        if act == "relu":
            slope = (pre > 0).double()
    dz = dz * slope
    if planes:
        dz, g = dz.movedim(1, -1), g.movedim(1, -1)
    N, K = w.shape
    dz, g, xr = dz.reshape(-1, N), g.double().reshape(-1, N), x.double().reshape(-1, K)
    return ((dz @ w.double()).view(x.shape), dz.t() @ xr, dz.sum(0)), ((dz.abs() @ w.double().abs()).view(x.shape), dz.abs().t() @ xr.abs(), dz.abs().sum(0)), \
        ((g.abs() @ w.double().abs()).view(x.shape), g.abs().t() @ xr.abs(), g.abs().sum(0))


def check_linear_grad(got, want, size, gsize, n, N, dtype):
    """dz is rounded once to the products' type (not for the bias), after about 16 roundings of values up to
    |g|; then as many sums as terms, and one rounding of the result."""
    for k, terms in (("x", N), ("weight", n), ("bias", n)):
        i = ("x", "weight", "bias").index(k)
        step = HALF[dtype] if k != "bias" and dtype != torch.float32 else 0.0
        tol = (U * (terms + 8) + step) * size[i] * 1.0001 + 24 * U * gsize[i] + HALF[dtype] * want[i].abs() * 1.0001 + SMALLEST[dtype]
        if dtype == torch.float16:
            tol = tol + terms * 2.0 ** -25 * 4      # a dz below 2^-14 is rounded to a step of 2^-24
        close("gradient of " + k, getattr(got, k), want[i], tol)


@pytest.mark.parametrize("dtype", TYPES, ids=ids_of)
@pytest.mark.parametrize("lead,K,N", [((1,), 1, 1), ((3,), 5, 7), ((2, 3), 129, 33), ((16,), 256, 40), ((70,), 72, 130), ((300,), 96, 65),
                                      ((1,), 515, 400), ((515,), 264, 136)])
def test_linear_grad_rows(lead, K, N, dtype):
    for i, act in enumerate(ACTS):
        out = dtype if i % 2 else torch.float32
        x, w, b, g = make_linear(lead, K, N, dtype, out, K + N + i)
        pre = (torch.randn(g.shape, generator=gen(i)) * 1.5).to(dtype) if act else None
        got = ssa.linear_grad(g.cuda(), x.cuda(), w.cuda(), activation=act, pre=None if pre is None else pre.cuda())
        want, size, gsize = plain_linear_grad(g, x, w, act, pre, False)
        check_linear_grad(got, want, size, gsize, x[..., 0].numel(), N, dtype)
        again = ssa.linear_grad(g.cuda(), x.cuda(), w.cuda(), activation=act, pre=None if pre is None else pre.cuda())
        for a, c in zip(got, again):
            assert torch.equal(a, c), "two calls differ"


@pytest.mark.parametrize("dtype", TYPES, ids=ids_of)
@pytest.mark.parametrize("lead,K,N", [((1, 1), 1, 1), ((2, 5), 7, 3), ((2, 16, 20), 256, 40), ((3, 65), 96, 150), ((2, 513), 130, 21)])
def test_linear_grad_planes(lead, K, N, dtype):
    for i, act in enumerate((None, "gelu")):
        out = dtype if i else torch.float32
        x, w, b, g = make_linear(lead, K, N, dtype, out, K + N + i, planes=True)
        pre = (torch.randn(g.shape, generator=gen(i)) * 1.5).to(dtype) if act else None
        got = ssa.linear_grad(g.cuda(), x.cuda(), w.cuda(), activation=act, pre=None if pre is None else pre.cuda(), planes=True)
        want, size, gsize = plain_linear_grad(g, x, w, act, pre, True)
        check_linear_grad(got, want, size, gsize, x[..., 0].numel(), N, dtype)


def test_linear_grad_views_and_parts():
    x, w, b, g = make_linear((2, 37), 72, 40, torch.bfloat16, torch.bfloat16, 4)
    wide_g = torch.full((2, 40, 43), math.nan, dtype=torch.bfloat16, device="cuda")
    wide_x = torch.full((2, 38, 75), math.nan, dtype=torch.bfloat16, device="cuda")
    wide_g[:, 1:38, 3:] = g.cuda()
    wide_x[:, 1:, 3:] = x.cuda()
    got = ssa.linear_grad(wide_g[:, 1:38, 3:], wide_x[:, 1:, 3:], w.cuda())
    want = ssa.linear_grad(g.cuda(), x.cuda(), w.cuda())
    for a, c in zip(got, want):
        assert torch.equal(a, c)
    part = ssa.linear_grad(g.cuda(), x.cuda(), w.cuda(), need_x=False, need_bias=False)
    assert part.x is None and part.bias is None and torch.equal(part.weight, want.weight)
    part = ssa.linear_grad(g.cuda(), x.cuda(), w.cuda(), need_weight=False, need_bias=False)
    assert torch.equal(part.x, want.x)
    part = ssa.linear_grad(g.cuda(), x.cuda(), w.cuda(), need_weight=False, need_x=False)
    assert torch.equal(part.bias, want.bias)
    # a gradient that is the same for every position, as a sum's is
    one = torch.randn((1, 1, 40), generator=gen(1)).bfloat16().cuda()
    got = ssa.linear_grad(one.expand(2, 37, 40), x.cuda(), w.cuda())
    want = ssa.linear_grad(one.expand(2, 37, 40).contiguous(), x.cuda(), w.cuda())
    for a, c in zip(got, want):
        assert torch.equal(a, c)


def check_grad_rounded_once(got, want, size, gsize, n, N, w, x, dtype):
    """dz counts with 2^-16 (bf16: two roundings of 2^-8) or 2^-22 (fp16: of 2^-11) of its size, after about 16 roundings
    of values up to |g|; the products sum two parts of it, and the result alone is rounded to 16 bits.  fp16 has steps of
    2^-24 at the least: what both parts leave of a value of dz is half of one."""
    keeps = {torch.bfloat16: 2.0 ** -16, torch.float16: 2.0 ** -22, torch.float32: 0.0}[dtype]
    floor = 2.0 ** -25 if dtype == torch.float16 else 0.0
    lost = (floor * w.double().abs().sum(0), floor * x.double().abs().reshape(-1, x.shape[-1]).sum(0), 0.0)
    for i, (k, terms) in enumerate((("x", N), ("weight", n), ("bias", n))):
        tol = (U * (2 * terms + 8) + keeps) * size[i] * 1.0001 + 24 * U * gsize[i] + lost[i] + HALF[dtype] * want[i].abs() * 1.0001 + SMALLEST[dtype]
        close("gradient of " + k, getattr(got, k), want[i].cpu(), tol.cpu())


@pytest.mark.parametrize("dtype", TYPES, ids=ids_of)
@pytest.mark.parametrize("lead,K,N,planes", [((1,), 1, 1, False), ((70,), 72, 130, False), ((300,), 96, 65, False), ((515,), 264, 136, False),
                                             ((1,), 515, 400, False), ((2, 16, 20), 256, 40, True), ((2, 513), 130, 21, True), ((3, 1), 8, 1, True)])
def test_linear_grad_is_rounded_once(lead, K, N, planes, dtype):
    """A gradient in float32, and one that an activation's slope multiplies, reach the products unrounded."""
    for act, out in ((None, torch.float32), ("gelu", dtype), ("relu", dtype), ("silu", torch.float32)):
        x, w, _, g = make_linear(lead, K, N, dtype, out, K + N, planes=planes)
        pre = (torch.randn(g.shape, generator=gen(K)) * 1.5).to(dtype) if act else None
        got = ssa.linear_grad(g.cuda(), x.cuda(), w.cuda(), activation=act, pre=None if pre is None else pre.cuda(), planes=planes)
        want, size, gsize = plain_linear_grad(g, x, w, act, pre, planes)
        check_grad_rounded_once(got, want, size, gsize, x[..., 0].numel(), N, w, x, dtype)


@pytest.mark.parametrize("dtype", TYPES, ids=ids_of)
@pytest.mark.parametrize("B,n,K,N,planes", [(1, 8190, 1000, 4088, False), (2, 701, 1001, 603, False), (3, 701, 1001, 603, True),
                                            (2, 3000, 512, 520, False), (2, 20000, 64, 40, True)])
def test_large_linear_grad_is_rounded_once(B, n, K, N, planes, dtype):
    """The largest tiles, split sums, copied operands and batches that do not merge, against 64-bit products."""
    g = torch.Generator(device="cuda").manual_seed(K)
    x = torch.full((B, n + 1, K), math.nan, device="cuda", dtype=dtype)[:, :n]
    x.copy_(torch.randn((B, n, K), device="cuda", generator=g))
    w = (torch.randn((N, K), device="cuda", generator=g) / math.sqrt(K)).to(dtype)
    dy = torch.randn((B, N, n) if planes else (B, n, N), device="cuda", generator=g).to(dtype)
    pre = (torch.randn(dy.shape, device="cuda", generator=g) * 1.5).to(dtype)
    got = ssa.linear_grad(dy, x, w, activation="silu", pre=pre, planes=planes)
    want, size, gsize = plain_linear_grad(dy, x, w, "silu", pre, planes)
    check_grad_rounded_once(got, want, size, gsize, B * n, N, w, x, dtype)


@pytest.mark.parametrize("planes", [False, True])
@pytest.mark.parametrize("size,scale", [(1e-12, 6e4), (1e-9, 3e4), (3e-7, 500.0), (1e-3, 1.0), (3e4, 1e-3), (1e7, 1e-4), (1e8, 1e-5)])
def test_linear_grad_of_float16_holds_any_float32_gradient(size, scale, planes):
    """Gradients far below and above what fp16 holds, into results that it does hold; an activation's slope on top."""
    B, n, K, N = 2, 150, 72, 64
    for act in (None, "gelu"):
        x, w, _, g = make_linear((B, n), K, N, torch.float16, torch.float32, 3, planes=planes)
        x, w, g = (x.float() * scale / 8).half(), (w.float() * scale).half(), g * size
        pre = (torch.randn(g.shape, generator=gen(K)) * 1.5).half() if act else None
        got = ssa.linear_grad(g.cuda(), x.cuda(), w.cuda(), activation=act, pre=None if pre is None else pre.cuda(), planes=planes)
        want, mag, gsize = plain_linear_grad(g, x, w, act, pre, planes)
        peak = float(g.abs().max())
        lost = (w.double().abs().sum(0), x.double().abs().reshape(-1, K).sum(0))
        for i, (k, terms) in enumerate((("x", N), ("weight", B * n))):
            # two roundings of 2^-11, sums of two parts, the slope's 16 roundings, 2^-38 of the peak a value, the result
            tol = (U * (2 * terms + 8) + 2.0 ** -22) * mag[i] * 1.0001 + 24 * U * gsize[i] + 2.0 ** -38 * peak * lost[i] + HALF[torch.float16] * want[i].abs() * 1.0001 + 2.0 ** -25
            close("gradient of " + k, getattr(got, k), want[i], tol)
            assert float(getattr(got, k).abs().max()) > 0


@pytest.mark.parametrize("planes", [False, True])
def test_linear_grad_of_float16_scales_by_finite_values(planes):
    """Infinities and NaN of a gradient stay in their positions and leave the scale alone; zeros stay zeros."""
    B, n, K, N = 2, 40, 24, 16
    x, w, _, g = make_linear((B, n), K, N, torch.float16, torch.float32, 4, planes=planes)
    w = w.abs() + 0.01
    g = g * 1e-6
    clean = ssa.linear_grad(g.cuda(), x.cuda(), w.cuda(), planes=planes, need_weight=False)
    bad = g.clone()
    at = (lambda e, r, o: (e, o, r)) if planes else (lambda e, r, o: (e, r, o))
    bad[at(0, 3, 5)], bad[at(1, 7, 2)] = math.inf, math.nan
    got = ssa.linear_grad(bad.cuda(), x.cuda(), w.cuda(), planes=planes)
    assert (got.x[0, 3] == math.inf).all() and torch.isnan(got.x[1, 7]).all()
    keep = torch.ones((B, n), dtype=torch.bool)
    keep[0, 3] = keep[1, 7] = False
    assert float(clean.x.abs().max()) > 0 and torch.equal(got.x.cpu()[keep], clean.x.cpu()[keep])
    others = [o for o in range(N) if o not in (2, 5)]
    assert torch.isfinite(got.weight[others]).all() and torch.isfinite(got.bias[others]).all()
    for t in ssa.linear_grad(torch.zeros_like(g).cuda(), x.cuda(), w.cuda(), planes=planes):
        assert not t.any()


@pytest.mark.parametrize("dtype", TYPES, ids=ids_of)
@pytest.mark.parametrize("K,N,n", [(65, 3, 40), (512, 512, 8191), (513, 70, 33000)])
def test_linear_of_sliding_windows(K, N, n, dtype):
    """Rows that overlap, one element on from each other, have a stride of 1 along both axes: features x and
    weights, forward and backward, below and above the size from which operands are copied."""
    g = torch.Generator(device="cuda").manual_seed(K)
    x = torch.randn(n + K - 1, device="cuda", generator=g).to(dtype).unfold(0, K, 1)
    dense = (torch.randn((N, K), device="cuda", generator=g) / math.sqrt(K)).to(dtype)
    slid = (torch.randn(N + K - 1, device="cuda", generator=g) / math.sqrt(K)).to(dtype).unfold(0, K, 1)
    assert x.stride() == (1, 1) and slid.stride() == (1, 1)
    dy = torch.randn((n, N), device="cuda", generator=g).to(dtype)
    d, xd = dy.double(), x.double()
    for w in (dense, slid):
        wd = w.double()
        tol = lambda want, size, terms: (U * (terms + 8) * size * 1.0001 + HALF[dtype] * want.abs() * 1.0001 + SMALLEST[dtype]).cpu()  # noqa: E731
        for planes in (False, True):
            move = (lambda t: t.t()[None].contiguous()) if planes else (lambda t: t)
            feat = x[None] if planes else x
            want, size = move(xd @ wd.t()), move(xd.abs() @ wd.abs().t())
            close("y", ssa.linear(feat, w, planes=planes), want.cpu(), tol(want, size, K))
            got = ssa.linear_grad(move(dy), feat, w, planes=planes)
            want, size = d @ wd, d.abs() @ wd.abs()
            close("gradient of x", got.x.view(n, K), want.cpu(), tol(want, size, N))
            want, size = d.t() @ xd, d.abs().t() @ xd.abs()
            close("gradient of weight", got.weight, want.cpu(), tol(want, size, n))


def test_linear_grad_of_a_single_class_whose_weight_is_a_turned_column():
    """[1, D] made by .t() is contiguous and has strides (1, 1).  One product a result: one rounding of it, in a
    product large enough that out of line operands are copied."""
    E, n, D = 4, 1 << 20, 256
    w = torch.randn((D, 1), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).bfloat16().t()
    assert w.is_contiguous() and w.stride() == (1, 1)
    x = torch.zeros((E, n, D), dtype=torch.bfloat16, device="cuda")
    dy = torch.randn((E, 1, n), device="cuda", generator=torch.Generator(device="cuda").manual_seed(2)).bfloat16()
    got = ssa.linear_grad(dy, x, w, planes=True, need_weight=False, need_bias=False)
    assert torch.equal(got.x, dy.transpose(1, 2) * w)
    x = x[:1].float()
    dy = dy[:1].float()
    got = ssa.linear_grad(dy, x, w.float(), planes=True, need_weight=False, need_bias=False)
    assert torch.equal(got.x, dy.transpose(1, 2) * w.float())


@pytest.mark.parametrize("act", ACTS[1:])
@pytest.mark.parametrize("dtype", TYPES, ids=ids_of)
def test_slope_where_pre_is_infinite(dtype, act):
    """fp16 keeps a value beyond 65504 as infinity for the backward pass, beside a finite float32 result: its slope is
    the limit, 1 or 0.  NaN stays NaN where the slope is computed from the value."""
    big = {torch.float16: 300.0, torch.bfloat16: 1e4, torch.float32: 1e4}[dtype]
    x = torch.tensor([[big, 1.0], [-big, 1.0], [0.5, 0.25]], dtype=dtype, device="cuda")
    w = torch.tensor([[big, 0.0], [0.0, 1.0]], dtype=dtype, device="cuda")
    y, pre = ssa.linear(x, w, activation=act, out_dtype=torch.float32, keep_pre=True)
    assert torch.isfinite(y).all() and (dtype != torch.float16 or torch.isinf(pre[:2, 0]).all())
    if dtype != torch.float16:
        pre[0, 0], pre[1, 0] = math.inf, -math.inf
    g = torch.tensor([[2.0, 0.0]] * 3, device="cuda")
    got = ssa.linear_grad(g, x, w, activation=act, pre=pre)
    assert got.x[0].tolist() == [2 * float(w[0, 0]), 0.0] and got.x[1].tolist() == [0.0, 0.0]
    assert torch.isfinite(got.x).all() and torch.isfinite(got.weight).all() and torch.isfinite(got.bias).all()
    pre[2, 0] = math.nan
    if act != "relu":
        assert torch.isnan(ssa.linear_grad(g, x, w, activation=act, pre=pre).x[2, 0])


def test_linear_grad_of_no_frames():
    for dtype in TYPES:
        w = torch.ones((4, 8), dtype=dtype, device="cuda")
        for act in (None, "silu"):
            dy = torch.zeros((0, 4, 9), dtype=torch.float32 if act is None else dtype, device="cuda")
            g = ssa.linear_grad(dy, torch.zeros((0, 9, 8), dtype=dtype, device="cuda"), w, activation=act, pre=dy.to(dtype) if act else None, planes=True)
            assert g.x.shape == (0, 9, 8) and not g.weight.any() and not g.bias.any() and g.weight.shape == (4, 8)
            dy = dy.new_zeros((0, 9, 4))
            g = ssa.linear_grad(dy, torch.zeros((0, 9, 8), dtype=dtype, device="cuda"), w, activation=act, pre=dy.to(dtype) if act else None)
            assert g.x.shape == (0, 9, 8) and not g.weight.any() and not g.bias.any()


@pytest.mark.parametrize("dtype", TYPES, ids=ids_of)
@pytest.mark.parametrize("n", [(1 << 21) + 3, (1 << 21) + 8])
def test_linear_grad_of_planes_past_the_direct_loads(n, dtype):
    """Planes of more than 2^21 positions, whose lines are too far apart for 32-bit offsets within a tile: loads
    through registers, dz in parts, two frames in the weight's sum."""
    E, K, N = 2, 8, 5
    g = torch.Generator(device="cuda").manual_seed(n)
    x = torch.randn((E, n, K), device="cuda", generator=g).to(dtype)
    w = (torch.randn((N, K), device="cuda", generator=g) / 4).to(dtype)
    dy = torch.randn((E, N, n), device="cuda", generator=g).to(dtype)
    pre = (torch.randn(dy.shape, device="cuda", generator=g) * 1.5).to(dtype)
    for act in (None, "silu"):
        got = ssa.linear_grad(dy, x, w, activation=act, pre=pre if act else None, planes=True)
        want, size, gsize = plain_linear_grad(dy, x, w, act, pre if act else None, True)
        check_grad_rounded_once(got, want, size, gsize, E * n, N, w, x, dtype)


@pytest.mark.parametrize("dtype", TYPES, ids=ids_of)
@pytest.mark.parametrize("planes", [False, True])
def test_linear_grad_of_expanded_operands(planes, dtype):
    """One frame's features, gradients and weights standing for several: strides of 0 along batch, rows and outputs."""
    B, n, K, N = 3, 300, 72, 70
    g = torch.Generator(device="cuda").manual_seed(6)
    x = torch.randn((1, n, K), device="cuda", generator=g).to(dtype).expand(B, n, K)
    w = (torch.randn((1, K), device="cuda", generator=g) / 8).to(dtype).expand(N, K)
    dy = torch.randn((1, N, n) if planes else (1, n, N), device="cuda", generator=g).to(dtype)
    dy = dy.expand((B,) + dy.shape[1:])
    pre = (torch.randn(dy.shape, device="cuda", generator=g) * 1.5).to(dtype)
    assert torch.equal(ssa.linear(x, w, planes=planes), ssa.linear(x.contiguous(), w.contiguous(), planes=planes))
    for act in (None, "gelu"):
        got = ssa.linear_grad(dy, x, w, activation=act, pre=pre if act else None, planes=planes)
        want, size, gsize = plain_linear_grad(dy, x, w, act, pre if act else None, planes)
        check_grad_rounded_once(got, want, size, gsize, B * n, N, w, x, dtype)


# ------------------------------------------------------------------ together, streams, graphs, the engine

def test_a_training_step_of_a_head():
    """features -> class planes -> log probabilities and entropy -> gradients, against autograd in 64 bits."""
    E, h, w_, D, C_, T = 2, 9, 14, 64, 40, 2.5
    g = gen(0)
    feat = torch.randn((E, h, w_, D), generator=g)
    wt, b = torch.randn((C_, D), generator=g) * 0.3, torch.randn(C_, generator=g)
    ids = torch.randint(0, C_, (E, h, w_), generator=g)
    ids[:, 0] = -100
    logits = ssa.linear(feat.cuda(), wt.cuda(), b.cuda(), planes=True)
    s = ssa.log_probs(logits, ids.cuda(), dim=1, temperature=T, top=2)
    g_l, g_e = torch.full((1, 1, 1), -0.5, device="cuda").expand(E, h, w_), torch.full((E, h, w_), 0.1, device="cuda")
    gl = ssa.log_probs_grad(logits, ids.cuda(), s, dim=1, temperature=T, grad_log_prob=g_l, grad_entropy=g_e)
    got = ssa.linear_grad(gl, feat.cuda(), wt.cuda(), planes=True)
    fd, wd, bd = (t.double().requires_grad_(True) for t in (feat, wt, b))
    lp = ((fd @ wd.t() + bd) / T).log_softmax(-1)
    picked = lp.gather(-1, ids.clamp(min=0)[..., None])[..., 0]
    loss = -0.5 * picked[ids >= 0].sum() + 0.1 * -(lp.exp() * lp).sum()
    want = torch.autograd.grad(loss, (fd, wd, bd))
    for a, c in zip(got, want):
        # float32 all the way: a few hundred roundings of values of the size of the largest gradient
        assert float((a.cpu().double() - c).abs().max()) < 1000 * U * float(c.abs().max())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=ids_of)
def test_engine_step_from_features(dtype):
    """step(features=...) is step(logits=linear(features)) with the same maps, bit for bit."""
    from tests import scenes
    E, h, w_, D, C_ = 2, 60, 80, 32, 8
    bounds = np.array([0.0, -0.2, 0.0, 4.5, 2.5, 4.5])
    g = gen(3)
    weight, bias = (torch.randn((C_, D), generator=g)).to(dtype).cuda(), torch.randn(C_, generator=g).cuda()
    engines = []
    for _ in range(2):
        eng = ssa.MapEngine(E, (h, w_), num_semantic_classes=9, depth_hfov=59.0, depth_range=(0.5, 5.0), probablistic_mapping=True,
                            prob_aggregate="height_map_avg_prob", seg_model_n_classes=C_, max_map_hw=ssa.map_size(bounds, 0.03))
        eng.set_schema(scenes.small_lut(C_))
        for e in range(E):
            eng.reset_env(e, bounds)
        engines.append(eng)
    with pytest.raises(RuntimeError, match="set_head"):
        engines[0].head_logits(torch.zeros((E, h, w_, D), dtype=dtype, device="cuda"))
    engines[0].set_head(torch.nn.Parameter(weight), bias)      # a module's own weight: the engine records nothing
    rng = np.random.default_rng(0)
    for i in range(2):
        frames = []
        for e in range(E):
            a, c = scenes.make_pose(1.2 + 0.2 * e, 0.0, 1.0 + 0.25 * i, np.pi + 0.75 + 0.1 * e)
            frames.append((scenes.room_frame(rng, h, w_, C_, 1.0, c, lut=scenes.small_lut(C_)), a, c))
        ag, cam = np.stack([f[1] for f in frames]), np.stack([f[2] for f in frames])
        depth = torch.from_numpy(np.stack([f[0]["depth"] for f in frames]).astype(np.float32).reshape(E, h, w_))
        gt = torch.from_numpy(np.stack([f[0]["semantic_gt"] for f in frames]).astype(np.int32).reshape(E, h, w_)).cuda()
        feat = torch.randn((E, h, w_, D), generator=g).to(dtype).cuda()
        logits = ssa.linear(feat, weight, bias, planes=True, out_dtype=torch.float32)
        engines[0].step(depth.cuda(), ag, cam, [3] * E, features=feat, temperature=2.0, semantic_gt=gt)
        engines[1].step(depth.cuda(), ag, cam, [3] * E, logits=logits, temperature=2.0, semantic_gt=gt)
        assert engines[0].results()[2].min() > 50
        with pytest.raises(ValueError, match="as well"):
            engines[0].step(depth.cuda(), ag, cam, [3] * E, features=feat, logits=logits)
    with pytest.raises(ValueError, match="features: expected"):
        engines[0].head_logits(feat[:, :-1])
    engines[1].results()
    for e in range(E):
        for k, t in engines[0].maps[e].items():
            assert torch.equal(t, engines[1].maps[e][k]), (e, k)
    for eng in engines:
        eng.close()


def _step_inputs(seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn((70, 96), device="cuda", generator=g).bfloat16()
    w = torch.randn((2500, 96), device="cuda", generator=g).bfloat16() * 0.2
    b = torch.randn((2500,), device="cuda", generator=g)
    ids = torch.randint(0, 2500, (70,), device="cuda", generator=g)
    return x, w, b, ids


def _step(x, w, b, ids):
    y, pre = ssa.linear(x, w, b, activation="gelu", out_dtype=torch.float32, keep_pre=True)
    s = ssa.log_probs(y, ids, top=5, temperature=0.9)
    gl = ssa.log_probs_grad(y, ids, s, temperature=0.9, grad_log_prob=torch.full_like(s.log_prob, -1.0), grad_entropy=torch.full_like(s.entropy, 0.1),
                            grad_top=torch.full_like(s.top_log_prob, 0.2))
    return (y,) + tuple(s) + (gl,) + tuple(ssa.linear_grad(gl, x, w, activation="gelu", pre=pre))


def test_two_graphs_replayed_in_turn():
    """A forward and backward pass captured twice, replayed alternately with eager work between, against
    the eager results for every set of inputs."""
    stills, graphs = [_step_inputs(1), _step_inputs(2)], []
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _step(*stills[0])
    torch.cuda.current_stream().wait_stream(side)
    outs = []
    for s in stills:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(_step(*s))
        graphs.append(graph)
    for turn in range(4):
        fresh = [_step_inputs(10 + 2 * turn + k) for k in range(2)]
        wants = [[t.clone() for t in _step(*f)] for f in fresh]
        for k in range(2):
            for a, f in zip(stills[k], fresh[k]):
                a.copy_(f)
        for k in (0, 1, 0):
            graphs[k].replay()
        torch.cuda.synchronize()
        for k in range(2):
            for a, want in zip(outs[k], wants[k]):
                assert torch.equal(a, want), (turn, k)


def test_two_streams_at_once():
    ins = [_step_inputs(5), _step_inputs(6)]
    wants = [[t.clone() for t in _step(*i)] for i in ins]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(5):
        for k in range(2):
            with torch.cuda.stream(streams[k]):
                got[k].append(_step(*ins[k]))
    torch.cuda.synchronize()
    for k in range(2):
        for run in got[k]:
            for a, want in zip(run, wants[k]):
                assert torch.equal(a, want)


def _head_step(x, w, b, ids):
    y, pre = ssa.linear(x, w, b, activation="gelu", planes=True, out_dtype=torch.float32, keep_pre=True)
    s = ssa.log_probs(y, ids, dim=1, top=2)
    gl = ssa.log_probs_grad(y, ids, s, dim=1, grad_log_prob=torch.full_like(s.log_prob, -1e-7), grad_top=torch.full_like(s.top_log_prob, 1e-8))
    return (y,) + tuple(s) + (gl,) + tuple(ssa.linear_grad(gl, x, w, activation="gelu", pre=pre, planes=True))


def _head_inputs(seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn((2, 600, 96), device="cuda", generator=g).half()
    w = torch.randn((21, 96), device="cuda", generator=g).half() * 0.2
    return x, w, torch.randn((21,), device="cuda", generator=g), torch.randint(0, 21, (2, 600), device="cuda", generator=g)


def test_a_float16_head_in_two_graphs_and_streams():
    """The gradient's scale comes from each call's own values: two graphs replayed in turn with eager work between
    them, and two streams at once, against eager results."""
    stills, graphs, outs = [_head_inputs(1), _head_inputs(2)], [], []
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _head_step(*stills[0])
    torch.cuda.current_stream().wait_stream(side)
    for s in stills:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(_head_step(*s))
        graphs.append(graph)
    for turn in range(4):
        fresh = [_head_inputs(10 + 2 * turn + k) for k in range(2)]
        fresh[1][1].mul_(3.0 ** turn)
        wants = [[t.clone() for t in _head_step(*f)] for f in fresh]
        for k in range(2):
            for a, f in zip(stills[k], fresh[k]):
                a.copy_(f)
        for k in (0, 1, 0):
            graphs[k].replay()
        torch.cuda.synchronize()
        for k in range(2):
            for a, want in zip(outs[k], wants[k]):
                assert torch.equal(a, want), (turn, k)
        assert wants[0][-2].any()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for _ in range(5):
        for k in range(2):
            with torch.cuda.stream(streams[k]):
                got[k].append(_head_step(*fresh[k]))
    torch.cuda.synchronize()
    for k in range(2):
        for run in got[k]:
            for a, want in zip(run, wants[k]):
                assert torch.equal(a, want)


def test_recorded_tensors_are_refused():
    x = torch.zeros((3, 5), device="cuda", requires_grad=True)
    ids = torch.zeros(3, dtype=torch.int64, device="cuda")
    with pytest.raises(RuntimeError, match="log_probs_grad"):
        ssa.log_probs(x, ids)
    with pytest.raises(RuntimeError, match="linear_grad"):
        ssa.linear(x, torch.zeros((4, 5), device="cuda"))
    with torch.no_grad():
        assert ssa.log_probs(x, ids).log_prob.shape == (3,)
    with pytest.raises(ValueError, match="ids: expected a tensor on cuda"):
        ssa.log_probs(x.detach(), ids.cpu())
    with pytest.raises(ssa._capi.EngineError, match="temperature"):
        ssa.log_probs(x.detach(), ids, temperature=0.0)


def test_tensors_with_a_tangent_are_refused():
    """Forward mode would lose the derivative without a word, under no_grad as well."""
    from torch.autograd import forward_ad
    x, w = torch.randn((3, 5), device="cuda"), torch.randn((4, 5), device="cuda")
    ids, y = torch.zeros(3, dtype=torch.int64, device="cuda"), torch.randn((3, 4), device="cuda")
    s = ssa.log_probs(x, ids)
    with forward_ad.dual_level(), torch.no_grad():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        for name, call in (("logits", lambda t: ssa.log_probs(t, ids)), ("logits", lambda t: ssa.log_probs_grad(t, ids, s)),
                           ("x", lambda t: ssa.linear(t, w)), ("x", lambda t: ssa.linear_grad(y, t, w))):
            with pytest.raises(RuntimeError, match=name + " carries a tangent"):
                call(dual)
            call(x)
        with pytest.raises(RuntimeError, match="residual carries a tangent"):
            ssa.linear(x, w, residual=forward_ad.make_dual(y, torch.ones_like(y)))


def test_views_that_negate_are_refused():
    """As the imaginary part of a lazy conjugate is one: memory holds the opposite of its values."""
    neg = torch._neg_view(torch.randn((3, 4), device="cuda"))
    assert neg.is_neg() and torch.randn((3, 8), device="cuda").view(torch.complex64).conj().imag[:, :1].is_neg()
    x, w, ids = torch.ones((3, 5), device="cuda"), torch.ones((4, 5), device="cuda"), torch.zeros(3, dtype=torch.int64, device="cuda")
    for name, call in (("logits", lambda t: ssa.log_probs(t, ids)), ("grad_top", lambda t: ssa.log_probs_grad(w.t()[:3].contiguous(), ids, s, grad_top=t)),
                       ("x", lambda t: ssa.linear(t, w[:, :4])), ("residual", lambda t: ssa.linear(x, w, residual=t)),
                       ("grad", lambda t: ssa.linear_grad(t, x, w))):
        s = ssa.log_probs(torch.ones((3, 4), device="cuda"), ids, top=4)
        with pytest.raises(ValueError, match=name + " is a view that negates"):
            call(neg)
        call(neg.resolve_neg())
