"""Cases of the framework's head operators: the log probabilities of given ids with entropy and top
alternatives, their gradient, the matrix product with a fused epilogue, and its gradients.

Two layouts run through all of them.  "rows": the classes (a vocabulary) lie last, as a language model
leaves its logits.  "planes": one plane per class, [envs, classes, height, width], as a segmentation head
leaves them and as the map engine reads them.
"""
import math

import torch

own = False
DEVICE = "cuda"

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
IGNORE = -100


def listed():
    return [
        # four sequences each want the log probability of their next token and 20 alternatives: latency
        dict(name="scores of 4 tokens", op="log_probs", layout="rows", batch=4, rows=1, vocab=131072, type="bf16",
             top=20, temperature=0.8),
        # scoring prompts: logits of positions 0..T-2 against tokens 1..T-1 (a view of a longer tensor), odd vocabulary
        dict(name="scores of prompts", op="log_probs", layout="rows", batch=4, rows=1024, vocab=32003, type="f16",
             top=5, temperature=1.0),
        # one row per token of a transformer's segmentation head with 150 classes
        dict(name="scores of head tokens", op="log_probs", layout="rows", batch=4, rows=16384, vocab=150, type="f32",
             top=2, temperature=2.5),
        # the engine's own frames: 16 envs, 640x480, 40 classes, T = 3.2, label likelihoods and three candidates
        dict(name="scores of frames", op="log_probs", layout="planes", batch=16, rows=480 * 640, vocab=40, type="f32",
             top=3, temperature=3.2),
        # a training step's loss gradient over a large vocabulary, with an entropy bonus
        dict(name="gradient of tokens", op="log_probs_grad", layout="rows", batch=8, rows=512, vocab=131072, type="bf16",
             top=0, temperature=1.0),
        # fine-tuning on frames of the 150-class head, with a term on the two best classes
        dict(name="gradient of frames", op="log_probs_grad", layout="planes", batch=4, rows=480 * 640, vocab=150,
             type="f32", top=2, temperature=2.5),
        # single tokens of three sequences through one layer: the weight is read once, nothing else counts
        dict(name="layer of 3 tokens", op="linear", layout="rows", batch=1, rows=3, inner=4096, outer=4096, type="bf16",
             out="bf16", act="silu", bias=True, residual=True),
        # a prompt or training batch through one layer with everything in the epilogue
        dict(name="layer of a batch", op="linear", layout="rows", batch=4, rows=2048, inner=4096, outer=8192, type="bf16",
             out="bf16", act="gelu", bias=True, residual=True),
        # a segmentation head: 256 features of every pixel of 4 frames to 40 class planes for the map engine
        dict(name="head of frames", op="linear", layout="planes", batch=4, rows=480 * 640, inner=256, outer=40,
             type="bf16", out="f32", act="none", bias=True, residual=False),
        # float32 with sizes that no tile divides
        dict(name="layer in float32", op="linear", layout="rows", batch=1, rows=1003, inner=515, outer=1501, type="f32",
             out="f32", act="relu", bias=True, residual=False),
        # the backward pass of a training batch's layer
        dict(name="gradients of a batch", op="linear_grad", layout="rows", batch=4, rows=2048, inner=4096, outer=4096,
             type="bf16", out="bf16", act="gelu", bias=True),
        # the backward pass of the 40-class head on one frame: plane gradients in float32, features in 16 bits
        dict(name="gradients of a head", op="linear_grad", layout="planes", batch=1, rows=480 * 640, inner=256, outer=40,
             type="f16", out="f32", act="none", bias=True),
    ]


def draw(rng):
    def spread(lo, hi):
        return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    op = rng.choice(["log_probs", "log_probs_grad", "linear", "linear_grad"])
    kind = rng.choice(["f32", "bf16", "f16"])
    if op.startswith("log_probs"):
        if rng.random() < 0.6:
            vocab = spread(8, 262144)
            rows = spread(1, max(1, min(65536, (1 << 27) // vocab)))
            batch = rng.choice([1, 2, 5])
            case = dict(op=op, layout="rows", batch=batch, rows=max(1, rows // batch), vocab=vocab)
        else:
            vocab = spread(2, 155)
            rows = spread(1, 480) * spread(1, 640)
            case = dict(op=op, layout="planes", batch=spread(1, max(1, min(16, (1 << 27) // (vocab * rows)))), rows=rows,
                        vocab=vocab)
        return dict(case, type=kind, top=min(rng.choice([0, 1, 2, 5, 20]), case["vocab"]),
                    temperature=rng.choice([0.7, 1.0, 2.5, 3.2]))
    inner, outer = spread(16, 8192), spread(2, 8192)
    most = (1 << 36) if kind == "f32" else (1 << 37)   # products of one pass
    if rng.random() < 0.75:
        rows = spread(1, max(1, min(65536, most // (inner * outer))))
        batch = rng.choice([1, 1, 2, 3])
        case = dict(op=op, layout="rows", batch=batch, rows=max(1, rows // batch), inner=inner, outer=outer)
    else:
        inner, outer = spread(16, 512), spread(2, 155)
        case = dict(op=op, layout="planes", batch=rng.choice([1, 2, 3]), rows=spread(1, 480) * spread(1, 640), inner=inner,
                    outer=outer)
    case = dict(case, type=kind, out=rng.choice([kind, "f32"]), act=rng.choice(["none", "relu", "gelu", "gelu_tanh", "silu"]),
                bias=rng.random() < 0.7)
    return dict(case, residual=rng.random() < 0.4) if op == "linear" else case


def _logits(case, g):
    """Logits of a trained model: a few classes stand out, some of a vocabulary are masked to -inf."""
    B, R, V, t = case["batch"], case["rows"], case["vocab"], TYPES[case["type"]]
    if case["layout"] == "planes":
        x = torch.randn((B, V, R), device=DEVICE, generator=g).mul_(3.0).to(t)
        ids = torch.randint(0, V, (B, R), device=DEVICE, generator=g)
        ids = torch.where(torch.rand((B, R), device=DEVICE, generator=g) < 0.02, IGNORE, ids).to(torch.int32)
        return x, ids
    whole = torch.randn((B, R + 1, V), device=DEVICE, generator=g, dtype=torch.float32 if case["type"] == "f32" else t)
    whole.mul_(2.5)
    if V >= 64:
        whole[:, :, torch.randint(0, V, (max(1, V // 512),), device=DEVICE, generator=g)] += 6.0
        whole[:, :, V - V // 64:] = -math.inf
    ids = torch.randint(0, V - V // 64, (B, R + 1), device=DEVICE, generator=g)
    ids = torch.where(torch.rand((B, R + 1), device=DEVICE, generator=g) < 0.05, IGNORE, ids)
    return whole, ids


def _parts(s):
    """The logits and ids that an operator is called with: positions 0..T-1 against tokens 1..T in rows."""
    return (s["x"], s["ids"]) if s["case"]["layout"] == "planes" else (s["x"][:, :-1], s["ids"][:, 1:])


def _dim(case):
    return 1 if case["layout"] == "planes" else -1


def prepare(case, seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(int(seed))
    s = {"case": dict(case)}
    B, R, t = case["batch"], case["rows"], TYPES[case["type"]]
    if case["op"].startswith("log_probs"):
        s["x"], s["ids"] = _logits(case, g)
        if case["op"] == "log_probs":
            return s
        x, ids = _parts(s)
        d, T, k = _dim(case), case["temperature"], case["top"]
        # what the forward pass left: its statistics and alternatives
        s["scores"] = _scores(x, ids, d, T, k)
        s["g_log_prob"] = torch.randn(ids.shape, device=DEVICE, generator=g) * 0.1 - 1.0
        s["g_entropy"] = torch.randn(ids.shape, device=DEVICE, generator=g) * 0.01
        s["g_top"] = torch.randn(s["scores"]["top_ids"].shape, device=DEVICE, generator=g) * 0.1 if k else None
        return s
    K, N, out = case["inner"], case["outer"], TYPES[case["out"]]
    planes = case["layout"] == "planes"
    y_shape = (B, N, R) if planes else (B, R, N)
    s["x"] = torch.randn((B, R, K), device=DEVICE, generator=g).to(t)
    s["w"] = (torch.randn((N, K), device=DEVICE, generator=g) / math.sqrt(K)).to(t)
    s["b"] = (torch.randn((N,), device=DEVICE, generator=g) * 0.5).to(t) if case["bias"] else None
    if case["op"] == "linear":
        s["r"] = torch.randn(y_shape, device=DEVICE, generator=g).to(out) if case["residual"] else None
        return s
    s["dy"] = torch.randn(y_shape, device=DEVICE, generator=g).to(out)
    # the forward pass's values before the activation
    s["pre"] = None if case["act"] == "none" else (torch.randn(y_shape, device=DEVICE, generator=g) * 1.1).to(t)
    return s


def _ranked(x, d):
    """Whole numbers in the order of x, largest first among equals at the lowest index."""
    bits = (x.float() + 0.0).view(torch.int32).to(torch.int64)
    bits = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits)
    shape = [1] * x.dim()
    shape[d] = x.shape[d]
    at = torch.arange(x.shape[d] - 1, -1, -1, device=x.device, dtype=torch.int64).view(shape)
    return bits * (1 << 32) + at


def _scores(x, ids, d, T, k):
    """Log probability of ids, entropy, and the k most probable classes along dimension d."""
    x = x.float()
    m = x.amax(d, keepdim=True)
    z = (x - m) / T
    e = z.exp()
    total = e.sum(d, keepdim=True)
    log_sum = total.log()
    entropy = log_sum - torch.where(e > 0, e * z, 0.0).sum(d, keepdim=True) / total
    at = ids.to(torch.int64).clamp(min=0).unsqueeze(d)
    given = torch.where(ids == IGNORE, 0.0, (z.gather(d, at) - log_sum).squeeze(d))
    got = {"log_prob": given, "entropy": entropy.squeeze(d), "row_max": m.squeeze(d), "log_sum": log_sum.squeeze(d)}
    shape = list(x.shape)
    shape[d] = 0
    top_ids, top = torch.zeros(shape, device=x.device, dtype=torch.int32), torch.zeros(shape, device=x.device)
    if k:
        top_ids = x.shape[d] - 1 - (_ranked(x, d).topk(k, d).values & 0xFFFFFFFF)
        top = z.gather(d, top_ids) - log_sum
        top_ids = torch.where(top == -math.inf, -1, top_ids).to(torch.int32)
    return dict(got, top_ids=top_ids, top_log_prob=top)


def _scores_grad(s, x, ids, d, T):
    f = s["scores"]
    z = (x.float() - f["row_max"].unsqueeze(d)) / T - f["log_sum"].unsqueeze(d)
    p = z.exp()
    g_l = torch.where(ids == IGNORE, 0.0, s["g_log_prob"]).unsqueeze(d)
    whole, valid = g_l, None
    if s["g_top"] is not None:
        valid = torch.where(f["top_ids"] < 0, 0.0, s["g_top"])
        whole = g_l + valid.sum(d, keepdim=True)
    z = torch.where(p > 0, z, 0.0)
    out = -p * (whole + s["g_entropy"].unsqueeze(d) * (z + f["entropy"].unsqueeze(d)))
    out.scatter_add_(d, ids.to(torch.int64).clamp(min=0).unsqueeze(d), g_l)
    if valid is not None:
        out.scatter_add_(d, f["top_ids"].to(torch.int64).clamp(min=0), valid)
    return (out / T).to(x.dtype)


def _act(z, name):
    if name == "relu":
        return torch.where(z > 0, z, 0.0)
    if name == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    if name == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z)))
    if name == "silu":
        return z / (1 + torch.exp(-z))
    return z


def _slope(z, name):
    if name == "relu":
        return torch.where(z > 0, 1.0, 0.0)
    if name == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    if name == "gelu_tanh":
        c = math.sqrt(2 / math.pi)
        t = torch.tanh(c * (z + 0.044715 * z * z * z))
        return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z)
    if name == "silu":
        q = 1 / (1 + torch.exp(-z))
        return q * (1 + z * (1 - q))
    return torch.ones_like(z)


def run(s):
    case = s["case"]
    planes = case["layout"] == "planes"
    if case["op"] == "log_probs":
        x, ids = _parts(s)
        if own:
            import semantic_search_amd as ssa
            got = ssa.log_probs(x, ids, dim=_dim(case), temperature=case["temperature"], top=case["top"], ignore_id=IGNORE)
            got = got._asdict()
        else:
            got = _scores(x, ids, _dim(case), case["temperature"], case["top"])
        return {k: got[k] for k in ("log_prob", "entropy", "top_ids", "top_log_prob")}
    if case["op"] == "log_probs_grad":
        x, ids = _parts(s)
        if own:
            import semantic_search_amd as ssa
            return ssa.log_probs_grad(x, ids, ssa.LogProbs(**s["scores"]), dim=_dim(case), temperature=case["temperature"],
                                      ignore_id=IGNORE, grad_log_prob=s["g_log_prob"], grad_entropy=s["g_entropy"],
                                      grad_top=s["g_top"])
        return _scores_grad(s, x, ids, _dim(case), case["temperature"])
    act = None if case["act"] == "none" else case["act"]
    if case["op"] == "linear":
        if own:
            import semantic_search_amd as ssa
            return ssa.linear(s["x"], s["w"], s["b"], activation=act, residual=s["r"], planes=planes,
                              out_dtype=TYPES[case["out"]])
        y = s["x"].float() @ s["w"].float().t()
        if s["b"] is not None:
            y = y + s["b"].float()
        y = _act(y, case["act"])
        if planes:
            y = y.transpose(1, 2)
        if s["r"] is not None:
            y = y + s["r"].float()
        return y.to(TYPES[case["out"]]).contiguous()
    if own:
        import semantic_search_amd as ssa
        got = ssa.linear_grad(s["dy"], s["x"], s["w"], activation=act, pre=s["pre"], planes=planes,
                              need_bias=case["bias"])
        return [t for t in got if t is not None]
    dz = s["dy"].float()
    if s["pre"] is not None:
        dz = dz * _slope(s["pre"].float(), case["act"])
    if planes:
        dz = dz.transpose(1, 2)
    dz = dz.reshape(-1, case["outer"]).contiguous()
    x = s["x"].float().reshape(-1, case["inner"])
    got = [(dz @ s["w"].float()).view(s["x"].shape).to(s["x"].dtype), (dz.t().contiguous() @ x).to(s["w"].dtype)]
    if case["bias"]:
        got.append(dz.sum(0).to(s["w"].dtype))
    return got


def work(case):
    rows = case["batch"] * case["rows"]
    b, k = SIZE[case["type"]], case.get("top", 0)
    if case["op"] == "log_probs":
        n = rows * case["vocab"]
        return {"bytes": n * b + rows * (16 + 8 * k), "flops": 5 * n}
    if case["op"] == "log_probs_grad":
        n = rows * case["vocab"]
        return {"bytes": 2 * n * b + rows * (28 + 8 * k), "flops": 6 * n}
    K, N, o = case["inner"], case["outer"], SIZE[case["out"]]
    if case["op"] == "linear":
        return {"bytes": rows * K * b + N * K * b + rows * N * o * (2 if case["residual"] else 1) + (N * b if case["bias"] else 0),
                "flops": 2 * rows * N * K}
    return {"bytes": 2 * rows * K * b + 2 * N * K * b + rows * N * (o + (0 if case["act"] == "none" else b)) +
            (N * b if case["bias"] else 0), "flops": 4 * rows * N * K}


# ---- the same from the definitions, in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    f64 = torch.float64
    if case["op"].startswith("log_probs"):
        x, ids = _parts(s)
        if case["layout"] == "planes":
            x = x.movedim(1, -1)
        V, T, k = case["vocab"], case["temperature"], case["top"]
        z = x.to(f64).reshape(-1, V) / T
        t = ids.reshape(-1).long()
        lse = torch.logsumexp(z, -1)
        logp = z - lse[:, None]
        p = logp.exp()
        plogp = torch.where(p == 0, torch.zeros((), dtype=f64, device=z.device), p * logp)
        h = -plogp.sum(-1)
        kept = t != IGNORE
        row = torch.arange(t.numel(), device=t.device)
        back = lambda v: v.reshape(ids.shape)  # noqa: E731
        if case["op"] == "log_probs":
            given = torch.zeros_like(lse)
            given[kept] = logp[row[kept], t[kept]]
            # the alternatives' values are the sorted ones whichever ids stand for equal ones
            best = logp.sort(-1, descending=True).values[:, :k]
            best = best.reshape(*ids.shape, k)
            return {"log_prob": back(given), "entropy": back(h), "top_ids": None,
                    "top_log_prob": best.movedim(-1, 1) if case["layout"] == "planes" else best}
        del z
        g_l = s["g_log_prob"].to(f64).reshape(-1) * kept
        g_h = s["g_entropy"].to(f64).reshape(-1)
        out = -g_h[:, None] * (plogp + p * h[:, None])
        # each chosen class c of a row adds g * (one at c - p)
        out -= p * g_l[:, None]
        out[row[kept], t[kept]] += g_l[kept]
        for j in range(k):
            one = s["scores"]["top_ids"].select(_dim(case), j).reshape(-1).long()
            g = s["g_top"].select(_dim(case), j).to(f64).reshape(-1)
            ok = one >= 0
            out -= p * (g * ok)[:, None]
            out[row[ok], one[ok]] += g[ok]
        out = (out / T).reshape(x.shape)
        return out.movedim(-1, 1).contiguous() if case["layout"] == "planes" else out
    w, x = s["w"].to(f64), s["x"].to(f64).flatten(0, 1)
    if case["op"] == "linear":
        z = torch.mm(x, w.t())
        if s["b"] is not None:
            z += s["b"].to(f64)
        a = case["act"]
        if a == "relu":
            z = z.clamp(min=0)
        elif a == "gelu":
            z = z * torch.erfc(-z / math.sqrt(2.0)) / 2
        elif a == "gelu_tanh":
            z = z * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))
        elif a == "silu":
            z = z * torch.sigmoid(z)
        z = z.view(case["batch"], case["rows"], -1)
        z = z.transpose(1, 2) if case["layout"] == "planes" else z
        return (z if s["r"] is None else z + s["r"].to(f64)).contiguous()
    dz = s["dy"].to(f64)
    if case["act"] != "none":
        # the activation's derivative by its definition, from autograd on the 64-bit function
        with torch.enable_grad():
            z = s["pre"].to(f64).requires_grad_(True)
            f = {"relu": lambda v: v.clamp(min=0) * (v > 0), "gelu": lambda v: v * torch.erfc(-v / math.sqrt(2.0)) / 2,
                 "gelu_tanh": lambda v: v * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3)),
                 "silu": lambda v: v * torch.sigmoid(v)}[case["act"]]
            dz = dz * torch.autograd.grad(f(z).sum(), z)[0]
    if case["layout"] == "planes":
        dz = dz.transpose(1, 2)
    dz = dz.reshape(-1, case["outer"])
    got = [torch.mm(dz, w).view(s["x"].shape), torch.mm(dz.t(), x)]
    return got + [dz.sum(0)] if case["bias"] else got
