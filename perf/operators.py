"""Measured cases of the token-model training operators: embedding lookup and its
gradient, layer norm and its backward pass, and the orthogonalised update.

Each case is one call of one operator on inputs that live on the GPU.  With `own`
False `run` computes the operator from elementary torch operations in 32 bits and
rounds once at the end; with `own` True it makes the call a user of the library makes.
`exact` evaluates the definition in 64 bits.

The operators (t a token, v a vocabulary row, r a row, j a column):

  embedding            out[t, :] = scale * table[ids[t], :], zero where ids[t] < 0 (padding)
  embedding_backward   dtable[v, :] = scale * sum over t with ids[t] == v of dout[t, :]
  layer_norm           mean[r], rstd[r] = (var[r] + eps)^-1/2,
                       y[r, j] = (x[r, j] - mean[r]) * rstd[r] * weight[j] + bias[j]
  layer_norm_backward  g = dy * weight, h = (x - mean) * rstd,
                       dx[r, :] = rstd[r] * (g - mean_j(g) - h * mean_j(g * h)),
                       dweight[j] = sum_r dy * h, dbias[j] = sum_r dy
  orthogonalize        X = G / (|G| + eps), then `steps` times
                       A = X X^T, X = a X + (b A + c A A) X   (on the shorter side of G)
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
INDEX = {32: torch.int32, 64: torch.int64}
LN_EPS = 1e-5
NS_STEPS = 5
NS_COEFFICIENTS = (3.4445, -4.7750, 2.0315)
NS_EPS = 1e-7

_context = None


def _ops():
    """The library's front end and the one context a program keeps per device and thread."""
    global _context
    from sapphire_b200 import ops
    if _context is None:
        _context = ops.Context(torch.cuda.current_device())
    return ops, _context


# ------------------------------------------------------------------------- cases

def listed():
    return [
        # the first layer of a generation step: a handful of tokens, nothing but latency
        {"name": "embedding 64 tokens", "op": "embedding", "tokens": 64, "vocab": 65536, "cols": 512,
         "table": "f32", "act": "f32", "index": 64, "padding": 0},
        # a large training batch with ragged, padded sequences, 16-bit table and activations
        {"name": "embedding 65536 tokens", "op": "embedding", "tokens": 65536, "vocab": 65536, "cols": 4096,
         "table": "bf16", "act": "bf16", "index": 64, "padding": 1},
        # a training batch of an ordinary model, 32 bits, a gradient row for every vocabulary row
        {"name": "embedding gradient 8192", "op": "embedding_backward", "tokens": 8192, "vocab": 32000, "cols": 1000,
         "table": "f32", "act": "f32", "index": 32, "padding": 0},
        # the gradient of the large batch: 16-bit activations into a 32-bit gradient
        {"name": "embedding gradient 65536", "op": "embedding_backward", "tokens": 65536, "vocab": 65536, "cols": 4096,
         "table": "f32", "act": "bf16", "index": 64, "padding": 1},
        # the batch of the MLP configuration, one launch's latency
        {"name": "layer norm 64x512", "op": "layer_norm", "rows": 64, "cols": 512, "act": "f32", "weight": "f32", "pad": 0},
        # ragged row count, a width that is no power of two, rows with a pitch (padded columns)
        {"name": "layer norm 8191x4000", "op": "layer_norm", "rows": 8191, "cols": 4000, "act": "f32", "weight": "f32", "pad": 8},
        # a large batch in 16 bits with 32-bit weights
        {"name": "layer norm 65536x4096", "op": "layer_norm", "rows": 65536, "cols": 4096, "act": "bf16", "weight": "f32", "pad": 0},
        # the backward pass of the MLP's batch
        {"name": "layer norm backward 64x512", "op": "layer_norm_backward", "rows": 64, "cols": 512, "act": "f32",
         "weight": "f32", "pad": 0},
        # the backward pass of a large batch: the column sums run over 32768 rows
        {"name": "layer norm backward 32768x4096", "op": "layer_norm_backward", "rows": 32768, "cols": 4096, "act": "f32",
         "weight": "f32", "pad": 0},
        # the first weight of the MLP configuration
        {"name": "orthogonalize 784x512", "op": "orthogonalize", "rows": 784, "cols": 512, "batch": 1, "act": "f32"},
        # the wide weights of four layers in one call, 16 bits
        {"name": "orthogonalize 4x1024x4096", "op": "orthogonalize", "rows": 1024, "cols": 4096, "batch": 4, "act": "bf16"},
        # the weight of the Linear configuration, 32 bits
        {"name": "orthogonalize 4096x4096", "op": "orthogonalize", "rows": 4096, "cols": 4096, "batch": 1, "act": "f32"},
    ]


def _spread(rng, low, high):
    """A whole number between low and high, uniform in its logarithm, odd or even as it falls."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["embedding", "embedding_backward", "layer_norm", "layer_norm_backward", "orthogonalize"])
    if op.startswith("embedding"):
        table, act = rng.choice([("f32", "f32"), ("bf16", "bf16"), ("f16", "f16"), ("f32", "bf16"), ("f32", "f16"),
                                 ("bf16", "f32"), ("f16", "f32")])
        return {"op": op, "tokens": _spread(rng, 1, 65536), "vocab": _spread(rng, 10, 65536), "cols": _spread(rng, 8, 4096),
                "table": table, "act": act, "index": rng.choice([32, 64]), "padding": rng.choice([0, 1])}
    if op.startswith("layer_norm"):
        act, weight = rng.choice([("f32", "f32"), ("bf16", "f32"), ("bf16", "bf16"), ("f16", "f32"), ("f16", "f16")])
        cols = _spread(rng, 8, 16384)
        most = 65536 * 4096 if op == "layer_norm" else 32768 * 4096
        return {"op": op, "rows": _spread(rng, 1, min(65536, most // cols)), "cols": cols, "act": act, "weight": weight,
                "pad": rng.choice([0, 0, 8, 3])}
    rows, cols = _spread(rng, 10, 4096), _spread(rng, 10, 4096)
    return {"op": op, "rows": rows, "cols": cols, "batch": rng.choice([1, 1, 2, 3, 4]) if rows * cols <= 1 << 22 else 1,
            "act": rng.choice(["f32", "bf16"])}


# ------------------------------------------------------------------------ inputs

def _normal(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32)


def _pitched(t, pad):
    """The same values with `pad` more elements from row to row (a view of a wider buffer)."""
    if not pad:
        return t
    wide = torch.zeros(t.shape[0], t.shape[1] + pad, dtype=t.dtype, device=t.device)
    wide[:, :t.shape[1]] = t
    return wide[:, :t.shape[1]]


def _tokens(gen, n, vocab, index, padding):
    """Token numbers as text has them: the k-th most frequent about 1 / k as often as the
    first (log-uniform ranks), frequent ones scattered over the vocabulary; with `padding`
    the last twentieth of every 256 positions is -1, a batch of sequences of unequal length."""
    u = torch.rand(n, generator=gen, device="cuda", dtype=torch.float64)
    rank = (torch.pow(float(vocab) + 1.0, u) - 1.0).floor().long().clamp_(0, vocab - 1)
    ids = (rank * _scatter(vocab)) % vocab
    if padding:
        at = torch.arange(n, device="cuda") % 256
        ids = torch.where(at >= 244, torch.full_like(ids, -1), ids)
    return ids.to(INDEX[index])


def _scatter(vocab):
    """A multiplier without a common factor with `vocab`: rank -> row is one to one."""
    m = max(1, int(vocab * 0.6180339887)) | 1
    while math.gcd(m, vocab) != 1:
        m += 2
    return m


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed))
    s = dict(case)
    op = case["op"]
    if op.startswith("embedding"):
        n, vocab, cols = case["tokens"], case["vocab"], case["cols"]
        s["ids"] = _tokens(gen, n, vocab, case["index"], case["padding"])
        s["scale"] = math.sqrt(cols)
        if op == "embedding":
            # small random weights; the lookup multiplies them by sqrt(cols)
            s["weights"] = (_normal(gen, vocab, cols) * 0.02).to(DTYPES[case["table"]])
        else:
            s["dout"] = (_normal(gen, n, cols) * 1e-2).to(DTYPES[case["act"]])
    elif op.startswith("layer_norm"):
        rows, cols = case["rows"], case["cols"]
        # rows of unequal size and offset, and a few channels far larger than the others
        x = _normal(gen, rows, cols) * (0.5 + torch.rand(rows, 1, generator=gen, device="cuda"))
        x += _normal(gen, rows, 1)
        x[:, ::61] *= 12.0
        s["x"] = _pitched(x.to(DTYPES[case["act"]]), case["pad"])
        s["w"] = (1.0 + 0.1 * _normal(gen, cols)).to(DTYPES[case["weight"]])
        s["b"] = (0.1 * _normal(gen, cols)).to(DTYPES[case["weight"]])
        if op == "layer_norm_backward":
            del x
            s["dy"] = _pitched((_normal(gen, rows, cols) * 1e-2).to(DTYPES[case["act"]]), case["pad"])
            xf = s["x"].double() if rows * cols <= 1 << 22 else s["x"].float()
            mean = xf.mean(1)
            var = (xf - mean[:, None]).square_().mean(1)
            s["mean"], s["rstd"] = mean.float(), (var + LN_EPS).rsqrt().float()
    else:
        rows, cols, batch = case["rows"], case["cols"], case["batch"]
        # a gradient: a few strong directions above a floor of noise
        rank = max(1, min(rows, cols) // 16)
        g = torch.bmm(_normal(gen, batch, rows, rank), _normal(gen, batch, rank, cols)) / math.sqrt(rank)
        g += 0.3 * _normal(gen, batch, rows, cols)
        g = (g * 1e-3).to(DTYPES[case["act"]])
        s["g"] = g if batch > 1 else g[0]
    return s


# --------------------------------------------------------------------- operators

def _embedding(s):
    ids = s["ids"].long()
    rows = s["weights"].index_select(0, ids.clamp_min(0)).float() * s["scale"]
    return torch.where((ids >= 0)[:, None], rows, torch.zeros((), device=rows.device)).to(DTYPES[s["act"]])


def _embedding_backward(s):
    ids = s["ids"].long()
    rows = torch.where((ids >= 0)[:, None], s["dout"].float(), torch.zeros((), device=ids.device))
    total = torch.zeros(s["vocab"], s["cols"], dtype=torch.float32, device=ids.device)
    total.index_add_(0, ids.clamp_min(0), rows)
    return (total * s["scale"]).to(DTYPES[s["table"]])


def _layer_norm(s):
    x = s["x"].float()
    mean = x.sum(1, keepdim=True) / s["cols"]
    d = x - mean
    rstd = torch.rsqrt((d * d).sum(1, keepdim=True) / s["cols"] + LN_EPS)
    y = d * rstd * s["w"].float() + s["b"].float()
    return y.to(s["x"].dtype), mean[:, 0], rstd[:, 0]


def _layer_norm_backward(s):
    dy, rstd = s["dy"].float(), s["rstd"][:, None]
    h = (s["x"].float() - s["mean"][:, None]) * rstd
    g = dy * s["w"].float()
    m1 = g.sum(1, keepdim=True) / s["cols"]
    m2 = (g * h).sum(1, keepdim=True) / s["cols"]
    dx = rstd * (g - m1 - h * m2)
    wt = s["w"].dtype
    return dx.to(s["x"].dtype), (dy * h).sum(0).to(wt), dy.sum(0).to(wt)


def _orthogonalize(s):
    a, b, c = NS_COEFFICIENTS
    g = s["g"].float()
    tall = g.shape[-2] > g.shape[-1]
    x = g.mT if tall else g
    x = x / (x.square().sum((-2, -1), keepdim=True).sqrt() + NS_EPS)
    for _ in range(NS_STEPS):
        m = x @ x.mT
        x = a * x + (b * m + c * (m @ m)) @ x
    return (x.mT if tall else x).contiguous().to(s["g"].dtype)


def run(state):
    op = state["op"]
    if own:
        ops, ctx = _ops()
        if op == "embedding":
            return ops.embedding(ctx, state["weights"], state["ids"], scale=state["scale"], out_dtype=DTYPES[state["act"]])
        if op == "embedding_backward":
            dtable = torch.empty(state["vocab"], state["cols"], dtype=DTYPES[state["table"]], device="cuda")
            return ops.embedding_backward(ctx, dtable, state["dout"], state["ids"], scale=state["scale"])
        if op == "layer_norm":
            return ops.layer_norm(ctx, state["x"], state["w"], state["b"], eps=LN_EPS)
        if op == "layer_norm_backward":
            return ops.layer_norm_backward(ctx, state["dy"], state["x"], state["mean"], state["rstd"], state["w"])
        return ops.orthogonalize(ctx, state["g"], steps=NS_STEPS, coefficients=NS_COEFFICIENTS, eps=NS_EPS)
    return {"embedding": _embedding, "embedding_backward": _embedding_backward, "layer_norm": _layer_norm,
            "layer_norm_backward": _layer_norm_backward, "orthogonalize": _orthogonalize}[op](state)


# -------------------------------------------------------------------------- work

_BYTES = {"f32": 4, "bf16": 2, "f16": 2}


def _distinct_rows(n, vocab):
    """Expected number of different vocabulary rows among n tokens of _tokens()."""
    top, total, v = math.log(vocab + 1.0), 0.0, 0
    while v < vocab:                                 # ranks in blocks whose probability hardly changes
        w = min(vocab, max(v + 1, int(v * 1.02)))
        p = math.log((w + 1.0) / (v + 1.0)) / top / (w - v)
        total += (w - v) * -math.expm1(n * math.log1p(-p)) if p < 1 else w - v
        v = w
    return total


def work(case):
    op = case["op"]
    if op.startswith("embedding"):
        n, vocab, cols = case["tokens"], case["vocab"], case["cols"]
        real = n - sum(max(0, min(256, n - at) - 244) for at in range(0, n, 256)) if case["padding"] else n
        ids, act, table = n * case["index"] // 8, _BYTES[case["act"]], _BYTES[case["table"]]
        if op == "embedding":
            return {"bytes": ids + _distinct_rows(real, vocab) * cols * table + n * cols * act, "flops": real * cols}
        return {"bytes": ids + real * cols * act + vocab * cols * table, "flops": 2 * real * cols}
    if op.startswith("layer_norm"):
        n, act, weight = case["rows"] * case["cols"], _BYTES[case["act"]], _BYTES[case["weight"]]
        if op == "layer_norm":
            return {"bytes": 2 * n * act + 2 * case["cols"] * weight + 8 * case["rows"], "flops": 8 * n}
        return {"bytes": 3 * n * act + 3 * case["cols"] * weight + 8 * case["rows"], "flops": 14 * n}
    r, c = sorted((case["rows"], case["cols"]))
    # A and A A are symmetric: half of their entries are enough
    step = r * (r + 1) * c + r * (r + 1) * r + 2 * r * r * c
    return {"bytes": 2 * case["batch"] * r * c * _BYTES[case["act"]], "flops": case["batch"] * NS_STEPS * step}


# ------------------------------------------------------------------------- exact

def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "embedding":
        t = s["weights"].double()
        pad = torch.cat([t, torch.zeros(1, case["cols"], dtype=torch.float64, device="cuda")])
        del t
        return pad[s["ids"].long()] * s["scale"]            # index -1 is the row of zeros behind the last
    if op == "embedding_backward":
        keep = (s["ids"] >= 0).nonzero()[:, 0]
        where = torch.stack([s["ids"][keep].long(), torch.arange(keep.numel(), device="cuda")])
        member = torch.sparse_coo_tensor(where, torch.ones(keep.numel(), dtype=torch.float64, device="cuda"),
                                         (case["vocab"], keep.numel()))
        return torch.sparse.mm(member, s["dout"][keep].double()) * s["scale"]
    if op == "layer_norm":
        ys, means, rstds = [], [], []
        for x in s["x"].split(8192):                        # a block of rows at a time: 64 bits take room
            x = x.double()
            var, mean = torch.var_mean(x, 1, correction=0)
            rstd = 1.0 / torch.sqrt(var + LN_EPS)
            ys.append(torch.addcmul(s["b"].double(), (x - mean[:, None]) * rstd[:, None], s["w"].double()))
            means.append(mean)
            rstds.append(rstd)
        return torch.cat(ys), torch.cat(means), torch.cat(rstds)
    if op == "layer_norm_backward":
        w, dxs = s["w"].double(), []
        dw = torch.zeros(case["cols"], dtype=torch.float64, device="cuda")
        db = torch.zeros_like(dw)
        for x, dy, mean, rstd in zip(s["x"].split(8192), s["dy"].split(8192), s["mean"].split(8192), s["rstd"].split(8192)):
            x, dy, mean, rstd = x.double(), dy.double(), mean.double()[:, None], rstd.double()[:, None]
            h = (x - mean) * rstd
            dxs.append(rstd * (dy * w - (dy @ w)[:, None] / case["cols"] - h * ((dy * h) @ w)[:, None] / case["cols"]))
            dw += torch.einsum("rj,rj->j", dy, h)
            db += torch.ones(1, dy.shape[0], dtype=torch.float64, device="cuda").mm(dy)[0]
        return torch.cat(dxs), dw, db
    a, b, c = NS_COEFFICIENTS
    g = s["g"].double()
    x = g / (torch.linalg.matrix_norm(g, keepdim=True) + NS_EPS)
    for _ in range(NS_STEPS):                               # X (a + b X^T X + c (X^T X)^2), products on the shorter side
        if g.shape[-2] < g.shape[-1]:
            m = x @ x.mT
            p = torch.addmm if m.dim() == 2 else torch.baddbmm
            x = p(a * x, p(b * m, m, m, alpha=c), x)
        else:
            m = x.mT @ x
            p = torch.addmm if m.dim() == 2 else torch.baddbmm
            x = p(a * x, x, p(b * m, m, m, alpha=c))
    return x
