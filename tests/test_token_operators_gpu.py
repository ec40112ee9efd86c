"""GPU parity of the token-model operators (embedding, layer norm, orthogonalised update)
with their definitions in 64 bits.

Tolerances are bounds, counted before the kernels ran.  u = 2^-24 is the rounding of an
fp32 operation, h(T) = finfo(T).eps / 2 the rounding of a result to T.  A sum of which each
term passes through D additions is off by at most D u times the sum of the absolute values
(first order; the bounds below count a few operations more than there are)."""
import math

import pytest
import torch

from sapphire_b200 import _lib as L
from sapphire_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def half_step(t):
    return torch.finfo(t).eps / 2


def tiny(t):
    """Half the spacing of T's subnormal numbers."""
    return torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2


def gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def randn(g, *shape, dtype=F32, pitch=None, offset=0):
    """Normal values on the device, as rows of `pitch` elements starting `offset` elements in."""
    x = torch.randn(*shape, generator=g).to(dtype)
    if pitch is None and not offset:
        return x.to(DEV)
    rows, cols = shape
    pitch = pitch or cols
    flat = torch.full((rows * pitch + offset + 16,), float("nan"), dtype=dtype, device=DEV)
    view = flat[offset:offset + rows * pitch].view(rows, pitch)[:, :cols]
    view.copy_(x.to(DEV))
    return view


def check(got, want, tol):
    got, want = got.double().cpu(), want.double().cpu()
    assert got.shape == want.shape
    off = (got - want).abs()
    bad = ~(off <= tol.double().cpu() if torch.is_tensor(tol) else off <= tol)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} values off, the worst by {float(off[bad].max()):.3g}"


# --------------------------------------------------------------------- embedding

COMBOS = [(F32, F32), (BF16, BF16), (F16, F16), (F32, BF16), (F32, F16), (BF16, F32), (F16, F32)]


def token_ids(g, n, vocab, dtype, pad=True):
    ids = (torch.rand(n, generator=g) ** 3 * vocab).long().clamp_(0, max(vocab - 1, 0))
    if pad and n > 2:
        ids[torch.randperm(n, generator=g)[: n // 5]] = -1
        ids[n // 2] = -100
    return ids.to(dtype)


@pytest.mark.parametrize("tt,ta", COMBOS)
@pytest.mark.parametrize("n,vocab,cols,index", [(1, 1, 1, torch.int64), (5, 10, 7, torch.int32), (64, 100, 512, torch.int64),
                                                (333, 1000, 264, torch.int32), (1025, 77, 1000, torch.int64), (3, 5, 8200, torch.int64)])
def test_embedding(ctx, tt, ta, n, vocab, cols, index):
    g = gen(n + cols)
    table = randn(g, vocab, cols, dtype=tt)
    ids = token_ids(g, n, vocab, index)
    scale = math.sqrt(cols)
    out = ops.embedding(ctx, table, ids.to(DEV), scale=scale, out_dtype=ta)
    assert out.dtype == ta and out.shape == (n, cols)
    s32 = float(torch.tensor(scale, dtype=F32))
    want = torch.where((ids >= 0)[:, None], table.cpu().double()[ids.long().clamp_min(0)] * s32, 0.0)
    check(out, want, want.abs() * (half_step(ta) + U) * 1.0001 + tiny(ta))
    ctx.check_device_status()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("pitch,offset", [(24, 0), (19, 0), (24, 1), (17, 3)])
def test_embedding_strides(ctx, dtype, pitch, offset):
    """Row pitches and base addresses that 16-byte accesses do not fit."""
    g = gen(3)
    table = randn(g, 40, 16, dtype=dtype, pitch=pitch, offset=offset)
    ids = token_ids(g, 100, 40, torch.int64).to(DEV)
    buf = torch.full((100, pitch), 7.0, dtype=dtype, device=DEV)
    out = ops.embedding(ctx, table, ids, scale=1.0, out=buf[:, :16])
    want = torch.where((ids >= 0)[:, None], table[ids.clamp_min(0)], 0.0)
    assert torch.equal(out, want)
    assert (buf[:, 16:] == 7.0).all()                      # what lies between the rows stays
    dt = torch.full((40, pitch), 5.0, dtype=dtype, device=DEV)
    ops.embedding_backward(ctx, dt[:, :16], out, ids)
    assert (dt[:, 16:] == 5.0).all()
    full = ops.embedding_backward(ctx, torch.empty(40, 16, dtype=dtype, device=DEV), out.contiguous(), ids)
    assert torch.equal(dt[:, :16], full)


def test_embedding_out_of_range_is_reported(ctx):
    table = torch.ones(10, 8, device=DEV)
    ids = torch.tensor([0, 9, 10, 1 << 40, -1], device=DEV)
    out = ops.embedding(ctx, table, ids)
    with pytest.raises(L.Sb200Error) as e:
        ctx.check_device_status()
    assert e.value.status == L.ERR_TOKEN_RANGE
    assert out.sum(1).tolist() == [8, 8, 0, 0, 0]
    ctx.check_device_status()                              # read once, then clear
    dt = ops.embedding_backward(ctx, torch.empty(10, 8, device=DEV), torch.ones(5, 8, device=DEV), ids)
    with pytest.raises(L.Sb200Error):
        ctx.check_device_status()
    assert dt.sum().item() == 16 and dt[0, 0] == 1 and dt[9, 0] == 1


@pytest.mark.parametrize("token_first", [True, False])
@pytest.mark.parametrize("product", ["gemm", "orthogonalize"])
def test_a_bad_token_hides_no_expired_wait(ctx, product, token_first):
    """A token number beyond the vocabulary and a wait that runs out are reported each, the
    wait first, in whatever order they came."""
    table = torch.ones(10, 8, device=DEV)
    ids = torch.tensor([3, 10], device=DEV)
    a = randn(gen(1), 320, 320)                            # (two k-blocks a slice: one of them is held back)

    def stalled():
        ctx.set_option(L.OPT_WAIT_LIMIT_US, 2000)
        ctx.set_option(L.OPT_TEST_STALL_KBLOCKS, 1)
        try:
            ops.gemm(ctx, a, a) if product == "gemm" else ops.orthogonalize(ctx, a, steps=1)
            torch.cuda.synchronize()
        finally:
            ctx.set_option(L.OPT_TEST_STALL_KBLOCKS, -1)
            ctx.set_option(L.OPT_WAIT_LIMIT_US, 2000000)

    ctx.check_device_status()
    if token_first:
        ops.embedding(ctx, table, ids)
        stalled()
    else:
        stalled()
        ops.embedding_backward(ctx, table, torch.ones(2, 8, device=DEV), ids)
    for status in (L.ERR_DEVICE_TIMEOUT, L.ERR_TOKEN_RANGE):
        with pytest.raises(L.Sb200Error) as e:
            ctx.check_device_status()
        assert e.value.status == status
    ctx.check_device_status()


def grad_reference(dout, ids, vocab, scale):
    keep = ids >= 0
    want = torch.zeros(vocab, dout.shape[1], dtype=torch.float64)
    size = torch.zeros(vocab, dout.shape[1], dtype=torch.float64)
    count = torch.zeros(vocab, dtype=torch.float64)
    at, d = ids[keep].long(), dout.cpu().double()[keep]
    want.index_add_(0, at, d)
    size.index_add_(0, at, d.abs())
    count.index_add_(0, at, torch.ones(len(at), dtype=torch.float64))
    return want * scale, size * abs(scale), count[:, None]


@pytest.mark.parametrize("tt,ta", COMBOS)
@pytest.mark.parametrize("n,vocab,cols,index", [(1, 1, 1, torch.int64), (7, 600, 7, torch.int32), (64, 100, 512, torch.int64),
                                                (2049, 1000, 264, torch.int32), (5000, 513, 33, torch.int64),
                                                (4100, 300000, 16, torch.int64), (700, 3, 2056, torch.int32)])
def test_embedding_backward(ctx, tt, ta, n, vocab, cols, index):
    g = gen(n + cols)
    dout = randn(g, n, cols, dtype=ta)
    ids = token_ids(g, n, vocab, index)
    dt = torch.full((vocab, cols), float("nan"), dtype=tt, device=DEV)
    ops.embedding_backward(ctx, dt, dout, ids.to(DEV), scale=0.5)
    want, size, count = grad_reference(dout, ids, vocab, 0.5)
    check(dt, want, (count + 2) * U * size + half_step(tt) * want.abs() * 1.001 + tiny(tt))
    again = ops.embedding_backward(ctx, torch.empty_like(dt), dout, ids.to(DEV), scale=0.5)
    assert torch.equal(again, dt)                          # fixed order of the sums
    # accumulating: rows in use are added to, the others not written
    before = randn(g, vocab, cols, dtype=tt)
    acc = ops.embedding_backward(ctx, before.clone(), dout, ids.to(DEV), scale=-0.25, accumulate=True)
    want, size, count = grad_reference(dout, ids, vocab, -0.25)
    total = before.cpu().double() + want
    check(acc, total, (count + 2) * U * (size + total.abs()) + half_step(tt) * total.abs() * 1.001 + tiny(tt))
    idle = (count[:, 0] == 0).to(DEV)
    assert torch.equal(acc[idle], before[idle])


@pytest.mark.parametrize("n,distinct", [(20000, 1), (20000, 2), (70001, 3), (33000, 33000)])
def test_embedding_backward_long_runs(ctx, n, distinct):
    """Runs over many pieces, and none: one token number, a few, all different."""
    g = gen(n)
    ids = torch.randint(0, distinct, (n,), generator=g) if distinct < n else torch.randperm(n, generator=g)
    dout = randn(g, n, 24)
    dt = ops.embedding_backward(ctx, torch.empty(distinct, 24, device=DEV), dout, ids.to(DEV))
    want, size, count = grad_reference(dout, ids, distinct, 1.0)
    check(dt, want, (count + 2) * U * size)


@pytest.mark.parametrize("tt,ta", [(F32, F32), (F32, BF16), (BF16, BF16), (F16, F32)])
@pytest.mark.parametrize("n,vocab,cols,index", [(16384, 3000, 24, torch.int64), (16385, 3000, 24, torch.int32), (16385, 300000, 16, torch.int64),
                                                (20011, 900, 2064, torch.int64), (70001, 5000, 33, torch.int32)])
@pytest.mark.parametrize("accumulate", [False, True])
def test_embedding_backward_sorted_by_several_blocks(ctx, tt, ta, n, vocab, cols, index, accumulate):
    """On both sides of 16384 tokens, from where on several blocks sort: padding and a number
    beyond the vocabulary among the tokens, rows that no token names, a token number that runs over
    many pieces, a third pass of the sort (300000 rows), several tiles of columns (2064)."""
    g = gen(n + cols)
    ids = token_ids(g, n, vocab // 2, index)
    ids[torch.randperm(n, generator=g)[: n // 4]] = vocab - 2        # behind the half that the others name
    ids[n // 3] = vocab
    dout = randn(g, n, cols, dtype=ta)
    before = randn(g, vocab, cols, dtype=tt) if accumulate else torch.full((vocab, cols), float("nan"), dtype=tt, device=DEV)
    dt = ops.embedding_backward(ctx, before.clone(), dout, ids.to(DEV), scale=-0.5, accumulate=accumulate)
    with pytest.raises(L.Sb200Error) as e:
        ctx.check_device_status()
    assert e.value.status == L.ERR_TOKEN_RANGE
    want, size, count = grad_reference(dout, torch.where(ids < vocab, ids, -1), vocab, -0.5)
    assert (count == 0).any() and count[vocab - 2] > 3000
    if accumulate:
        want = want + before.cpu().double()
        idle = (count[:, 0] == 0).to(DEV)
        assert torch.equal(dt[idle], before[idle])
        size = size + want.abs()
    check(dt, want, (count + 2) * U * size + half_step(tt) * want.abs() * 1.001 + tiny(tt))
    again = ops.embedding_backward(ctx, before.clone(), dout, ids.to(DEV), scale=-0.5, accumulate=accumulate)
    assert torch.equal(again, dt)
    with pytest.raises(L.Sb200Error):
        ctx.check_device_status()


def test_embedding_backward_all_padding(ctx):
    dt = torch.full((33, 12), float("nan"), device=DEV)
    ids = torch.full((100,), -1, dtype=torch.int32, device=DEV)
    ops.embedding_backward(ctx, dt, torch.full((100, 12), float("nan"), device=DEV), ids)
    assert (dt == 0).all()
    ops.embedding_backward(ctx, dt.fill_(3.0), torch.ones(0, 12, device=DEV), ids[:0])
    assert (dt == 0).all()


def test_embedding_padding_rows_are_not_read_into_sums(ctx):
    """What stands in the gradient rows of padding (NaN, infinities) reaches nothing."""
    ids = torch.tensor([0, -1, 1, -1, 0, 1, -7], device=DEV)
    dout = torch.ones(7, 20, device=DEV)
    dout[ids < 0] = torch.tensor([float("nan"), float("inf"), -float("inf")], device=DEV)[:, None]
    dt = ops.embedding_backward(ctx, torch.empty(4, 20, device=DEV), dout, ids)
    assert torch.equal(dt.cpu(), torch.tensor([2.0, 2.0, 0.0, 0.0])[:, None].expand(4, 20))


# -------------------------------------------------------------------- layer norm

LN_TYPES = [(F32, F32), (BF16, F32), (BF16, BF16), (F16, F32), (F16, F16)]
LN_SHAPES = [(1, 1), (3, 2), (64, 512), (1000, 8), (37, 40), (17, 1000), (300, 4096), (5, 4001), (9, 8192), (4, 8200),
             (3, 20000), (2500, 129)]


def depth(cols):
    """Additions a term of a row sum passes through: a thread's own, lanes, warps."""
    return 16 + 5 + 16 + cols // 512


def ln_reference(x, w, b, eps):
    x = x.cpu().double()
    mean = x.mean(-1, keepdim=True)
    rstd = 1.0 / (x.var(-1, correction=0, keepdim=True) + eps).sqrt()
    h = (x - mean) * rstd
    w = torch.ones(x.shape[-1], dtype=torch.float64) if w is None else w.cpu().double()
    b = torch.zeros(x.shape[-1], dtype=torch.float64) if b is None else b.cpu().double()
    return x, mean, rstd, h, w, b


@pytest.mark.parametrize("t,wt", LN_TYPES)
@pytest.mark.parametrize("rows,cols", LN_SHAPES)
def test_layer_norm(ctx, t, wt, rows, cols):
    g = gen(rows * 31 + cols)
    x = (randn(g, rows, cols) + 3.0 * randn(g, rows, 1)).to(t)
    w, b = randn(g, cols, dtype=wt), randn(g, cols, dtype=wt)
    eps = 1e-3
    y, mean, rstd = ops.layer_norm(ctx, x, w, b, eps=eps)
    x, m, r, h, w, b = ln_reference(x, w, b, eps)
    D = depth(cols) + 8
    dm = D * U * x.abs().mean(-1, keepdim=True)            # of the mean; enters the differences whole
    check(mean, m[:, 0], dm[:, 0])
    dr = (D * U + dm ** 2 * r ** 2) * r                    # the variance moves by the mean's error squared
    check(rstd, r[:, 0], dr[:, 0])
    want = h * w + b
    tol = w.abs() * (r * dm + h.abs() * (dr / r + 4 * U)) + 4 * U * (b.abs() + want.abs())
    check(y, want, tol + half_step(t) * (want.abs() + tol) * 1.001 + tiny(t))


@pytest.mark.parametrize("t,wt", LN_TYPES)
@pytest.mark.parametrize("rows,cols", LN_SHAPES)
@pytest.mark.parametrize("accumulate", [False, True])
def test_layer_norm_backward(ctx, t, wt, rows, cols, accumulate):
    g = gen(rows * 31 + cols)
    x = (randn(g, rows, cols) + randn(g, rows, 1)).to(t)
    dy, w = randn(g, rows, cols, dtype=t), randn(g, cols, dtype=wt)
    _, mean, rstd = ops.layer_norm(ctx, x, w, None, eps=1e-3)
    kw, dx0, dw0, db0 = {}, 0.0, 0.0, 0.0
    if accumulate:
        dx0, dw0, db0 = randn(g, rows, cols, dtype=t), randn(g, cols, dtype=wt), randn(g, cols, dtype=wt)
        kw = dict(dx=dx0.clone(), dweight=dw0.clone(), dbias=db0.clone(), accumulate_dx=True, accumulate_weight=True)
        dx0, dw0, db0 = dx0.cpu().double(), dw0.cpu().double(), db0.cpu().double()
    dx, dw, db = ops.layer_norm_backward(ctx, dy, x, mean, rstd, w, **kw)
    m, r = mean.cpu().double()[:, None], rstd.cpu().double()[:, None]       # the call's own inputs
    dy, w = dy.cpu().double(), w.cpu().double()
    h = (x.cpu().double() - m) * r
    gw = dy * w
    m1, m2 = gw.mean(-1, keepdim=True), (gw * h).mean(-1, keepdim=True)
    want = r * (gw - m1 - h * m2) + dx0
    D = (depth(cols) + 10) * U
    size = r * (gw.abs() * 6 * U + D * gw.abs().mean(-1, keepdim=True) + h.abs() * (D * (gw * h).abs().mean(-1, keepdim=True)) +
                6 * U * (m1.abs() + (h * m2).abs())) + 2 * U * want.abs()
    check(dx, want, size + half_step(t) * (want.abs() + size) * 1.001 + tiny(t))
    R = (rows + 70) * U
    for got, terms, start in ((dw, dy * h, dw0), (db, dy, db0)):
        total = terms.sum(0) + start
        tol = (R + 4 * U) * terms.abs().sum(0) + 2 * U * total.abs()
        check(got, total, tol + half_step(wt) * (total.abs() + tol) * 1.001 + tiny(wt))


def test_layer_norm_backward_against_differences(ctx):
    """sum(dy * y) has the gradients dx, dweight, dbias: central differences of the 64-bit definition."""
    g = gen(5)
    x, w, b, dy = randn(g, 6, 24), randn(g, 24), randn(g, 24), randn(g, 6, 24)
    _, mean, rstd = ops.layer_norm(ctx, x, w, b)
    grads = ops.layer_norm_backward(ctx, dy, x, mean, rstd, w)

    def loss(x, w, b):
        m = x.mean(-1, keepdim=True)
        v = ((x - m) ** 2).mean(-1, keepdim=True)
        return (dy.cpu().double() * ((x - m) / (v + 1e-5).sqrt() * w + b)).sum()

    args = [t.cpu().double() for t in (x, w, b)]
    step = 1e-5
    for k, got in enumerate(grads):
        want = torch.zeros_like(args[k]).reshape(-1)
        for i in range(want.numel()):
            moved = [[t.clone() for t in args] for _ in range(2)]
            for sign, m in zip((1, -1), moved):
                m[k].view(-1)[i] += sign * step
            want[i] = (loss(*moved[0]) - loss(*moved[1])) / (2 * step)
        # differences: step^2 times a third derivative (values here are of order 10) and 1e-16 / step of rounding
        check(got.reshape(-1), want, 1e-5 * (1 + want.abs().max()))


@pytest.mark.parametrize("t", [F32, BF16])
@pytest.mark.parametrize("cols,pitch,offset", [(16, 24, 0), (16, 19, 0), (512, 520, 1), (4096, 4104, 0), (4000, 4003, 2), (8200, 8208, 0)])
def test_layer_norm_strides_and_in_place(ctx, t, cols, pitch, offset):
    g = gen(cols)
    x = randn(g, 21, cols, dtype=t, pitch=pitch, offset=offset)
    dy = randn(g, 21, cols, dtype=t, pitch=pitch, offset=offset)
    w, b = randn(g, cols), randn(g, cols)
    y, mean, rstd = ops.layer_norm(ctx, x.contiguous(), w, b)
    buf = torch.full((21, pitch), 7.0, dtype=t, device=DEV)
    y2, mean2, rstd2 = ops.layer_norm(ctx, x, w, b, out=buf[:, :cols])
    # another access width adds in another order: both are within the bound of the definition
    D = depth(cols) + 8
    off = 2 * D * U * (1 + x.double().abs().mean(-1, keepdim=True) * rstd[:, None].double())
    wy = w.double().abs() * off * (1 + ((y.double() - b.double()) / w.double()).abs()) + 4 * U * (b.abs() + y.abs().double())
    check(y2, y, wy + 2 * half_step(t) * y.double().abs() * 1.01 + tiny(t))
    assert (buf[:, cols:] == 7.0).all()
    x3 = x.contiguous()
    y3, _, _ = ops.layer_norm(ctx, x3, w, b, out=x3)
    assert y3.data_ptr() == x3.data_ptr() and torch.equal(y3, y)
    dx, dw, db = ops.layer_norm_backward(ctx, dy.contiguous(), x.contiguous(), mean, rstd, w)
    dy3 = dy.contiguous()
    dx3, dw3, db3 = ops.layer_norm_backward(ctx, dy3, x.contiguous(), mean, rstd, w, dx=dy3)
    assert torch.equal(dx3, dx) and torch.equal(dw3, dw) and torch.equal(db3, db)
    buf.fill_(9.0)
    ops.layer_norm_backward(ctx, dy, x, mean, rstd, w, dx=buf[:, :cols])
    assert (buf[:, cols:] == 9.0).all()
    scale = rstd.double()[:, None] * (w.double().abs() * dy.double().abs()).mean(-1, keepdim=True)
    check(buf[:, :cols], dx, 64 * D * U * scale * (1 + ((x.double() - mean.double()[:, None]) * rstd.double()[:, None]).abs()) +
          2 * half_step(t) * dx.double().abs() * 1.01 + 4 * U * dx.double().abs() + tiny(t))


@pytest.mark.parametrize("t,wt", LN_TYPES)
@pytest.mark.parametrize("rows,cols,pitch,offset", [(3, 1, 1, 5), (40, 1, 1, 0), (700, 3, 3, 1), (100, 5, 8, 3), (40, 17, 17, 7), (9000, 63, 63, 0),
                                                    (20, 505, 505, 2), (20, 506, 508, 1), (5000, 1001, 1001, 0), (30, 1024, 1027, 5),
                                                    (1000, 4003, 4003, 0), (9, 8185, 8185, 3), (9, 8187, 8190, 1), (5, 16376, 16379, 1)])
def test_layer_norm_rows_that_start_anywhere(ctx, t, wt, rows, cols, pitch, offset):
    """Rows at the same odd distances in all arrays give what aligned rows give, up to the order
    of the sums, in place too, and nothing around them is read into a sum or written."""
    g = gen(rows + cols)
    x = randn(g, rows, cols, dtype=t, pitch=pitch, offset=offset)
    dy = randn(g, rows, cols, dtype=t, pitch=pitch, offset=offset)
    w, b = randn(g, cols, dtype=wt), randn(g, cols, dtype=wt)

    def like():
        flat = torch.full((rows * pitch + offset + 16,), 7.0, dtype=t, device=DEV)
        return flat, flat[offset:offset + rows * pitch].view(rows, pitch)[:, :cols]

    eps = 1e-3
    flat, y = like()
    _, mean, rstd = ops.layer_norm(ctx, x, w, b, eps=eps, out=y)
    xr, m, r, h, wr, br = ln_reference(x, w, b, eps)
    D = depth(cols) + 8
    dm = D * U * xr.abs().mean(-1, keepdim=True)
    check(mean, m[:, 0], dm[:, 0])
    dr = (D * U + dm ** 2 * r ** 2) * r
    check(rstd, r[:, 0], dr[:, 0])
    want = h * wr + br
    tol = wr.abs() * (r * dm + h.abs() * (dr / r + 4 * U)) + 4 * U * (br.abs() + want.abs())
    check(y, want, tol + half_step(t) * (want.abs() + tol) * 1.001 + tiny(t))
    kept = torch.ones_like(flat, dtype=torch.bool)
    kept[offset:offset + rows * pitch].view(rows, pitch)[:, :cols] = False
    assert (flat[kept] == 7.0).all()

    flat, dx = like()
    dx.copy_(x)
    dx0 = x.cpu().double()
    got, dw, db = ops.layer_norm_backward(ctx, dy, x, mean, rstd, w, dx=dx, accumulate_dx=True)
    assert (flat[kept] == 7.0).all()
    m, r = mean.cpu().double()[:, None], rstd.cpu().double()[:, None]       # the call's own inputs
    d = dy.cpu().double()
    h = (xr - m) * r
    gw = d * wr
    m1, m2 = gw.mean(-1, keepdim=True), (gw * h).mean(-1, keepdim=True)
    want = r * (gw - m1 - h * m2) + dx0
    D = (depth(cols) + 10) * U
    size = r * (gw.abs() * 6 * U + D * gw.abs().mean(-1, keepdim=True) + h.abs() * (D * (gw * h).abs().mean(-1, keepdim=True)) +
                6 * U * (m1.abs() + (h * m2).abs())) + 2 * U * want.abs()
    check(got, want, size + half_step(t) * (want.abs() + size) * 1.001 + tiny(t))
    R = (rows + 70) * U
    for out, terms in ((dw, d * h), (db, d)):
        tol = (R + 4 * U) * terms.abs().sum(0) + 2 * U * terms.sum(0).abs()
        check(out, terms.sum(0), tol + half_step(wt) * (terms.sum(0).abs() + tol) * 1.001 + tiny(wt))
    # in place
    z = y.clone() if offset == 0 and pitch == cols else y
    plain, _, _ = ops.layer_norm_backward(ctx, dy, x, mean, rstd, w)
    over = dy
    ops.layer_norm_backward(ctx, over, x, mean, rstd, w, dx=over)
    check(over, plain.double().cpu(), 4 * size + 2 * half_step(t) * (plain.double().cpu().abs() + size) + tiny(t))
    ops.layer_norm(ctx, x, w, b, eps=eps, out=x)
    assert torch.equal(x, z)


def test_layer_norm_without_weights_and_leading_dimensions(ctx):
    g = gen(8)
    x = randn(g, 12, 96).view(3, 4, 96)
    y, mean, rstd = ops.layer_norm(ctx, x)
    assert y.shape == x.shape and mean.shape == (3, 4)
    one, zero = torch.ones(96, device=DEV), torch.zeros(96, device=DEV)
    y1, _, _ = ops.layer_norm(ctx, x, one, zero)
    assert torch.equal(y, y1)
    a = ops.layer_norm_backward(ctx, y, x, mean, rstd)
    b = ops.layer_norm_backward(ctx, y, x, mean, rstd, one)
    assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_layer_norm_constant_rows_and_bad_values(ctx):
    """A row without variance gives the bias; a row with NaN or infinity stays its own affair."""
    x = torch.full((4, 64), 5.0, device=DEV)
    x[1] = torch.arange(64, device=DEV)
    x[2, 7] = float("nan")
    x[3, 9] = float("inf")
    b = torch.arange(64, dtype=F32, device=DEV)
    y, mean, rstd = ops.layer_norm(ctx, x, None, b)
    assert torch.equal(y[0], b)
    assert torch.isfinite(y[1]).all() and torch.isnan(y[2]).all() and torch.isnan(y[3]).all()
    alone, _, _ = ops.layer_norm(ctx, x[1:2].contiguous(), None, b)
    assert torch.equal(alone[0], y[1])


@pytest.mark.parametrize("t", [F32, BF16])
@pytest.mark.parametrize("cols", [3, 8, 100, 1100, 4004])
def test_layer_norm_backward_of_constant_rows_of_large_numbers(ctx, t, cols):
    """h is 0 in such a row, but (0 - mean) * rstd, which lanes beyond the row could take for
    theirs, is not finite: 2^120 * 316 > 2^128."""
    g = gen(cols)
    x = torch.full((5, cols), 2.0 ** 120, dtype=t, device=DEV)
    dy, w = randn(g, 5, cols, dtype=t), randn(g, cols)
    mean, rstd = torch.full((5,), 2.0 ** 120, device=DEV), torch.full((5,), 316.0, device=DEV)
    dx, dw, _ = ops.layer_norm_backward(ctx, dy, x, mean, rstd, w)
    gw = dy.cpu().double() * w.cpu().double()
    m1 = gw.mean(-1, keepdim=True)
    want = 316.0 * (gw - m1)
    size = 316.0 * (gw.abs() * 6 * U + (depth(cols) + 10) * U * gw.abs().mean(-1, keepdim=True) + 6 * U * m1.abs()) + 2 * U * want.abs()
    check(dx, want, size + half_step(t) * (want.abs() + size) * 1.001 + tiny(t))
    assert (dw == 0).all()


def test_layer_norm_large_offsets(ctx):
    """Rows far from zero: the variance comes from differences to the mean."""
    g = gen(2)
    x = randn(g, 16, 1024) * 0.5 + 1000.0
    y, _, rstd = ops.layer_norm(ctx, x, eps=0.0)
    _, m, r, h, _, _ = ln_reference(x, None, None, 0.0)
    # the mean's error (depth x u x 1000) against a deviation of 0.5
    tol = (depth(1024) + 8) * U * 1000.0 * r
    check(y, h, tol * (1 + h.abs()) + 8 * U * h.abs())


def test_layer_norm_row_lengths_in_any_order(ctx):
    """One kernel serves several block sizes with different amounts of shared memory: what a
    shorter row needs must not be all that a longer one gets afterwards."""
    g = gen(12)
    xs = {cols: randn(g, 5, cols) for cols in (16000, 8000, 4000, 2000, 1100)}
    first = {}
    for cols in (16000, 8000, 4000, 2000, 1100, 16000, 2000, 8000, 1100, 4000):
        y, mean, rstd = ops.layer_norm(ctx, xs[cols])
        dx, dw, db = ops.layer_norm_backward(ctx, y, xs[cols], mean, rstd)
        got = first.setdefault(cols, (y, dx, dw))
        assert all(torch.equal(p, q) for p, q in zip(got, (y, dx, dw)))


def test_layer_norm_no_rows(ctx):
    dw, db = torch.full((16,), 3.0, device=DEV), torch.full((16,), 3.0, device=DEV)
    empty, stat = torch.empty(0, 16, device=DEV), torch.empty(0, device=DEV)
    ops.layer_norm(ctx, empty)
    ops.layer_norm_backward(ctx, empty, empty, stat, stat, dweight=dw, dbias=db, dx=empty, accumulate_weight=True)
    assert (dw == 3).all() and (db == 3).all()
    ops.layer_norm_backward(ctx, empty, empty, stat, stat, dweight=dw, dbias=db)
    assert (dw == 0).all() and (db == 0).all()


# ----------------------------------------------------------------- orthogonalize

COEF = (3.4445, -4.7750, 2.0315)


def ns_reference(g, steps=5, coef=COEF, eps=1e-7):
    a, b, c = coef
    x = g.cpu().double()
    tall = x.shape[-2] > x.shape[-1]
    x = x.mT if tall else x
    x = x / (x.square().sum((-2, -1), keepdim=True).sqrt() + eps)
    for _ in range(steps):
        m = x @ x.mT
        x = a * x + (b * m + c * (m @ m)) @ x
    return x.mT if tall else x


def ns_tolerance(t, steps=5):
    """Relative, 2-norm.  The operands' roundings, three matrices a step, carried along
    (a step multiplies an error in a direction by no more than it multiplies the direction
    itself, about), then the result's own.  Two parts: 22 bits and chains of 24 cut
    additions, a few u each: 1e-5 is the bar of the library's other fp32-accurate products."""
    if t == BF16:
        return steps * 3 * 2.0 ** -12 + half_step(t)
    return 1e-5 + (half_step(t) if t == F16 else 0.0)


def rel(got, want):
    got, want = got.cpu().double(), want.cpu().double()
    return float((got - want).norm() / want.norm())


def gradient(g, *shape, dtype=F32):
    """A few strong directions over noise, small values as gradients have them."""
    rows, cols = shape[-2:]
    rank = max(1, min(rows, cols) // 8)
    x = torch.randn(*shape[:-1], rank, generator=g) @ torch.randn(*shape[:-2], rank, cols, generator=g) / rank ** 0.5
    return ((x + 0.3 * torch.randn(*shape, generator=g)) * 1e-3).to(dtype).to(DEV)


NS_SHAPES = [(1, 1), (1, 7), (5, 3), (10, 256), (64, 64), (65, 127), (128, 128), (129, 300), (784, 512), (256, 1000),
             (640, 640), (1, 5000), (1300, 260), (128, 300), (100, 1000), (128, 2048), (2048, 128), (1500, 37), (128, 2049), (520, 9),
             (128, 4096), (128, 4097), (3000, 90)]


@pytest.mark.parametrize("t", [F32, BF16, F16])
@pytest.mark.parametrize("rows,cols", NS_SHAPES)
def test_orthogonalize(ctx, t, rows, cols):
    g = gradient(gen(rows + 7 * cols), rows, cols, dtype=t)
    out = ops.orthogonalize(ctx, g)
    ctx.check_device_status()
    assert rel(out, ns_reference(g)) <= ns_tolerance(t)
    assert torch.equal(ops.orthogonalize(ctx, g), out)


@pytest.mark.parametrize("t", [F32, BF16])
@pytest.mark.parametrize("batch,rows,cols", [(3, 100, 60), (2, 300, 700), (9, 512, 512), (5, 33, 33), (3, 1300, 1024),
                                             (4, 128, 700), (40, 70, 1030), (200, 16, 24)])
def test_orthogonalize_batches(ctx, t, batch, rows, cols):
    """Every matrix of a batch as alone; the larger ones take tiles of 256 on pairs of SMs."""
    g = gradient(gen(batch), batch, rows, cols, dtype=t)
    out = ops.orthogonalize(ctx, g)
    ctx.check_device_status()
    for k in range(batch):
        assert rel(out[k], ns_reference(g[k])) <= ns_tolerance(t)


@pytest.mark.parametrize("t", [F32, BF16])
@pytest.mark.parametrize("rows,cols", [(2500, 2300), (2048, 4096)])
def test_orthogonalize_large(ctx, t, rows, cols):
    g = gradient(gen(rows), rows, cols, dtype=t)
    out = ops.orthogonalize(ctx, g)
    ctx.check_device_status()
    want = g.double()
    x = want.mT if rows > cols else want
    x = x / (x.norm() + 1e-7)
    for _ in range(5):
        m = x @ x.mT
        x = COEF[0] * x + (COEF[1] * m + COEF[2] * (m @ m)) @ x
    assert rel(out, x.mT if rows > cols else x) <= ns_tolerance(t)


@pytest.mark.parametrize("batch,rows,cols", [(1, 45, 813), (3, 128, 128), (2, 700, 100), (1, 17, 4096)])
def test_orthogonalize_narrow_bf16(ctx, batch, rows, cols):
    """With a side of at most 128 the operands have 22 bits for bf16 too: what is left is the
    bar of the fp32-accurate products and the result's own rounding."""
    g = gradient(gen(rows + cols), batch, rows, cols, dtype=BF16)
    assert rel(ops.orthogonalize(ctx, g), ns_reference(g)) <= 1e-5 + half_step(BF16)


@pytest.mark.parametrize("batch,rows,cols", [(1, 128, 4097), (1, 45, 6000), (2, 4500, 100), (1, 128, 4096)])
def test_orthogonalize_narrow_bf16_of_any_length(ctx, batch, rows, cols):
    """22 bits whichever kernel such a matrix takes.  A result d away from the definition rounds
    to another number than it with a probability of |d| / spacing, and is then one spacing off:
    the squares add up to sum |d| spacing <= 1e-5 |x| 2^-7 |x| (operands of 11 bits: 2e-3 |x|)."""
    g = gradient(gen(rows + cols), batch, rows, cols, dtype=BF16)
    out = ops.orthogonalize(ctx, g)
    ctx.check_device_status()
    assert rel(out, ns_reference(g).to(BF16)) <= (1e-5 * 2.0 ** -7) ** 0.5


@pytest.mark.parametrize("rows", [2048, 2304])
def test_orthogonalize_bf16_long_sums(ctx, rows):
    """X X^T over 2^19 columns whose terms are all positive: the tensor core cuts every
    accumulation, so one chain over all of them loses 3.0e-3 of the sum, always to one side.
    (2048 rows take tiles of one SM, 2304 of pairs.)

    The rows are s_i times orthogonal signs, so with a = c = 0, b = 1 a step gives
    x_ij * (2^19 x_ij^2).  A row's result has the rounding of x (half a step of fp16, three
    times over), of A and of the result; their mean over the rows has a deviation of a
    rows^1/2-th of that, four of which are allowed, and a chain of at most 256 accumulations
    may lose four units of 2^-23 each."""
    g, cols = gen(rows), 1 << 19
    signs = torch.ones(1, 1, device=DEV)
    while signs.shape[0] < 4096:
        signs = torch.cat([torch.cat([signs, signs], 1), torch.cat([signs, -signs], 1)], 0)
    signs = signs[:rows]
    s = (1 + torch.rand(rows, generator=g)).to(BF16).to(DEV)
    out = ops.orthogonalize(ctx, (signs * s[:, None]).to(BF16).repeat(1, cols // 4096), steps=1, coefficients=(0.0, 1.0, 0.0))
    ctx.check_device_status()
    x = s.double() / (cols * s.double().square().sum()).sqrt()
    off = (out[:, -4096:].double() * signs / (cols * x ** 3)[:, None]).mean() - 1
    spread = (half_step(BF16) ** 2 + (3 * half_step(F16)) ** 2 + half_step(F16) ** 2) ** 0.5 / 3 ** 0.5
    assert abs(float(off)) <= 256 * 4 * 2.0 ** -23 + 4 * spread / rows ** 0.5


def test_orthogonalize_strides_steps_and_in_place(ctx):
    g = gen(4)
    wide = gradient(g, 90, 200)
    for view in (wide[:, :120], wide[:, 3:124], wide[:60, 5:]):
        out = torch.full((view.shape[0], 211), 2.0, device=DEV)
        got = ops.orthogonalize(ctx, view, out=out[:, 1:1 + view.shape[1]])
        assert rel(got, ns_reference(view)) <= ns_tolerance(F32)
        assert (out[:, 0] == 2).all() and (out[:, 1 + view.shape[1]:] == 2).all()
    for steps, coef in ((1, COEF), (2, COEF), (12, (1.5, -0.5, 0.0))):
        got = ops.orthogonalize(ctx, wide, steps=steps, coefficients=coef)
        assert rel(got, ns_reference(wide, steps, coef)) <= ns_tolerance(F32, steps)
    want = ops.orthogonalize(ctx, wide)
    same = wide.clone()
    assert torch.equal(ops.orthogonalize(ctx, same, out=same), want)
    batch = gradient(g, 4, 50, 70)
    got = ops.orthogonalize(ctx, batch[::2])
    assert torch.equal(got[1], ops.orthogonalize(ctx, batch[2]))


def test_orthogonalize_range_of_inputs(ctx):
    """Magnitudes at both ends of fp32, zero, and values that are not finite."""
    # (bits may differ from one magnitude to the other: the squares are added in fp32 inside its
    # range and in fp64 beyond, and at 2^-112 the smallest inputs are subnormal; each result is
    # held to the definition on its own input)
    g, wide = gradient(gen(6), 40, 70), gradient(gen(7), 140, 200)
    for power in (-112, -90, 0, 100):
        for m in (g * 2.0 ** power, wide * 2.0 ** power):
            assert rel(ops.orthogonalize(ctx, m, eps=0.0), ns_reference(m, eps=0.0)) <= ns_tolerance(F32)
    assert (ops.orthogonalize(ctx, torch.zeros(30, 20, device=DEV)) == 0).all()
    bad = g.clone()
    bad[3, 5] = float("nan")
    assert torch.isnan(ops.orthogonalize(ctx, bad)).all()


def test_orthogonalize_bounded_waits(ctx):
    """The waits of all kernels run out, the status says so and the context goes on."""
    small, large = gradient(gen(1), 130, 300), gradient(gen(2), 2300, 2300)
    one, some = gradient(gen(3), 40, 50), gradient(gen(4), 90, 900)
    want = ops.orthogonalize(ctx, small)
    ctx.check_device_status()
    ctx.set_option(L.OPT_WAIT_LIMIT_US, 2000)
    ctx.set_option(L.OPT_TEST_STALL_KBLOCKS, 1)
    try:
        for g in (small, large, one, some):
            ops.orthogonalize(ctx, g, steps=2)
            with pytest.raises(L.Sb200Error) as e:
                ctx.check_device_status()
            assert e.value.status == L.ERR_DEVICE_TIMEOUT
    finally:
        ctx.set_option(L.OPT_TEST_STALL_KBLOCKS, -1)
        ctx.set_option(L.OPT_WAIT_LIMIT_US, 2000000)
    assert torch.equal(ops.orthogonalize(ctx, small), want)


@pytest.mark.parametrize("batch,rows,cols", [(1, 128, 2048), (700, 2000, 100), (3, 40, 50)])
def test_orthogonalize_reads_and_writes_no_workspace_where_it_needs_none(ctx, batch, rows, cols):
    """The page such a call asks for stays as it was, and the buffer behind it too."""
    g = gradient(gen(batch), batch, rows, cols)
    want = ops.orthogonalize(ctx, g)
    need = L.lib().sb200_orthogonalize_workspace(rows, cols, batch, L.F32)
    assert need == 4096
    ws = torch.full((2 * need,), 0xA5, dtype=torch.uint8, device=DEV)
    out = torch.full_like(g, float("nan"))
    torch.cuda.synchronize()
    status = L.lib().sb200_orthogonalize(ctx.handle, out.data_ptr(), cols, rows * cols, g.data_ptr(), cols, rows * cols, rows, cols,
                                         batch, 5, *COEF, 1e-7, L.F32, ws.data_ptr(), need, torch.cuda.current_stream().cuda_stream)
    assert status == L.OK
    ctx.check_device_status()
    assert torch.equal(out, want) and (ws == 0xA5).all()


def test_expired_waits_leave_what_comes_behind_alone(ctx):
    """A product that gave up stays on its SMs until what it has issued has landed: the kernels
    enqueued right behind it, which get its shared memory and tensor memory, are as ever."""
    g = gen(9)
    ms = [gradient(g, 130, 300), gradient(g, 2300, 2300), gradient(g, 90, 900), gradient(g, 1024, 1024, dtype=BF16)]
    x, a = randn(g, 4096, 2048), randn(g, 512, 512)
    want = [*ops.layer_norm(ctx, x), ops.gemm(ctx, a, a), *(ops.orthogonalize(ctx, m) for m in ms)]
    ctx.check_device_status()
    ctx.set_option(L.OPT_WAIT_LIMIT_US, 5000)
    try:
        for m in ms:
            ctx.set_option(L.OPT_TEST_STALL_KBLOCKS, 1)
            ops.orthogonalize(ctx, m, steps=1)
            ctx.set_option(L.OPT_TEST_STALL_KBLOCKS, -1)
            got = [*ops.layer_norm(ctx, x), ops.gemm(ctx, a, a), *(ops.orthogonalize(ctx, m) for m in ms)]
            with pytest.raises(L.Sb200Error) as e:
                ctx.check_device_status()
            assert e.value.status == L.ERR_DEVICE_TIMEOUT
            ctx.check_device_status()
            assert all(torch.equal(p, q) for p, q in zip(got, want))
    finally:
        ctx.set_option(L.OPT_TEST_STALL_KBLOCKS, -1)
        ctx.set_option(L.OPT_WAIT_LIMIT_US, 2000000)


# ----------------------------------------------------------- streams and graphs

def test_other_streams_and_captured_graphs(ctx):
    """The calls on another stream than the tensors', and two captured graphs that share
    one context, replayed in turn after larger calls have run."""
    g = gen(11)
    table, ids = randn(g, 50, 64), token_ids(g, 200, 50, torch.int64).to(DEV)
    dout, x, w, b = randn(g, 200, 64), randn(g, 200, 64), randn(g, 64), randn(g, 64)
    m = gradient(g, 70, 40)

    def step(k):
        e = ops.embedding(ctx, table, ids, scale=2.0)
        y, mean, rstd = ops.layer_norm(ctx, e + x * k, w, b)
        dx, dw, db = ops.layer_norm_backward(ctx, dout, e + x * k, mean, rstd, w)
        dt = ops.embedding_backward(ctx, torch.empty_like(table), dx, ids, scale=2.0)
        return [e, y, dx, dw, db, dt, ops.orthogonalize(ctx, m * k)]

    want = {k: [t.clone() for t in step(k)] for k in (1, 3)}
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = step(1)
    side.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(got, want[1]))
    graphs, outs = {}, {}
    for k in (1, 3):
        graphs[k] = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graphs[k]):
            outs[k] = step(k)
    big = randn(g, 3000, 512)
    ops.layer_norm_backward(ctx, big, big, torch.zeros(3000, device=DEV), torch.ones(3000, device=DEV))
    ops.orthogonalize(ctx, big)
    for k in (3, 1, 3, 1):
        for t in outs[k]:
            t.fill_(float("nan"))
        graphs[k].replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(outs[k], want[k]))


@pytest.mark.parametrize("rows,cols", [(300, 700), (2304, 2500)])
def test_captured_products_and_long_sorts(ctx, rows, cols):
    """The larger ways of the calls in a graph, replayed after their inputs have changed."""
    g = gen(13)
    m, ids, dout = gradient(g, rows, cols), token_ids(g, 20000, 3000, torch.int64).to(DEV), randn(g, 20000, 24)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = ops.orthogonalize(ctx, m)
        dt = ops.embedding_backward(ctx, torch.empty(3000, 24, device=DEV), dout, ids)
    for _ in range(2):
        m.copy_(gradient(g, rows, cols))
        ids.copy_(ids.flip(0))
        o.fill_(float("nan"))
        dt.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(o, ops.orthogonalize(ctx, m))
        assert torch.equal(dt, ops.embedding_backward(ctx, torch.empty(3000, 24, device=DEV), dout, ids))
    ctx.check_device_status()


def test_two_streams_at_once(ctx):
    """Calls of one context on two streams, in flight together: nothing of theirs is shared."""
    g = gen(15)
    ms = [gradient(g, 300, 700), gradient(g, 2304, 2500), gradient(g, 100, 900)]
    ids = [token_ids(g, n, 3000, torch.int64).to(DEV) for n in (20000, 5000)]
    douts = [randn(g, len(i), 136) for i in ids]
    x, w = randn(g, 4001, 999, dtype=BF16), randn(g, 999)

    def work():
        out = [ops.orthogonalize(ctx, m) for m in ms]
        out += [ops.embedding_backward(ctx, torch.empty(3000, 136, device=DEV), d, i) for d, i in zip(douts, ids)]
        y, mean, rstd = ops.layer_norm(ctx, x, w)
        return out + [y, *ops.layer_norm_backward(ctx, y, x, mean, rstd, w)]

    want = work()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for _ in range(4):
        for st in streams:
            with torch.cuda.stream(st):
                got.append(work())
    torch.cuda.synchronize()
    ctx.check_device_status()
    assert all(torch.equal(p, q) for out in got for p, q in zip(out, want))


def test_two_host_threads_with_a_context_each(ctx):
    """A context per host thread, as documented: the calls of two threads at the same time."""
    import threading
    g = gen(16)
    ms = [gradient(g, 300, 700), gradient(g, 100, 900, dtype=BF16), gradient(g, 1100, 1300, dtype=BF16)]
    ids, dout = token_ids(g, 20000, 3000, torch.int64).to(DEV), randn(g, 20000, 40)
    x, w = randn(g, 2001, 999, dtype=BF16), randn(g, 999)

    def work(c):
        out = [ops.orthogonalize(c, m) for m in ms]
        out += [ops.embedding_backward(c, torch.empty(3000, 40, device=DEV), dout[:n], ids[:n]) for n in (20000, 5000)]
        y, mean, rstd = ops.layer_norm(c, x, w)
        return out + [y, *ops.layer_norm_backward(c, y, x, mean, rstd, w)]

    want = work(ctx)
    torch.cuda.synchronize()
    got, failed = [], []

    def thread():
        try:
            own = ops.Context(0)
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(10):
                    got.append(work(own))
                own.check_device_status()
        except Exception as e:
            failed.append(e)

    threads = [threading.Thread(target=thread) for _ in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not failed and len(got) == 20
    assert all(torch.equal(p, q) for out in got for p, q in zip(out, want))


def test_offsets_beyond_32_bits(ctx):
    """Rows so far apart that the last ones start more than 2^32 elements in."""
    g = gen(14)
    rows, cols, pitch = 300, 200, 1 << 24
    def far():
        return torch.empty(rows * pitch, dtype=BF16, device=DEV).view(rows, pitch)[:, :cols]
    a, b = far(), far()
    small = randn(g, rows, cols, dtype=BF16)
    a.copy_(small)
    ids = torch.randint(0, rows, (500,), generator=g)
    ids[:3] = torch.tensor([rows - 1, 0, rows - 1])
    ids = ids.to(DEV)
    e = ops.embedding(ctx, a, ids)
    assert torch.equal(e, small[ids])
    b.zero_()
    ops.embedding(ctx, small, torch.arange(rows, device=DEV), out=b)
    assert torch.equal(b, small)
    ops.embedding_backward(ctx, b, e, ids)
    assert torch.equal(b, ops.embedding_backward(ctx, torch.empty_like(small), e, ids))
    y, mean, rstd = ops.layer_norm(ctx, small)
    ops.layer_norm(ctx, a, out=b)
    assert torch.equal(b, y)
    dx, _, _ = ops.layer_norm_backward(ctx, small, small, mean, rstd)
    ops.layer_norm_backward(ctx, a, a, mean, rstd, dx=b)
    assert torch.equal(b, dx)
    ops.orthogonalize(ctx, a, out=b)
    assert torch.equal(b, ops.orthogonalize(ctx, small))


# ------------------------------------------------------------ a run of them together

def test_training_step_of_a_token_model(ctx):
    """Embedding, layer norm, Linear, softmax cross-entropy, and back: every gradient and
    the updated parameters against autograd in 64 bits.  The matrix weight takes the
    orthogonalised update, the vectors and the table SGD."""
    g = gen(21)
    vocab, width, classes, n, lr = 300, 96, 52, 257, 0.02
    table, W = randn(g, vocab, width) * 0.1, randn(g, width, classes) * 0.1
    bias, lw, lb = randn(g, classes) * 0.1, 1 + 0.1 * randn(g, width), 0.1 * randn(g, width)
    ids = token_ids(g, n, vocab, torch.int64).to(DEV)
    target = torch.randint(0, classes, (n,), generator=g).to(DEV)
    onehot = torch.nn.functional.one_hot(target, classes).float()
    scale = width ** 0.5

    e = ops.embedding(ctx, table, ids, scale=scale)
    y, mean, rstd = ops.layer_norm(ctx, e, lw, lb)
    logits = ops.gemm(ctx, y, W, bias=bias, mode=L.MODE_TF32X3)
    _, loss, dlogits = ops.softmax_cross_entropy(ctx, logits, onehot)
    dy = ops.gemm(ctx, dlogits, W, trans_b=True, mode=L.MODE_TF32X3)
    dbias = torch.empty(classes, device=DEV)
    dW = ops.gemm(ctx, y, dlogits, trans_a=True, mode=L.MODE_TF32X3, colsum_out=dbias)
    de, dlw, dlb = ops.layer_norm_backward(ctx, dy, e, mean, rstd, lw)
    dtable = ops.embedding_backward(ctx, torch.empty_like(table), de, ids, scale=scale)

    p = [t.cpu().double().requires_grad_() for t in (table, lw, lb, W, bias)]
    rows = p[0][ids.cpu().clamp_min(0)] * (ids.cpu() >= 0)[:, None] * scale
    out = torch.nn.functional.layer_norm(rows, (width,), p[1], p[2], 1e-5) @ p[3] + p[4]
    want_loss = torch.nn.functional.cross_entropy(out, target.cpu(), reduction="none")
    want_loss.sum().backward()
    # the products are good to 1e-5, the sums around them to a few u: one bar for all
    assert rel(loss, want_loss.detach()) <= 3e-5
    for got, want in zip((dtable, dlw, dlb, dW, dbias), p):
        assert rel(got, want.grad) <= 3e-5
    # padding rows are constant (zero): their layer norm has rstd = eps^-1/2 and their gradient goes nowhere

    new_W = ops.sgd_update(ctx, W.clone(), ops.orthogonalize(ctx, dW), lr)
    want_W = p[3].detach() - lr * ns_reference(p[3].grad)
    assert rel(new_W, want_W) <= 3e-5
    new_table = ops.embedding_backward(ctx, table.clone(), de, ids, scale=-lr * scale, accumulate=True)
    assert rel(new_table, p[0].detach() - lr * p[0].grad) <= 3e-5
