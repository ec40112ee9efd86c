"""Argument checks of the token-model operators through the C ABI, without a device: the
context is a stand-in of which the calls only read the first two words (device, SM count)
before they refuse."""
import ctypes as C

import pytest
import torch

from sapphire_b200 import _lib as L

BUF = C.create_string_buffer(1 << 16)
P = (C.addressof(BUF) + 255) // 256 * 256          # a 256-byte aligned address, never read


@pytest.fixture()
def fake():
    words = (C.c_int * 4096)()
    words[0], words[1] = 0, 148
    return words


def embedding(fake, out=P, ldo=8, table=P, ldt=8, ids=P, bits=64, n=4, vocab=10, cols=8, tt=L.F32, ta=L.F32):
    return L.lib().sb200_embedding(fake, out, ldo, table, ldt, ids, bits, n, vocab, cols, 1.0, tt, ta, None)


def embedding_backward(fake, dtable=P, ldt=8, dout=P, ldo=8, ids=P, bits=64, n=4, vocab=10, cols=8, tt=L.F32, ta=L.F32,
                       acc=0, ws=P, nbytes=1 << 40):
    return L.lib().sb200_embedding_backward(fake, dtable, ldt, dout, ldo, ids, bits, n, vocab, cols, 1.0, tt, ta, acc, ws,
                                            nbytes, None)


def layer_norm(fake, y=P, ldy=8, x=P, ldx=8, rows=4, cols=8, eps=1e-5, t=L.F32, w=L.F32):
    return L.lib().sb200_layer_norm(fake, y, ldy, P, P, x, ldx, P, P, rows, cols, eps, t, w, None)


def layer_norm_backward(fake, dx=P, lddx=8, dw=P, db=P, dy=P, lddy=8, x=P, ldx=8, mean=P, rstd=P, rows=4, cols=8, t=L.F32,
                        w=L.F32, ws=P, nbytes=1 << 40):
    return L.lib().sb200_layer_norm_backward(fake, dx, lddx, dw, db, dy, lddy, x, ldx, P, mean, rstd, rows, cols, t, w, 0, 0,
                                             ws, nbytes, None)


def orthogonalize(fake, out=P, ldo=8, so=64, g=P, ldg=8, sg=64, rows=8, cols=8, batch=2, steps=5, coef=(3.4445, -4.775, 2.0315),
                  eps=1e-7, t=L.F32, ws=P, nbytes=1 << 40):
    return L.lib().sb200_orthogonalize(fake, out, ldo, so, g, ldg, sg, rows, cols, batch, steps, *coef, eps, t, ws, nbytes,
                                       None)


REFUSED = [
    (embedding, dict(n=-1), L.ERR_INVALID_ARG),
    (embedding, dict(cols=-1), L.ERR_INVALID_ARG),
    (embedding, dict(ldo=7), L.ERR_INVALID_ARG),
    (embedding, dict(ldt=7), L.ERR_INVALID_ARG),
    (embedding, dict(bits=16), L.ERR_INVALID_ARG),
    (embedding, dict(tt=3), L.ERR_INVALID_ARG),
    (embedding, dict(ta=-1), L.ERR_INVALID_ARG),
    (embedding, dict(tt=L.BF16, ta=L.F16), L.ERR_UNSUPPORTED),
    (embedding, dict(out=None), L.ERR_INVALID_ARG),
    (embedding, dict(table=None), L.ERR_INVALID_ARG),
    (embedding, dict(ids=None), L.ERR_INVALID_ARG),
    (embedding, dict(ids=P + 4), L.ERR_INVALID_ARG),
    (embedding, dict(out=P + 2), L.ERR_INVALID_ARG),
    (embedding, dict(table=P + 1, tt=L.BF16, ta=L.BF16), L.ERR_INVALID_ARG),
    (embedding_backward, dict(dtable=P + 2), L.ERR_INVALID_ARG),
    (embedding_backward, dict(dout=P + 1, ta=L.F16), L.ERR_INVALID_ARG),
    (layer_norm, dict(x=P + 2), L.ERR_INVALID_ARG),
    (layer_norm, dict(y=P + 1, t=L.BF16), L.ERR_INVALID_ARG),
    (layer_norm_backward, dict(dy=P + 2), L.ERR_INVALID_ARG),
    (layer_norm_backward, dict(dx=P + 1, t=L.F16), L.ERR_INVALID_ARG),
    (layer_norm_backward, dict(dw=P + 2), L.ERR_INVALID_ARG),
    (layer_norm_backward, dict(mean=P + 2), L.ERR_INVALID_ARG),
    (orthogonalize, dict(g=P + 2), L.ERR_INVALID_ARG),
    (orthogonalize, dict(out=P + 1, t=L.BF16), L.ERR_INVALID_ARG),
    (embedding, dict(n=(1 << 30) + 1), L.ERR_TOO_LARGE),
    (embedding, dict(vocab=(1 << 31) - 1), L.ERR_TOO_LARGE),
    (embedding, dict(cols=(1 << 20) + 1, ldo=1 << 21, ldt=1 << 21), L.ERR_TOO_LARGE),
    (embedding_backward, dict(n=-1), L.ERR_INVALID_ARG),
    (embedding_backward, dict(vocab=-1), L.ERR_INVALID_ARG),
    (embedding_backward, dict(ldt=7), L.ERR_INVALID_ARG),
    (embedding_backward, dict(ldo=7), L.ERR_INVALID_ARG),
    (embedding_backward, dict(dtable=None), L.ERR_INVALID_ARG),
    (embedding_backward, dict(dout=None), L.ERR_INVALID_ARG),
    (embedding_backward, dict(ids=None), L.ERR_INVALID_ARG),
    (embedding_backward, dict(tt=L.F16, ta=L.BF16), L.ERR_UNSUPPORTED),
    (embedding_backward, dict(ws=None), L.ERR_INVALID_ARG),
    (embedding_backward, dict(ws=P + 4), L.ERR_INVALID_ARG),
    (embedding_backward, dict(nbytes=16), L.ERR_INVALID_ARG),
    (embedding_backward, dict(n=(1 << 30) + 1), L.ERR_TOO_LARGE),
    (layer_norm, dict(rows=-1), L.ERR_INVALID_ARG),
    (layer_norm, dict(cols=0), L.ERR_INVALID_ARG),
    (layer_norm, dict(ldx=7), L.ERR_INVALID_ARG),
    (layer_norm, dict(ldy=7), L.ERR_INVALID_ARG),
    (layer_norm, dict(eps=-1.0), L.ERR_INVALID_ARG),
    (layer_norm, dict(eps=float("nan")), L.ERR_INVALID_ARG),
    (layer_norm, dict(x=None), L.ERR_INVALID_ARG),
    (layer_norm, dict(y=None), L.ERR_INVALID_ARG),
    (layer_norm, dict(t=5), L.ERR_INVALID_ARG),
    (layer_norm, dict(t=L.F32, w=L.BF16), L.ERR_UNSUPPORTED),
    (layer_norm, dict(t=L.F16, w=L.BF16), L.ERR_UNSUPPORTED),
    (layer_norm_backward, dict(rows=-1), L.ERR_INVALID_ARG),
    (layer_norm_backward, dict(cols=0), L.ERR_INVALID_ARG),
    (layer_norm_backward, dict(lddx=7), L.ERR_INVALID_ARG),
    (layer_norm_backward, dict(lddy=7), L.ERR_INVALID_ARG),
    (layer_norm_backward, dict(ldx=7), L.ERR_INVALID_ARG),
    (layer_norm_backward, dict(dy=None), L.ERR_INVALID_ARG),
    (layer_norm_backward, dict(mean=None), L.ERR_INVALID_ARG),
    (layer_norm_backward, dict(rstd=None), L.ERR_INVALID_ARG),
    (layer_norm_backward, dict(ws=None), L.ERR_INVALID_ARG),
    (layer_norm_backward, dict(nbytes=4), L.ERR_INVALID_ARG),
    (layer_norm_backward, dict(t=L.BF16, w=L.F16), L.ERR_UNSUPPORTED),
    (orthogonalize, dict(rows=-1), L.ERR_INVALID_ARG),
    (orthogonalize, dict(ldo=7), L.ERR_INVALID_ARG),
    (orthogonalize, dict(ldg=7), L.ERR_INVALID_ARG),
    (orthogonalize, dict(so=60), L.ERR_INVALID_ARG),
    (orthogonalize, dict(sg=-1), L.ERR_INVALID_ARG),
    (orthogonalize, dict(steps=0), L.ERR_INVALID_ARG),
    (orthogonalize, dict(steps=65), L.ERR_TOO_LARGE),
    (orthogonalize, dict(eps=-1e-7), L.ERR_INVALID_ARG),
    (orthogonalize, dict(t=9), L.ERR_INVALID_ARG),
    (orthogonalize, dict(out=None), L.ERR_INVALID_ARG),
    (orthogonalize, dict(g=None), L.ERR_INVALID_ARG),
    (orthogonalize, dict(ws=None), L.ERR_INVALID_ARG),
    (orthogonalize, dict(nbytes=1024), L.ERR_INVALID_ARG),
    (orthogonalize, dict(rows=1 << 21, batch=1), L.ERR_TOO_LARGE),
    (orthogonalize, dict(batch=65536), L.ERR_TOO_LARGE),
    (orthogonalize, dict(coef=(10.0, 0.0, 0.0)), L.ERR_UNSUPPORTED),        # |X| grows tenfold a step
    (orthogonalize, dict(coef=(1.0, 8.0, 0.0)), L.ERR_UNSUPPORTED),         # |b s^2| = 8 at once
    (orthogonalize, dict(coef=(float("nan"), 0.0, 0.0)), L.ERR_UNSUPPORTED),
    (orthogonalize, dict(coef=(1.5, float("inf"), 0.0)), L.ERR_UNSUPPORTED),
]


@pytest.mark.parametrize("call,args,status", REFUSED, ids=[f"{c.__name__}-{next(iter(a))}-{i}" for i, (c, a, _) in enumerate(REFUSED)])
def test_refusals(fake, call, args, status):
    assert call(fake, **args) == status
    assert call(None) == L.ERR_INVALID_ARG


def test_empty_calls_touch_nothing(fake):
    assert embedding(fake, n=0, out=None, ids=None) == L.OK
    assert embedding(fake, cols=0, ldo=0, ldt=0) == L.OK
    assert embedding_backward(fake, vocab=0, ws=None) == L.OK
    assert embedding_backward(fake, n=0, acc=1, ws=None) == L.OK
    assert layer_norm(fake, rows=0, x=None, y=None) == L.OK
    assert layer_norm_backward(fake, rows=0, dw=None, db=None, x=None, dy=None, ws=None) == L.OK
    assert orthogonalize(fake, rows=0) == L.OK
    assert orthogonalize(fake, batch=0) == L.OK


@pytest.mark.parametrize("rows,cols", [(1 << 41, 8), (4, 1 << 36), (1 << 20, 1 << 61), (1 << 62, 1 << 13)])
def test_layer_norm_sizes_beyond_any_memory(fake, rows, cols):
    """Refused before a size in bytes or a grid's extent wraps (rows of 2^61 columns would have
    had a workspace of no bytes)."""
    assert layer_norm(fake, rows=rows, cols=cols, ldx=cols, ldy=cols) == L.ERR_TOO_LARGE
    assert layer_norm_backward(fake, rows=rows, cols=cols, ldx=cols, lddx=cols, lddy=cols) == L.ERR_TOO_LARGE
    assert L.lib().sb200_layer_norm_backward_workspace(fake, rows, cols) == -1


def test_workspace_sizes(fake):
    lib = L.lib()
    assert lib.sb200_embedding_backward_workspace(None, 4, 10, 8) == -1
    assert lib.sb200_embedding_backward_workspace(fake, -1, 10, 8) == -1
    assert lib.sb200_layer_norm_backward_workspace(fake, 4, 0) == -1
    assert lib.sb200_orthogonalize_workspace(8, 8, 1, 7) == -1
    for n in (0, 1, 7, 4096, 1 << 20):
        need = lib.sb200_embedding_backward_workspace(fake, n, 65536, 64)
        assert need >= 16 * n                     # two sets of keys and positions
    for rows in (0, 1, 64, 1 << 16):
        assert lib.sb200_layer_norm_backward_workspace(fake, rows, 512) >= 2 * 512 * 4
    # four fp16 arrays of the matrix, four of its Gram matrix
    assert lib.sb200_orthogonalize_workspace(512, 784, 1, L.F32) >= 2 * (4 * 512 * 784 + 4 * 512 * 512)


@pytest.mark.parametrize("t", [L.F32, L.BF16, L.F16])
def test_workspace_of_matrices_that_need_none(t):
    """What one cluster of any device holds asks for a page, whatever the batch; the next size
    up, which another device may take the general way with, for all its matrices."""
    size = L.lib().sb200_orthogonalize_workspace
    for rows, cols in ((1, 1), (128, 2048), (2048, 128), (50, 60)):
        for batch in (0, 1, 65535):
            assert size(rows, cols, batch, t) == 4096
    for rows, cols in ((128, 2049), (129, 129)):
        assert size(rows, cols, 10, t) > 10 * rows * cols * 2 * 4


def test_workspace_of_narrow_bf16(fake):
    """With a side of at most 128 every operand has two parts, for bf16 as for fp32; with both
    sides longer A and B have one."""
    size = L.lib().sb200_orthogonalize_workspace
    for rows, cols in ((128, 4097), (45, 6000), (6000, 100), (1, 5000)):
        assert size(rows, cols, 2, L.BF16) == size(rows, cols, 2, L.F32)
    assert size(129, 4097, 2, L.BF16) < size(129, 4097, 2, L.F32)


@pytest.mark.skipif(torch.cuda.is_available(), reason="would launch on a stand-in context")
def test_valid_calls_reach_the_device_and_fail_there(fake):
    """The checks let these pass: without a device the next thing is a CUDA error."""
    for call in (embedding, embedding_backward, layer_norm, layer_norm_backward, orthogonalize):
        assert call(fake) == L.ERR_CUDA
    assert embedding(fake, tt=L.BF16, ta=L.F32, bits=32) == L.ERR_CUDA
    assert layer_norm(fake, t=L.F16, w=L.F32) == L.ERR_CUDA
    assert orthogonalize(fake, coef=(1.5, -0.5, 0.0), steps=30) == L.ERR_CUDA


def test_front_end_refuses_host_tensors():
    from sapphire_b200 import ops

    class Ctx:
        device, handle = 0, None

    x = torch.zeros(4, 8)
    for call in (lambda: ops.layer_norm(Ctx, x), lambda: ops.embedding(Ctx, x, torch.zeros(3, dtype=torch.int64)),
                 lambda: ops.orthogonalize(Ctx, x), lambda: ops.embedding_backward(Ctx, x, x, torch.zeros(4, dtype=torch.int64))):
        with pytest.raises(ValueError):
            call()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float64])
def test_fp32_calls_refuse_other_types(dtype):
    """What takes fp32 addresses refuses the 16-bit tensors that the token operators produce,
    in every place of its arguments, before the library is called."""
    from sapphire_b200 import conv, ops

    class Ctx:
        device, handle = 0, None

    f, h = torch.zeros(4, 4), torch.zeros(4, 4, dtype=dtype)
    idx = torch.zeros(5, dtype=torch.int32)
    csr, image = ops.CsrMatrix(idx, idx[:0], h[0, :0], 4, 4), torch.zeros(1, 1, 4, 4)
    good = ops.CsrMatrix(idx, idx[:0], f[0, :0], 4, 4)
    for call in (
            lambda: ops.relu(Ctx, h), lambda: ops.relu(Ctx, f, h),
            lambda: ops.relu_backward(Ctx, h, f, f), lambda: ops.relu_backward(Ctx, f, h, f), lambda: ops.relu_backward(Ctx, f, f, h),
            lambda: ops.softmax(Ctx, h), lambda: ops.softmax(Ctx, f, h),
            lambda: ops.softmax_backward(Ctx, h, f, f), lambda: ops.softmax_backward(Ctx, f, h, f), lambda: ops.softmax_backward(Ctx, f, f, h),
            lambda: ops.cross_entropy(Ctx, h, f), lambda: ops.cross_entropy(Ctx, f, h), lambda: ops.cross_entropy(Ctx, f, f, h[0]),
            lambda: ops.cross_entropy_backward(Ctx, h, f, f), lambda: ops.cross_entropy_backward(Ctx, f, h, f),
            lambda: ops.cross_entropy_backward(Ctx, f, f, h),
            lambda: ops.softmax_cross_entropy(Ctx, h, f), lambda: ops.softmax_cross_entropy(Ctx, f, h),
            lambda: ops.softmax_cross_entropy(Ctx, f, f, prob=h), lambda: ops.softmax_cross_entropy(Ctx, f, f, loss=h[0]),
            lambda: ops.softmax_cross_entropy(Ctx, f, f, dlogits=h),
            lambda: ops.sgd_update(Ctx, h, f, 0.1), lambda: ops.sgd_update(Ctx, f, h, 0.1),
            lambda: ops.scale(Ctx, h, 2.0), lambda: ops.scale(Ctx, f, 2.0, h),
            lambda: ops.sum_blocks(Ctx, h, f[None]), lambda: ops.sum_blocks(Ctx, f, h[None]),
            lambda: ops.gemm(Ctx, f, f, bias=h[0]), lambda: ops.gemm(Ctx, f, f, colsum_out=h[0]),
            lambda: ops.dense_to_csr(Ctx, h), lambda: ops.csr_to_dense(Ctx, csr), lambda: ops.csr_to_dense(Ctx, good, h),
            lambda: ops.spgemm(Ctx, csr, good), lambda: ops.spgemm(Ctx, good, csr), lambda: ops.spgemm_callee_alloc(Ctx, csr, good),
            lambda: conv.im2col(Ctx, image.to(dtype), 3, 3), lambda: conv.col2im(Ctx, image.to(dtype), image, 3, 3),
            lambda: conv.col2im(Ctx, image, image.to(dtype), 3, 3)):
        with pytest.raises(TypeError):
            call()
