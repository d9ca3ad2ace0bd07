"""The training operators' refusals, which come before any device is touched: C entry points on made-up addresses,
and the Python binding on CPU tensors.  A context that was never created stands in (zeroed memory): the calls
below are all refused before it is looked at."""
import ctypes
import math

import pytest
import torch

INVALID, UNSUPPORTED, TOO_LARGE = -1, -3, -6


@pytest.fixture(scope="module")
def lib():
    from gern_b200 import api
    return api.lib


@pytest.fixture(scope="module")
def fake():
    buf = ctypes.create_string_buffer(1 << 16)
    return ctypes.addressof(buf), buf


A, B, C, D, E = (0x10000000 * i for i in range(1, 6))   # operands far apart


def refused(lib, rc, code, text):
    assert rc == code, lib.gb200_last_error_string()
    assert text in lib.gb200_last_error_string().decode()


def norm_args(**kw):
    a = dict(x=A, ldx=64, res=B, ldr=64, w=C, y=D, ldy=64, h=E, ldh=64, rows=10, cols=64, eps=1e-6)
    a.update(kw)
    return [a[k] for k in ("x", "ldx", "res", "ldr", "w", "y", "ldy", "h", "ldh", "rows", "cols", "eps")]


@pytest.mark.parametrize("kw,text", [
    (dict(rows=-1), "negative extent"), (dict(eps=-1e-6), "eps"), (dict(eps=math.nan), "eps"), (dict(eps=math.inf), "eps"),
    (dict(x=None), "NULL"), (dict(w=None), "NULL"), (dict(y=None), "NULL"), (dict(ldx=63), "leading dimension"),
    (dict(ldr=0), "leading dimension"), (dict(ldh=10), "leading dimension"), (dict(x=A + 1), "aligned"),
    (dict(y=A + 4), "overlaps"), (dict(y=A, ldy=128), "overlaps"), (dict(y=D, h=D), "overlaps"), (dict(y=C), "overlaps")])
def test_rmsnorm(lib, fake, kw, text):
    for name in ("gb200_rmsnorm_f32", "gb200_rmsnorm_bf16"):
        refused(lib, getattr(lib, name)(fake[0], *norm_args(**kw), None), INVALID, text)
        refused(lib, getattr(lib, name)(None, *norm_args(), None), INVALID, "ctx is NULL")


def test_rmsnorm_too_large(lib, fake):
    refused(lib, lib.gb200_rmsnorm_f32(fake[0], *norm_args(cols=1 << 31), None), TOO_LARGE, "columns")
    refused(lib, lib.gb200_rmsnorm_f32(fake[0], *norm_args(rows=1 << 62), None), TOO_LARGE, "does not fit")


@pytest.mark.parametrize("group,scales,lds,code,text", [
    (48, E, 10, UNSUPPORTED, "group"), (-32, E, 10, UNSUPPORTED, "group"), (32, None, 2, INVALID, "scales is NULL"),
    (32, E, 1, INVALID, "scales"), (32, A, 2, INVALID, "overlaps"), (32, E + 2, 2, INVALID, "aligned")])
def test_rmsnorm_e4m3(lib, fake, group, scales, lds, code, text):
    for name in ("gb200_rmsnorm_f32_e4m3", "gb200_rmsnorm_bf16_e4m3"):
        rc = getattr(lib, name)(fake[0], A, 64, B, 64, C, D, 64, scales, lds, None, 0, 10, 64, group, 1e-6, None)
        refused(lib, rc, code, text)


@pytest.mark.parametrize("kw,text", [
    (dict(dy=None), "NULL"), (dict(dx=None), "NULL"), (dict(lddx=3), "leading dimension"), (dict(dx=A + 8), "overlaps"),
    (dict(dw=A), "overlaps"), (dict(dw=E + 2), "aligned"), (dict(dx=C), "overlaps")])
def test_rmsnorm_backward(lib, fake, kw, text):
    a = dict(dy=A, lddy=64, h=B, ldh=64, w=C, dres=None, lddr=0, dx=D, lddx=64, dw=E, acc=0, rows=10, cols=64, eps=1e-6)
    a.update(kw)
    for name in ("gb200_rmsnorm_backward_f32", "gb200_rmsnorm_backward_bf16"):
        refused(lib, getattr(lib, name)(fake[0], *a.values(), None), INVALID, text)


@pytest.mark.parametrize("kw,code,text", [
    (dict(T=-1), INVALID, "negative"), (dict(V=0), INVALID, "no classes"), (dict(D=0), INVALID, "without elements"),
    (dict(V=1 << 27), TOO_LARGE, "2^26"), (dict(h=None), INVALID, "NULL"), (dict(t=None), INVALID, "NULL"),
    (dict(ldh=63), INVALID, "leading dimension"), (dict(ldw=63), INVALID, "leading dimension"), (dict(h=A + 1), INVALID, "aligned"),
    (dict(t=C + 4), INVALID, "aligned"), (dict(loss=None, lse=None, total=None), INVALID, "nothing to produce"),
    (dict(loss=A), INVALID, "overlaps"), (dict(lse=D + 8), INVALID, "overlaps"), (dict(total=E + 2), INVALID, "aligned")])
def test_linear_xent(lib, fake, kw, code, text):
    a = dict(h=A, ldh=64, w=B, ldw=64, t=C, T=10, V=100, D=64, ignore=-100, loss=D, lse=D + 4096, total=E)
    a.update(kw)
    refused(lib, lib.gb200_linear_xent_bf16(fake[0], *a.values(), None), code, text)
    refused(lib, lib.gb200_linear_xent_bf16(None, *a.values(), None), INVALID, "ctx is NULL")


@pytest.mark.parametrize("kw,text", [
    (dict(dh=None, dw=None), "nothing to produce"), (dict(dloss=None, total=None), "either dloss"), (dict(total=E + 64), "either dloss"),
    (dict(lse=None), "lse is NULL"), (dict(lddh=3), "leading dimension"), (dict(lddw=3), "leading dimension"), (dict(dh=A), "overlaps"),
    (dict(dw=B + 128), "overlaps"), (dict(dw=D + 0x800000), "overlaps"), (dict(dh=E - 128), "overlaps")])
def test_linear_xent_backward(lib, fake, kw, text):
    a = dict(h=A, ldh=64, w=B, ldw=64, t=C, lse=C + 4096, dloss=E, total=None, T=10, V=100, D=64, ignore=-100, scale=1.0,
             dh=D + 0x800000, lddh=64, dw=D, lddw=64)
    a.update(kw)
    refused(lib, lib.gb200_linear_xent_bf16_backward(fake[0], *a.values(), None), INVALID, text)


def tensors(*rows):
    from gern_b200 import api  # noqa: F401
    import struct
    return struct.pack("QQqii" * len(rows), *[v for r in rows for v in r]), len(rows)


@pytest.mark.parametrize("rows,code,text", [
    ([(A, 0, 100, 7, 0)], UNSUPPORTED, "element type"), ([(0, 0, 100, 0, 0)], INVALID, "NULL"),
    ([(A + 2, 0, 100, 0, 0)], INVALID, "aligned"), ([(A, 0, -1, 0, 0)], INVALID, "elements"),
    ([(A, B + 1, 100, 1, 1)], INVALID, "aligned"), ([(A, B, 100, 0, 1)], UNSUPPORTED, "fp32 result"),
    ([(A, 0, 100, 0, 0), (A, 0, 100, 0, 0)], INVALID, "overlaps"), ([(A, 0, 100, 0, 0), (A + 396, 0, 5, 0, 0)], INVALID, "overlaps"),
    ([(A, A, 100, 1, 0)], INVALID, "overlaps"), ([(A, B, 100, 0, 0), (B, C, 100, 0, 0)], INVALID, "overlaps"),
    ([(E - 396, 0, 100, 0, 0)], INVALID, "overlaps")])
def test_grad_clip(lib, fake, rows, code, text):
    buf, n = tensors(*rows)
    refused(lib, lib.gb200_grad_clip(fake[0], buf, n, 1.0, E, None), code, text)


def test_grad_clip_scalars(lib, fake):
    buf, n = tensors((A, 0, 100, 0, 0))
    refused(lib, lib.gb200_grad_clip(fake[0], buf, n, -1.0, E, None), INVALID, "max_norm")
    refused(lib, lib.gb200_grad_clip(fake[0], buf, n, math.nan, E, None), INVALID, "max_norm")
    refused(lib, lib.gb200_grad_clip(fake[0], buf, n, 1.0, None, None), INVALID, "norm is NULL")
    refused(lib, lib.gb200_grad_norm(fake[0], None, 1, E, None), INVALID, "tensors is NULL")
    refused(lib, lib.gb200_grad_norm(fake[0], buf, -1, E, None), INVALID, "negative number")
    refused(lib, lib.gb200_grad_norm(None, buf, n, E, None), INVALID, "ctx is NULL")


def test_python_binding_refuses_cpu_tensors_wrong_types_and_shapes():
    from gern_b200 import api
    ctx = api.Context.__new__(api.Context)       # no device: every call below is refused before the library is called
    ctx.handle, ctx.device = None, 0
    x, w = torch.zeros(4, 8), torch.zeros(8)
    with pytest.raises(ValueError, match="context's device"):
        ctx.rmsnorm(x, w, x.clone(), 1e-6)
    with pytest.raises(TypeError, match="bfloat16"):
        ctx.rmsnorm(x.half(), w, x, 1e-6)
    with pytest.raises(ValueError, match="4 x 8"):
        ctx.rmsnorm_backward(x[:3], x, w, x, None, 1e-6)
    with pytest.raises(TypeError, match="bfloat16"):
        ctx.linear_xent(x, w[None], torch.zeros(4, dtype=torch.int64), w[:4], w[:4])
    with pytest.raises(ValueError, match="contiguous fp32 or bf16"):
        ctx.grad_clip([x], 1.0, _Cuda())


class _Cuda:
    """Stands in for a one-element fp32 vector on the device."""
    dtype, shape = torch.float32, (1,)

    def dim(self):
        return 1

    def get_device(self):
        return 0


@pytest.mark.parametrize("kw", [
    dict(y=A + 4 * 63), dict(y=A + 4 * 160 - 4), dict(y=A + 4 * 97), dict(y=A + 4 * 160 * 4 + 4 * 40),
    dict(y=A + 4 * 64, ldy=161), dict(h=D + 4 * 60), dict(y=A - 4 * 63), dict(y=A - 4 * 97), dict(w=A + 4 * 160 * 3 + 4 * 97, y=A + 4 * 64)])
def test_columns_of_one_buffer_that_share_bytes(lib, fake, kw):
    """Rows of one pitch whose columns cross, at either end or across a row's end into the next; other pitches.  (A case
    that ends beside its neighbours without crossing them is taken: those run on the GPU.)"""
    a = dict(ldx=160, ldy=160, ldh=160, ldr=160, cols=64)
    a.update(kw)
    refused(lib, lib.gb200_rmsnorm_f32(fake[0], *norm_args(**a), None), INVALID, "overlaps")
