"""The linear and LayerNorm training launchers between guards: outputs and workspaces of exactly the size asked for lie in
memory that has to stay as it was, inputs in memory full of NaN that must not reach a result.  Results equal the tensor calls'
bit for bit."""
import pytest
import torch
from linear_sizes import SIZES

from forward_amd import lib, ops

pytestmark = pytest.mark.gpu
TYPES = {torch.float32: lib.F32, torch.float16: lib.F16, torch.bfloat16: lib.BF16}
ROOM = 1 << 12                                       # bytes in front of and behind what is used


class Space:
    """`shape` of `dtype` from `shift` elements past a 512-byte boundary on, between bytes of `fill`."""

    def __init__(self, shape, dtype, fill, shift=0):
        size = torch.empty((), dtype=dtype).element_size()
        n = torch.Size(shape).numel()
        self.first, self.bytes = ROOM + shift * size, n * size
        self.all = torch.full((self.first + self.bytes + ROOM,), fill, dtype=torch.uint8, device="cuda")
        self.fill = fill
        self.t = self.all[self.first:self.first + self.bytes].view(dtype).view(shape)

    def ptr(self):
        return self.t.data_ptr()

    def untouched(self):
        return bool((self.all[:self.first] == self.fill).all() and (self.all[self.first + self.bytes:] == self.fill).all())


def held(shape, dtype, g, std=1.0, mean=0.0, shift=0):
    """Normal values between NaN (all bits set are one in every floating type here)."""
    s = Space(shape, dtype, 0xff, shift)
    s.t.copy_(torch.randn(shape, generator=g, device="cuda") * std + mean)
    return s


def room(shape, dtype, shift=0):
    return Space(shape, dtype, 0x5a, shift)


def settle(outputs, names, want):
    torch.cuda.synchronize()
    for name, out, w in zip(names, outputs, want):
        assert out.untouched(), "written around " + name
        if w is not None:
            assert torch.equal(out.t, w), name


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("size", SIZES)
def test_linear(size, dtype):
    m, n, k, on_boundary, with_act = size
    dt, shift = TYPES[dtype], 0 if on_boundary else 1
    g = torch.Generator(device="cuda").manual_seed(m + n + k)
    x, w, r, dy, z = (held(s, dtype, g, shift=shift) for s in ((m, k), (n, k), (m, n), (m, n), (m, n)))
    b = held((n,), torch.float32, g, shift=shift)
    act = lib.ACT_GELU if with_act else lib.ACT_NONE
    name = "gelu" if with_act else "none"

    y, keep = room((m, n), dtype, shift), room((m, n), dtype, shift)
    need = lib.dll.fwdmi_linear_workspace(m, n, k, dt)
    ws = room((need,), torch.uint8)
    lib.check(lib.dll.fwdmi_linear(None, m, n, k, x.ptr(), w.ptr(), b.ptr(), r.ptr(), y.ptr(), keep.ptr(), act, dt,
                                   ws.ptr() if need else None, need))
    settle((y, keep, ws), ("y", "preact", "workspace"),
           ops.linear(x.t, w.t, bias=b.t, activation=name, residual=r.t, want_preact=True) + (None,))
    assert torch.isfinite(y.t).all() and torch.isfinite(keep.t).all()

    need = lib.dll.fwdmi_linear_backward_workspace(m, n, k, act, dt)
    for want_dx, want_dw in ((True, True), (True, False), (False, True)):
        dx, dw, db = room((m, k), dtype, shift), room((n, k), dtype, shift), room((n,), torch.float32, shift)
        ws = room((need,), torch.uint8)
        lib.check(lib.dll.fwdmi_linear_backward(None, m, n, k, dy.ptr(), x.ptr(), w.ptr(), z.ptr() if with_act else None,
                                                dx.ptr() if want_dx else None, dw.ptr() if want_dw else None, db.ptr(), act, dt,
                                                ws.ptr() if need else None, need))
        got = iter(ops.linear_backward(dy.t, x.t, w.t, preact=z.t if with_act else None, activation=name, want_dx=want_dx,
                                       want_dweight=want_dw))
        want = [next(got) if want_dx else None, next(got) if want_dw else None, next(got), None]
        settle((dx, dw, db, ws), ("dx", "dw", "dbias", "workspace"), want)
        for unwanted in ([dx] if not want_dx else []) + ([dw] if not want_dw else []):
            assert (unwanted.all == unwanted.fill).all()
        assert all(torch.isfinite(t).all() for t in want if t is not None)


# every lane layout whole and ragged, rows of more than 16 elements a lane, streamed rows; few rows (one launch) and many
ROWS = [(ld, rows) for ld in (1, 3, 7, 8, 31, 64, 127, 200, 256, 509, 1000, 1024, 1531, 2048, 4097, 8192) for rows in (1, 37, 1100)] + \
       [(ld, rows) for ld in (9999, 12288, 16384, 16401) for rows in (1, 9, 150)]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("ld, rows", ROWS)
def test_layer_norm(ld, rows, dtype):
    dt, n = TYPES[dtype], ld * rows
    g = torch.Generator(device="cuda").manual_seed(ld + rows)
    for bias, extra, shift in ((False, False, 0), (True, True, 1), (False, True, 3)):
        x, skip, dy, dsum = (held((rows, ld), dtype, g, shift=shift) for _ in range(4))
        gamma, beta, b = (held((ld,), torch.float32, g, std=0.3, mean=mean, shift=shift) for mean in (1.0, 0.0, 0.0))
        opt = lambda s, there: s.ptr() if there else None
        some = lambda s, there: s.t if there else None
        y, h = room((rows, ld), dtype, shift), room((rows, ld), dtype, shift)
        mean, rstd = room((rows,), torch.float32, shift), room((rows,), torch.float32, shift)
        lib.check(lib.dll.fwdmi_layer_norm_forward(None, ld, n, x.ptr(), opt(skip, extra), beta.ptr(), gamma.ptr(), opt(b, bias),
                                                   y.ptr(), h.ptr(), mean.ptr(), rstd.ptr(), dt, 1e-5))
        want = ops.layer_norm_forward(x.t, gamma.t, beta.t, skip=some(skip, extra), bias=some(b, bias), eps=1e-5, want_sum=True)
        settle((y, mean, rstd, h), ("y", "mean", "rstd", "sum"), want)
        assert all(torch.isfinite(t).all() for t in want)

        stats = [Space((rows,), torch.float32, 0xff, shift) for _ in range(2)]
        for s, t in zip(stats, want[1:3]):
            s.t.copy_(t)
        dx, dg, dbeta, db = room((rows, ld), dtype, shift), *(room((ld,), torch.float32, shift) for _ in range(3))
        need = lib.dll.fwdmi_layer_norm_backward_workspace(ld, n, bias, dt)
        ws = room((need,), torch.uint8)
        lib.check(lib.dll.fwdmi_layer_norm_backward(None, ld, n, dy.ptr(), x.ptr(), opt(skip, extra), opt(dsum, extra), gamma.ptr(),
                                                    opt(b, bias), stats[0].ptr(), stats[1].ptr(), dx.ptr(), dg.ptr(), dbeta.ptr(),
                                                    opt(db, bias), ws.ptr() if need else None, need, dt))
        want = ops.layer_norm_backward(dy.t, x.t, gamma.t, stats[0].t, stats[1].t, skip=some(skip, extra), bias=some(b, bias),
                                       dsum=some(dsum, extra))
        settle((dx, dg, dbeta, db, ws), ("dx", "dgamma", "dbeta", "dbias", "workspace"), list(want) + [None] * (5 - len(want)))
        if not bias:
            assert (db.all == db.fill).all()
        assert all(torch.isfinite(t).all() for t in want)
