"""gsp_rms_norm and gsp_quantize_fp8 against their formulas in 64 bits.

Tolerances.  A thread adds at most 32 squares one after the other (rows past 32768 values: dim / 1024) and
the workgroup's sums meet in 6 + 16 steps, so a mean of squares is off by less than (32 + 22 + 2) 2^-24
relatively (or dim / 1024 + 24), its root's inverse by half of that and two roundings, y by two more: under 40
steps of 2^-24 for the rows here.  The gated SiLU is one exponential (2 steps), an addition, a division and a
product.  Codes: fp8_helpers.check_codes.
"""
import numpy as np
import pytest

from fp8_helpers import E4M3, check_codes, norm64

pytestmark = pytest.mark.gpu
EPS24 = 2.0 ** -24

# (rows, dim): one value, less than a wave, odd lengths, every register count of both access widths, past
# the registers; single rows, many rows.
SHAPES = [(1, 1), (3, 2), (5, 63), (2, 64), (1, 896), (64, 3584), (7, 1001), (3, 4098), (9, 4096), (600, 2050),
          (700, 1024), (520, 8192), (513, 16384), (2, 16387), (3, 18944), (515, 18945), (2, 32768), (2, 32767),
          (2, 32769), (1, 50000)]
GUARD = 64


def _dev(torch, a, offset=0):
    """`a` on the device, `offset` elements behind an aligned start."""
    flat = np.concatenate([np.zeros(offset, a.dtype), a.reshape(-1)])
    return torch.from_numpy(flat).cuda()[offset:].view(a.shape)


class Out:
    """An output with sentinels on both sides of what the call may write."""

    def __init__(self, torch, shape, dtype, offset=0):
        n = int(np.prod(shape))
        self.buf = torch.full((GUARD + offset + n + GUARD,), 77, dtype=dtype, device="cuda")
        self.lo, self.shape = GUARD + offset, shape
        self.ptr = self.buf[self.lo:].data_ptr()

    def get(self):
        b = self.buf.cpu().numpy()
        n = int(np.prod(self.shape))
        assert np.all(b[: self.lo] == 77) and np.all(b[self.lo + n:] == 77)
        return b[self.lo: self.lo + n].reshape(self.shape)


def _norm_tol(dim):
    return (max(32, dim / 1024) / 2 + 24) * EPS24


def _case(rng, rows, dim, residual=True):
    x = rng.standard_normal((rows, dim)).astype(np.float32) * rng.choice([1e-3, 1.0, 50.0], (rows, 1)).astype(np.float32)
    x[:, rng.integers(0, dim)] *= 12
    r = (rng.standard_normal((rows, dim)) * 5).astype(np.float32) if residual else None
    w = (1 + 0.2 * rng.standard_normal(dim)).astype(np.float32)
    return x, r, w


def _check_norm(x, r, w, eps, total, y, codes, scale):
    s, want = norm64(x, r, w, eps)
    rel = _norm_tol(x.shape[1])
    if total is not None:
        assert np.array_equal(total, s)
    if y is not None:
        assert np.all(np.abs(y - want) <= rel * np.abs(want) + 1e-44)
    if codes is not None:
        check_codes(codes, scale, want, rel)


@pytest.mark.parametrize("outs", ["all", "fp8", "f32", "plain"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: f"{s[0]}x{s[1]}")
def test_norm(torch_mod, ctx, shape, outs):
    torch = torch_mod
    print(f"case norm {shape} {outs}", flush=True)
    rows, dim = shape
    rng = np.random.default_rng(rows * 131 + dim)
    x, r, w = _case(rng, rows, dim, outs != "plain")
    xd, wd = _dev(torch, x), _dev(torch, w)
    rd = _dev(torch, r) if r is not None else None
    total = Out(torch, shape, torch.float32) if outs == "all" else None
    y = Out(torch, shape, torch.float32) if outs in ("all", "f32") else None
    codes = Out(torch, shape, torch.uint8) if outs != "f32" else None
    scale = Out(torch, (rows,), torch.float32) if outs != "f32" else None
    at = lambda o: o.ptr if o is not None else 0  # noqa: E731
    torch.cuda.synchronize()
    ctx.rms_norm(rows, dim, xd.data_ptr(), wd.data_ptr(), 1e-5, residual_ptr=rd.data_ptr() if rd is not None else 0,
                 sum_ptr=at(total), y_ptr=at(y), y_fp8_ptr=at(codes), y_scale_ptr=at(scale))
    ctx.sync()
    got = [o.get() if o is not None else None for o in (total, y, codes, scale)]
    _check_norm(x, r, w, 1e-5, *got)


@pytest.mark.parametrize("shape", [(5, 896), (600, 1024), (3, 40000), (4, 1001)], ids=str)
@pytest.mark.parametrize("alias", ["sum=x", "sum=residual", "y=x", "y=residual", "sum=x,y=residual", "sum=residual,y=x"])
def test_norm_in_place(torch_mod, ctx, shape, alias):
    torch = torch_mod
    rows, dim = shape
    x, r, w = _case(np.random.default_rng(dim), rows, dim)
    d = {"x": _dev(torch, x), "residual": _dev(torch, r)}
    put = dict(p.split("=") for p in alias.split(","))
    for o in ("sum", "y"):
        d[o] = d[put[o]] if o in put else torch.zeros(shape, device="cuda")
    codes = torch.zeros(shape, dtype=torch.uint8, device="cuda")
    scale = torch.zeros(rows, device="cuda")
    wd = _dev(torch, w)
    torch.cuda.synchronize()
    ctx.rms_norm(rows, dim, d["x"].data_ptr(), wd.data_ptr(), 1e-6, residual_ptr=d["residual"].data_ptr(),
                 sum_ptr=d["sum"].data_ptr(), y_ptr=d["y"].data_ptr(), y_fp8_ptr=codes.data_ptr(),
                 y_scale_ptr=scale.data_ptr())
    ctx.sync()
    _check_norm(x, r, w, 1e-6, d["sum"].cpu().numpy(), d["y"].cpu().numpy(), codes.cpu().numpy(), scale.cpu().numpy())


@pytest.mark.parametrize("which", ["x", "residual", "weight", "sum", "y", "codes", "scale"])
def test_norm_of_unaligned_buffers(torch_mod, ctx, which):
    """4-byte aligned fp32 buffers (codes: any address) give the same as aligned ones."""
    torch = torch_mod
    rows, dim = 6, 1024
    x, r, w = _case(np.random.default_rng(9), rows, dim)
    off = lambda name: 1 if name == which else 0  # noqa: E731
    xd, rd, wd = _dev(torch, x, off("x")), _dev(torch, r, off("residual")), _dev(torch, w, off("weight"))
    total, y = Out(torch, x.shape, torch.float32, off("sum")), Out(torch, x.shape, torch.float32, off("y"))
    codes, scale = Out(torch, x.shape, torch.uint8, off("codes")), Out(torch, (rows,), torch.float32, off("scale"))
    torch.cuda.synchronize()
    ctx.rms_norm(rows, dim, xd.data_ptr(), wd.data_ptr(), 0.0, residual_ptr=rd.data_ptr(), sum_ptr=total.ptr,
                 y_ptr=y.ptr, y_fp8_ptr=codes.ptr, y_scale_ptr=scale.ptr)
    ctx.sync()
    _check_norm(x, r, w, 0.0, total.get(), y.get(), codes.get(), scale.get())


@pytest.mark.parametrize("dim", [256, 257, 40000])
def test_norm_of_special_rows(torch_mod, ctx, dim):
    """Zero rows, rows of one value, subnormal rows, infinities and NaN; no row touches another."""
    torch = torch_mod
    x = np.random.default_rng(3).standard_normal((7, dim)).astype(np.float32)
    x[0] = 0
    x[1] = 0
    x[1, dim - 1] = 3e-39
    x[2] *= 1e-30
    x[3, 5] = np.inf
    x[4, dim // 2] = np.nan
    w = np.ones(dim, np.float32)
    w[0] = 0
    y, codes = Out(torch, x.shape, torch.float32), Out(torch, x.shape, torch.uint8)
    scale = Out(torch, (7,), torch.float32)
    xd, wd = _dev(torch, x), _dev(torch, w)
    torch.cuda.synchronize()
    ctx.rms_norm(7, dim, xd.data_ptr(), wd.data_ptr(), 1e-6, y_ptr=y.ptr, y_fp8_ptr=codes.ptr, y_scale_ptr=scale.ptr)
    ctx.sync()
    y, codes, scale = y.get(), codes.get(), scale.get()
    fine = [0, 1, 2, 5, 6]
    _check_norm(x[fine], None, w, 1e-6, None, y[fine], codes[fine], scale[fine])
    assert np.all(E4M3[codes[0]] == 0) and scale[0] > 0
    # 1 / sqrt(inf) is 0: finite values go to 0, infinity and NaN to NaN.
    assert np.isnan(y[3, 5]) and not np.any(np.delete(y[3], 5)) and np.isnan(scale[3])
    assert np.all(np.isnan(y[4])) and np.isnan(scale[4])


def _silu64(a, b):
    a = a.astype(np.float64)
    return a / (1 + np.exp(-a)) * b.astype(np.float64)


@pytest.mark.parametrize("act", ["none", "silu"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: f"{s[0]}x{s[1]}")
def test_quantize(torch_mod, gsp, ctx, shape, act):
    torch = torch_mod
    print(f"case quantize {shape} {act}", flush=True)
    rows, dim = shape
    rng = np.random.default_rng(rows * 17 + dim)
    for pad, offset in ((0, 0), (4 - dim % 4, 0), (3, 1)):
        halves = 2 if act == "silu" else 1
        a = (rng.standard_normal((rows, halves * dim + pad)) * 3).astype(np.float32)
        a[:, dim // 2] = -150.0  # exp overflows: the gate is -0
        ad = _dev(torch, a, offset)
        codes, scale = Out(torch, shape, torch.uint8), Out(torch, (rows,), torch.float32)
        torch.cuda.synchronize()
        ctx.quantize_fp8(gsp.ACT_SILU_MUL if act == "silu" else gsp.ACT_NONE, rows, dim, a.shape[1], ad.data_ptr(),
                         ad.data_ptr() + 4 * dim if act == "silu" else 0, codes.ptr, scale.ptr)
        ctx.sync()
        y = _silu64(a[:, :dim], a[:, dim: 2 * dim]) if act == "silu" else a[:, :dim].astype(np.float64)
        check_codes(codes.get(), scale.get(), y, 8 * EPS24 if act == "silu" else 0.0)


def test_quantize_special_rows(torch_mod, gsp, ctx):
    torch = torch_mod
    a = np.random.default_rng(4).standard_normal((8, 320)).astype(np.float32)
    a[0] = 0
    a[1] = 0
    a[1, 7] = 1e-45
    a[2] *= np.float32(2.0 ** -110)
    a[3] = -3e38
    a[4, 9] = np.nan
    a[5, 9] = -np.inf
    a[6, :] = np.float32(2.0 ** -100) * np.linspace(-1, 1, 320, dtype=np.float32)
    ad = _dev(torch, a)
    codes, scale = Out(torch, a.shape, torch.uint8), Out(torch, (8,), torch.float32)
    torch.cuda.synchronize()
    ctx.quantize_fp8(gsp.ACT_NONE, 8, 320, 320, ad.data_ptr(), 0, codes.ptr, scale.ptr)
    ctx.sync()
    codes, scale = codes.get(), scale.get()
    fine = [0, 1, 2, 3, 6, 7]
    check_codes(codes[fine], scale[fine], a[fine].astype(np.float64), 0.0)
    assert np.all(E4M3[codes[0]] == 0) and np.all(E4M3[codes[3]] == -448)
    assert np.isnan(scale[4]) and np.isnan(E4M3[codes[4, 9]])
    assert np.isinf(scale[5]) and np.isnan(E4M3[codes[5, 9]])


def test_quantize_ties_go_to_even(torch_mod, gsp, ctx):
    """With 448 in the row the factor is 1: every e4m3 value stays, every middle goes to the even code."""
    torch = torch_mod
    pos = E4M3[:127]
    mids = (pos[:-1] + pos[1:]) / 2
    a = np.concatenate([pos, -pos, mids, -mids]).astype(np.float32)[None]
    ad = _dev(torch, a)
    codes = torch.zeros(a.shape, dtype=torch.uint8, device="cuda")
    scale = torch.zeros(1, device="cuda")
    torch.cuda.synchronize()
    ctx.quantize_fp8(gsp.ACT_NONE, 1, a.shape[1], a.shape[1], ad.data_ptr(), 0, codes.data_ptr(), scale.data_ptr())
    ctx.sync()
    got = codes.cpu().numpy()[0]
    even = np.array([c if c % 2 == 0 else c + 1 for c in range(126)])
    assert scale.item() == 1.0
    assert np.array_equal(E4M3[got[:127]], pos) and np.array_equal(E4M3[got[127:254]], -pos)
    assert np.array_equal(E4M3[got[254:380]], E4M3[even]) and np.array_equal(E4M3[got[380:]], -E4M3[even])
