"""gsp_rms_norm and gsp_quantize_fp8 on rows that one workgroup's registers do not hold."""
import numpy as np
import pytest

from fp8_helpers import E4M3

pytestmark = pytest.mark.gpu


def test_the_longest_row(torch_mod, gsp, ctx):
    """dim 2^31 - 1: a thread's place passes 2^31 behind its last value.  Zeros but for a few values, so that every
    result is known: with 448 in the row a code is the value itself."""
    torch = torch_mod
    dim = 2 ** 31 - 1
    print(f"case longest row {dim}", flush=True)
    places = [0, 1, 1023, 1024, 2 ** 30, dim - 1025, dim - 1024, dim - 2, dim - 1]
    values = np.array([448, -2, 3, 0.5, -448, 64, 1, -26, 7], np.float32)
    x = torch.zeros(dim + 64, device="cuda")
    x[dim:] = 9.0
    at = torch.tensor(places, device="cuda")
    x[at] = torch.from_numpy(values).cuda()
    codes = torch.zeros(dim + 64, dtype=torch.uint8, device="cuda")
    codes[dim:] = 77
    scale = torch.zeros(1, device="cuda")
    torch.cuda.synchronize()
    ctx.quantize_fp8(gsp.ACT_NONE, 1, dim, dim, x.data_ptr(), 0, codes.data_ptr(), scale.data_ptr())
    ctx.sync()
    assert scale.item() == 1.0
    assert np.array_equal(E4M3[codes[at].cpu().numpy()], values)
    assert torch.count_nonzero(codes[:dim]).item() == len(places) and torch.all(codes[dim:] == 77)
    # y over x, with weight 1: f = 1 / sqrt(sum of squares / dim), and the codes are the same.
    codes[:dim] = 0
    w = torch.ones(dim, device="cuda")
    torch.cuda.synchronize()
    ctx.rms_norm(1, dim, x.data_ptr(), w.data_ptr(), 0.0, y_ptr=x.data_ptr(), y_fp8_ptr=codes.data_ptr(),
                 y_scale_ptr=scale.data_ptr())
    ctx.sync()
    want = values / np.sqrt(np.sum(values.astype(np.float64) ** 2) / dim)
    # nine squares are added exactly in 32 bits; the mean, the root, its inverse and two products round once each
    assert np.all(np.abs(x[at].cpu().numpy() - want) <= 6 * 2.0 ** -24 * np.abs(want))
    assert np.array_equal(E4M3[codes[at].cpu().numpy()], values)
    assert torch.count_nonzero(x[:dim]).item() == len(places) and torch.all(x[dim:] == 9.0)
    assert torch.all(codes[dim:] == 77)
    del x, codes, w
    torch.cuda.empty_cache()


def _rows64(x, w, eps):
    """y in 64 bits on the device."""
    d = x.double()
    return d / (d.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()


@pytest.mark.parametrize("value", [None, 1.1, 0.3], ids=["random", "1.1", "0.3"])
def test_sums_of_long_rows(torch_mod, ctx, value):
    """A thread adds dim / 1024 squares; with equal values every addition can round the same way.

    The squares, their sum and the root hold 64 bits, so y is off by its two roundings and the factor's: 3 steps."""
    torch = torch_mod
    rows, dim = 2, (1 << 24) + 3
    g = torch.Generator(device="cuda").manual_seed(5)
    x = torch.randn((rows, dim), generator=g, device="cuda") if value is None else torch.full((rows, dim), value, device="cuda")
    w = 1 + 0.2 * torch.randn(dim, generator=g, device="cuda")
    y, codes = torch.zeros_like(x), torch.zeros((rows, dim), dtype=torch.uint8, device="cuda")
    scale = torch.zeros(rows, device="cuda")
    torch.cuda.synchronize()
    ctx.rms_norm(rows, dim, x.data_ptr(), w.data_ptr(), 1e-5, y_ptr=y.data_ptr(), y_fp8_ptr=codes.data_ptr(),
                 y_scale_ptr=scale.data_ptr())
    ctx.sync()
    want = _rows64(x, w, float(np.float32(1e-5)))
    worst = ((y.double() - want).abs() / want.abs().clamp(min=1e-30)).max().item()
    print(f"largest error {worst * 2 ** 24:.1f} steps", flush=True)
    assert worst <= 3 * 2.0 ** -24
    top = want.abs().amax(-1)
    assert ((scale.double() - top / 448).abs() <= 5 * 2.0 ** -24 * top / 448).all()


@pytest.mark.parametrize("dim", [32769, 40000])
@pytest.mark.parametrize("eps", [0.0, 1e-6, 1e-42])
def test_range_of_long_rows(torch_mod, ctx, dim, eps):
    """Rows whose squares leave fp32: y is off by 3 steps, or a few of the least subnormals."""
    torch = torch_mod
    mags = [2.0 ** -140, 2.0 ** -100, 1e-24, 1e-19, 1.0, 2.0 ** 59, 2.0 ** 64, 2.0 ** 100, 2.0 ** 124]
    g = torch.Generator(device="cuda").manual_seed(6)
    x = torch.randn((len(mags), dim), generator=g, device="cuda").double() * torch.tensor(mags, dtype=torch.float64, device="cuda")[:, None]
    x = x.float()
    assert torch.isfinite(x).all()
    w = 1 + 0.2 * torch.randn(dim, generator=g, device="cuda")
    y = torch.zeros_like(x)
    torch.cuda.synchronize()
    ctx.rms_norm(len(mags), dim, x.data_ptr(), w.data_ptr(), eps, y_ptr=y.data_ptr())
    ctx.sync()
    want = _rows64(x, w, float(np.float32(eps)))
    off = (y.double() - want).abs()
    print([f"{(o / t.abs().clamp(min=1e-44)).max().item():.2g}" for o, t in zip(off, want)], flush=True)
    assert (off <= 3 * 2.0 ** -24 * want.abs() + 4 * 2.0 ** -149).all()
