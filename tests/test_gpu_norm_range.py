"""gsp_rms_norm on rows whose squares leave fp32's range, up to the lengths that a workgroup's registers hold.

The formula has no trouble there: y is about 1 whatever the row's magnitude, unless eps is larger.  A sum of squares is
off by at most 32 + 22 steps of 2^-24, its root's inverse by half of that, and y by a few more roundings, also where the
row was scaled by a power of two before: 40 steps in all.  Results below 2^-126 are off by a few of the least subnormals.
"""
import numpy as np
import pytest

from fp8_helpers import check_codes, norm64

pytestmark = pytest.mark.gpu
REL = 40 * 2.0 ** -24
MAGS = [2.0 ** -149, 2.0 ** -140, 2.0 ** -126, 2.0 ** -100, 1e-24, 2.0 ** -63, 1e-19, 1e-10, 1.0, 1e10, 2.0 ** 52, 2.0 ** 59,
        2.0 ** 63, 2.0 ** 64, 2.0 ** 100, 2.0 ** 125]


def _run(torch, ctx, x, r, w, eps):
    rows, dim = x.shape
    dev = lambda a: torch.from_numpy(a).cuda()  # noqa: E731
    xd, rd, wd = dev(x), dev(r) if r is not None else None, dev(w)
    y, total = torch.full((rows, dim), 77.0, device="cuda"), torch.full((rows, dim), 77.0, device="cuda")
    codes, scale = torch.zeros((rows, dim), dtype=torch.uint8, device="cuda"), torch.zeros(rows, device="cuda")
    torch.cuda.synchronize()
    ctx.rms_norm(rows, dim, xd.data_ptr(), wd.data_ptr(), eps, residual_ptr=rd.data_ptr() if r is not None else 0,
                 sum_ptr=total.data_ptr() if r is not None else 0, y_ptr=y.data_ptr(), y_fp8_ptr=codes.data_ptr(),
                 y_scale_ptr=scale.data_ptr())
    ctx.sync()
    return [t.cpu().numpy() for t in (total, y, codes, scale)]


def _check(x, r, w, eps, total, y, codes, scale):
    s, want = norm64(x, r, w, eps)
    if r is not None:
        assert np.array_equal(total, s)
    off = np.abs(y - want)
    assert np.all(off <= REL * np.abs(want) + 4 * 2.0 ** -149), [i for i in range(len(x)) if not np.all(off[i] <= REL * np.abs(want[i]) + 4 * 2.0 ** -149)]
    check_codes(codes, scale, want, REL)


@pytest.mark.parametrize("eps", [0.0, 1e-42, 1e-6, 1e30])
@pytest.mark.parametrize("dim", [1, 4, 63, 256, 1001, 4096, 16387, 18944, 32768])
def test_rows_of_every_magnitude(torch_mod, ctx, dim, eps):
    """Random rows and rows of equal values, one magnitude a row, beside ordinary ones."""
    print(f"case norm range {dim} {eps}", flush=True)
    rng = np.random.default_rng(dim)
    x = np.concatenate([rng.standard_normal((len(MAGS), dim)) * 0.5, np.ones((len(MAGS), dim))]) * np.array(MAGS * 2)[:, None]
    x = x.astype(np.float32)
    if eps == 0.0:
        x = x[np.any(x != 0, 1)]  # a row of zeros is 0 / 0
    w = (1 + 0.2 * rng.standard_normal(dim)).astype(np.float32)
    got = _run(torch_mod, ctx, x, None, w, eps)
    _check(x, None, w, eps, *got)


@pytest.mark.parametrize("dim", [256, 1001, 8192])
def test_rows_of_mixed_magnitudes(torch_mod, ctx, dim):
    """One value far above or below the others, and a sum with the residual that cancels: the sum comes out unscaled."""
    rng = np.random.default_rng(dim + 1)
    x = rng.standard_normal((6, dim)).astype(np.float32)
    r = rng.standard_normal((6, dim)).astype(np.float32)
    x[0, 3] = 2.0 ** 126
    x[1] *= np.float32(2.0 ** -120)
    r[1] = 0
    x[1, dim - 1] = 2.0 ** -70
    x[2] *= np.float32(2.0 ** 70)
    r[2] = -x[2] * np.float32(1 - 2.0 ** -20)
    x[3], r[3] = np.float32(1.5e38), np.float32(1.5e38)
    x[4] *= np.float32(2.0 ** 63)
    for eps in (0.0, 1e-6):
        _check(x, r, np.ones(dim, np.float32), eps, *_run(torch_mod, ctx, x, r, np.ones(dim, np.float32), eps))


@pytest.mark.parametrize("dim", [64, 1001, 4096])
def test_what_has_no_norm(torch_mod, ctx, dim):
    """Zeros with eps 0, an infinity, a sum that overflows, a NaN: NaN and 0 as in the formula, and nothing in other rows."""
    x = np.ones((5, dim), np.float32)
    r = np.zeros((5, dim), np.float32)
    x[0] = 0
    x[1, 7] = -np.inf
    x[2, 7], r[2, 7] = 3e38, 3e38
    x[3, 7] = np.nan
    total, y, codes, scale = _run(torch_mod, ctx, x, r, np.ones(dim, np.float32), 0.0)
    assert np.all(np.isnan(y[0])) and np.isnan(scale[0])
    for i in (1, 2):
        assert np.isnan(y[i, 7]) and not np.any(np.delete(y[i], 7)) and np.isnan(scale[i])
    assert np.all(np.isnan(y[3])) and np.isnan(scale[3])
    assert np.all(np.abs(y[4] - 1) <= REL) and abs(scale[4] * 448 - 1) <= 2 * REL
