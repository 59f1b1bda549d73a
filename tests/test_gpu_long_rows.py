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
