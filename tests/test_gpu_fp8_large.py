"""The 8-bit operators where offsets pass 32 bits: the last rows of buffers of several GB."""
import numpy as np
import pytest

from fp8_helpers import E4M3, Q4_0, Q4_1, check_codes, decode_weights, norm64, random_weights

pytestmark = pytest.mark.gpu


def _free(torch):
    torch.cuda.empty_cache()


def test_norm_and_quantiser(torch_mod, gsp, ctx):
    torch = torch_mod
    rows, dim = 80001, 32768  # 2.6e9 values, 10.5 GB
    x = torch.zeros((rows, dim), device="cuda")
    tail = np.random.default_rng(1).standard_normal((3, dim)).astype(np.float32)
    x[-3:] = torch.from_numpy(tail).cuda()
    w = torch.ones(dim, device="cuda")
    codes = torch.full((rows, dim), 77, dtype=torch.uint8, device="cuda")
    scale = torch.zeros(rows, device="cuda")
    torch.cuda.synchronize()
    ctx.rms_norm(rows, dim, x.data_ptr(), w.data_ptr(), 1e-6, y_ptr=x.data_ptr(), y_fp8_ptr=codes.data_ptr(),
                 y_scale_ptr=scale.data_ptr())
    ctx.sync()
    _, y = norm64(tail, None, np.ones(dim, np.float32), 1e-6)
    check_codes(codes[-3:].cpu().numpy(), scale[-3:].cpu().numpy(), y, 40 * 2.0 ** -24)
    assert not codes[: rows - 3].any() and not x[: rows - 3].any()
    got = x[-3:].cpu().numpy()
    codes.fill_(77)
    torch.cuda.synchronize()
    ctx.quantize_fp8(gsp.ACT_SILU_MUL, rows, dim // 2, dim, x.data_ptr(), x.data_ptr() + 2 * dim, codes.data_ptr(),
                     scale.data_ptr())
    ctx.sync()
    g, u = got[:, : dim // 2].astype(np.float64), got[:, dim // 2:].astype(np.float64)
    flat = codes.view(-1)
    n = rows * (dim // 2)
    check_codes(flat[n - 3 * (dim // 2): n].view(3, -1).cpu().numpy(), scale[-3:].cpu().numpy(), g / (1 + np.exp(-g)) * u,
                8 * 2.0 ** -24)
    assert torch.all(flat[n: n + 4096] == 77) and torch.all(flat[-4096:] == 77)
    del x, codes, flat
    _free(torch)


def test_weights_past_4_gb(torch_mod, gsp, ctx):
    torch = torch_mod
    rng = np.random.default_rng(2)
    in_dim, out_dim = 18944, 420001  # 4.5 GB
    rb = in_dim // 64 * 36
    w = torch.zeros((out_dim, rb), dtype=torch.uint8, device="cuda")
    raw = random_weights(rng, Q4_0, 5, in_dim)
    w[-5:] = torch.from_numpy(raw).cuda()
    wm, mag = decode_weights(Q4_0, raw, in_dim)
    for batch in (1, 6, 40):
        codes = rng.integers(0, 120, (batch, in_dim)).astype(np.uint8)
        x, s, y = torch.from_numpy(codes).cuda(), torch.ones(batch, device="cuda"), torch.ones((batch, out_dim), device="cuda")
        torch.cuda.synchronize()
        ctx.matmul_batch_fp8(Q4_0, w.data_ptr(), x.data_ptr(), s.data_ptr(), y.data_ptr(), in_dim, out_dim, batch)
        ctx.sync()
        X = E4M3[codes]
        bound = (37 + in_dim / 16) * 2.0 ** -23 * (np.abs(X) @ mag.T) + 1e-40
        assert np.all(np.abs(y[:, -5:].cpu().numpy() - X @ wm.T) <= bound)
        assert not y[:, :-5].any()
    del w
    _free(torch)


@pytest.mark.parametrize("in_dim", [64, 256])
def test_outputs_past_8_gb(torch_mod, gsp, ctx, in_dim):
    torch = torch_mod
    rng = np.random.default_rng(3)
    out_dim, batch = 32800, 70001  # 2.3e9 outputs
    raw = random_weights(rng, Q4_0, out_dim, in_dim)
    wm, mag = decode_weights(Q4_0, raw, in_dim)
    x = torch.zeros((batch, in_dim), dtype=torch.uint8, device="cuda")
    codes = rng.integers(0, 120, (130, in_dim)).astype(np.uint8)
    x[-130:] = torch.from_numpy(codes).cuda()
    w, s = torch.from_numpy(raw).cuda(), torch.ones(batch, device="cuda")
    y = torch.ones((batch, out_dim), device="cuda")
    torch.cuda.synchronize()
    ctx.matmul_batch_fp8(Q4_0, w.data_ptr(), x.data_ptr(), s.data_ptr(), y.data_ptr(), in_dim, out_dim, batch)
    ctx.sync()
    X = E4M3[codes]
    bound = (37 + in_dim / 16) * 2.0 ** -23 * (np.abs(X) @ mag.T) + 1e-40
    assert np.all(np.abs(y[-130:].cpu().numpy() - X @ wm.T) <= bound)
    assert not any(part.any() for part in y[:-130].split(8192))
    del y
    _free(torch)


def test_rows_in_pieces(torch_mod, gsp, ctx):
    """More converted activations than the workspace holds at once: 3840 rows a piece at 512 units of K."""
    torch = torch_mod
    rng = np.random.default_rng(4)
    in_dim, out_dim, batch = 131072, 520, 9001
    raw = random_weights(rng, Q4_1, out_dim, in_dim)
    x = torch.randint(0, 120, (batch, in_dim), dtype=torch.uint8, device="cuda")
    w, s = torch.from_numpy(raw).cuda(), torch.ones(batch, device="cuda")
    y = torch.zeros((batch, out_dim), device="cuda")
    torch.cuda.synchronize()
    ctx.matmul_batch_fp8(Q4_1, w.data_ptr(), x.data_ptr(), s.data_ptr(), y.data_ptr(), in_dim, out_dim, batch)
    ctx.sync()
    rows = [0, 1, 3711, 3839, 3840, 3841, 3967, 7679, 7680, 7681, 8999, 9000]
    wm, mag = decode_weights(Q4_1, raw, in_dim)
    X = E4M3[x[rows].cpu().numpy()]
    bound = (37 + in_dim / 16) * 2.0 ** -23 * (np.abs(X) @ mag.T)
    assert np.all(np.abs(y[rows].cpu().numpy() - X @ wm.T) <= bound)
    assert not (y == 0).all(dim=1).any()
    del x, y
    _free(torch)
