"""gsp_matmul_batch_fp8 against float64 on the same codes and weight bytes.

Products of codes and 4-bit quants are exact.  A group of 32 and its offset's product is one fp32 sum of at most 33
terms, and an output adds in_dim / 32 such sums (twice as many with a minimum): in any order of these additions an
output is off by at most (33 + 2 in_dim / 32 + 4) roundings of the magnitudes they pass through, which are the codes'
part and the offset's part of every weight without their signs.  2^-23 a rounding: the matrix instruction's own sums
may cut instead of rounding.
"""
import numpy as np
import pytest

from fp8_helpers import E4M3, Q4_0, Q4_1, Q4_K, decode_weights, random_codes, random_weights

pytestmark = pytest.mark.gpu

TYPES = {"q4_0": Q4_0, "q4_1": Q4_1, "q4_k": Q4_K}
# (in_dim, out_dim, batch); K-quants skip in_dim that is no multiple of 256.
SHAPES = [(64, 1, 1), (64, 16, 3), (128, 17, 2), (192, 40, 5), (256, 16, 16), (256, 5, 1), (320, 33, 17), (512, 64, 32),
          (896, 1152, 8), (1024, 100, 33), (3584, 512, 64), (3584, 37, 65), (4864, 896, 1), (18944, 48, 4),
          (18944, 20, 64), (256, 130, 200), (512, 257, 129), (1280, 96, 300), (64, 300, 1000), (2048, 256, 512),
          # the tile forms: each tile height, with and without ranges of K, ragged ends, K that ends inside a unit
          (1024, 4000, 65), (4864, 130, 70), (4928, 900, 515), (3584, 3600, 1030), (576, 5000, 1290), (18944, 300, 66)]


def _reference(w_type, raw, codes, scale, in_dim):
    w, mag = decode_weights(w_type, raw, in_dim)
    x = E4M3[codes] * scale.astype(np.float64)[:, None]
    bound = (37 + in_dim / 16) * 2.0 ** -23 * (np.abs(x) @ mag.T)
    return x @ w.T, bound


def _inputs(rng, w_type, in_dim, out_dim, batch):
    raw = random_weights(rng, w_type, out_dim, in_dim)
    codes = random_codes(rng, (batch, in_dim))
    scale = np.exp(rng.uniform(-8, 3, batch)).astype(np.float32)
    return raw, codes, scale


@pytest.mark.parametrize("name", list(TYPES))
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: f"in{s[0]}_out{s[1]}_b{s[2]}")
def test_matches_64_bits(torch_mod, ctx, shape, name):
    torch = torch_mod
    in_dim, out_dim, batch = shape
    w_type = TYPES[name]
    if w_type == Q4_K and in_dim % 256:
        in_dim += 256 - in_dim % 256
    print(f"case matmul_fp8 {name} {in_dim} {out_dim} {batch}", flush=True)
    rng = np.random.default_rng(in_dim * 7 + out_dim * 3 + batch + w_type)
    raw, codes, scale = _inputs(rng, w_type, in_dim, out_dim, batch)
    w = torch.from_numpy(raw).cuda()
    x = torch.from_numpy(codes).cuda()
    s = torch.from_numpy(scale).cuda()
    y = torch.full((64 + batch * out_dim + 64,), 77.0, device="cuda")
    torch.cuda.synchronize()

    def run():
        ctx.matmul_batch_fp8(w_type, w.data_ptr(), x.data_ptr(), s.data_ptr(), y[64:].data_ptr(), in_dim, out_dim, batch)
        ctx.sync()
        return y.cpu().numpy()

    got = run()
    assert np.all(got[:64] == 77) and np.all(got[64 + batch * out_dim:] == 77)
    want, bound = _reference(w_type, raw, codes, scale, in_dim)
    err = np.abs(got[64:-64].reshape(batch, out_dim) - want)
    print(f"largest error {np.max(err / np.maximum(bound, 1e-300)):.3f} of its bound", flush=True)
    assert np.all(err <= bound + 1e-40)
    assert np.array_equal(got, run())


@pytest.mark.parametrize("name", list(TYPES))
def test_every_code_of_both_operands(torch_mod, ctx, name):
    """One activation per row, one at a time at every place of two groups: exact products, exactly."""
    torch = torch_mod
    w_type = TYPES[name]
    in_dim, out_dim = 256, 64
    rng = np.random.default_rng(11)
    raw = random_weights(rng, w_type, out_dim, in_dim)
    # Scales of one power of two each: the products then have no rounding at all.
    per = raw.reshape(out_dim, -1, {Q4_0: 18, Q4_1: 20, Q4_K: 144}[w_type])
    per[..., 0:2] = np.array([2.0 ** -3], np.float16).view(np.uint8)
    if w_type != Q4_0:
        per[..., 2:4] = np.array([-2.0 ** -2], np.float16).view(np.uint8)
    codes = np.zeros((256, in_dim), np.uint8)
    values = np.array([c for c in range(256) if c & 127 != 127])
    codes[np.arange(256), np.arange(256)] = values[np.arange(256) % len(values)]
    w, _ = decode_weights(w_type, raw, in_dim)
    wd, xd = torch.from_numpy(raw).cuda(), torch.from_numpy(codes).cuda()
    s, y = torch.ones(256, device="cuda"), torch.zeros((256, out_dim), device="cuda")
    torch.cuda.synchronize()
    ctx.matmul_batch_fp8(w_type, wd.data_ptr(), xd.data_ptr(), s.data_ptr(), y.data_ptr(), in_dim, out_dim, 256)
    ctx.sync()
    assert np.array_equal(y.cpu().numpy().astype(np.float64), E4M3[codes] @ w.T)


@pytest.mark.parametrize("batch", [3, 40, 300])
def test_nan_codes_and_scales_stay_in_their_rows(torch_mod, ctx, batch):
    torch = torch_mod
    rng = np.random.default_rng(2)
    in_dim, out_dim = 320, 70
    raw, codes, scale = _inputs(rng, Q4_0, in_dim, out_dim, batch)
    codes[1, 319] = 0x7f
    scale[2] = np.nan
    wd, xd, sd = (torch.from_numpy(a).cuda() for a in (raw, codes, scale))
    y = torch.zeros((batch, out_dim), device="cuda")
    torch.cuda.synchronize()
    ctx.matmul_batch_fp8(Q4_0, wd.data_ptr(), xd.data_ptr(), sd.data_ptr(), y.data_ptr(), in_dim, out_dim, batch)
    ctx.sync()
    got = y.cpu().numpy()
    assert np.all(np.isnan(got[1])) and np.all(np.isnan(got[2]))
    rest = [b for b in range(batch) if b not in (1, 2)]
    want, bound = _reference(Q4_0, raw, codes[rest], scale[rest], in_dim)
    assert np.all(np.abs(got[rest] - want) <= bound + 1e-40)


def test_weights_at_four_byte_addresses(torch_mod, ctx):
    torch = torch_mod
    rng = np.random.default_rng(5)
    in_dim, out_dim, batch = 512, 50, 9
    for w_type in TYPES.values():
        raw, codes, scale = _inputs(rng, w_type, in_dim, out_dim, batch)
        buf = torch.zeros(raw.size + 12, dtype=torch.uint8, device="cuda")
        xd, sd = torch.from_numpy(codes).cuda(), torch.from_numpy(scale).cuda()
        want, bound = _reference(w_type, raw, codes, scale, in_dim)
        for off in (4, 8, 12):
            buf[off: off + raw.size] = torch.from_numpy(raw.reshape(-1)).cuda()
            y = torch.zeros((batch, out_dim), device="cuda")
            torch.cuda.synchronize()
            ctx.matmul_batch_fp8(w_type, buf.data_ptr() + off, xd.data_ptr(), sd.data_ptr(), y.data_ptr(), in_dim,
                                 out_dim, batch)
            ctx.sync()
            assert np.all(np.abs(y.cpu().numpy() - want) <= bound + 1e-40)


# 17 to 64 rows in tiles of 32 by 32: one round of workgroups, several, ragged rows and outputs, K of one unit and of
# many; the last two are wide enough that the tile forms are weighed against them.
STREAM32 = [(256, 4500, 17), (1024, 4611, 31), (2560, 3590, 37), (4864, 4100, 32), (512, 8300, 40), (768, 5000, 64),
            (256, 16411, 32), (512, 17000, 50), (256, 33000, 64)]


@pytest.mark.parametrize("name", list(TYPES))
@pytest.mark.parametrize("shape", STREAM32, ids=lambda s: f"in{s[0]}_out{s[1]}_b{s[2]}")
def test_tiles_of_32_rows_that_share_k(torch_mod, ctx, shape, name):
    test_matches_64_bits(torch_mod, ctx, shape, name)


@pytest.mark.parametrize("name", list(TYPES))
def test_nan_rows_in_tiles_of_32(torch_mod, ctx, name):
    torch = torch_mod
    rng = np.random.default_rng(3)
    in_dim, out_dim, batch = 512, 4500, 29
    raw, codes, scale = _inputs(rng, TYPES[name], in_dim, out_dim, batch)
    codes[1, 511], codes[7, 0], codes[28, 300] = 0x7f, 0xff, 0x7f
    wd, xd, sd = (torch.from_numpy(a).cuda() for a in (raw, codes, scale))
    y = torch.zeros((batch, out_dim), device="cuda")
    torch.cuda.synchronize()
    ctx.matmul_batch_fp8(TYPES[name], wd.data_ptr(), xd.data_ptr(), sd.data_ptr(), y.data_ptr(), in_dim, out_dim, batch)
    ctx.sync()
    bad = torch.isnan(y)
    assert set(np.nonzero(bad.any(1).cpu().numpy())[0]) == {1, 7, 28}
    assert bad[[1, 7, 28]].all()
