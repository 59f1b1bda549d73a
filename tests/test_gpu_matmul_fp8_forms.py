"""gsp_matmul_batch_fp8 in each of its forms: every output in 64 bits, and where every step is exact, exactly.

The bound is that of tests/test_gpu_matmul_fp8.py, one more addition for each range of K.
"""
import numpy as np
import pytest

from fp8_forms import CUS, STREAM32, STREAMS, TILES
from fp8_helpers import E4M3, GROUP_BYTES, Q4_0, Q4_1, Q4_K, decode_weights, random_codes, random_weights

pytestmark = pytest.mark.gpu
TYPES = {"q4_0": Q4_0, "q4_1": Q4_1, "q4_k": Q4_K}


@pytest.fixture(scope="module", autouse=True)
def planned_for(gsp):
    assert gsp.device_info(0).compute_units == CUS


def _runs(torch, ctx, w_type, raw, codes, scale, offset, times=1):
    """The outputs, with the weights `offset` bytes behind a 16-byte address."""
    (out_dim, _), (batch, in_dim) = raw.shape, codes.shape
    w = torch.zeros(raw.size + 16, dtype=torch.uint8, device="cuda")
    w[offset: offset + raw.size] = torch.from_numpy(raw.reshape(-1)).cuda()
    x, s = torch.from_numpy(codes).cuda(), torch.from_numpy(scale).cuda()
    got = []
    for _ in range(times):
        y = torch.full((64 + batch * out_dim + 64,), 77.0, device="cuda")
        torch.cuda.synchronize()
        ctx.matmul_batch_fp8(w_type, w.data_ptr() + offset, x.data_ptr(), s.data_ptr(), y[64:].data_ptr(), in_dim, out_dim,
                             batch)
        ctx.sync()
        assert torch.all(y[:64] == 77) and torch.all(y[-64:] == 77)
        got.append(y[64:-64].view(batch, out_dim))
    return got


def _id(case):
    return f"{case[3]}_{case[4]}x{case[5]}_in{case[0]}_out{case[1]}_b{case[2]}"


@pytest.mark.parametrize("case,name", [pytest.param(c, n, id=f"{_id(c)}-{n}") for c in TILES + STREAMS + STREAM32
                                       for n in TYPES if n != "q4_k" or c[0] % 256 == 0])
def test_every_output(torch_mod, ctx, case, name):
    torch = torch_mod
    in_dim, out_dim, batch, form, ranges, _ = case
    w_type = TYPES[name]
    print(f"case forms {name} {case}", flush=True)
    rng = np.random.default_rng(in_dim + 3 * out_dim + batch + w_type)
    raw, codes = random_weights(rng, w_type, out_dim, in_dim), random_codes(rng, (batch, in_dim))
    scale = np.exp(rng.uniform(-8, 3, batch)).astype(np.float32)
    w, mag = (torch.from_numpy(a).cuda() for a in decode_weights(w_type, raw, in_dim))
    x = torch.from_numpy(E4M3[codes] * scale.astype(np.float64)[:, None]).cuda()
    want = x @ w.t()
    bound = (37 + in_dim / 16 + ranges) * 2.0 ** -23 * (x.abs() @ mag.t()) + 1e-40
    # Whole units: once with 16-byte loads, once at a 4-byte address.  STREAMS are what the latter take.
    for offset in ([0] if in_dim % 256 or form == "stream32" else [4] if form == "stream" else [0, 4]):
        first, second = _runs(torch, ctx, w_type, raw, codes, scale, offset, 2)
        err = (first.double() - want).abs()
        print(f"offset {offset}: largest error {(err / bound).max().item():.3f} of its bound", flush=True)
        assert (err <= bound).all()
        assert torch.equal(first, second)


# A size for each form; streams both with 16-byte loads and without.
EXACT = [(256, 70, 1), (256, 5000, 4), (512, 70, 8), (512, 5000, 7), (256, 70, 16), (256, 5000, 13), (256, 70, 40),
         (256, 4001, 37), (256, 5001, 40), (256, 16403, 20), (256, 4500, 32), (256, 8001, 64), (256, 130, 200),
         (512, 1208, 845), (1280, 2469, 1604), (3584, 1797, 1371)]


@pytest.mark.parametrize("name", list(TYPES))
@pytest.mark.parametrize("size", EXACT, ids=lambda s: f"in{s[0]}_out{s[1]}_b{s[2]}")
def test_small_terms_beside_large_ones(torch_mod, ctx, size, name):
    """448 and -448 beside 2^-9 among neighbours that one step of the matrix cores adds: nothing of 2^-9 is lost.

    A row's few codes lie in one dword.  Scales are powers of two, and every sum on the way fits 24 bits: with d 2^-3
    and Q4_K scales of 1 to 16 a sum is at most 16 * 15 * 448 = 2^16.7 in steps of its scale times 2^-9, an output at most
    2^13.8 in steps of 2^-9 or 2^9.8 in steps of 2^-12.  Q4_K's rows have both 448 and -448, so that minimums meet a sum of
    2^-9 alone; the others' also 448 alone."""
    torch = torch_mod
    in_dim, out_dim, batch = size
    w_type = TYPES[name]
    rng = np.random.default_rng(batch + w_type)
    raw = random_weights(rng, w_type, out_dim, in_dim)
    blocks = raw.reshape(out_dim, -1, GROUP_BYTES[w_type][1])
    half = lambda v: np.array([v], np.float16).view(np.uint8)  # noqa: E731
    blocks[..., 0:2] = half(2.0 ** -3)
    if w_type == Q4_1:
        blocks[..., 2:4] = half(-2.0 ** -2)
    if w_type == Q4_K:
        blocks[..., 2:4] = half(-1.0)
        blocks[..., 4:8] = 1 << rng.integers(0, 5, blocks[..., 4:8].shape)
        blocks[..., 12:16] = (blocks[..., 12:16] & 0xf0) | 1 << rng.integers(0, 4, blocks[..., 12:16].shape)
    codes = np.zeros((batch, in_dim), np.uint8)
    for b in range(batch):
        at = 4 * ((b * 37 + batch) % (in_dim // 4)) + rng.permutation(4)
        codes[b, at[0]] = 0x7e
        codes[b, at[1]] = 0xfe if w_type == Q4_K or b % 2 else 0
        codes[b, at[2]] = 0x01
    w = torch.from_numpy(decode_weights(w_type, raw, in_dim)[0]).cuda()
    want = torch.from_numpy(E4M3[codes]).cuda() @ w.t()
    assert torch.equal(want.float().double(), want)
    for offset in (0, 4):
        got = _runs(torch, ctx, w_type, raw, codes, np.ones(batch, np.float32), offset)[0]
        off = got.double() != want
        assert not off.any(), f"offset {offset}: {int(off.sum())} of {off.numel()} outputs"
