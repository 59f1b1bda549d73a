"""gsp_matmul_batch_fp8 at the longest K that its sizes allow, 2^31 - 64 (Q4_K: 2^31 - 256).

Blocks of zeros (scale 0) but for a few groups of random weights, so that the other codes add nothing: an output is
off by at most the 37 roundings of a group (twice for a minimum) and one for each of the groups.
"""
import numpy as np
import pytest

from fp8_helpers import E4M3, GROUP_BYTES, Q4_0, Q4_1, Q4_K, decode_weights, random_weights

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("batch", [1, 9, 20])
@pytest.mark.parametrize("w_type", [Q4_0, Q4_1, Q4_K], ids=["q4_0", "q4_1", "q4_k"])
def test_longest_k(torch_mod, ctx, w_type, batch):
    torch = torch_mod
    per, size = GROUP_BYTES[w_type]
    in_dim = 2 ** 31 - max(64, per)
    print(f"case longest k {w_type} {in_dim} rows {batch}", flush=True)
    rng = np.random.default_rng(batch)
    blocks = in_dim // per
    at = [0, 1, 9, blocks // 3, blocks // 2, blocks - 10, blocks - 2, blocks - 1]
    raw = random_weights(rng, w_type, 1, per * len(at)).reshape(len(at), size)
    w = torch.zeros((blocks, size), dtype=torch.uint8, device="cuda")
    w[torch.tensor(at, device="cuda")] = torch.from_numpy(raw).cuda()
    x = torch.empty((batch, in_dim), dtype=torch.uint8, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(batch)
    for b in range(batch):
        x[b].random_(0, 120, generator=g)
    s = torch.full((batch,), 0.5, device="cuda")
    y = torch.full((batch + 2,), 77.0, device="cuda")
    torch.cuda.synchronize()
    ctx.matmul_batch_fp8(w_type, w.data_ptr(), x.data_ptr(), s.data_ptr(), y[1:].data_ptr(), in_dim, 1, batch)
    ctx.sync()
    got = y.cpu().numpy()
    assert got[0] == 77 and got[-1] == 77
    wm, mag = decode_weights(w_type, raw.reshape(1, -1), per * len(at))
    codes = x.view(batch, blocks, per)[:, torch.tensor(at, device="cuda")].cpu().numpy().reshape(batch, -1)
    X = E4M3[codes] * 0.5
    bound = (37 + 2 * per // 32 * len(at)) * 2.0 ** -23 * (np.abs(X) @ mag.T)
    err = np.abs(got[1:-1, None] - X @ wm.T)
    print(f"largest error {np.max(err / bound):.3f} of its bound", flush=True)
    assert np.all(err <= bound)
    del x, w
    torch.cuda.empty_cache()
