"""gsp_mrope_write_step at the widest tokens it takes."""
import numpy as np
import pytest

from fp8_helpers import axis_of_pair, rotate64

pytestmark = pytest.mark.gpu
ITEMS = 65535 * 256  # pairs of Q and K and values of V


def _pool(gsp, ctx, d, dv):
    pool = gsp.Pool.create(ctx, 4, 1, 1, d, v_head_dim=dv)
    ctx.pack_step(pool, [3], [5], [0, 1], [2], 64, q_lens=[2])
    return pool


def test_wider_tokens_are_refused(torch_mod, gsp, ctx):
    """Up to head counts whose pairs leave 32 bits; nothing is enqueued."""
    torch = torch_mod
    pool = _pool(gsp, ctx, 256, 256)
    t = torch.full((4096,), 7.0, device="cuda")
    pos = torch.zeros((1, 2), dtype=torch.int32, device="cuda")
    out = torch.full((64,), 7.0, device="cuda")
    torch.cuda.synchronize()
    for heads in (ITEMS // 128 - 2, 1 << 23, (1 << 24) - 1, 1 << 24, (1 << 31) - 1):
        with pytest.raises(gsp.Unsupported):
            pool.mrope_write_step(0, heads, gsp.MRope(1e4, (128,)), pos.data_ptr(), t.data_ptr(), out.data_ptr(),
                                  t.data_ptr(), t.data_ptr() + 2048)
    ctx.sync()
    assert torch.all(out == 7.0) and torch.all(t == 7.0) and not pool.download(0, pool.arenas()[2]).any()
    pool.destroy()


@pytest.mark.parametrize("d,dv", [(256, 256), (6, 5)])
def test_widest_tokens(torch_mod, gsp, ctx, d, dv):
    """As many heads as fit, in fours and one by one: every head turns."""
    torch = torch_mod
    pool = _pool(gsp, ctx, d, dv)
    heads = (ITEMS - dv) // (d // 2) - 1
    print(f"case widest tokens {heads} heads of {d}", flush=True)
    g = torch.Generator(device="cuda").manual_seed(1)
    q = torch.randn((2, heads, d), generator=g, device="cuda")
    k, v = torch.randn((2, d), generator=g, device="cuda"), torch.randn((2, dv), generator=g, device="cuda")
    out = torch.full((2 * heads * d + 64,), 7.0, device="cuda")
    pos = torch.tensor([[5, 70000]], dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    pool.mrope_write_step(0, heads, gsp.MRope(1e4, (d // 2,)), pos.data_ptr(), q.data_ptr(), out.data_ptr(), k.data_ptr(),
                          v.data_ptr())
    ctx.sync()
    assert torch.all(out[2 * heads * d:] == 7.0)
    got = out[:2 * heads * d].view(2, heads, d)
    some = np.unique(np.concatenate([[0, 1, heads - 2, heads - 1], np.random.default_rng(2).integers(0, heads, 500)]))
    at = torch.from_numpy(some).cuda()
    rates = 1e4 ** (-2.0 * np.arange(d // 2) / d)
    turn = lambda x: rotate64(x, pos.cpu().numpy(), axis_of_pair((d // 2,), False), rates, d, False)  # noqa: E731
    want, mag = turn(q[:, at].cpu().numpy())
    assert np.all(np.abs(got[:, at].cpu().numpy() - want) <= 5e-7 * mag + 1e-12)
    # pairs keep their length, in every head: four roundings of 2^-24 each way and the cosine's and sine's two steps
    norm = lambda x: x.view(2, heads, d // 2, 2).double().square().sum(-1)  # noqa: E731
    assert ((norm(got) - norm(q)).abs() <= 2e-6 * norm(q) + 1e-12).all()
    want, mag = turn(k.cpu().numpy()[:, None])
    K = pool.download(0, pool.arenas()[2]).view(np.float32).reshape(4, 16, d)
    V = pool.download(1, pool.arenas()[3]).view(np.float32).reshape(4, 16, dv)
    assert np.all(np.abs(K[2, 3:5] - want[:, 0]) <= 5e-7 * mag[:, 0] + 1e-12)
    assert np.array_equal(V[2, 3:5], v.cpu().numpy())
    pool.destroy()
    del q, out, got
    torch.cuda.empty_cache()
