"""What gsp_matmul_batch_fp8 keeps of device memory, and batches that go piece by piece for it."""
import numpy as np
import pytest

from fp8_forms import PIECES, TILES
from fp8_helpers import E4M3, Q4_0, Q4_1, Q4_K, decode_weights, random_weights

pytestmark = pytest.mark.gpu


def test_converted_activations_do_not_double_past_a_gigabyte(torch_mod, gsp):
    """A product of 0.93 GB, then one of the most, 1.07 GB: the context keeps 1.07 GB and the split sums' few MB."""
    torch = torch_mod
    ctx = gsp.Context(0)
    in_dim, out_dim = 131072, 520
    w = torch.zeros((out_dim, in_dim // 32 * 20), dtype=torch.uint8, device="cuda")
    x = torch.zeros((9001, in_dim), dtype=torch.uint8, device="cuda")
    s, y = torch.ones(9001, device="cuda"), torch.ones((9001, out_dim), device="cuda")
    torch.cuda.synchronize()
    free = torch.cuda.mem_get_info()[0]
    kept = []
    for batch in (3300, 9001):
        ctx.matmul_batch_fp8(Q4_1, w.data_ptr(), x.data_ptr(), s.data_ptr(), y.data_ptr(), in_dim, out_dim, batch)
        ctx.sync()
        kept.append(free - torch.cuda.mem_get_info()[0])
    print(f"kept {kept}", flush=True)
    assert not y.any()
    assert 0.9e9 < kept[0] <= 1.0e9 and 1.0e9 < kept[1] <= 1.15e9
    ctx.close()
    del x, w
    torch.cuda.empty_cache()


@pytest.mark.parametrize("case,w_type", [pytest.param(c, t, id=f"in{c[0]}_out{c[1]}_b{c[2]}-{n}") for c in PIECES
                                         for n, t in (("q4_0", Q4_0), ("q4_1", Q4_1), ("q4_k", Q4_K))
                                         if t != Q4_K or c[0] % 256 == 0])
def test_pieces_of_a_batch_with_ranges_of_k(torch_mod, ctx, case, w_type):
    """Every piece adds up its own ranges.  The weights are eight rows over and over, so that every output has its 64 bits."""
    torch = torch_mod
    in_dim, out_dim, batch, _, ranges, _ = case
    print(f"case pieces {w_type} {case}", flush=True)
    rng = np.random.default_rng(out_dim)
    eight = random_weights(rng, w_type, 8, in_dim)
    which = torch.from_numpy(rng.integers(0, 8, out_dim)).cuda()
    w = torch.from_numpy(eight).cuda()[which]
    x = torch.randint(0, 254, (batch, in_dim), dtype=torch.uint8, device="cuda")
    x[x == 0x7f] = 0xfe  # every code but NaN
    s = torch.rand(batch, device="cuda") + 0.5
    y = torch.full((64 + batch * out_dim + 64,), 77.0, device="cuda")
    torch.cuda.synchronize()
    ctx.matmul_batch_fp8(w_type, w.data_ptr(), x.data_ptr(), s.data_ptr(), y[64:].data_ptr(), in_dim, out_dim, batch)
    ctx.sync()
    assert torch.all(y[:64] == 77) and torch.all(y[-64:] == 77)
    wm, mag = (torch.from_numpy(a.T.copy()).cuda() for a in decode_weights(w_type, eight, in_dim))
    table = torch.from_numpy(E4M3).cuda()
    got = y[64:-64].view(batch, out_dim)
    for at in range(0, batch, 200):
        part = table[x[at: at + 200].int()] * s[at: at + 200, None].double()
        want, bound = (part @ wm)[:, which], (37 + in_dim / 16 + ranges) * 2.0 ** -23 * (part.abs() @ mag)[:, which]
        err = (got[at: at + 200].double() - want).abs()
        assert (err <= bound).all(), at
        # the bound grows with K's length, the error of sums in any order hardly: a lost range would be a large part
        assert (err <= 1e-4 * (part.abs() @ mag)[:, which]).all(), at
    del x, y
    torch.cuda.empty_cache()


def test_captured_wide_products_keep_their_buffers(torch_mod, gsp):
    """Two captured products of the wide form, the second of which needs more than the first, with eager products of
    other sizes between the replays: each replay gives what the eager call gave.  A first call while the stream captures
    is refused and leaves the capture whole."""
    torch = torch_mod
    ctx = gsp.Context(0)
    stream = torch.cuda.Stream()
    ctx.set_stream(stream.cuda_stream)
    rng = np.random.default_rng(3)
    sizes = [c[:3] for c in TILES if c[3] == "wide" and c[0] % 256 == 0]
    small, large = [next(s for s in sizes if s[0] == k) for k in (2816, 3584)]
    prods = []
    for w_type, (in_dim, out_dim, batch) in ((Q4_1, small), (Q4_K, large), (Q4_0, sizes[0])):
        raw = random_weights(rng, w_type, out_dim, in_dim)
        x = torch.randint(0, 120, (batch, in_dim), dtype=torch.uint8, device="cuda")
        prods.append((w_type, torch.from_numpy(raw).cuda(), x, torch.rand(batch, device="cuda"),
                      torch.zeros((batch, out_dim), device="cuda"), in_dim, out_dim, batch))

    def call(p):
        t, w, x, s, y, *sizes = p
        ctx.matmul_batch_fp8(t, w.data_ptr(), x.data_ptr(), s.data_ptr(), y.data_ptr(), *sizes)

    cold, z = torch.cuda.CUDAGraph(), torch.zeros(4, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.graph(cold, stream=stream):
        z.add_(1)
        with pytest.raises(gsp.StateError):
            call(prods[0])
    cold.replay()
    torch.cuda.synchronize()
    assert torch.all(z == 1) and not prods[0][4].any()
    wants = []
    for p in prods:
        call(p)
        ctx.sync()
        wants.append(p[4].clone())
    graphs = []
    for p in prods[:2]:
        g = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(g, stream=stream):
            call(p)
        graphs.append(g)
    for _ in range(3):
        for g, p, want in zip(graphs, prods, wants):
            p[4].fill_(77)
            torch.cuda.synchronize()
            with torch.cuda.stream(stream):
                g.replay()
            call(prods[2])
            torch.cuda.synchronize()
            assert torch.equal(p[4], want) and torch.equal(prods[2][4], wants[2])
            prods[2][4].fill_(77)
    del graphs, cold
    ctx.close()
