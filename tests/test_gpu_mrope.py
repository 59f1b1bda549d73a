"""gsp_mrope_write_step against the rotation in 64 bits.

An angle is reduced in 64 bits and rounded once to fp32 (half a step of pi, 1.2e-7), cosine and sine are within two steps
of 1 (1.2e-7), and the two products, their sum and mscale round once each: every value is within 5e-7 of the pair's
|x0| + |x1|.  fp16 pools add half a step of the value, 2^-11 (2^-25 for subnormals).
"""
import numpy as np
import pytest

from fp8_helpers import axis_of_pair, rotate64

pytestmark = pytest.mark.gpu

# (heads, kv heads, head_dim, v_head_dim, rope_dim, sections, kv dtype, page)
CASES = [
    (28, 4, 128, 128, 128, (16, 24, 24), "f16", 16),
    (14, 2, 64, 64, 64, (12, 10, 10), "f32", 16),
    (6, 2, 80, 80, 64, (11, 11, 10), "f16", 8),
    (4, 4, 36, 36, 36, (6, 6, 6), "f32", 16),      # no multiple of 8: single values
    (3, 1, 64, 33, 32, (8, 8), "f16", 24),         # two axes, odd v_head_dim
    (8, 8, 256, 128, 256, (128,), "f32", 32),      # one axis: plain positions
    (2, 1, 32, 32, 32, (4, 4, 4, 4), "f32", 16),
]
BASE = 1.0e6


def _step(gsp, ctx, rng, case, n_rows=5, layers=2, new_hi=40):
    heads, kvh, d, dv, _, _, kv, page = case
    new = rng.integers(1, new_hi, n_rows).astype(np.int32)
    before = rng.integers(0, 70, n_rows).astype(np.int32)
    total = before + new
    pages = -(-total // page)
    blocks = int(pages.sum()) + 3
    off = np.concatenate([[0], np.cumsum(pages)]).astype(np.int32)
    ids = rng.permutation(blocks)[: off[-1]].astype(np.int32)
    pool = gsp.Pool.create(ctx, blocks, layers, kvh, d, gsp.KV_F16 if kv == "f16" else gsp.KV_F32, v_head_dim=dv,
                           block_size=page)
    ctx.pack_step(pool, before, total, off, ids, 4096, q_lens=new)
    row = np.repeat(np.arange(n_rows), new)
    at = np.concatenate([b + np.arange(n) for b, n in zip(before, new)])
    return pool, blocks, ids[off[row] + at // page], at % page


def _arenas(pool, blocks, layers, case):
    heads, kvh, d, dv, _, _, kv, page = case
    t = np.float16 if kv == "f16" else np.float32
    _, _, kb, vb = pool.arenas()
    return (pool.download(0, kb).view(t).reshape(blocks, layers, kvh, page, d),
            pool.download(1, vb).view(t).reshape(blocks, layers, kvh, page, dv))


def _tol(mag, want, kv):
    t = 5e-7 * mag + 1e-12
    return t + (np.maximum(np.abs(want) * 2.0 ** -11, 2.0 ** -25) if kv == "f16" else 0)


@pytest.mark.parametrize("fused", [False, True], ids=["dense", "fused"])
@pytest.mark.parametrize("style", ["pairs", "halves"])
@pytest.mark.parametrize("layout", ["sections", "interleaved"])
@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{c[0]}q{c[1]}kv_d{c[2]}_{c[3]}_{c[6]}_{len(c[5])}axes")
def test_matches_64_bits(torch_mod, gsp, ctx, case, layout, style, fused):
    torch = torch_mod
    heads, kvh, d, dv, rope_dim, sections, kv, page = case
    print(f"case mrope {case} {layout} {style} fused={fused}", flush=True)
    rng = np.random.default_rng(d + len(sections) + heads)
    pool, blocks, blk, slot = _step(gsp, ctx, rng, case)
    n, na = len(blk), len(sections)
    axes = rng.integers(0, 60000, (na, n)).astype(np.int32)
    axes[:, 0], axes[:, 1] = 0, 1
    axes[-1, 2] = -5
    axes[0, 3] = 2 ** 31 - 1
    wq, wk, wv = heads * d, kvh * d, kvh * dv
    rows = rng.standard_normal((n, wq + wk + wv + (3 if dv == 33 else 4))).astype(np.float32)
    q, k, v = rows[:, :wq], rows[:, wq: wq + wk], rows[:, wq + wk: wq + wk + wv]
    pos = torch.from_numpy(axes).cuda()
    out = torch.full((64 + n * wq + 64,), 77.0, device="cuda")
    rope = gsp.MRope(BASE, sections, style=gsp.ROPE_HALVES if style == "halves" else gsp.ROPE_PAIRS,
                     layout=gsp.MROPE_INTERLEAVED if layout == "interleaved" else gsp.MROPE_SECTIONS, rope_dim=rope_dim,
                     mscale=1.25 if fused else 0.0)
    if fused:
        rd = torch.from_numpy(rows).cuda()
        st = rows.shape[1]
        ptr = [rd.data_ptr(), rd.data_ptr() + 4 * wq, rd.data_ptr() + 4 * (wq + wk)]
        keep = rd
    else:
        st = 0
        keep = [torch.from_numpy(np.ascontiguousarray(t)).cuda() for t in (q, k, v)]
        ptr = [t.data_ptr() for t in keep]
    torch.cuda.synchronize()

    def call():
        pool.mrope_write_step(1, heads, rope, pos.data_ptr(), ptr[0], out[64:].data_ptr(), ptr[1], ptr[2], q_stride=st,
                              k_stride=st, v_stride=st)
        ctx.sync()

    if layout == "interleaved" and any(na * (s - 1) + a >= rope_dim // 2 for a, s in enumerate(sections) if a):
        with pytest.raises(gsp.InvalidArgument):  # an axis does not find its pairs dealt out one by one
            call()
        pool.destroy()
        return
    call()
    del keep
    K, V = _arenas(pool, blocks, 2, case)
    axis = axis_of_pair(sections, layout == "interleaved")
    rates = BASE ** (-2.0 * np.arange(rope_dim // 2) / rope_dim)
    ms = 1.25 if fused else 1.0
    wantq, magq = rotate64(q.reshape(n, heads, d), axes, axis, rates, rope_dim, style == "halves", ms)
    wantk, magk = rotate64(k.reshape(n, kvh, d), axes, axis, rates, rope_dim, style == "halves", ms)
    got = out.cpu().numpy()
    assert np.all(got[:64] == 77) and np.all(got[-64:] == 77)
    # The far position's angle is itself off by 2^31 2^-53 in 64 bits.
    assert np.all(np.abs(got[64:-64].reshape(wantq.shape) - wantq) <= _tol(magq, wantq, "f32") + 5e-7 * magq)
    gk = K[blk, 1, :, slot].astype(np.float64)
    assert np.all(np.abs(gk - wantk) <= _tol(magk, wantk, kv) + 5e-7 * magk)
    assert np.array_equal(V[blk, 1, :, slot], v.reshape(n, kvh, dv).astype(V.dtype))
    mask = np.ones(K.shape[:1] + K.shape[3:4], bool)
    mask[blk, slot] = False
    assert not K[:, 0].any() and not V[:, 0].any()
    assert not K[:, 1].transpose(0, 2, 1, 3)[mask].any() and not V[:, 1].transpose(0, 2, 1, 3)[mask].any()
    pool.destroy()


@pytest.mark.parametrize("case", [CASES[0], CASES[1], CASES[4]], ids=["d128", "d64", "odd"])
def test_many_tokens(torch_mod, gsp, ctx, case):
    """A prefill of over 512 tokens, whose threads take several items each."""
    torch = torch_mod
    heads, kvh, d, dv, rope_dim, sections, kv, page = case
    rng = np.random.default_rng(31)
    pool, blocks, blk, slot = _step(gsp, ctx, rng, case, n_rows=30, new_hi=50)
    n = len(blk)
    assert n >= 512
    axes = rng.integers(0, 60000, (len(sections), n)).astype(np.int32)
    q, k, v = (rng.standard_normal((n, w)).astype(np.float32) for w in (heads * d, kvh * d, kvh * dv))
    qd, kd, vd, pos = (torch.from_numpy(t).cuda() for t in (q, k, v, axes))
    torch.cuda.synchronize()
    pool.mrope_write_step(0, heads, gsp.MRope(BASE, sections, 1, rope_dim=rope_dim), pos.data_ptr(), qd.data_ptr(),
                          qd.data_ptr(), kd.data_ptr(), vd.data_ptr())
    ctx.sync()
    K, V = _arenas(pool, blocks, 2, case)
    rates = BASE ** (-2.0 * np.arange(rope_dim // 2) / rope_dim)
    axis = axis_of_pair(sections, False)
    wantq, magq = rotate64(q.reshape(n, heads, d), axes, axis, rates, rope_dim, True)
    wantk, magk = rotate64(k.reshape(n, kvh, d), axes, axis, rates, rope_dim, True)
    assert np.all(np.abs(qd.cpu().numpy().reshape(wantq.shape) - wantq) <= _tol(magq, wantq, "f32"))
    assert np.all(np.abs(K[blk, 0, :, slot].astype(np.float64) - wantk) <= _tol(magk, wantk, kv))
    assert np.array_equal(V[blk, 0, :, slot], v.reshape(n, kvh, dv).astype(V.dtype))
    pool.destroy()


@pytest.mark.parametrize("tables", ["inv_freq", "factors"])
def test_equal_axes_are_plain_rope(torch_mod, gsp, ctx, tables):
    """Text: the same position on every axis, at the token's place in its row, is gsp_rope_write_step_ex.

    The two kernels' compilations may contract the two products and their sum differently, so each is
    within 5e-7 of the pair's |x0| + |x1| of the exact value, and they of each other within twice that (keys
    plus one fp16 step, 2^-10 of the value, where the difference crosses a rounding border)."""
    torch = torch_mod
    case = (12, 4, 128, 128, 96, (20, 20, 8), "f16", 16)
    heads, kvh, d, dv, rope_dim, sections, kv, page = case
    rng = np.random.default_rng(8)
    tab = rng.uniform(0.5, 2.0, rope_dim // 2).astype(np.float32)
    kw = {"inv_freq": tab} if tables == "inv_freq" else {"freq_factors": tab}
    pool, blocks, blk, slot = _step(gsp, ctx, rng, case)
    n = len(blk)
    rng2 = np.random.default_rng(8)
    rng2.uniform(0.5, 2.0, rope_dim // 2)
    new = rng2.integers(1, 40, 5)
    before = rng2.integers(0, 70, 5)
    at = np.concatenate([b + np.arange(m) for b, m in zip(before, new)]).astype(np.int32)
    pos = torch.from_numpy(np.stack([at] * 3)).cuda()
    q, k, v = (torch.from_numpy(rng.standard_normal((n, w)).astype(np.float32)).cuda()
               for w in (heads * d, kvh * d, kvh * dv))
    q2, q0 = q.clone(), q.clone()
    torch.cuda.synchronize()
    pool.rope_write_step_ex(0, heads, gsp.Rope(1e4, 1, rope_dim, mscale=0.7, **kw), q.data_ptr(), k.data_ptr(), v.data_ptr())
    # in place
    pool.mrope_write_step(1, heads, gsp.MRope(1e4, sections, 1, rope_dim=rope_dim, mscale=0.7, **kw), pos.data_ptr(),
                          q2.data_ptr(), q2.data_ptr(), k.data_ptr(), v.data_ptr())
    ctx.sync()
    K, V = _arenas(pool, blocks, 2, case)
    halves = rope_dim // 2

    def pair_mag(x):
        m = np.abs(x)
        m[..., :rope_dim] = np.concatenate([m[..., :halves] + m[..., halves:rope_dim]] * 2, -1)
        return m

    mq = pair_mag(q0.cpu().numpy().reshape(n, heads, d))
    mk = pair_mag(k.cpu().numpy().reshape(n, kvh, d))
    assert np.all(np.abs((q - q2).cpu().numpy().reshape(mq.shape)) <= 1e-6 * mq)
    a, b = K[blk, 0, :, slot].astype(np.float64), K[blk, 1, :, slot].astype(np.float64)
    assert np.all(np.abs(a - b) <= 1e-6 * mk + np.maximum(np.abs(a) * 2.0 ** -10, 2.0 ** -24))
    assert np.mean(a == b) > 0.99 and np.array_equal(V[:, 0], V[:, 1])
    pool.destroy()


def test_tokens_without_a_slot_and_without_q(torch_mod, gsp, ctx):
    """A row whose token count ends before its new tokens stores those that have a slot; Q turns all the same."""
    torch = torch_mod
    pool = gsp.Pool.create(ctx, 4, 1, 2, 64)
    ctx.pack_step(pool, [0, 6], [3, 8], [0, 1, 2], [2, 0], 64, q_lens=[5, 2])
    pos = torch.zeros((3, 7), dtype=torch.int32, device="cuda")
    q = torch.ones((7, 4, 64), device="cuda")
    out = torch.zeros((7, 4, 64), device="cuda")
    k, v = torch.full((7, 2, 64), 2.0, device="cuda"), torch.full((7, 2, 64), 3.0, device="cuda")
    rope = gsp.MRope(1e4, (12, 10, 10))
    torch.cuda.synchronize()
    pool.mrope_write_step(0, 4, rope, pos.data_ptr(), q.data_ptr(), out.data_ptr(), k.data_ptr(), v.data_ptr())
    pool.mrope_write_step(0, 0, rope, pos.data_ptr(), 0, 0, k.data_ptr(), v.data_ptr())
    ctx.sync()
    K = pool.download(0, pool.arenas()[2]).view(np.float32).reshape(4, 2, 16, 64)
    assert torch.equal(out, q)
    assert np.all(K[2, :, :3] == 2) and not K[2, :, 3:].any()
    assert np.all(K[0, :, 6:8] == 2) and not K[0, :, :6].any() and not K[0, :, 8:].any() and not K[[1, 3]].any()
    pool.destroy()


def test_refusals(torch_mod, gsp, ctx):
    torch = torch_mod
    pool = gsp.Pool.create(ctx, 4, 1, 2, 64)
    ctx.pack_step(pool, [0], [5], [0, 1], [1], 64, q_lens=[5])
    q = torch.zeros((5 * 4 * 64 + 64,), device="cuda")
    k = torch.zeros((5 * 2 * 64,), device="cuda")
    v = torch.zeros_like(k)
    pos = torch.zeros((3, 5), dtype=torch.int32, device="cuda")
    out = torch.zeros((5, 4, 64), device="cuda")

    def call(sections=(12, 10, 10), layout=0, heads=4, layer=0, pos_p=pos.data_ptr(), q_p=q.data_ptr(),
             out_p=out.data_ptr(), k_p=k.data_ptr(), v_p=v.data_ptr(), **kw):
        pool.mrope_write_step(layer, heads, gsp.MRope(1e4, sections, layout=layout), pos_p, q_p, out_p, k_p, v_p, **kw)

    for bad in (dict(sections=()), dict(sections=(12, 10, 9)), dict(sections=(-2, 24, 10)), dict(layout=2),
                dict(layout=gsp.MROPE_INTERLEAVED, sections=(2, 15, 15)), dict(layer=1), dict(heads=-1), dict(pos_p=None),
                dict(q_p=0), dict(out_p=0), dict(k_p=None), dict(v_p=None), dict(q_stride=255), dict(k_stride=-128),
                dict(v_stride=127), dict(k_stride=1 << 61), dict(out_p=q.data_ptr() + 256), dict(out_p=k.data_ptr()),
                dict(out_p=pos.data_ptr()), dict(out_p=q.data_ptr(), q_stride=260), dict(k_p=k.data_ptr() + 2),
                dict(pos_p=pos.data_ptr() + 1)):
        with pytest.raises(gsp.InvalidArgument):
            call(**bad)
    odd = gsp.Pool.create(ctx, 4, 1, 2, 63)
    with pytest.raises(gsp.Unsupported):
        odd.mrope_write_step(0, 4, gsp.MRope(1e4, (12, 10, 10)), pos.data_ptr(), q.data_ptr(), out.data_ptr(),
                             k.data_ptr(), v.data_ptr())
    fresh = gsp.Context(0)
    p2 = gsp.Pool.create(fresh, 4, 1, 2, 64)
    with pytest.raises(gsp.StateError):
        p2.mrope_write_step(0, 4, gsp.MRope(1e4, (12, 10, 10)), pos.data_ptr(), q.data_ptr(), out.data_ptr(),
                            k.data_ptr(), v.data_ptr())
    call()
    ctx.sync()
    for p in (pool, odd, p2):
        p.destroy()
    fresh.close()
