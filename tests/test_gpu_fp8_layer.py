"""The 8-bit operators as a serving layer uses them: one after the other, captured, on other streams, side by side.

A layer: norm -> Q, K and V in one projection -> rotary axes and KV write -> attention -> quantiser -> projection ->
norm with the residual -> gate and up in one projection -> gated quantiser -> projection.  Every stage is checked in
64 bits on what the device gave the stage before it, so that a code that falls on the other side of a rounding border does
not make the rest incomparable.  Tolerances: those of each operator's own tests.
"""
import math
import threading

import numpy as np
import pytest

from fp8_helpers import E4M3, Q4_0, Q4_1, Q4_K, axis_of_pair, check_codes, decode_weights, norm64, random_weights, rotate64

pytestmark = pytest.mark.gpu
EPS = 1e-6
SECTIONS = (8, 12, 12)


class Layer:
    """One decoder layer's buffers for the packed step of `ctx`; 14/2 heads of 64, hidden 896, FFN 1216."""

    def __init__(self, torch, gsp, ctx, rng, q_lens, types=(Q4_0, Q4_1, Q4_0, Q4_1)):
        self.torch, self.gsp, self.ctx, self.types = torch, gsp, ctx, types
        self.heads, self.kvh, self.d, self.hidden, self.ffn = 14, 2, 64, 896, 1216
        before = rng.integers(0, 90, len(q_lens)).astype(np.int32)
        total = before + q_lens
        pages = -(-total // 16)
        self.blocks = int(pages.sum()) + 2
        off = np.concatenate([[0], np.cumsum(pages)]).astype(np.int32)
        ids = rng.permutation(self.blocks)[: off[-1]].astype(np.int32)
        self.step = (before, total, off, ids, np.asarray(q_lens, np.int32))
        n = self.n = int(np.sum(q_lens))
        row = np.repeat(np.arange(len(q_lens)), q_lens)
        at = np.concatenate([b + np.arange(m) for b, m in zip(before, q_lens)])
        self.blk, self.slot, self.row, self.at = ids[off[row] + at // 16], at % 16, row, at
        self.pool = gsp.Pool.create(ctx, self.blocks, 1, self.kvh, self.d)
        kv = rng.standard_normal((self.blocks, 1, self.kvh, 16, self.d)).astype(np.float32)
        self.pool.upload(0, kv)
        self.pool.upload(1, -kv)
        self.qkv_dim = (self.heads + 2 * self.kvh) * self.d
        self.raw = [random_weights(rng, t, o, i) for t, o, i in zip(
            types, (self.qkv_dim, self.hidden, 2 * self.ffn, self.hidden),
            (self.hidden, self.heads * self.d, self.hidden, self.ffn))]
        dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
        f32 = lambda *s: torch.zeros(s, device="cuda")  # noqa: E731
        u8 = lambda *s: torch.zeros(s, dtype=torch.uint8, device="cuda")  # noqa: E731
        self.w = [dev(r) for r in self.raw]
        self.x0 = rng.standard_normal((n, self.hidden)).astype(np.float32)
        self.x, self.res = dev(self.x0), f32(n, self.hidden)
        self.nw = (1 + 0.2 * rng.standard_normal((2, self.hidden))).astype(np.float32)
        self.nwd = dev(self.nw)
        self.axes = np.stack([at + 3, at // 2, at % 7]).astype(np.int32)
        self.pos = dev(self.axes)
        self.c = [u8(n, self.hidden), u8(n, self.heads * self.d), u8(n, self.hidden), u8(n, self.ffn)]
        self.s = [f32(n) for _ in range(4)]
        self.qkv, self.q, self.o = f32(n, self.qkv_dim), f32(n, self.heads, self.d), f32(n, self.heads, self.d)
        self.att, self.gu, self.y = f32(n, self.hidden), f32(n, 2 * self.ffn), f32(n, self.hidden)
        self.rope = gsp.MRope(1e4, SECTIONS, style=gsp.ROPE_HALVES)
        torch.cuda.synchronize()

    def pack(self):
        before, total, off, ids, q_lens = self.step
        self.ctx.pack_step(self.pool, before, total, off, ids, 4096, q_lens=q_lens)

    def run(self):
        ctx, gsp, n, p = self.ctx, self.gsp, self.n, lambda t: t.data_ptr()  # noqa: E731
        wide, kv = self.heads * self.d, self.kvh * self.d
        ctx.rms_norm(n, self.hidden, p(self.x), p(self.nwd), EPS, y_fp8_ptr=p(self.c[0]), y_scale_ptr=p(self.s[0]))
        ctx.matmul_batch_fp8(self.types[0], p(self.w[0]), p(self.c[0]), p(self.s[0]), p(self.qkv), self.hidden,
                             self.qkv_dim, n)
        self.pool.mrope_write_step(0, self.heads, self.rope, p(self.pos), p(self.qkv), p(self.q), p(self.qkv) + 4 * wide,
                                   p(self.qkv) + 4 * (wide + kv), q_stride=self.qkv_dim, k_stride=self.qkv_dim,
                                   v_stride=self.qkv_dim)
        ctx.attention_step(self.pool, 0, self.heads, p(self.q), p(self.o), 1 / math.sqrt(self.d))
        ctx.quantize_fp8(gsp.ACT_NONE, n, wide, wide, p(self.o), 0, p(self.c[1]), p(self.s[1]))
        ctx.matmul_batch_fp8(self.types[1], p(self.w[1]), p(self.c[1]), p(self.s[1]), p(self.att), wide, self.hidden, n)
        ctx.rms_norm(n, self.hidden, p(self.att), p(self.nwd) + 4 * self.hidden, EPS, residual_ptr=p(self.x),
                     sum_ptr=p(self.res), y_fp8_ptr=p(self.c[2]), y_scale_ptr=p(self.s[2]))
        ctx.matmul_batch_fp8(self.types[2], p(self.w[2]), p(self.c[2]), p(self.s[2]), p(self.gu), self.hidden, 2 * self.ffn, n)
        ctx.quantize_fp8(gsp.ACT_SILU_MUL, n, self.ffn, 2 * self.ffn, p(self.gu), p(self.gu) + 4 * self.ffn, p(self.c[3]),
                         p(self.s[3]))
        ctx.matmul_batch_fp8(self.types[3], p(self.w[3]), p(self.c[3]), p(self.s[3]), p(self.y), self.ffn, self.hidden, n)

    def outputs(self):
        got = [t.cpu().numpy().copy() for t in (*self.c, *self.s, self.qkv, self.q, self.o, self.att, self.res, self.gu, self.y)]
        return got + [self.pool.download(i, self.pool.arenas()[2 + i]) for i in (0, 1)]

    def check(self):
        n, d = self.n, self.d
        wide, kv = self.heads * d, self.kvh * d
        c = [t.cpu().numpy() for t in self.c]
        s = [t.cpu().numpy() for t in self.s]
        qkv, q, o, att, res, gu, y = (t.cpu().numpy() for t in (self.qkv, self.q, self.o, self.att, self.res, self.gu, self.y))

        def product(i, codes, scale, in_dim, got):
            w, mag = decode_weights(self.types[i], self.raw[i], in_dim)
            x = E4M3[codes] * scale.astype(np.float64)[:, None]
            bound = (37 + in_dim / 16) * 2.0 ** -23 * (np.abs(x) @ mag.T) + 1e-40
            assert np.all(np.abs(got - x @ w.T) <= bound), f"projection {i}"

        _, y64 = norm64(self.x0, None, self.nw[0], EPS)
        check_codes(c[0], s[0], y64, 40 * 2.0 ** -24)
        product(0, c[0], s[0], self.hidden, qkv)
        axis = axis_of_pair(SECTIONS, False)
        rates = 1e4 ** (-2.0 * np.arange(d // 2) / d)
        wq, mq = rotate64(qkv[:, :wide].reshape(n, self.heads, d), self.axes, axis, rates, d, True)
        wk, mk = rotate64(qkv[:, wide: wide + kv].reshape(n, self.kvh, d), self.axes, axis, rates, d, True)
        K, V = (self.pool.download(i, self.pool.arenas()[2 + i]).view(np.float32).reshape(self.blocks, self.kvh, 16, d)
                for i in (0, 1))
        assert np.all(np.abs(q - wq) <= 5e-7 * mq + 1e-12)
        assert np.all(np.abs(K[self.blk, :, self.slot] - wk) <= 5e-7 * mk + 1e-12)
        assert np.array_equal(V[self.blk, :, self.slot], qkv[:, wide + kv:].reshape(n, self.kvh, d))
        self.check_attention(q.astype(np.float64), K.astype(np.float64), V.astype(np.float64), o)
        check_codes(c[1], s[1], o.reshape(n, wide).astype(np.float64), 0.0)
        product(1, c[1], s[1], wide, att)
        total, y64 = norm64(att, self.x0, self.nw[1], EPS)
        assert np.array_equal(res, total)
        check_codes(c[2], s[2], y64, 40 * 2.0 ** -24)
        product(2, c[2], s[2], self.hidden, gu)
        g, u = gu[:, : self.ffn].astype(np.float64), gu[:, self.ffn:].astype(np.float64)
        with np.errstate(over="ignore"):
            check_codes(c[3], s[3], g / (1 + np.exp(-g)) * u, 8 * 2.0 ** -24)
        product(3, c[3], s[3], self.ffn, y)

    def check_attention(self, q, K, V, o):
        _, _, off, ids, _ = self.step
        for t in range(self.n):
            b, total = self.row[t], self.at[t] + 1
            pages = ids[off[b]: off[b + 1]]
            kk = K[pages].transpose(1, 0, 2, 3).reshape(self.kvh, -1, self.d)[:, :total]
            vv = V[pages].transpose(1, 0, 2, 3).reshape(self.kvh, -1, self.d)[:, :total]
            g = self.heads // self.kvh
            sc = np.einsum("hgd,htd->hgt", q[t].reshape(self.kvh, g, self.d), kk) / math.sqrt(self.d)
            p = np.exp(sc - sc.max(-1, keepdims=True))
            want = np.einsum("hgt,htd->hgd", p / p.sum(-1, keepdims=True), vv).reshape(self.heads, self.d)
            # the attention step's own bar is 1e-4 for values of unit size; scores and values here are larger
            assert np.max(np.abs(o[t] - want)) <= 1e-4 * max(1.0, np.abs(vv).max(), np.abs(sc).max())


ROWS = {"decode": [1] * 9, "mixed": [1, 1, 40, 1, 33, 1], "prefill": [200, 61, 300]}


@pytest.mark.parametrize("rows", list(ROWS))
def test_layer(torch_mod, gsp, ctx, rows):
    layer = Layer(torch_mod, gsp, ctx, np.random.default_rng(5), np.array(ROWS[rows]))
    layer.pack()
    layer.run()
    ctx.sync()
    layer.check()
    layer.pool.destroy()


@pytest.mark.parametrize("rows", list(ROWS))
def test_layer_captured_and_replayed(torch_mod, gsp, rows):
    """Replays between eager work of other sizes give what the eager layer gave, bit for bit, each time."""
    torch = torch_mod
    ctx = gsp.Context(0)
    stream = torch.cuda.Stream()
    ctx.set_stream(stream.cuda_stream)
    rng = np.random.default_rng(6)
    layer = Layer(torch, gsp, ctx, rng, np.array(ROWS[rows]))
    big = torch.zeros((700, 896), dtype=torch.uint8, device="cuda")
    ones, by = torch.ones(700, device="cuda"), torch.zeros((700, layer.qkv_dim), device="cuda")
    torch.cuda.synchronize()
    layer.pack()
    layer.run()
    ctx.sync()
    want = layer.outputs()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=stream):
        layer.run()
    for _ in range(3):
        for t in (*layer.c, *layer.s, layer.qkv, layer.q, layer.o, layer.att, layer.res, layer.gu, layer.y):
            t.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            g.replay()
        # an eager product that needs more workspace than the captured ones
        ctx.matmul_batch_fp8(Q4_0, layer.w[0].data_ptr(), big.data_ptr(), ones.data_ptr(), by.data_ptr(), 896, layer.qkv_dim, 700)
        torch.cuda.synchronize()
        for a, b in zip(layer.outputs(), want):
            assert np.array_equal(a, b)
    del g
    layer.pool.destroy()
    ctx.close()


def test_cold_capture_of_a_split_product_is_refused(torch_mod, gsp):
    torch = torch_mod
    ctx = gsp.Context(0)
    stream = torch.cuda.Stream()
    ctx.set_stream(stream.cuda_stream)
    rng = np.random.default_rng(1)
    in_dim, out_dim, batch = 4864, 130, 70
    w = torch.from_numpy(random_weights(rng, Q4_1, out_dim, in_dim)).cuda()
    x = torch.randint(0, 120, (batch, in_dim), dtype=torch.uint8, device="cuda")
    s, y, z = torch.ones(batch, device="cuda"), torch.full((batch, out_dim), 7.0, device="cuda"), torch.zeros(4, device="cuda")

    def call():
        ctx.matmul_batch_fp8(Q4_1, w.data_ptr(), x.data_ptr(), s.data_ptr(), y.data_ptr(), in_dim, out_dim, batch)

    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=stream):
        z.add_(1)
        with pytest.raises(gsp.StateError):
            call()
    g.replay()
    torch.cuda.synchronize()
    assert torch.all(y == 7.0) and torch.all(z == 1.0)
    call()
    torch.cuda.synchronize()
    want = y.clone()
    g2 = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g2, stream=stream):
        call()
    for _ in range(3):
        y.zero_()
        torch.cuda.synchronize()
        g2.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want)
    del g, g2
    ctx.close()


def test_two_contexts_side_by_side(torch_mod, gsp):
    """Two engine threads, a context and a stream each, give what each gives alone."""
    torch = torch_mod
    ctxs = [gsp.Context(0) for _ in range(2)]
    layers = [Layer(torch, gsp, c, np.random.default_rng(20 + i), np.array(ROWS["mixed" if i else "prefill"]))
              for i, c in enumerate(ctxs)]
    alone = []
    for layer in layers:
        layer.pack()
        layer.run()
        layer.ctx.sync()
        alone.append(layer.outputs())
    errors = []

    def work(layer):
        try:
            for _ in range(10):
                layer.run()
            layer.ctx.sync()
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(layer,)) for layer in layers]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    assert not errors
    for layer, want in zip(layers, alone):
        for a, b in zip(layer.outputs(), want):
            assert np.array_equal(a, b)
        layer.pool.destroy()
        layer.ctx.close()


def test_k_quant_weights_through_every_form(torch_mod, gsp, ctx):
    """The same rows at every batch size class: a row's outputs agree between the forms within the bound of either."""
    torch = torch_mod
    rng = np.random.default_rng(8)
    in_dim, out_dim = 1536, 5000
    for w_type in (Q4_0, Q4_1, Q4_K):
        raw = random_weights(rng, w_type, out_dim, in_dim)
        codes = rng.integers(0, 120, (1300, in_dim)).astype(np.uint8) | (rng.integers(0, 2, (1300, in_dim)).astype(np.uint8) << 7)
        w, mag = decode_weights(w_type, raw, in_dim)
        wd, xd, s = torch.from_numpy(raw).cuda(), torch.from_numpy(codes).cuda(), torch.full((1300,), 0.01, device="cuda")
        x = E4M3[codes[-1]] * float(np.float32(0.01))
        bound = (37 + in_dim / 16) * 2.0 ** -23 * (np.abs(x) @ mag.T) + 1e-40
        for batch in (1, 4, 5, 8, 9, 16, 17, 33, 64, 65, 200, 1300):
            y = torch.full((batch, out_dim), float("nan"), device="cuda")
            torch.cuda.synchronize()
            at = 1300 - batch
            ctx.matmul_batch_fp8(w_type, wd.data_ptr(), xd.data_ptr() + at * in_dim, s.data_ptr(), y.data_ptr(), in_dim,
                                 out_dim, batch)
            ctx.sync()
            got = y.cpu().numpy()
            assert np.all(np.isfinite(got))
            assert np.all(np.abs(got[-1] - x @ w.T) <= bound), (w_type, batch)


def test_nan_rows_in_the_128_row_form(torch_mod, gsp, ctx):
    torch = torch_mod
    rng = np.random.default_rng(9)
    in_dim, out_dim, batch = 576, 5000, 1290
    raw = random_weights(rng, Q4_1, out_dim, in_dim)
    codes = rng.integers(0, 120, (batch, in_dim)).astype(np.uint8)
    codes[3, 575], codes[200, 0] = 0x7f, 0xff
    wd, xd, s = torch.from_numpy(raw).cuda(), torch.from_numpy(codes).cuda(), torch.ones(batch, device="cuda")
    y = torch.zeros((batch, out_dim), device="cuda")
    torch.cuda.synchronize()
    ctx.matmul_batch_fp8(Q4_1, wd.data_ptr(), xd.data_ptr(), s.data_ptr(), y.data_ptr(), in_dim, out_dim, batch)
    ctx.sync()
    bad = torch.isnan(y).any(1).cpu().numpy()
    assert set(np.nonzero(bad)[0]) == {3, 200}
    assert torch.isnan(y[[3, 200]]).all()


@pytest.mark.parametrize("out_dim", [130, 16400, 70000])
@pytest.mark.parametrize("batch", [1, 33, 64])
def test_cold_capture_up_to_64_rows(torch_mod, gsp, batch, out_dim):
    """Products of up to 64 rows need no workspace: a context's first call may be captured."""
    torch = torch_mod
    ctx = gsp.Context(0)
    stream = torch.cuda.Stream()
    ctx.set_stream(stream.cuda_stream)
    rng = np.random.default_rng(batch)
    in_dim = 320
    raw = random_weights(rng, Q4_1, out_dim, in_dim)
    codes = rng.integers(0, 120, (batch, in_dim)).astype(np.uint8)
    w, x = torch.from_numpy(raw).cuda(), torch.from_numpy(codes).cuda()
    s, y = torch.ones(batch, device="cuda"), torch.zeros((batch, out_dim), device="cuda")
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=stream):
        ctx.matmul_batch_fp8(Q4_1, w.data_ptr(), x.data_ptr(), s.data_ptr(), y.data_ptr(), in_dim, out_dim, batch)
    wm, mag = decode_weights(Q4_1, raw, in_dim)
    X = E4M3[codes]
    bound = (37 + in_dim / 16) * 2.0 ** -23 * (np.abs(X) @ mag.T)
    for _ in range(2):
        y.zero_()
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert np.all(np.abs(y.cpu().numpy() - X @ wm.T) <= bound)
    del g
    ctx.close()
