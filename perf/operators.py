"""The measured operators around the attention step: what a decoder layer does in 8 bits between two attentions.

  norm    residual addition and root-mean-square norm of the hidden states (Context.rms_norm), its result in fp32,
          in e4m3 with one scale a row, or both.
  quant   activations into e4m3 with one scale a row (Context.quantize_fp8): the attention's output as it is, or the
          gated SiLU of the FFN's two halves, which one fused projection leaves side by side in its rows.
  matmul  a projection of e4m3 activations by 4-bit weights in their GGUF bytes (Context.matmul_batch_fp8).
  mrope   rotary positions of several axes (time, height, width) on the new tokens' queries and keys, and the write of
          keys and values into the paged pool (Pool.mrope_write_step).

`run` computes them in elementary torch operations, or, where `own` is true, through the framework's entry points.
"""
import math
import sys
from pathlib import Path

import numpy as np
import torch

own = False

EPS = 1e-6
FREQ_BASE = 1.0e6
MAX_SEQ = 65536
E4M3_MAX = 448.0
LEAST = 2.0 ** -100  # the least largest magnitude that a row's scale is taken from
E4M3 = torch.float8_e4m3fn
BLOCK = {"q4_0": (32, 18), "q4_1": (32, 20), "q4_k": (256, 144)}  # weights and bytes of a block
# Pairs of a head that turn with each axis: the first ones by time, the next by height, the last by width; or the axes in
# turn as far as each one's count goes, the rest by time.
SECTIONS = {(64, "sections"): (8, 12, 12), (128, "sections"): (16, 24, 24), (64, "interleaved"): (12, 10, 10),
            (128, "interleaved"): (24, 20, 20)}


def _norm(name, rows, dim, residual, out):
    return {"name": name, "op": "norm", "rows": rows, "dim": dim, "residual": residual, "out": out}


def _quant(name, act, rows, dim, pad):
    return {"name": name, "op": "quant", "act": act, "rows": rows, "dim": dim, "pad": pad}


def _matmul(name, w, rows, in_dim, out_dim):
    return {"name": name, "op": "matmul", "w": w, "rows": rows, "in_dim": in_dim, "out_dim": out_dim}


def _mrope(name, heads, kv_heads, head_dim, kv, page, rows, new_lo, new_hi, layout, fused, lens):
    return {"name": name, "op": "mrope", "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim, "kv": kv,
            "page": page, "rows": rows, "new_lo": new_lo, "new_hi": new_hi, "layout": layout, "fused": fused,
            "lens": lens}


def listed():
    return [
        # A small model (hidden 896) serving 8 short chats: launch latency.
        _norm("norm_8x896_fp8", 8, 896, True, "fp8"),
        # The decode tick of 64 rows (hidden 3584), a norm before an 8-bit projection.
        _norm("norm_64x3584_fp8", 64, 3584, True, "fp8"),
        # Prefill chunks of 8192 tokens, an odd one over: both results, for a layer that mixes projection kinds.
        _norm("norm_8193x4096_both", 8193, 4096, True, "both"),
        # The FFN's gate and up halves of a decode tick into the down projection's input.
        _quant("silu_64x18944", "silu", 64, 18944, 0),
        # The attention's output of a prefill chunk before the output projection.
        _quant("quant_4099x3584", "none", 4099, 3584, 0),
        # One chat alone: the fused gate and up projection, 37888 outputs. Reads 76 MB of weights.
        _matmul("mm_q4_0_1x3584x37888", "q4_0", 1, 3584, 37888),
        # The small model's fused QKV projection for 8 chats: latency.
        _matmul("mm_q4_1_8x896x1152", "q4_1", 8, 896, 1152),
        # A decode tick's down projection, its longest sums.
        _matmul("mm_q4_0_64x18944x3584", "q4_0", 64, 18944, 3584),
        # The same tick's fused QKV projection with K-quant weights, an odd batch.
        _matmul("mm_q4_k_37x3584x4608", "q4_k", 37, 3584, 4608),
        # A prefill chunk's widest projection.
        _matmul("mm_q4_0_2048x3584x18944", "q4_0", 2048, 3584, 18944),
        # A decode tick over image and text tokens, keys and values into fp16 pages, Q, K and V side by side in the
        # fused projection's rows.
        _mrope("mrope_decode_64", 28, 4, 128, "f16", 16, 64, 1, 1, "sections", True, 21),
        # Sixteen prompts with images, a few hundred tokens each, into fp32 pages.
        _mrope("mrope_prefill", 28, 4, 128, "f32", 16, 16, 300, 700, "interleaved", False, 22),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the listed ranges; it costs no more than the largest of its operator."""
    op = rng.choice(["norm", "quant", "matmul", "matmul", "mrope"])
    if op == "norm":
        dim = _log_int(rng, 64, 16384)
        if rng.random() < 0.6:
            dim += -dim % 64
        rows = max(1, min(_log_int(rng, 1, 8193), 8193 * 4096 // dim))
        c = _norm("", rows, dim, rng.random() < 0.7, rng.choice(["fp8", "f32", "both"]))
    elif op == "quant":
        dim = _log_int(rng, 64, 18944)
        if rng.random() < 0.6:
            dim += -dim % 64
        rows = max(1, min(_log_int(rng, 1, 4099), 4099 * 3584 // dim))
        c = _quant("", rng.choice(["none", "silu"]), rows, dim, rng.choice([0, 0, 64, 7]))
    elif op == "matmul":
        w = rng.choice(["q4_0", "q4_1", "q4_k"])
        unit = 256 if w == "q4_k" else 64
        in_dim = unit * _log_int(rng, 256 // unit, 18944 // unit)
        out_dim = _log_int(rng, 16, 37888)
        if rng.random() < 0.6:
            out_dim += -out_dim % 16
        rows = max(1, min(_log_int(rng, 1, 4096), 2048 * 3584 * 18944 // (in_dim * out_dim)))
        c = _matmul("", w, rows, in_dim, out_dim)
    else:
        heads, kv_heads, head_dim = rng.choice([(14, 2, 64), (28, 4, 128), (32, 8, 128), (64, 8, 128)])
        hi = _log_int(rng, 1, 700)
        lo = _log_int(rng, 1, hi)
        rows = max(1, min(_log_int(rng, 1, 256), 16 * 700 * 28 * 128 // (hi * heads * head_dim)))
        c = _mrope("", heads, kv_heads, head_dim, rng.choice(["f32", "f16"]), rng.choice([8, 16, 32]), rows, lo, hi,
                   rng.choice(["sections", "interleaved"]), rng.random() < 0.5, rng.randrange(1 << 30))
    del c["name"]
    return c


# ---- what a program has in hand ---------------------------------------------

_GSP = None
_CTX = None


def _gsp():
    global _GSP
    if _GSP is None:
        sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "glacier.serve_amd"))
        import glacier_paged
        _GSP = glacier_paged
    return _GSP


def _context():
    """The engine's one context, on a stream of its own."""
    global _CTX
    if _CTX is None:
        _CTX = _gsp().Context(0)
    return _CTX


class _State:
    """Device buffers, and for the rotary write the context that holds the packed step and the pool over the arenas."""

    def __init__(self, case):
        self.case, self.ctx, self.pool = case, None, None

    def __del__(self):
        if self.pool is not None:
            self.pool.destroy()
            self.ctx.close()


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _activations(rows, dim, g):
    """Hidden states: unit scale with a few channels an order of magnitude larger."""
    x = torch.randn((rows, dim), generator=g, device="cuda")
    loud = torch.rand((dim,), generator=g, device="cuda") < 0.005
    return x.mul_(torch.where(loud, 12.0, 1.0))


def _le16(t):
    return t.to(torch.float16).contiguous().view(torch.uint8)


def _encode(w_type, w):
    """Rows of fp32 weights in the GGUF bytes of `w_type`, rounded to its grid."""
    n, k = w.shape
    if w_type == "q4_0":
        b = w.view(n, k // 32, 32)
        top = b.gather(-1, b.abs().argmax(-1, keepdim=True))
        d = (top / -8).to(torch.float16)
        q = torch.clamp(torch.round(b / d.float()) + 8, 0, 15).to(torch.uint8)
        return torch.cat([_le16(d), q[..., :16] | q[..., 16:] << 4], -1).reshape(n, -1).contiguous()
    if w_type == "q4_1":
        b = w.view(n, k // 32, 32)
        m = b.amin(-1, keepdim=True).to(torch.float16)
        d = ((b.amax(-1, keepdim=True) - m.float()) / 15).to(torch.float16)
        q = torch.clamp(torch.round((b - m.float()) / d.float()), 0, 15).to(torch.uint8)
        return torch.cat([_le16(d), _le16(m), q[..., :16] | q[..., 16:] << 4], -1).reshape(n, -1).contiguous()
    b = w.view(n, k // 256, 8, 32)
    lo = torch.clamp(b.amin(-1), max=0.0)
    step = (b.amax(-1) - lo) / 15
    d = (step.amax(-1, keepdim=True) / 63).to(torch.float16)
    dmin = (-lo.amin(-1, keepdim=True) / 63).to(torch.float16)
    sc = torch.clamp(torch.round(step / d.float()), 1, 63)
    m = torch.clamp(torch.round(-lo / dmin.float()), 0, 63)
    q = torch.round((b + (dmin.float() * m).unsqueeze(-1)) / (d.float() * sc).unsqueeze(-1))
    q = torch.clamp(q, 0, 15).to(torch.uint8)
    sc, m = sc.to(torch.uint8), m.to(torch.uint8)
    head = [sc[..., :4] | (sc[..., 4:] >> 4 << 6), m[..., :4] | (m[..., 4:] >> 4 << 6),
            (sc[..., 4:] & 15) | (m[..., 4:] & 15) << 4]
    qs = (q[..., 0::2, :] | q[..., 1::2, :] << 4).reshape(n, k // 256, 128)
    return torch.cat([_le16(d), _le16(dmin), *head, qs], -1).reshape(n, -1).contiguous()


def _weights(w_type, out_dim, in_dim, g):
    per, size = BLOCK[w_type]
    raw = torch.empty((out_dim, in_dim // per * size), dtype=torch.uint8, device="cuda")
    step = max(1, (1 << 25) // in_dim)
    for at in range(0, out_dim, step):
        w = torch.randn((min(step, out_dim - at), in_dim), generator=g, device="cuda")
        raw[at: at + step] = _encode(w_type, w.div_(math.sqrt(in_dim)))
    return raw


def _positions(case, g):
    """(tokens in the cache, new tokens) of each row, and the new tokens' positions on the three axes [3, tokens]: text
    advances all three together; an image is a grid of rows and columns at one time, and the text behind it starts past
    its longest side."""
    n = case["rows"]
    new = g.integers(case["new_lo"], case["new_hi"] + 1, n)
    before = g.integers(0, 200, n)
    axes = []
    for b in range(n):
        at, parts, left = int(g.integers(0, 30000)), [], int(new[b])
        while left > 0:
            if left > 8 and g.random() < 0.6:
                wide = int(g.integers(2, max(3, math.isqrt(left) + 1)))
                high = int(g.integers(2, max(3, left // wide + 1)))
                cells = np.arange(wide * high)[:left]
                parts.append(np.stack([np.full_like(cells, at), at + cells // wide, at + cells % wide]))
                at += max(wide, high)
            else:
                run_of = int(g.integers(1, left + 1))
                parts.append(np.broadcast_to(at + np.arange(run_of), (3, run_of)))
                at += run_of
            left -= parts[-1].shape[1]
        axes.append(np.concatenate(parts, 1))
    return before, new, np.concatenate(axes, 1).astype(np.int32)


def _prepare_mrope(s, case, seed):
    before, new, axes = _positions(case, np.random.default_rng([case["lens"], 1]))
    page, heads, kvh, d = case["page"], case["heads"], case["kv_heads"], case["head_dim"]
    total = before + new
    pages = -(-total // page)
    rng = np.random.default_rng([case["lens"], seed])
    blocks = int(pages.sum()) * 6 // 5 + 1
    offsets = np.concatenate([[0], np.cumsum(pages)]).astype(np.int32)
    ids = rng.permutation(blocks)[: int(pages.sum())].astype(np.int32)
    n = int(new.sum())
    row = np.repeat(np.arange(case["rows"]), new)
    at = np.concatenate([p + np.arange(m) for p, m in zip(before, new)])
    g = _gen(seed)
    s.block = torch.from_numpy(ids[offsets[row] + at // page].astype(np.int64)).cuda()
    s.slot = torch.from_numpy(at % page).cuda()
    s.axes = torch.from_numpy(axes).cuda()
    shape = (blocks, 2, kvh, page, d)
    dtype = torch.float32 if case["kv"] == "f32" else torch.float16
    s.keys = torch.randn(shape, generator=g, device="cuda").to(dtype)
    s.values = torch.randn(shape, generator=g, device="cuda").to(dtype)
    wide, kv = heads * d, kvh * d
    if case["fused"]:
        rows = torch.randn((n, wide + 2 * kv), generator=g, device="cuda")
        s.q, s.k, s.v = rows[:, :wide], rows[:, wide: wide + kv], rows[:, wide + kv:]
    else:
        s.q, s.k, s.v = (torch.randn((n, w), generator=g, device="cuda") for w in (wide, kv, kv))
    s.q_out = torch.zeros((n, heads, d), device="cuda")
    if own:
        s.axes = s.axes.contiguous()  # the call takes the address of dense [3, tokens], which numpy's order need not be
        # The engine packs a tick once for all its layers.
        gsp = _gsp()
        s.ctx = gsp.Context(0)
        s.pool = gsp.Pool.wrap(s.ctx, s.keys.data_ptr(), s.values.data_ptr(), blocks, 2, kvh, d,
                               gsp.KV_F32 if case["kv"] == "f32" else gsp.KV_F16, block_size=page)
        s.ctx.pack_step(s.pool, before, total, offsets, ids, MAX_SEQ, q_lens=new, want_info=False)
        s.rope = gsp.MRope(FREQ_BASE, SECTIONS[d, case["layout"]], style=gsp.ROPE_HALVES,
                           layout=gsp.MROPE_INTERLEAVED if case["layout"] == "interleaved" else gsp.MROPE_SECTIONS)


def prepare(case, seed):
    s = _State(case)
    g = _gen(seed)
    if case["op"] == "mrope":
        _prepare_mrope(s, case, seed)
        torch.cuda.synchronize()
        return s
    rows = case["rows"]
    if case["op"] == "matmul":
        s.w = _weights(case["w"], case["out_dim"], case["in_dim"], g)
        x = _activations(rows, case["in_dim"], g)
        s.scale = x.abs().amax(-1) / E4M3_MAX
        s.x = torch.clamp(x / s.scale[:, None], -E4M3_MAX, E4M3_MAX).to(E4M3)
        s.y = torch.zeros((rows, case["out_dim"]), device="cuda")
        torch.cuda.synchronize()
        return s
    dim = case["dim"]
    if case["op"] == "norm":
        s.x = _activations(rows, dim, g)
        s.residual = _activations(rows, dim, g).mul_(5.0) if case["residual"] else None
        s.total = torch.zeros((rows, dim), device="cuda") if case["residual"] else None
        s.weight = 1.0 + 0.2 * torch.randn((dim,), generator=g, device="cuda")
        s.y = torch.zeros((rows, dim), device="cuda") if case["out"] != "fp8" else None
    else:
        halves = 2 if case["act"] == "silu" else 1
        s.a = _activations(rows, halves * dim + case["pad"], g)
    if case["op"] == "quant" or case["out"] != "f32":
        s.codes = torch.zeros((rows, dim), dtype=torch.uint8, device="cuda")
        s.scale = torch.zeros((rows,), device="cuda")
    torch.cuda.synchronize()
    return s


# ---- one pass ----------------------------------------------------------------

def _to_e4m3(y):
    top = torch.clamp(y.abs().amax(-1, keepdim=True), min=LEAST)
    codes = torch.clamp(y * (E4M3_MAX / top), -E4M3_MAX, E4M3_MAX).to(E4M3)
    return {"codes": codes, "scale": top[:, 0] / E4M3_MAX}


def _plain_norm(s):
    x = s.x if s.residual is None else s.x + s.residual
    y = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * s.weight
    got = {} if s.residual is None else {"sum": x}
    if s.case["out"] != "fp8":
        got["y"] = y
    if s.case["out"] != "f32":
        got.update(_to_e4m3(y))
    return got


def _plain_quant(s):
    dim = s.case["dim"]
    if s.case["act"] == "none":
        return _to_e4m3(s.a[:, :dim])
    gate, up = s.a[:, :dim], s.a[:, dim: 2 * dim]
    return _to_e4m3(gate / (1.0 + torch.exp(-gate)) * up)


def _plain_weights(w_type, raw, in_dim):
    """The fp32 weights that rows of `w_type` stand for."""
    n = raw.shape[0]
    half = lambda b: b.contiguous().view(torch.float16).float()  # noqa: E731
    if w_type != "q4_k":
        per, size = BLOCK[w_type]
        b = raw.view(n, in_dim // 32, size)
        q = torch.cat([b[..., -16:] & 15, b[..., -16:] >> 4], -1).float()
        w = half(b[..., :2]) * (q - 8.0) if w_type == "q4_0" else half(b[..., :2]) * q + half(b[..., 2:4])
        return w.view(n, in_dim)
    b = raw.view(n, in_dim // 256, 144)
    s0, s1, s2 = b[..., 4:8], b[..., 8:12], b[..., 12:16]
    sc = torch.cat([s0 & 63, (s2 & 15) | (s0 >> 6 << 4)], -1).float()
    m = torch.cat([s1 & 63, (s2 >> 4) | (s1 >> 6 << 4)], -1).float()
    qs = b[..., 16:].reshape(n, -1, 4, 32)
    q = torch.stack([qs & 15, qs >> 4], -2).view(n, -1, 8, 32).float()
    return ((half(b[..., 0:2]) * sc).unsqueeze(-1) * q - (half(b[..., 2:4]) * m).unsqueeze(-1)).view(n, in_dim)


def _plain_matmul(s):
    case = s.case
    w = _plain_weights(case["w"], s.w, case["in_dim"])
    return torch.matmul(s.x.float(), w.t()) * s.scale[:, None]


def _axis_of_pair(d, layout):
    sec, half = SECTIONS[d, layout], d // 2
    j = np.arange(half)
    if layout == "sections":
        return np.repeat(np.arange(3), sec)
    return np.where((j % 3 == 1) & (j < 3 * sec[1]), 1, np.where((j % 3 == 2) & (j < 3 * sec[2]), 2, 0))


def _plain_mrope(s):
    case = s.case
    d, half = case["head_dim"], case["head_dim"] // 2
    axis = torch.from_numpy(_axis_of_pair(d, case["layout"])).to("cuda", non_blocking=True)
    rate = FREQ_BASE ** (-torch.arange(half, dtype=torch.float64, device="cuda") / half)
    angle = s.axes[axis].t().double() * rate  # [tokens, pairs]; far positions need 64 bits
    c, sn = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]

    def turned(x, heads):
        x = x.reshape(-1, heads, d)
        a, b = x[..., :half], x[..., half:]
        return torch.cat([a * c - b * sn, a * sn + b * c], -1)

    q = turned(s.q, case["heads"])
    s.keys[s.block, 1, :, s.slot] = turned(s.k, case["kv_heads"]).to(s.keys.dtype)
    s.values[s.block, 1, :, s.slot] = s.v.reshape(-1, case["kv_heads"], d).to(s.values.dtype)
    return {"q": q, "keys": s.keys, "values": s.values}


PLAIN = {"norm": _plain_norm, "quant": _plain_quant, "matmul": _plain_matmul, "mrope": _plain_mrope}


def _own_norm(s):
    case, at = s.case, lambda t: 0 if t is None else t.data_ptr()  # noqa: E731
    fp8 = case["out"] != "f32"
    _context().rms_norm(case["rows"], case["dim"], at(s.x), at(s.weight), EPS, residual_ptr=at(s.residual),
                        sum_ptr=at(s.total), y_ptr=at(s.y), y_fp8_ptr=at(s.codes) if fp8 else 0,
                        y_scale_ptr=at(s.scale) if fp8 else 0)
    got = {} if s.residual is None else {"sum": s.total}
    if case["out"] != "fp8":
        got["y"] = s.y
    if fp8:
        got.update(codes=s.codes.view(E4M3), scale=s.scale)
    return got


def _own_quant(s):
    case, gsp = s.case, _gsp()
    gated = case["act"] == "silu"
    a = s.a.data_ptr()
    _context().quantize_fp8(gsp.ACT_SILU_MUL if gated else gsp.ACT_NONE, case["rows"], case["dim"], s.a.stride(0), a,
                            a + 4 * case["dim"] if gated else 0, s.codes.data_ptr(), s.scale.data_ptr())
    return {"codes": s.codes.view(E4M3), "scale": s.scale}


def _own_matmul(s):
    case, gsp = s.case, _gsp()
    w_type = {"q4_0": gsp.WTYPE_Q4_0, "q4_1": gsp.WTYPE_Q4_1, "q4_k": gsp.WTYPE_Q4_K}[case["w"]]
    _context().matmul_batch_fp8(w_type, s.w.data_ptr(), s.x.data_ptr(), s.scale.data_ptr(), s.y.data_ptr(),
                                case["in_dim"], case["out_dim"], case["rows"])
    return s.y


def _own_mrope(s):
    s.pool.mrope_write_step(1, s.case["heads"], s.rope, s.axes.data_ptr(), s.q.data_ptr(), s.q_out.data_ptr(),
                            s.k.data_ptr(), s.v.data_ptr(), q_stride=s.q.stride(0), k_stride=s.k.stride(0),
                            v_stride=s.v.stride(0))
    return {"q": s.q_out, "keys": s.keys, "values": s.values}


OWN = {"norm": _own_norm, "quant": _own_quant, "matmul": _own_matmul, "mrope": _own_mrope}


def run(s):
    return (OWN if own else PLAIN)[s.case["op"]](s)


# ---- what a pass cannot do without -------------------------------------------

def work(case):
    op = case["op"]
    if op == "norm":
        cells = case["rows"] * case["dim"]
        per = 4 + 8 * case["residual"] + {"fp8": 1, "f32": 4, "both": 5}[case["out"]]
        return {"bytes": cells * per + 4 * case["dim"] + 4 * case["rows"] * (case["out"] != "f32"), "flops": 6 * cells}
    if op == "quant":
        cells, gated = case["rows"] * case["dim"], case["act"] == "silu"
        return {"bytes": cells * (9 if gated else 5) + 4 * case["rows"], "flops": cells * (8 if gated else 3)}
    if op == "matmul":
        b, i, o = case["rows"], case["in_dim"], case["out_dim"]
        per, size = BLOCK[case["w"]]
        return {"bytes": o * (i // per) * size + b * i + 4 * b + 4 * b * o, "flops": 2 * b * i * o}
    n = int(_positions(case, np.random.default_rng([case["lens"], 1]))[1].sum())
    wide, kv = case["heads"] * case["head_dim"], case["kv_heads"] * case["head_dim"]
    elem = 4 if case["kv"] == "f32" else 2
    return {"bytes": n * (8 * wide + 2 * kv * (4 + elem) + 12), "flops": n * 3 * (wide + kv)}


# ---- the same in 64 bits -----------------------------------------------------

def _exact_codes(y):
    """The values that the codes of y round, and the scales."""
    scale = torch.clamp(y.abs().amax(-1), min=LEAST) / E4M3_MAX
    return {"codes": y / scale[:, None], "scale": scale}


def _exact_weights(w_type, raw, in_dim):
    """Each weight from its block's bytes, one group of 32 after the other."""
    n = raw.shape[0]
    out = torch.empty((n, in_dim), dtype=torch.float64, device="cuda")

    def half(lo, hi):
        bits = lo.to(torch.int32) | hi.to(torch.int32) << 8
        return bits.to(torch.int16).view(torch.float16).double()

    per, size = BLOCK[w_type]
    for g in range(in_dim // 32):
        b = raw[:, g * 32 // per * size:][:, :size]
        if w_type == "q4_k":
            i = g % 8
            if i < 4:
                sc, m = b[:, 4 + i] % 64, b[:, 8 + i] % 64
            else:
                sc = b[:, 8 + i] % 16 + 16 * (b[:, i] // 64)
                m = b[:, 8 + i] // 16 + 16 * (b[:, 4 + i] // 64)
            codes = b[:, 16 + 32 * (i // 2): 48 + 32 * (i // 2)]
            q = (codes // 16 if i % 2 else codes % 16).double()
            w = (half(b[:, 0], b[:, 1]) * sc.double())[:, None] * q - (half(b[:, 2], b[:, 3]) * m.double())[:, None]
        else:
            codes = b[:, size - 16:]
            q = torch.cat([codes % 16, codes // 16], 1).double()
            d = half(b[:, 0], b[:, 1])[:, None]
            w = d * (q - 8) if w_type == "q4_0" else d * q + half(b[:, 2], b[:, 3])[:, None]
        out[:, 32 * g: 32 * g + 32] = w
    return out


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "norm":
        x = s.x.double()
        got = {}
        if s.residual is not None:
            x = x + s.residual.double()
            got["sum"] = x
        y = x / torch.sqrt((x * x).sum(-1, keepdim=True) / case["dim"] + EPS) * s.weight.double()
        if case["out"] != "fp8":
            got["y"] = y
        if case["out"] != "f32":
            got.update(_exact_codes(y))
        return got
    if op == "quant":
        a, dim = s.a.double(), case["dim"]
        y = a[:, :dim]
        return _exact_codes(y if case["act"] == "none" else y * torch.sigmoid(y) * a[:, dim: 2 * dim])
    if op == "matmul":
        w = _exact_weights(case["w"], s.w, case["in_dim"])
        x = s.x.float().double() * s.scale.double()[:, None]
        return torch.matmul(x, w.t().contiguous())
    d, half = case["head_dim"], case["head_dim"] // 2
    axis = _axis_of_pair(d, case["layout"])
    at = s.axes.double()
    keys, values = s.keys.double(), s.values.double()
    q = s.q.double().reshape(-1, case["heads"], d).clone()
    k = s.k.double().reshape(-1, case["kv_heads"], d).clone()
    for j in range(half):
        angle = at[int(axis[j])] * math.exp(-math.log(FREQ_BASE) * j / half)
        turn = torch.polar(torch.ones_like(angle), angle)[:, None]
        for x in (q, k):
            z = torch.complex(x[..., j], x[..., half + j]) * turn
            x[..., j], x[..., half + j] = z.real, z.imag
    keys[s.block, 1, :, s.slot] = k
    values[s.block, 1, :, s.slot] = s.v.double().reshape(-1, case["kv_heads"], d)
    return {"q": q, "keys": keys, "values": values}
