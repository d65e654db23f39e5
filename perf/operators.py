"""Cases of the low-precision serving operators and of the root-mean-square norm: what each has to
compute, in plain torch operations, beside the calls a user makes of ``mmltk_b200.ops``.

A quantised tensor is kept as *codes* (4-bit codes two to a byte, the even element in the low
half; 8-bit codes as float8_e4m3fn) whose rows are padded to 16 bytes, and *scales*, one byte per
block of a row's elements, in tiles of 128 rows x 4 blocks: byte ``[r / 128, b / 4, r % 32,
(r / 32) % 4, b % 4]`` belongs to row r, block b; rows and blocks past the end are zero bytes.
"""
import math

import torch

own = False

FORMATS = {  # elements per scale, largest element, bits, power-of-two scales
    "mxfp4": (32, 6.0, 4, True),
    "nvfp4": (16, 6.0, 4, False),
    "mxfp8": (32, 448.0, 8, True),
}
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
EPS = 1e-6


def listed():
    return [
        # pre-norm block of the ViT in training: 8 images x 1300 tokens, width 384
        {"name": "norm_train_vit", "op": "norm", "rows": 10400, "dim": 384, "dtype": "bf16", "residual": True},
        # a width that no vector load divides, fp32, a plain norm with nothing to add
        {"name": "norm_train_odd", "op": "norm", "rows": 2999, "dim": 1111, "dtype": "f32", "residual": False},
        # wide rows of a large model's training step
        {"name": "norm_train_wide", "op": "norm", "rows": 16384, "dim": 8192, "dtype": "bf16", "residual": True},
        # one token on its way into an 8-bit product
        {"name": "norm_q8_token", "op": "norm_q", "rows": 1, "dim": 2048, "dtype": "bf16", "residual": True},
        # a large serving batch
        {"name": "norm_q8_wide", "op": "norm_q", "rows": 32768, "dim": 4096, "dtype": "bf16", "residual": True},
        # the ViT's first MLP weight, quantised and read back
        {"name": "quant4_mx_fc1", "op": "quant", "rows": 1536, "dim": 384, "dtype": "bf16", "fmt": "mxfp4"},
        # a large weight, with the scale of the whole tensor found first
        {"name": "quant4_nv_wide", "op": "quant", "rows": 16384, "dim": 8192, "dtype": "bf16", "fmt": "nvfp4"},
        # one token through a 4-bit weight: the weight's bytes are the work
        {"name": "linear4_token", "op": "linear", "m": 1, "n": 4096, "k": 4096, "dtype": "bf16", "fmt": "nvfp4",
         "act": "none", "out": "same"},
        # the ViT's first MLP product, 8 images
        {"name": "linear4_vit", "op": "linear", "m": 10400, "n": 1536, "k": 384, "dtype": "bf16", "fmt": "mxfp4",
         "act": "gelu", "out": "same"},
        # a long prompt or a large batch against a large weight: the tensor cores' case
        {"name": "linear4_large", "op": "linear", "m": 8192, "n": 8192, "k": 8192, "dtype": "bf16", "fmt": "nvfp4",
         "act": "none", "out": "same"},
        # a few tokens, sizes that no tile divides
        {"name": "linear8_few", "op": "linear", "m": 17, "n": 2050, "k": 1000, "dtype": "f16", "fmt": "mxfp8",
         "act": "none", "out": "same"},
        # the decoder's first FFN product (8 images x 3900 queries), whose output feeds the second in 8 bits
        {"name": "linear8_dec", "op": "linear", "m": 31200, "n": 2048, "k": 256, "dtype": "bf16", "fmt": "mxfp8",
         "act": "relu", "out": "mxfp8"},
    ]


def _between(rng, lo, hi):
    """A whole number, spread over the logarithm of its range."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "norm", "norm_q", "quant", "linear", "linear", "linear"])
    if op == "linear":
        fmt = rng.choice(["mxfp4", "nvfp4", "mxfp8"])
        n, k = _between(rng, 64, 8192), _between(rng, 64, 8192)
        if rng.random() < 0.5:      # a model's own sizes; else whatever comes
            n, k = -(-n // 64) * 64, -(-k // 64) * 64
        return {"op": op, "m": _between(rng, 1, 16384 if n * k <= 4096 * 8192 else 8192), "n": n, "k": k,
                "dtype": rng.choice(["bf16", "f16"]), "fmt": fmt, "act": rng.choice(["none", "relu", "gelu"]),
                "out": rng.choice(["same", "same", "same", "mxfp8"])}
    dim = _between(rng, 64, 8192)
    if rng.random() < 0.6:
        dim = -(-dim // 64) * 64
    rows = _between(rng, 1, min(65536, 16384 * 8192 // dim))
    c = {"op": op, "rows": rows, "dim": dim, "dtype": rng.choice(["bf16", "bf16", "f16", "f32"])}
    if c["dtype"] == "f32":
        c["rows"] = (rows + 1) // 2
    if op == "quant":
        return {**c, "fmt": rng.choice(["mxfp4", "nvfp4"])}
    return {**c, "residual": rng.random() < 0.7}


# ---------------------------------------------------------------- the formats in plain torch
def _blocks(x, size):
    """[rows, dim] -> [rows, blocks, size], zeros behind the last element."""
    rows, dim = x.shape
    nb = -(-dim // size)
    return torch.nn.functional.pad(x, (0, nb * size - dim)).view(rows, nb, size)


def _round_e2m1(x):
    """Nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 (ties to the even code), as the value; sign kept."""
    a = x.abs()
    step = torch.where(a < 2.0, 0.5, torch.where(a < 4.0, 1.0, 2.0))   # grid spacing around a (a tie sits between)
    return torch.copysign((torch.round(a / step) * step).clamp(max=6.0), x)


def _round_elements(x, fmt):
    if FORMATS[fmt][2] == 4:
        return _round_e2m1(x)
    return x.clamp(-448.0, 448.0).to(torch.float8_e4m3fn).float()


def _scale_of(amax, fmt, g):
    """(scale byte, scale value, factor that takes x to the element grid) of blocks with this largest magnitude."""
    size, top, bits, pow2 = FORMATS[fmt]
    if pow2:
        m, e = torch.frexp(amax)                            # amax = m 2^e, m in [0.5, 1)
        p = (e - (3 if bits == 4 else 9) + (m > top / (8.0 if bits == 4 else 512.0)).int()).clamp(-127, 127)
        p = torch.where(amax > 0, p, torch.full_like(p, -127))
        byte = (p + 127).to(torch.uint8)
        return byte, byte.view(torch.float8_e8m0fnu).float(), ((127 - p) << 23).view(torch.float32)
    s8 = (amax / (6.0 * g)).clamp(max=448.0).to(torch.float8_e4m3fn)
    s = s8.float()
    return s8.view(torch.uint8), s, torch.where(s > 0, 1.0 / (s * g), 0.0)


def _quantize(x, fmt, g):
    """fp32 [rows, dim] -> (elements [rows, dim] as values, scale bytes [rows, blocks], values [rows, dim])."""
    rows, dim = x.shape
    xb = _blocks(x, FORMATS[fmt][0])
    byte, s, inv = _scale_of(xb.abs().amax(-1), fmt, g)
    q = _round_elements(xb * inv[..., None], fmt)
    v = q * s[..., None]
    return q.reshape(rows, -1)[:, :dim], byte, v.reshape(rows, -1)[:, :dim]


def _tensor_scale(x):
    """fp32 scale of a whole tensor that puts its largest block scale at the top of e4m3."""
    a = x.abs().amax()
    return torch.where(a > 0, (a / 2688.0).clamp(min=2.0 ** -100), 1.0).reshape(1)


def _tile_scales(byte):
    rows, nb = byte.shape
    rt, kt = -(-rows // 128), -(-nb // 4)
    full = torch.nn.functional.pad(byte, (0, kt * 4 - nb, 0, rt * 128 - rows))
    return full.view(rt, 4, 32, kt, 4).permute(0, 3, 2, 1, 4).contiguous()


def _pack(q, fmt):
    """Element values [rows, dim] -> codes, rows padded to 16 bytes."""
    dim = q.shape[1]
    if FORMATS[fmt][2] == 8:
        return torch.nn.functional.pad(q, (0, -dim % 16)).to(torch.float8_e4m3fn)
    grid = torch.tensor(E2M1, device=q.device)
    code = torch.bucketize(q.abs(), grid).to(torch.uint8) | (torch.signbit(q).to(torch.uint8) << 3)
    code = torch.nn.functional.pad(code, (0, -dim % 32))
    return code[:, 0::2] | (code[:, 1::2] << 4)


def _elements(codes, fmt, dim):
    if FORMATS[fmt][2] == 8:
        return codes[:, :dim].float()
    grid = torch.tensor(E2M1 + tuple(-v for v in E2M1), device=codes.device)
    return grid[torch.stack((codes & 15, codes >> 4), -1).view(codes.shape[0], -1)[:, :dim].long()]


# ---------------------------------------------------------------- inputs
def prepare(case, seed):
    dev = "cuda"
    gen = torch.Generator(device=dev).manual_seed(seed)

    def normal(*shape, scale=1.0):
        return torch.randn(*shape, device=dev, generator=gen) * scale

    def activations(rows, dim):
        # a few channels far louder than the rest, as between the layers of a transformer
        return normal(rows, dim) * (1 + 12 * (torch.rand(dim, device=dev, generator=gen) < 0.01))

    dt = DTYPES[case["dtype"]]
    st = {"case": dict(case)}
    if case["op"] in ("norm", "norm_q"):
        rows, dim = case["rows"], case["dim"]
        st["x"] = activations(rows, dim).to(dt)
        st["r"] = normal(rows, dim, scale=2.0).to(dt) if case["residual"] else None
        st["w"] = (1 + normal(dim, scale=0.2)).to(dt)
        if case["op"] == "norm":
            st["gy"] = normal(rows, dim).to(dt)
            st["gh"] = normal(rows, dim).to(dt) if case["residual"] else None
            for n in ("x", "r", "w"):
                if st[n] is not None:
                    st[n].requires_grad_()
    elif case["op"] == "quant":
        st["x"] = (normal(case["rows"], case["dim"]) * case["dim"] ** -0.5).to(dt)
    else:
        m, n, k, fmt = case["m"], case["n"], case["k"], case["fmt"]
        st["x"] = activations(m, k).to(dt)
        st["bias"] = normal(n, scale=0.1).to(dt)
        w = normal(n, k, scale=k ** -0.5)
        st["g"] = _tensor_scale(w) if fmt == "nvfp4" else None
        q, byte, _ = _quantize(w, fmt, st["g"])
        # the weight as it is kept: codes and tiled scales, and its scales row by row
        st["codes"], st["scales"], st["row_scales"] = _pack(q, fmt), _tile_scales(byte), byte
    return st


# ---------------------------------------------------------------- one pass
def run(state):
    return (_run_own if own else _run_plain)(state)


def _grads(y, h, st):
    ins = [t for t in (st["x"], st["r"], st["w"]) if t is not None]
    outs, gs = ([y], [st["gy"]]) if h is None else ([y, h], [st["gy"], st["gh"]])
    return torch.autograd.grad(outs, ins, gs)


def _run_own(st):
    from mmltk_b200 import ops
    c = st["case"]
    if c["op"] == "norm":
        if st["r"] is None:
            y = ops.rms_norm(st["x"], st["w"], EPS)
            return y.detach(), *_grads(y, None, st)
        y, h = ops.add_rms_norm(st["x"], st["r"], st["w"], EPS)
        return y.detach(), h.detach(), *_grads(y, h, st)
    if c["op"] == "norm_q":
        t, h = ops.rms_norm_quantized(st["x"], st["w"], EPS, residual=st["r"], fmt="mxfp8")
        out = (t.codes[:, :c["dim"]], t.scales.view(torch.float8_e8m0fnu))
        return out if st["r"] is None else (*out, h)
    if c["op"] == "quant":
        t = ops.mx_quantize(st["x"], c["fmt"])
        v = t.dequantize(torch.bfloat16)
        return v if t.global_scale is None else (v, t.global_scale)
    w = ops.MXTensor(st["codes"], st["scales"], c["fmt"], (c["n"], c["k"]), st["g"])
    act = None if c["act"] == "none" else c["act"]
    if c["out"] == "same":
        return ops.mx_linear(st["x"], w, st["bias"], act=act)
    t = ops.mx_linear(st["x"], w, st["bias"], act=act, out_fmt=c["out"])
    return t.codes[:, :c["n"]], t.scales.view(torch.float8_e8m0fnu)


def _rms(h, w):
    return h * torch.rsqrt(h.square().mean(-1, keepdim=True) + EPS) * w


class _Round(torch.autograd.Function):
    """Rounds a sum to its stored type; the gradient passes."""

    @staticmethod
    def forward(ctx, x, dt):
        return x.to(dt).float()

    @staticmethod
    def backward(ctx, g):
        return g, None


def _run_plain(st):
    c = st["case"]
    dt = DTYPES[c["dtype"]]
    if c["op"] == "norm":
        h = st["x"].float() if st["r"] is None else _Round.apply(st["x"].float() + st["r"].float(), dt)
        y = _rms(h, st["w"].float())
        if st["r"] is None:
            return y.detach().to(dt), *_grads32(y, None, st)
        return y.detach().to(dt), h.detach().to(dt), *_grads32(y, h, st)
    if c["op"] == "norm_q":
        h = st["x"].float() if st["r"] is None else (st["x"].float() + st["r"].float()).to(dt).float()
        q, byte, _ = _quantize(_rms(h, st["w"].float()), "mxfp8", None)
        out = (q.to(torch.float8_e4m3fn), _tile_scales(byte).view(torch.float8_e8m0fnu))
        return out if st["r"] is None else (*out, h.to(dt))
    if c["op"] == "quant":
        x = st["x"].float()
        g = _tensor_scale(x) if c["fmt"] == "nvfp4" else None
        v = _quantize(x, c["fmt"], g)[2]
        return v.to(torch.bfloat16) if g is None else ((v * g).to(torch.bfloat16), g)
    fmt, k = c["fmt"], c["k"]
    one = torch.ones(1, device="cuda")
    xv = _quantize(st["x"].float(), fmt, one)[2]
    size, _, _, pow2 = FORMATS[fmt]
    s = st["row_scales"].view(torch.float8_e8m0fnu if pow2 else torch.float8_e4m3fn).float()
    wv = _elements(st["codes"], fmt, k) * s.repeat_interleave(size, 1)[:, :k]
    y = xv @ wv.t()
    if st["g"] is not None:
        y = y * st["g"]
    y = y + st["bias"].float()
    if c["act"] == "relu":
        y = y.clamp(min=0)
    elif c["act"] == "gelu":
        y = 0.5 * y * (1 + torch.erf(y * 0.7071067811865476))
    if c["out"] == "same":
        return y.to(dt)
    q, byte, _ = _quantize(y, c["out"], None)
    return q.to(torch.float8_e4m3fn), _tile_scales(byte).view(torch.float8_e8m0fnu)


def _grads32(y, h, st):
    """Gradients through the 32-bit graph, each rounded once to its input's type (autograd's own casts)."""
    ins = [t for t in (st["x"], st["r"], st["w"]) if t is not None]
    outs, gs = ([y], [st["gy"].float()]) if h is None else ([y, h], [st["gy"].float(), st["gh"].float()])
    return torch.autograd.grad(outs, ins, gs)


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    e = {"bf16": 2, "f16": 2, "f32": 4}[case["dtype"]]
    if case["op"] == "linear":
        m, n, k, fmt = case["m"], case["n"], case["k"], case["fmt"]
        size, _, bits, _ = FORMATS[fmt]
        w = n * k * bits / 8 + n * k / size
        y = m * n * e if case["out"] == "same" else m * n * (1 + 1 / 32)
        return {"bytes": w + n * e + m * k * e + y, "flops": 2.0 * m * n * k}
    t = case["rows"] * case["dim"]
    if case["op"] == "quant":
        size = FORMATS[case["fmt"]][0]
        q = t / 2 + t / size        # written by one half of the pass, read by the other
        return {"bytes": t * e + 2 * q + t * 2, "flops": 4.0 * t}
    r = 1 if case["residual"] else 0
    if case["op"] == "norm_q":
        return {"bytes": t * e * (1 + 2 * r) + t * (1 + 1 / 32) + case["dim"] * e, "flops": 6.0 * t}
    # forward: x (and the residual) in, y (and the sum) out; backward: the sum, its gradients in, theirs out
    return {"bytes": t * e * (2 + 2 * r) + t * e * (2 + r) + t * e + 3 * case["dim"] * e, "flops": 14.0 * t}


# ---------------------------------------------------------------- the definition in 64 bits
def _grid64(y, fmt):
    """Scale of each block by the format's rule, in 64 bits: (scale bytes' values [rows, blocks], per-element scale)."""
    size, top, bits, pow2 = FORMATS[fmt]
    rows, dim = y.shape
    nb = (dim + size - 1) // size
    z = torch.zeros(rows, nb * size, dtype=torch.float64, device=y.device)
    z[:, :dim] = y
    amax = z.reshape(rows, nb, size).abs().max(-1).values
    if pow2:
        p = torch.ceil(torch.log2(amax / top)).clamp(-127, 127)
        p = torch.where(amax > top * torch.exp2(p), p + 1, torch.where(amax <= top * torch.exp2(p - 1), p - 1, p))
        s = torch.exp2(p.clamp(-127, 127))
    else:
        s = (amax / 6).clamp(max=448).float().to(torch.float8_e4m3fn).double()
    return s, s[:, :, None].expand(-1, -1, size).reshape(rows, nb * size)[:, :dim]


def _nearest64(v, fmt):
    """Nearest element, ties to the even one, by the exponent of each value."""
    lo, mant, top = (0, 1, 6.0) if FORMATS[fmt][2] == 4 else (-6, 3, 448.0)
    e = torch.frexp(v)[1].double() - 1
    ulp = torch.exp2(e.clamp(min=lo) - mant)
    return (torch.round(v / ulp) * ulp).clamp(-top, top)


def _values64(y, fmt):
    _, s = _grid64(y, fmt)
    return torch.where(s > 0, _nearest64(torch.where(s > 0, y / s, 0.0), fmt) * s, 0.0)


def _quantised64(y):
    """8-bit output: the elements before their rounding (they are within half a step of them), and the tiled scales."""
    s, se = _grid64(y, "mxfp8")
    rows, nb = s.shape
    tiled = torch.full((-(-rows // 128), -(-nb // 4), 32, 4, 4), 2.0 ** -127, dtype=torch.float64, device=y.device)
    r = torch.arange(rows, device=y.device)[:, None]
    b = torch.arange(nb, device=y.device)[None, :]
    tiled[r // 128, b // 4, r % 32, (r // 32) % 4, b % 4] = s
    return y / se, tiled


def exact(case, seed):
    st = prepare(case, seed)
    x = st["x"].detach().double()
    if case["op"] == "quant":
        if case["fmt"] == "mxfp4":
            return _values64(x, "mxfp4")
        g = (st["x"].abs().max().float() / 2688).double()
        return _values64(x / g, "nvfp4") * g, g.reshape(1)
    if case["op"] == "linear":
        fmt, k = case["fmt"], case["k"]
        size, _, bits, pow2 = FORMATS[fmt]
        c = st["codes"].view(torch.uint8)
        if bits == 4:
            c = torch.stack((c % 16, c // 16), -1).flatten(1)
            mag = c % 8
            el = torch.where(mag < 2, mag * 0.5, (1 + 0.5 * (mag % 2)) * torch.exp2((mag // 2).double() - 1))
            el = torch.where(c >= 8, -el, el)
        else:
            el = c.view(torch.float8_e4m3fn).double()
        s = st["row_scales"]
        s = torch.exp2(s.double() - 127) if pow2 else s.view(torch.float8_e4m3fn).double()
        j = torch.arange(k, device=x.device)
        w = el[:, :k].double() * s[:, j // size]
        y = _values64(x, fmt) @ w.t()
        y = y * (1.0 if st["g"] is None else st["g"].double()) + st["bias"].double()
        y = {"none": lambda v: v, "relu": torch.relu, "gelu": torch.nn.functional.gelu}[case["act"]](y)
        return y if case["out"] == "same" else _quantised64(y)
    w = st["w"].detach().double()
    h = x if st["r"] is None else (x + st["r"].detach().double()).to(DTYPES[case["dtype"]]).double()
    rstd = (h.pow(2).sum(-1, keepdim=True) / case["dim"] + EPS) ** -0.5
    xh = h * rstd
    if case["op"] == "norm_q":
        return _quantised64(xh * w) if st["r"] is None else (*_quantised64(xh * w), h)
    gy = st["gy"].double()
    gx = rstd * (gy * w - xh * (gy * w * xh).mean(-1, keepdim=True))
    gw = (gy * xh).sum(0)
    if st["r"] is None:
        return xh * w, gx, gw
    gx = gx + st["gh"].double()
    return xh * w, h, gx, gx, gw
