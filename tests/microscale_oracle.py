"""Plain 64-bit definitions of the microscaled formats, written value by value (tests only)."""
import numpy as np
import torch

FORMATS = ("mxfp4", "nvfp4", "mxfp8")
BLOCK = {"mxfp4": 32, "nvfp4": 16, "mxfp8": 32}


def _grid(mant, emin, top):
    v = [i * 2.0 ** (emin - mant) for i in range(2 ** mant)]
    e = emin
    while v[-1] < top:
        v += [2.0 ** e * (1 + i / 2 ** mant) for i in range(2 ** mant)]
        e += 1
    return np.array([x for x in v if x <= top])


GRID = {4: _grid(1, 0, 6.0), 8: _grid(3, -6, 448.0)}    # non-negative values, index = code


def nearest(v, bits):
    """Index of the nearest grid value of |v|, ties to the even code, saturating."""
    g = GRID[bits]
    a = np.minimum(np.abs(v), g[-1])
    hi = np.clip(np.searchsorted(g, a), 1, len(g) - 1)
    lo = hi - 1
    dl, dh = a - g[lo], g[hi] - a
    return np.where(dl < dh, lo, np.where(dh < dl, hi, np.where(lo % 2 == 0, lo, hi)))


def quantize(x, fmt, g=None):
    """numpy fp64 [rows, dim] -> (signed codes, scale bytes [rows, blocks], values).  Non-finite blocks: NaN scale."""
    size, bits = BLOCK[fmt], 8 if fmt == "mxfp8" else 4
    rows, dim = x.shape
    nb = -(-dim // size)
    codes = np.zeros((rows, dim), np.int64)
    byte = np.zeros((rows, nb), np.int64)
    val = np.zeros((rows, dim))
    for b in range(nb):
        s = slice(b * size, min(dim, (b + 1) * size))
        xb = x[:, s]
        with np.errstate(invalid="ignore"):
            amax = np.abs(xb).max(1)
        bad = ~np.isfinite(amax)
        am = np.where(bad, 0, amax)
        if fmt == "nvfp4":
            f32 = np.float32
            t = np.minimum((am.astype(f32) / (f32(6) * f32(g))), f32(448))      # in fp32, as stated
            byte[:, b] = nearest(t.astype(np.float64), 8)
            sv = GRID[8][byte[:, b]]
            with np.errstate(divide="ignore"):
                inv = np.where(sv > 0, f32(1) / (sv.astype(f32) * f32(g)), f32(0)).astype(f32)
            q = (np.where(bad[:, None], 0, xb).astype(f32) * inv[:, None]).astype(np.float64)
            scale = sv * float(f32(g))
            byte[bad, b] = 0x7F
        else:
            top = GRID[bits][-1]
            e = np.frexp(am)[1]                                  # am < 2^e: the answer is one of three
            p = np.clip(e - (3 if bits == 4 else 9), -127, 127)
            for _ in range(2):
                p = np.where((p < 127) & (am > top * 2.0 ** p.astype(np.float64)), p + 1, p)
            p = np.where(am > 0, p, -127)
            scale = 2.0 ** p.astype(np.float64)
            q = np.where(bad[:, None], 0, xb) / scale[:, None]
            byte[:, b] = np.where(bad, 255, p + 127)
        c = nearest(q, bits)
        val[:, s] = np.where(bad[:, None], np.nan, np.copysign(GRID[bits][c], q) * scale[:, None])
        codes[:, s] = c | (np.signbit(q).astype(np.int64) << (bits - 1))
    return codes, byte, val


def tensor_scale(x):
    a = np.abs(x).max()
    return np.float32(1) if not np.isfinite(a) or a == 0 else max(np.float32(a) * np.float32(1 / 2688), np.float32(2.0 ** -100))


def unpack(t):
    """(codes, scale bytes [rows, blocks]) of an MXTensor on any device, and that its padding is zero."""
    rows, dim = t.rows, t.shape[-1]
    c = t.codes.cpu().view(torch.uint8).long()
    if t.fmt != "mxfp8":
        c = torch.stack((c % 16, c // 16), -1).reshape(rows, -1)
    assert (c[:, dim:] == 0).all()
    s = t.scales.cpu().long()
    rt, kt = s.shape[:2]
    r, b = torch.meshgrid(torch.arange(rt * 128), torch.arange(kt * 4), indexing="ij")
    s = s[r // 128, b // 4, r % 32, r // 32 % 4, b % 4]
    nb = -(-dim // BLOCK[t.fmt])
    assert (s[rows:] == 0).all() and (s[:, nb:] == 0).all()
    return c[:, :dim].numpy(), s[:rows, :nb].numpy()


def hard_rows(dim, seed=0):
    """fp32 rows whose blocks sit where a format can go wrong: zeros, subnormals, the edges between two scales,
    ties between two elements, the largest numbers, infinities, NaN."""
    gen = torch.Generator().manual_seed(seed)
    base = torch.randn(12, dim, generator=gen)
    base[1] = 0
    base[2] *= 2.0 ** -140
    base[3] = 6.0 * 2.0 ** 5
    base[4] = 6.0 * 2.0 ** 5 * (1 + 2.0 ** -7)
    base[5] = 448.0
    base[6] = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0]).repeat(dim // 8 + 1)[:dim]
    base[7] = -base[6]
    base[8] *= 1e38
    base[9, dim // 2] = float("inf")
    base[10, 0] = float("nan")
    base[11, dim - 1] = -float("inf")
    return base
