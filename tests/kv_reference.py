"""Plain 64-bit forms of the paged-cache calls for their tests: the row formats, and attention over decoded rows."""
import numpy as np

from yuuka_b200 import cuda

FORMATS = {"f32": cuda.KV_F32, "f16": cuda.KV_F16, "q8_0": cuda.KV_Q8_0, "f8": cuda.KV_F8}
DTYPES = {"f32": cuda.F32, "f16": cuda.F16, "bf16": cuda.BF16}
# half a unit in the last place, relative
HALF_STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}


def to_dtype(x, dtype):
    """float32 -> array whose bytes are the values in dtype."""
    x = np.ascontiguousarray(x, np.float32)
    return x if dtype == "f32" else x.astype(np.float16) if dtype == "f16" else cuda.to_bf16(x)


def from_dtype(a, dtype):
    return a.astype(np.float64) if dtype != "bf16" else cuda.from_bf16(a).astype(np.float64)


def storage(dtype):
    return {"f32": np.float32, "f16": np.float16, "bf16": np.uint16}[dtype]


# E4M3 by its definition: sign, four exponent bits with a bias of 7, three mantissa bits; 0x7f is NaN
_B = np.arange(256)
_E, _M = (_B >> 3) & 15, _B & 7
E4M3 = np.where(_E == 0, _M * 2.0 ** -9, (1 + _M / 8.0) * 2.0 ** (_E - 7.0)) * np.where(_B >= 128, -1.0, 1.0)
E4M3[(_B & 127) == 127] = np.nan


def encode_e4m3(y):
    """Nearest, ties to an even last bit, saturating; y float."""
    mag = np.minimum(np.abs(y.astype(np.float64)), 448.0)
    grid = E4M3[:127]
    hi = np.clip(np.searchsorted(grid, mag), 0, 126)
    lo = np.maximum(hi - 1, 0)
    dh, dl = grid[hi] - mag, mag - grid[lo]
    pick = np.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)
    return (pick | np.where(np.signbit(y), 128, 0)).astype(np.uint8)


def encode(x, fmt, oracle):
    """Rows [n, heads, dim] f32 -> bytes [n, row_bytes]; f32 and f16 numbers by the oracle's codec (the sessions' own)."""
    n, h, d = x.shape
    x = np.ascontiguousarray(x, np.float32)
    if fmt in ("f32", "f16"):
        return np.stack([oracle.kv_encode_row(FORMATS[fmt], r) for r in x.reshape(n, h * d)])
    if fmt == "q8_0":
        blocks = x.reshape(n, h * d // 32, 32)
        scale = np.fmax.reduce(np.abs(blocks), -1) * (np.float32(1) / np.float32(127))
        with np.errstate(divide="ignore", invalid="ignore", over="ignore"):
            y = (blocks / scale[..., None]).astype(np.float64)
            q = np.trunc(y + np.copysign(0.5, y))
        q = np.where(np.isfinite(q) & (scale[..., None] != 0), q, 0).astype(np.int64).astype(np.int8)
        bits = oracle.kv_encode_row(FORMATS["f16"], np.ascontiguousarray(scale.reshape(-1))).reshape(n, h * d // 32, 2)
        return np.concatenate([bits, q.view(np.uint8)], -1).reshape(n, -1)
    out = np.zeros((n, cuda.kv_row_bytes(cuda.KV_F8, h, d)), np.uint8)
    amax = np.abs(x).max(-1).astype(np.float32)
    with np.errstate(divide="ignore"):
        inv = np.float32(1.0) / amax * np.float32(448.0)
    live = inv <= np.float32(3e38)
    inv = np.where(live, inv, np.float32(0))
    out[:, :h * d] = encode_e4m3((x * inv[..., None]).astype(np.float32)).reshape(n, h * d)
    out[:, h * d:h * d + 4 * h] = np.where(live, amax * (np.float32(1) / np.float32(448)), np.float32(0)).astype(np.float32).view(np.uint8).reshape(n, 4 * h)
    return out


def decode(rows, fmt, h, d):
    """bytes [n, row_bytes] -> float64 [n, heads, dim]."""
    rows = np.ascontiguousarray(rows)
    n = rows.shape[0]
    if fmt == "f32":
        return rows.view(np.float32).astype(np.float64).reshape(n, h, d)
    if fmt == "f16":
        return rows.view(np.float16).astype(np.float64).reshape(n, h, d)
    if fmt == "q8_0":
        b = rows.reshape(n, h * d // 32, 34)
        scale = np.ascontiguousarray(b[:, :, :2]).view(np.float16).astype(np.float64)
        return (scale * np.ascontiguousarray(b[:, :, 2:]).view(np.int8)).reshape(n, h, d)
    scale = np.ascontiguousarray(rows[:, h * d:h * d + 4 * h]).view(np.float32).astype(np.float64)
    return E4M3[rows[:, :h * d]].reshape(n, h, d) * scale[:, :, None]


class Paged:
    """K and V pools on the device with pages in no order; what no token has been written to is NaN in every format."""

    def __init__(self, dev, rng, fmt, heads, dim, block, lens, spare=2, extra_pages=0):
        self.dev, self.fmt, self.heads, self.dim, self.block = dev, fmt, heads, dim, block
        self.row = cuda.kv_row_bytes(FORMATS[fmt], heads, dim)
        need = [max(1, -(-n // block)) + extra_pages for n in lens]
        self.blocks = sum(need) + spare
        order = rng.permutation(self.blocks).astype(np.int32)
        self.tables = np.full((len(lens), max(need)), -7, np.int32)  # (ids that are never to be used)
        at = 0
        for i, k in enumerate(need):
            self.tables[i, :k] = order[at:at + k]
            at += k
        self.k = np.full((self.blocks * block, self.row), 255, np.uint8)
        self.v = self.k.copy()
        self.kb, self.vb, self.tb = dev.upload(self.k), dev.upload(self.v), dev.upload(self.tables)
        self.cache = cuda.KvCache(self.kb, self.vb, self.tb, FORMATS[fmt], heads, dim, block, self.blocks, len(lens), self.tables.shape[1])

    def slots(self, seq, pos):
        pos = np.asarray(pos)
        return self.tables[seq, pos // self.block].astype(np.int64) * self.block + pos % self.block

    def upload(self):
        self.kb.write(self.k)
        self.vb.write(self.v)
        self.tb.write(self.tables)

    def download(self):
        n = self.k.size
        return self.kb.read(np.uint8, n).reshape(self.k.shape), self.vb.read(np.uint8, n).reshape(self.v.shape)

    def free(self):
        for b in (self.kb, self.vb, self.tb):
            b.free()


def attend(q, k, v, scale):
    """One head in 64 bits: q [d], k, v [n, d]. Returns out, lse, sum p|v| / sum p, max_j sum_i |q_i k_ij| |scale|."""
    if k.shape[0] == 0:
        return np.zeros(v.shape[1]), -np.inf, np.zeros(v.shape[1]), 0.0
    s = (k @ q) * scale
    m = s.max()
    p = np.exp(s - m)
    return p @ v / p.sum(), m + np.log(p.sum()), p @ np.abs(v) / p.sum(), (np.abs(k) @ np.abs(q)).max() * abs(scale)


def attend_bounds(out, lse, weight, reach, dim, dtype):
    """How far an output and its log-sum-exp may be off.

    A score is a sum of `dim` products whose factors carry 22 bits (queries in two parts, or exact) in f32: each of the dim/8
    or dim/16 steps of the product (at most dim/8 + 4 with the joining of partial sums) may cut off 2^-23 of the largest
    partial sum, at most `reach`; dropping the product of the two low parts and the parts' own rounding is 2^-21 of it. So a
    score is off by ds = reach (2^-21 + (dim/8 + 4) 2^-23) and a probability by 2 ds (with the maximum's) + 2^-20 for the
    exponential and the sums. Queries and outputs of 16 bits take probabilities of 11 bits: 2^-11 more. All of it is relative
    to sum p|v| / sum p. The output's own rounding and the gate's few f32 steps come on top."""
    ds = reach * (2.0 ** -21 + (dim / 8 + 4) * 2.0 ** -23)
    eps = 2 * ds + 2.0 ** -20 + (0.0 if dtype == "f32" else 2.0 ** -11)
    return weight * eps + np.abs(out) * (HALF_STEP[dtype] + 2.0 ** -20) + 1e-30, ds + 2.0 ** -20 + abs(lse) * 2.0 ** -22 if np.isfinite(lse) else 0.0
