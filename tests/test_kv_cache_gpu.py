"""kv_write and kv_read against the row formats, byte for byte."""
import numpy as np
import pytest

from tests.kv_reference import DTYPES, FORMATS, Paged, decode, encode, from_dtype, storage, to_dtype
from yuuka_b200 import cuda

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    d = cuda.Device(0)
    yield d
    d.close()


@pytest.fixture(scope="module")
def stream(dev):
    s = dev.stream()
    yield s
    s.destroy()


def numbers(rng, rows, heads, dim, dtype):
    """Rows with the values that roundings turn on: magnitudes from tiny to large, exact halves of steps, zeros, signed zeros."""
    x = (rng.standard_normal((rows, heads, dim)) * np.exp2(rng.uniform(-8, 4, (rows, heads, 1)))).astype(np.float32)
    x[rng.random(x.shape) < 0.02] = 0.0
    x[rng.random(x.shape) < 0.01] = -0.0
    # blocks whose scale is a power of two, with values on halves of steps
    if rows > 1:
        x[1, 0, :32] = np.linspace(-127, 127, 32, dtype=np.float32)
        x[1, 0, 1:31] = np.floor(x[1, 0, 1:31]) + 0.5
        x[1, 0, 0], x[1, 0, 31] = -127.0, 127.0
    if rows > 2:
        x[2] = 0.0
    if rows > 3:
        x[3] *= 1e-6  # f16 subnormals
    if rows > 4 and dtype == "f32":
        x[4] *= 1e-33  # scales whose inverse is not finite, or barely
    return to_dtype(x, dtype)


def place(rng, rows, lens, block):
    """Distinct tokens of several sequences in no order, some of them without a token (-1)."""
    tokens = [(s, p) for s, n in enumerate(lens) for p in range(n)]
    pick = rng.permutation(len(tokens))[:rows]
    seq, pos = np.array([tokens[i][0] for i in pick], np.int32), np.array([tokens[i][1] for i in pick], np.int32)
    return seq, pos


CASES = [
    # format, type, heads, dim, block, rows
    ("f32", "f32", 1, 64, 16, 1), ("f32", "bf16", 3, 64, 5, 9), ("f32", "f16", 2, 256, 16, 40),
    ("f16", "f32", 4, 256, 16, 1), ("f16", "f32", 5, 64, 7, 33), ("f16", "bf16", 1, 128, 1, 12), ("f16", "f16", 3, 128, 64, 70),
    ("q8_0", "f32", 1, 64, 16, 1), ("q8_0", "f32", 3, 64, 3, 37), ("q8_0", "bf16", 4, 256, 16, 50), ("q8_0", "f16", 5, 128, 24, 21),
    ("f8", "f32", 1, 64, 16, 1), ("f8", "f32", 3, 64, 11, 31), ("f8", "bf16", 8, 128, 32, 64), ("f8", "f16", 2, 256, 16, 17),
    ("f8", "f32", 5, 256, 2, 8),
]


@pytest.mark.parametrize("fmt,dtype,heads,dim,block,rows", CASES)
def test_write_then_read(dev, stream, oracle, fmt, dtype, heads, dim, block, rows):
    rng = np.random.default_rng(heads * 1000 + dim + rows)
    lens = [max(1, rows // 2), rows + 3, 4]
    paged = Paged(dev, rng, fmt, heads, dim, block, lens)
    seq, pos = place(rng, rows, lens, block)
    pad = 3
    x = {c: numbers(rng, rows + pad, heads, dim, dtype) for c in "kv"}
    seq_all = np.concatenate([seq, np.array([0, 99, -5], np.int32)])  # (rows without a token: their sequence does not matter)
    pos_all = np.concatenate([pos, np.array([-1, -1, -2147483648], np.int32)])
    bufs = {c: dev.upload(x[c]) for c in "kv"}
    sb, pb, status = dev.upload(seq_all), dev.upload(pos_all), dev.upload(np.zeros(4, np.int32))
    cuda.kv_write(stream, paged.cache, cuda.KvRows(bufs["k"], bufs["v"], pb, rows + pad, DTYPES[dtype], seq=sb, status=status))
    stream.synchronize()
    slots = paged.slots(seq, pos)
    want = {}
    for c, before in (("k", paged.k), ("v", paged.v)):
        want[c] = before.copy()
        want[c][slots] = encode(from_dtype(x[c], dtype).astype(np.float32)[:rows], fmt, oracle)
    got = dict(zip("kv", paged.download()))
    for c in "kv":
        assert np.array_equal(got[c], want[c]), (c, np.argwhere(got[c] != want[c])[:5])  # untouched rows among them

    # read back, into rows that hold something already
    was = to_dtype(np.full((rows + pad, heads, dim), 7.0, np.float32), dtype)
    for c in "kv":
        bufs[c].write(was)
    cuda.kv_read(stream, paged.cache, cuda.KvRows(bufs["k"], bufs["v"], pb, rows + pad, DTYPES[dtype], seq=sb, status=status))
    stream.synchronize()
    for c in "kv":
        back = bufs[c].read(storage(dtype), was.size).reshape(was.shape)
        exact = decode(want[c][slots], fmt, heads, dim)
        assert np.array_equal(back[:rows], to_dtype(exact.astype(np.float32), dtype)), c
        assert np.array_equal(back[rows:], was[rows:])
    assert status.read(np.int32, 1)[0] == 0
    for b in (*bufs.values(), sb, pb, status):
        b.free()
    paged.free()


def test_q8_rows_are_within_a_rounding_of_a_sessions(dev, stream, oracle):
    """The sessions' codec takes the quotient amax / 127, kv_write the product with 1 / 127: the f16 scales are the same or
    neighbours, and the whole numbers the same or one apart where a value lies next to a half."""
    rng = np.random.default_rng(8)
    x = (rng.standard_normal((400, 8, 256)) * np.exp2(rng.uniform(-6, 6, (400, 8, 1)))).astype(np.float32)
    paged = Paged(dev, rng, "q8_0", 8, 256, 16, [400])
    b, pb, sb = dev.upload(x), dev.upload(np.arange(400, dtype=np.int32)), dev.upload(np.zeros(400, np.int32))
    cuda.kv_write(stream, paged.cache, cuda.KvRows(b, b, pb, 400, seq=sb))
    stream.synchronize()
    got = paged.download()[0][paged.slots(0, np.arange(400))].reshape(400, -1, 34)
    want = np.stack([oracle.kv_encode_row(cuda.KV_Q8_0, r) for r in x.reshape(400, -1)]).reshape(400, -1, 34)
    scales = [np.ascontiguousarray(a[:, :, :2]).view(np.uint16).astype(int) for a in (got, want)]
    apart = np.abs(scales[0] - scales[1])
    assert apart.max() <= 1 and apart.mean() < 1e-3
    off = np.abs(got[:, :, 2:].view(np.int8).astype(int) - want[:, :, 2:].view(np.int8).astype(int))
    assert off.max() <= 1 and off.mean() < 1e-4
    for q in (b, pb, sb):
        q.free()
    paged.free()


@pytest.mark.parametrize("fmt", list(FORMATS))
def test_strided_rows_of_a_fused_projection(dev, stream, oracle, fmt):
    """K and V as columns of one array, written from and read into; what lies between the columns stays."""
    rng = np.random.default_rng(5)
    heads, dim, block, rows, wide = 2, 64, 16, 19, 7 * 64
    paged = Paged(dev, rng, fmt, heads, dim, block, [rows])
    x = rng.standard_normal((rows, wide)).astype(np.float32)
    buf, pb = dev.upload(x), dev.upload(np.arange(rows, dtype=np.int32))
    sb = dev.upload(np.zeros(rows, np.int32))
    at = dict(k_stride=wide, v_stride=wide, k_offset=64 * 4, v_offset=4 * 64 * 4, seq=sb)
    cuda.kv_write(stream, paged.cache, cuda.KvRows(buf, buf, pb, rows, **at))
    stream.synchronize()
    slots = paged.slots(0, np.arange(rows))
    rows_k, rows_v = x[:, 64:192].reshape(rows, heads, dim), x[:, 256:384].reshape(rows, heads, dim)
    got_k, got_v = paged.download()
    assert np.array_equal(got_k[slots], encode(rows_k, fmt, oracle)) and np.array_equal(got_v[slots], encode(rows_v, fmt, oracle))
    buf.write(np.full_like(x, 3.0))
    cuda.kv_read(stream, paged.cache, cuda.KvRows(buf, buf, pb, rows, **at))
    stream.synchronize()
    back = buf.read(np.float32, x.size).reshape(x.shape)
    assert np.array_equal(back[:, 64:192].reshape(rows, heads, dim), decode(got_k[slots], fmt, heads, dim).astype(np.float32))
    assert np.array_equal(back[:, 256:384].reshape(rows, heads, dim), decode(got_v[slots], fmt, heads, dim).astype(np.float32))
    rest = np.delete(back, np.r_[64:192, 256:384], axis=1)
    assert np.all(rest == 3.0)
    for b in (buf, pb, sb):
        b.free()
    paged.free()


@pytest.mark.parametrize("fmt", list(FORMATS))
def test_ids_out_of_range(dev, stream, fmt):
    """Bad blocks, sequences and positions: nothing is written, NaN is read, the status says which."""
    rng = np.random.default_rng(9)
    heads, dim, block = 2, 64, 4
    paged = Paged(dev, rng, fmt, heads, dim, block, [8, 8])
    paged.tables[0] = [1, paged.blocks]   # beyond the pool
    paged.tables[1] = [-1, 2]
    paged.upload()
    cases = [([0], [0], 0), ([0], [4], 1), ([1], [3], 1), ([2], [0], 2), ([-1], [0], 2), ([1], [8], 4), ([0], [2147483647], 4)]
    x = dev.upload(rng.standard_normal((1, heads, dim)).astype(np.float32))
    y = dev.upload(np.zeros((1, heads, dim), np.float32))
    for seq, pos, bit in cases:
        sb, pb, status = dev.upload(np.array(seq, np.int32)), dev.upload(np.array(pos, np.int32)), dev.upload(np.zeros(4, np.int32))
        before = paged.download()
        cuda.kv_write(stream, paged.cache, cuda.KvRows(x, x, pb, 1, seq=sb, status=status))
        stream.synchronize()
        assert status.read(np.int32, 1)[0] == bit
        after = paged.download()
        changed = any(not np.array_equal(a, b) for a, b in zip(before, after))
        assert changed == (bit == 0)
        status.write(np.zeros(4, np.int32))
        for b in (x, y):
            b.write(np.ones((1, heads, dim), np.float32))
        cuda.kv_read(stream, paged.cache, cuda.KvRows(x, y, pb, 1, seq=sb, status=status))
        stream.synchronize()
        assert status.read(np.int32, 1)[0] == bit
        back = np.concatenate([b.read(np.float32, heads * dim) for b in (x, y)])
        assert np.all(np.isnan(back)) if bit else np.all(np.isfinite(back))
        x.write(rng.standard_normal((1, heads, dim)).astype(np.float32))
        for b in (sb, pb, status):
            b.free()
    for b in (x, y):
        b.free()
    paged.free()


def test_row_r_is_sequence_r_without_a_list(dev, stream, oracle):
    rng = np.random.default_rng(2)
    lens = [3, 9, 1, 6]
    paged = Paged(dev, rng, "f16", 1, 64, 4, lens)
    x = rng.standard_normal((4, 1, 64)).astype(np.float32)
    b, pb = dev.upload(x), dev.upload(np.array([n - 1 for n in lens], np.int32))
    cuda.kv_write(stream, paged.cache, cuda.KvRows(b, b, pb, 4))
    stream.synchronize()
    slots = paged.slots(np.arange(4), np.array(lens) - 1)
    assert np.array_equal(paged.download()[1][slots], encode(x, "f16", oracle))
    for q in (b, pb):
        q.free()
    paged.free()


@pytest.mark.parametrize("fmt", list(FORMATS))
def test_values_that_are_not_finite(dev, stream, oracle, fmt):
    """A NaN or an infinity stays within its own head (its block in Q8_0), and finite heads beside it keep their bytes."""
    rng = np.random.default_rng(3)
    x = rng.standard_normal((3, 4, 64)).astype(np.float32)
    clean = x.copy()
    x[0, 1, 5], x[1, 2, 40], x[2, 3, 63] = np.nan, np.inf, -np.inf
    paged = Paged(dev, rng, fmt, 4, 64, 4, [3])
    b, pb = dev.upload(x), dev.upload(np.arange(3, dtype=np.int32))
    sb = dev.upload(np.zeros(3, np.int32))
    cuda.kv_write(stream, paged.cache, cuda.KvRows(b, b, pb, 3, seq=sb))
    stream.synchronize()
    rows = paged.download()[0][paged.slots(0, np.arange(3))]
    with np.errstate(invalid="ignore"):
        got = decode(rows, fmt, 4, 64)
    want = decode(encode(clean, fmt, oracle), fmt, 4, 64)
    other = np.ones((3, 4), bool)
    other[[0, 1, 2], [1, 2, 3]] = False
    assert np.array_equal(got[other], want[other])
    if fmt in ("f32", "f16"):
        assert np.isnan(got[0, 1, 5]) and np.isposinf(got[1, 2, 40]) and np.isneginf(got[2, 3, 63])
    if fmt == "f8":
        assert np.isnan(got[0, 1, 5]) and np.isnan(got[1, 2, 40]) and np.isnan(got[2, 3, 63])
    for q in (b, pb, sb):
        q.free()
    paged.free()


def test_a_pool_behind_two_gigabytes(dev, stream):
    """Row offsets pass 32 bits: the last rows of a 4.3 GB pool."""
    heads, dim, block, blocks = 8, 256, 64, 8225  # 8192 bytes a row
    row = cuda.kv_row_bytes(cuda.KV_F32, heads, dim)
    k, v = (dev.alloc(row * block * blocks) for _ in range(2))
    tables = dev.upload(np.array([[blocks - 1, 0]], np.int32))
    cache = cuda.KvCache(k, v, tables, cuda.KV_F32, heads, dim, block, blocks, 1, 2)
    x = np.random.default_rng(1).standard_normal((2, heads, dim)).astype(np.float32)
    b, y, z = dev.upload(x), dev.upload(np.zeros_like(x)), dev.upload(np.zeros_like(x))
    pb, sb = dev.upload(np.array([block - 1, block], np.int32)), dev.upload(np.zeros(2, np.int32))
    cuda.kv_write(stream, cache, cuda.KvRows(b, b, pb, 2, seq=sb))
    cuda.kv_read(stream, cache, cuda.KvRows(y, z, pb, 2, seq=sb))
    stream.synchronize()
    assert np.array_equal(y.read(np.float32, x.size).reshape(x.shape), x) and np.array_equal(z.read(np.float32, x.size).reshape(x.shape), x)
    last = v.read(np.float32, heads * dim, offset=row * (block * blocks - 1))
    assert np.array_equal(last, x[0].ravel())
    for q in (k, v, tables, b, y, z, pb, sb):
        q.free()
