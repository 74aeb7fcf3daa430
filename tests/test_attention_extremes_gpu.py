"""attention_decode where numbers leave the ordinary: infinite keys and values, values far apart, strong gates."""
import numpy as np
import pytest

from tests.kv_reference import DTYPES, HALF_STEP, attend, attend_bounds, decode, encode, from_dtype, to_dtype
from tests.test_attention_decode_gpu import Step, dev, scratch, stream  # noqa: F401  (fixtures)
from yuuka_b200 import cuda

pytestmark = pytest.mark.gpu


def check_keys(step, out, lse, keep, rows, more=None):
    """The formula over the keys `keep(sequence)` alone; `more`: allowed beyond attend_bounds, by sequence."""
    more = [0.0] * len(step.lens) if more is None else more
    q = from_dtype(step.qg, step.dtype)
    for b in rows:
        seq = step.rows[b][0]
        slots = step.paged.slots(seq, keep(seq))
        k, v = decode(step.paged.k[slots], step.fmt, step.kv_heads, step.dim), decode(step.paged.v[slots], step.fmt, step.kv_heads, step.dim)
        for h in range(step.heads):
            j = h // step.group
            want, want_lse, weight, reach = attend(q[b, h, :step.dim], k[:, j], v[:, j], step.scale)
            far, far_lse = attend_bounds(want, want_lse, weight, reach, step.dim, step.dtype)
            off = np.abs(out[b, h] - want)
            assert np.all(off <= far + more[seq]), (b, h, len(slots), float(np.nanmax(off)), float(np.nanmax(off / (far + more[seq]))))
            if np.isfinite(want_lse):
                assert abs(lse[b, h] - want_lse) <= far_lse, (b, h, lse[b, h], want_lse)
            else:
                assert np.isneginf(lse[b, h]) and np.all(out[b, h] == 0)


def set_pool(step, c, slots, dims, value):
    """Numbers of an F32 or F16 pool, all heads."""
    pool = getattr(step.paged, c).view({"f32": np.float32, "f16": np.float16}[step.fmt])
    pool = pool.reshape(-1, step.kv_heads, step.dim)
    pool[slots[:, None], :, dims] = value


# one tile; several in one team's run and in several; a row of infinite keys alone; many joined partials
INF_LENS = [20, 300, 57, 41, 40, 5000]


@pytest.mark.parametrize("fmt", ["f16", "f32"])
@pytest.mark.parametrize("dtype,exact", [("f32", False), ("f32", True), ("bf16", False), ("f16", False)])
@pytest.mark.parametrize("dim,group", [(64, 2), (128, 3), (256, 9)])
@pytest.mark.parametrize("crowd", [1, 60])
def test_infinite_keys_weigh_nothing(dev, stream, scratch, fmt, dtype, exact, dim, group, crowd):  # noqa: F811
    """Keys with a component of -infinity where the queries are positive, or of infinity where they are negative, score
    -infinity: as if they were not there, in whole tiles and between others. `exact`: queries without a second part.
    crowd: the batch so often that teams have whole rows in their runs."""
    if crowd > 1 and (dim, group) != (128, 3):
        pytest.skip("one shape is enough")
    step = Step(dev, stream, dim + group, fmt, dtype, 1, group, dim, 16, INF_LENS, seq_ids=list(range(6)) * crowd)
    q = from_dtype(step.qg, dtype)
    if exact:
        q = np.round(q * 4) / 4 + 0.0
    q[..., 5], q[..., dim - 7], q[..., 33] = np.abs(q[..., 5]) + 0.25, -np.abs(q[..., dim - 7]) - 0.25, 1e-7 if dtype == "f16" else 1e-15
    step.qg = to_dtype(q.astype(np.float32), dtype)
    step.qb.write(step.qg)
    rng = np.random.default_rng(dim)
    gone = [set(range(min(40, n))) | {int(i) for i in rng.integers(0, n, n // 9)} if n >= 40 else {0, 3, 19} for n in INF_LENS]
    gone[4] = set(range(40))
    for s in range(6):
        at = step.paged.slots(s, np.array(sorted(gone[s])))
        set_pool(step, "k", at[0::3], 5, -np.inf)
        set_pool(step, "k", at[1::3], dim - 7, np.inf)
        set_pool(step, "k", at[2::3], 33, -np.inf)
    step.paged.upload()
    out, lse = step.run(scratch)
    rows = range(6) if crowd == 1 else [0, 1, 2, 3, 4, 5, 6 * crowd - 1, 6 * crowd - 2, 6 * crowd - 5]
    check_keys(step, out, lse, lambda s: np.array([i for i in range(INF_LENS[s]) if i not in gone[s]], np.int64), rows)
    step.free()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("dim", [64, 256])
@pytest.mark.parametrize("size", [1e30, 1e35, 1e-30])
def test_large_and_small_values_over_f32_pools(dev, stream, scratch, dtype, dim, size):  # noqa: F811
    """Sums of values near the ends of f32, over rows that are whole, shared by few runs and by many."""
    step = Step(dev, stream, dim, "f32", dtype, 1, 3, dim, 16, [20, 300, 3000])
    for s, n in enumerate(step.lens):
        at = step.paged.slots(s, np.arange(n))
        pool = step.paged.v.view(np.float32)
        pool[at] = np.clip(pool[at], -4, 4) * np.float32(size)
    step.paged.upload()
    step.check(*step.run(scratch))
    step.free()


@pytest.mark.parametrize("fmt", ["f16", "f32", "q8_0", "f8"])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_infinite_queries(dev, stream, scratch, fmt, dtype, dim):  # noqa: F811
    """A query of -infinity where all keys are positive scores -infinity alone: a row without keys. One of infinity, or with a NaN, is
    a NaN. The other heads of the tile do not notice."""
    lens = [20, 33, 700, 3000]
    step = Step(dev, stream, dim, fmt, dtype, 1, 4, dim, 16, lens)
    rng = np.random.default_rng(dim)
    for s, n in enumerate(lens):
        k = rng.standard_normal((n, 1, dim))
        k[..., 7] = np.abs(k[..., 7]) + 0.5
        bufs = [dev.upload(np.ascontiguousarray(a, t)) for a, t in ((k, np.float32), (rng.standard_normal((n, 1, dim)), np.float32), (np.arange(n), np.int32), (np.full(n, s), np.int32))]
        cuda.kv_write(stream, step.paged.cache, cuda.KvRows(bufs[0], bufs[1], bufs[2], n, seq=bufs[3]))
        stream.synchronize()
        for b in bufs:
            b.free()
    step.paged.k, step.paged.v = step.paged.download()
    q = from_dtype(step.qg, dtype)
    good = to_dtype(q.astype(np.float32), dtype)
    q[:, 0, 7], q[:, 1, 7], q[:, 2, 9] = -np.inf, np.inf, np.nan
    step.qb.write(to_dtype(q.astype(np.float32), dtype))
    out, lse = step.run(scratch)
    assert np.all(out[:, 0] == 0) and np.all(np.isneginf(lse[:, 0]))
    assert np.all(np.isnan(out[:, 1:3]))
    step.qg = good
    bad_out, bad_lse = out.copy(), lse.copy()
    step.qb.write(good)
    out, lse = step.run(scratch)
    assert np.array_equal(out[:, 3], bad_out[:, 3]) and np.array_equal(lse[:, 3], bad_lse[:, 3])
    step.check(out, lse)
    step.free()


@pytest.mark.parametrize("fmt,dtype", [("f16", "f32"), ("f16", "bf16"), ("f32", "f32"), ("f32", "f16"), ("q8_0", "f32"), ("q8_0", "bf16")])
@pytest.mark.parametrize("dim", [64, 256])
def test_values_that_are_not_finite_stay_in_their_place(dev, stream, scratch, fmt, dtype, dim):  # noqa: F811
    """Infinities and NaN of V make their dimensions of out infinite or NaN, over Q8_0 those of their blocks, and no others."""
    step = Step(dev, stream, dim, fmt, dtype, 1, 3, dim, 16, [20, 33, 700])
    bad = [3, 40] if fmt != "q8_0" else [*range(32, 64)]
    for s, n in enumerate(step.lens):
        at = step.paged.slots(s, np.array([n // 2, n - 1]))
        if fmt == "q8_0":  # the scale of the second block: NaN, and an infinity
            blocks = step.paged.v.reshape(step.paged.v.shape[0], -1, 34)
            blocks[at[0], 1, :2] = np.array([0x7e00], np.uint16).view(np.uint8)
            blocks[at[1], 1, :2] = np.array([0x7c00], np.uint16).view(np.uint8)
        else:
            set_pool(step, "v", at[:1], 3, np.inf)
            set_pool(step, "v", at[1:], 40, np.nan)
    step.paged.upload()
    out, lse = step.run(scratch)
    assert not np.any(np.isfinite(out[..., bad]))
    q = from_dtype(step.qg, dtype)
    good = np.setdiff1d(np.arange(dim), bad)
    for b, (s, n) in enumerate(step.rows):
        slots = step.paged.slots(s, np.arange(n))
        k = decode(step.paged.k[slots], fmt, 1, dim)[:, 0]
        with np.errstate(invalid="ignore"):
            v = decode(step.paged.v[slots], fmt, 1, dim)[:, 0][:, good]
        for h in range(step.heads):
            want, want_lse, weight, reach = attend(q[b, h], k, v, step.scale)
            far, far_lse = attend_bounds(want, want_lse, weight, reach, dim, dtype)
            assert np.all(np.abs(out[b, h, good] - want) <= far) and abs(lse[b, h] - want_lse) <= far_lse
    step.free()


def apart(step, ratio, gap, where, blocks, only=None):
    """V of magnitude 2^-6 (F8: 1), and of 2^ratio times that in every 50th key from `where` on; the queries of even heads score
    those keys `gap` nats below the others, of odd heads as much above. blocks: in the second 32 dimensions alone. only: of these sequences."""
    rng, d, dt = np.random.default_rng(100 + ratio), step.dim, step.dtype
    u = np.where(rng.random(d) < 0.5, -1.0, 1.0)
    q = np.broadcast_to(u, (step.batch, step.heads, d)).copy()
    q[:, 1::2] *= -1.0
    step.qg = to_dtype(q.astype(np.float32), dt)
    step.qb.write(step.qg)
    small = 1.0 if step.fmt in ("f8", "f32") else 2.0 ** -6
    for s, n in enumerate(step.lens):
        k = rng.standard_normal((n, 1, d)) * 0.25
        v = rng.standard_normal((n, 1, d)) * small
        far = np.arange(where % n, n, 50) if only is None or s in only else np.zeros(0, np.int64)
        k[far, 0] = -u * (gap / (d * step.scale)) + 0.01 * rng.standard_normal((len(far), d))
        v[far, :, 32:64] *= 2.0 ** ratio
        if not blocks:
            v[far, :, :32] *= 2.0 ** ratio
            v[far, :, 64:] *= 2.0 ** ratio
        bufs = [step.dev.upload(np.ascontiguousarray(a, t)) for a, t in ((k, np.float32), (v, np.float32), (np.arange(n), np.int32), (np.full(n, s), np.int32))]
        cuda.kv_write(step.stream, step.paged.cache, cuda.KvRows(bufs[0], bufs[1], bufs[2], n, seq=bufs[3]))
        step.stream.synchronize()
        for b in bufs:
            b.free()
    step.paged.k, step.paged.v = step.paged.download()


@pytest.mark.parametrize("fmt,dtype", [("q8_0", "f32"), ("q8_0", "bf16"), ("f8", "f32"), ("f8", "bf16"), ("f32", "f32"), ("f16", "f32")])
@pytest.mark.parametrize("dim,group", [(64, 2), (128, 16), (256, 4)])
@pytest.mark.parametrize("ratio,gap,where", [(4, 12, 7), (8, 20, 7), (12, 20, 40), (16, 24, 7), (20, 24, 0), (24, 28, 31), (-16, 0, 9)])
def test_values_far_apart(dev, stream, scratch, fmt, dtype, dim, group, ratio, gap, where):  # noqa: F811
    """Large values of next to no weight beside ordinary ones that have it all, and the other way round, in one batch. All of
    it within the bounds that hold for ordinary values. Besides, f16 ends at 2^-24, which probabilities are rounded to: half of it in units
    of the largest scale (over F16 1), less than twice the largest value's, where the row's largest probability is 2^11 at least. So each key
    may be off by 2^-35 of the largest value. Rows over Q8_0 and F8 with scales further apart than 2^10 (f32 queries) or 2^14 are
    summed in f32 and have no such term (the ratios between are not tested without it)."""
    if fmt == "f16" and ratio > 16:
        pytest.skip("infinities in f16")
    for blocks in ((False, True) if fmt == "q8_0" else (False,)):
        step = Step(dev, stream, 3, fmt, dtype, 1, group, dim, 16, [70, 1, 333, 2600])
        apart(step, ratio, gap, where, blocks)
        out, lse = step.run(scratch)
        near = fmt == "f16" or (fmt in ("q8_0", "f8") and abs(ratio) < (12 if dtype == "f32" else 16))
        more = [2.0 ** -35 * n * np.abs(decode(step.paged.v[step.paged.slots(s, np.arange(n))], fmt, 1, dim)).max() if near else 0.0 for s, n in enumerate(step.lens)]
        check_keys(step, out, lse, lambda s: np.arange(step.lens[s]), range(4), more)
        again, lse2 = step.run(scratch)
        assert np.array_equal(out, again) and np.array_equal(lse, lse2)
        step.free()


@pytest.mark.parametrize("fmt,dtype", [("q8_0", "f32"), ("f8", "f32"), ("q8_0", "bf16"), ("f8", "f16")])
@pytest.mark.parametrize("dim,group,crowd", [(64, 2, 60), (128, 16, 25), (256, 4, 400)])
def test_values_far_apart_in_rows_of_any_split(dev, stream, scratch, fmt, dtype, dim, group, crowd):  # noqa: F811
    """The batch so often that rows lie whole within a team's run, or are joined from a few of them, gates included."""
    lens = [70, 1, 333, 2600]
    step = Step(dev, stream, 3, fmt, dtype, 1, group, dim, 16, lens, seq_ids=list(range(4)) * crowd)
    apart(step, 18 if dtype == "f16" else 24, 26, 5, False)
    if dtype == "f16":  # outputs of f16 end at 65504
        step.paged.v.view(np.float32)[:, dim // 4] *= np.float32(2.0 ** -8)
        step.paged.upload()
    gate = np.random.default_rng(0).standard_normal((step.batch, step.heads, dim)).astype(np.float32)
    gb = dev.upload(to_dtype(gate, dtype))
    step.args = cuda.DecodeArgs(step.qb, step.ob, step.nb, step.batch, step.heads, DTYPES[dtype], gate=gb, lse=step.lb, seq_ids=step.ib, status=step.status)
    out, lse = step.run(scratch)
    out = out * (1 + np.exp(-from_dtype(to_dtype(gate, dtype), dtype)))  # (a factor of up to 2^6 on what is allowed for a rounding alone)
    rows = [0, 1, 2, 3, step.batch // 2 // 4 * 4 + 2, step.batch - 4, step.batch - 3, step.batch - 2, step.batch - 1]
    check_keys(step, out, lse, lambda s: np.arange(lens[s]), rows)
    for b in range(step.batch):  # the same row in every split: sums of another order
        assert np.allclose(out[b], out[b % 4], rtol=1e-4 if dtype == "f32" else 0.03, atol=1e-4 * np.abs(out[b]).max()), b
    gb.free()
    step.free()


@pytest.mark.parametrize("fmt,dtype", [("q8_0", "f32"), ("f8", "bf16")])
@pytest.mark.parametrize("crowd", [1, 7, 60])
@pytest.mark.parametrize("only", [0, 2, 3])
def test_one_sequence_with_values_far_apart(dev, stream, scratch, fmt, dtype, crowd, only):  # noqa: F811
    """Rows that are done again between rows that are not, whole, joined from a few runs and from many."""
    lens = [70, 1, 333, 2600, 500, 90]
    step = Step(dev, stream, 3, fmt, dtype, 1, 5, 128, 16, lens, seq_ids=list(range(6)) * crowd)
    apart(step, 22, 24, 5, False, [only])
    out, lse = step.run(scratch)
    check_keys(step, out, lse, lambda s: np.arange(lens[s]), sorted({*range(6), *range(step.batch - 6, step.batch), step.batch // 12 * 6 + only}))
    step.free()


@pytest.mark.parametrize("fmt", ["q8_0", "f8"])
def test_values_far_apart_in_more_heads_than_warps(dev, stream, scratch, fmt):  # noqa: F811
    heads, dim, lens = 1000, 64, [40, 3]
    step = Step(dev, stream, 4, fmt, "f32", heads, 17, dim, 16, lens)  # (17 query heads: two units to a KV head)
    rng = np.random.default_rng(7)
    q = np.repeat(rng.standard_normal((2, heads, 1, dim)), 17, 2).reshape(2, heads * 17, dim).astype(np.float32)
    step.qg = q
    step.qb.write(q)
    for s, n in enumerate(lens):
        k, v = rng.standard_normal((n, heads, dim)) * 0.25, rng.standard_normal((n, heads, dim)) * 2.0 ** -6
        u = q[s, ::17]
        k[1] = -24.0 * u / (step.scale * (u * u).sum(-1, keepdims=True)) * np.where(np.arange(heads) % 2, 1.0, -1.0)[:, None]
        v[1] *= 2.0 ** 20
        bufs = [dev.upload(np.ascontiguousarray(a, t)) for a, t in ((k, np.float32), (v, np.float32), (np.arange(n), np.int32), (np.full(n, s), np.int32))]
        cuda.kv_write(stream, step.paged.cache, cuda.KvRows(bufs[0], bufs[1], bufs[2], n, seq=bufs[3]))
        stream.synchronize()
        for b in bufs:
            b.free()
    step.paged.k, step.paged.v = step.paged.download()
    out, lse = step.run(scratch)
    for b, n in enumerate(lens):
        slots = step.paged.slots(b, np.arange(n))
        k, v = decode(step.paged.k[slots], fmt, heads, dim), decode(step.paged.v[slots], fmt, heads, dim)
        for h in [0, 8, 9, 16, 17, 33, 8500, 8509, 16983, 16999]:
            want, want_lse, weight, reach = attend(q[b, h].astype(np.float64), k[:, h // 17], v[:, h // 17], step.scale)
            far, far_lse = attend_bounds(want, want_lse, weight, reach, dim, "f32")
            assert np.all(np.abs(out[b, h] - want) <= far) and abs(lse[b, h] - want_lse) <= far_lse, (b, h)
    step.free()


@pytest.mark.parametrize("fmt,dtype", [("f16", "f32"), ("q8_0", "f32"), ("f8", "f32"), ("f32", "f32"), ("f16", "f16"), ("f8", "bf16")])
def test_strong_gates(dev, stream, scratch, fmt, dtype):  # noqa: F811
    """Gates from -100 to 100, over one key (the output is its value times the gate) and over joined runs. An exponential is off by
    an f32 step, sum, quotient and product by half of one each: 2^-22 at most, with the value's own 2^-22 beside it."""
    step = Step(dev, stream, 9, fmt, dtype, 2, 2, 128, 16, [1, 1, 1500], gate=True)
    q = from_dtype(step.qg, dtype)
    q[..., 128:] = np.linspace(-1, 1, 128) * np.array([30.0, 100.0, 30.0])[:, None, None]
    step.qg = to_dtype(q.astype(np.float32), dtype)
    step.qb.write(step.qg)
    q = from_dtype(step.qg, dtype)
    out, lse = step.run(scratch)
    if dtype != "f16":  # (f16 outputs below 2^-14 have no relative bound: 2^-25 below)
        step.check(out, lse)
    for b in range(2):
        v = decode(step.paged.v[step.paged.slots(b, np.array([0]))], fmt, 2, 128)[0]
        want = np.repeat(v, 2, axis=0) / (1 + np.exp(-q[b, :, 128:]))
        bound = np.abs(want) * (HALF_STEP[dtype] + 2.0 ** -21 + (0 if dtype == "f32" else 2.0 ** -11)) + (1e-36 if dtype != "f16" else 2.0 ** -25)
        assert np.all(np.abs(out[b] - want) <= bound), float(np.max(np.abs(out[b] - want) / bound))
    step.free()
