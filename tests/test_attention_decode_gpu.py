"""attention_decode against the formula in 64 bits, over caches written by kv_write."""
import numpy as np
import pytest

from tests.kv_reference import DTYPES, FORMATS, HALF_STEP, Paged, attend, attend_bounds, decode, encode, from_dtype, storage, to_dtype
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


@pytest.fixture(scope="module")
def scratch(dev):
    s = cuda.AttentionScratch(dev)
    yield s
    s.destroy()


class Step:
    """A cache of sequences of the given lengths and one token's queries for each row of the batch."""

    def __init__(self, dev, stream, seed, fmt, dtype, kv_heads, group, dim, block, lens, gate=False, window=0, scale=0.0, seq_ids=None,
                 spread=1.0, extra_pages=0):
        self.__dict__.update(dev=dev, stream=stream, fmt=fmt, dtype=dtype, kv_heads=kv_heads, group=group, dim=dim, gate=gate, window=window)
        rng = self.rng = np.random.default_rng(seed)
        self.lens = np.asarray(lens, np.int32)
        self.paged = Paged(dev, rng, fmt, kv_heads, dim, block, lens, extra_pages=extra_pages)
        self.seq_ids = seq_ids
        ids = np.arange(len(lens)) if seq_ids is None else np.asarray(seq_ids)
        self.rows = [(int(s), int(self.lens[s])) for s in ids]
        self.batch, self.heads = len(ids), kv_heads * group
        self.scale = scale or dim ** -0.5
        # written by the library itself
        total = int(self.lens.sum())
        if total:
            seq = np.repeat(np.arange(len(lens)), self.lens).astype(np.int32)
            pos = np.concatenate([np.arange(n) for n in self.lens]).astype(np.int32)
            mix = rng.permutation(total)
            seq, pos = seq[mix], pos[mix]
            x = [(rng.standard_normal((total, kv_heads, dim)) * f).astype(np.float32) for f in (1.0, np.exp2(rng.uniform(-3, 3, (total, kv_heads, 1))))]
            bufs = [dev.upload(a) for a in (*x, seq, pos)]
            cuda.kv_write(stream, self.paged.cache, cuda.KvRows(bufs[0], bufs[1], bufs[3], total, seq=bufs[2]))
            stream.synchronize()
            for b in bufs:
                b.free()
        self.paged.k, self.paged.v = self.paged.download()
        width = 2 * dim if gate else dim
        qg = (rng.standard_normal((self.batch, self.heads, width)) * spread).astype(np.float32)
        self.qg = to_dtype(qg, dtype)
        size = self.qg.itemsize
        self.qb = dev.upload(self.qg)
        self.ob, self.lb = dev.alloc(self.batch * self.heads * dim * size), dev.alloc(self.batch * self.heads * 4)
        row_lens = np.array([n for _, n in self.rows], np.int32)
        self.nb = dev.upload(row_lens)
        self.ib = dev.upload(ids.astype(np.int32)) if seq_ids is not None else None
        self.status = dev.upload(np.zeros(4, np.int32))
        self.args = cuda.DecodeArgs(self.qb, self.ob, self.nb, self.batch, self.heads, DTYPES[dtype], scale=scale, window=window,
                                    gate=self.qb if gate else None, gate_offset=dim * size if gate else 0, q_head_stride=width, lse=self.lb,
                                    seq_ids=self.ib, status=self.status)

    def run(self, scratch):
        self.ob.write(np.full(self.ob.nbytes, 0xAA, np.uint8))
        cuda.attention_decode(self.stream, scratch, self.paged.cache, self.args)
        self.stream.synchronize()
        return self.result()

    def result(self):
        out = from_dtype(self.ob.read(storage(self.dtype), self.batch * self.heads * self.dim), self.dtype)
        return out.reshape(self.batch, self.heads, self.dim), self.lb.read(np.float32, self.batch * self.heads).reshape(self.batch, self.heads)

    def check(self, out, lse, skip=()):
        qg = from_dtype(self.qg, self.dtype)
        for b, (seq, n) in enumerate(self.rows):
            if b in skip:
                continue
            first = max(0, n - self.window) if self.window else 0
            slots = self.paged.slots(seq, np.arange(first, n)) if n else np.zeros(0, np.int64)
            k, v = decode(self.paged.k[slots], self.fmt, self.kv_heads, self.dim), decode(self.paged.v[slots], self.fmt, self.kv_heads, self.dim)
            for h in range(self.heads):
                j = h // self.group
                want, want_lse, weight, reach = attend(qg[b, h, :self.dim], k[:, j], v[:, j], self.scale)
                if self.gate:
                    s = 1 / (1 + np.exp(-qg[b, h, self.dim:]))
                    want, weight = want * s, weight * s
                far, far_lse = attend_bounds(want, want_lse, weight, reach, self.dim, self.dtype)
                off = np.abs(out[b, h] - want)
                assert np.all(off <= far), (b, h, n, float(off.max()), float((off / far).max()))
                if np.isfinite(want_lse):
                    assert abs(lse[b, h] - want_lse) <= far_lse, (b, h, n, lse[b, h], want_lse, far_lse)
                else:
                    assert np.isneginf(lse[b, h])

    def free(self):
        for b in (self.qb, self.ob, self.lb, self.nb, self.status, *([self.ib] if self.ib else [])):
            b.free()
        self.paged.free()


EDGE = [1, 2, 15, 16, 17, 31, 33, 64, 65, 0, 127, 300]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("fmt", list(FORMATS))
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_lengths_around_tiles(dev, stream, scratch, fmt, dtype, dim):
    """Lengths from zero over one to several warps' runs, pages that end inside tiles."""
    step = Step(dev, stream, dim, fmt, dtype, 2, 4, dim, 5, EDGE)
    out, lse = step.run(scratch)
    step.check(out, lse)
    assert np.all(out[EDGE.index(0)] == 0)
    assert step.status.read(np.int32, 1)[0] == 0
    step.free()


@pytest.mark.parametrize("fmt,dtype,dim", [("f16", "f32", 128), ("f16", "bf16", 256), ("q8_0", "f32", 256), ("q8_0", "f16", 64),
                                           ("f8", "bf16", 128), ("f8", "f32", 256), ("f32", "f32", 64), ("f32", "bf16", 256)])
@pytest.mark.parametrize("group", [1, 3, 8, 9, 16, 17, 40])
def test_query_heads_per_kv_head(dev, stream, scratch, fmt, dtype, dim, group):
    step = Step(dev, stream, group, fmt, dtype, 1 if group > 8 else 3, group, dim, 16, [70, 1, 260])
    step.check(*step.run(scratch))
    step.free()


@pytest.mark.parametrize("fmt", list(FORMATS))
@pytest.mark.parametrize("lens,kv_heads,dim", [([9000], 1, 128), ([4100, 1, 700], 2, 256), ([3000] * 3, 3, 64)])
def test_long_sequences_are_split_and_joined(dev, stream, scratch, fmt, lens, kv_heads, dim):
    """Runs of warps, CTAs and many CTAs within one unit; twice the same bits."""
    step = Step(dev, stream, 1, fmt, "f32", kv_heads, 4, dim, 16, lens, gate=True)
    out, lse = step.run(scratch)
    step.check(out, lse)
    again, lse2 = step.run(scratch)
    assert np.array_equal(out, again) and np.array_equal(lse, lse2)
    step.free()


@pytest.mark.parametrize("fmt,dtype", [("f16", "bf16"), ("q8_0", "f32"), ("f8", "f16"), ("f32", "f32")])
def test_many_rows_of_ragged_lengths(dev, stream, scratch, fmt, dtype):
    rng = np.random.default_rng(4)
    lens = np.exp(rng.uniform(0, np.log(600), 150)).astype(int)
    lens[[3, 50, 149]] = 0
    step = Step(dev, stream, 6, fmt, dtype, 4, 2, 64, 24, lens)
    step.check(*step.run(scratch))
    step.free()


@pytest.mark.parametrize("fmt,kv_heads,group,dim", [("f32", 640, 1, 256), ("f16", 300, 3, 64), ("f8", 40, 40, 128)])
def test_more_heads_than_warps(dev, stream, scratch, fmt, kv_heads, group, dim):
    """Units (KV heads times tiles of query heads) that pass the warps of the machine, or take a good part of them."""
    step = Step(dev, stream, 3, fmt, "f32", kv_heads, group, dim, 16, [3, 0, 35])
    step.check(*step.run(scratch))
    step.free()


@pytest.mark.parametrize("fmt", ["q8_0", "f8"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("kv_heads,dim", [(1, 64), (3, 64), (5, 64), (1, 128), (3, 128), (1, 256)])
def test_rows_that_are_no_whole_lines(dev, stream, scratch, fmt, dtype, kv_heads, dim):
    """Heads that begin anywhere in 16 bytes, differently from key to key, in a pool whose last row is in use."""
    step = Step(dev, stream, kv_heads, fmt, dtype, kv_heads, 2, dim, 3, [60, 7, 1])
    pages, last = step.paged, step.paged.blocks - 1
    if last not in pages.tables:  # the first sequence's last page moves there
        old = int(pages.tables[0, 19])
        for pool in (pages.k, pages.v):
            pool[3 * last:3 * last + 3] = pool[3 * old:3 * old + 3]
            pool[3 * old:3 * old + 3] = 255
        pages.tables[0, 19] = last
        pages.tb.write(pages.tables)
        pages.upload()
    step.check(*step.run(scratch))
    step.free()


def test_a_batch_of_thousands(dev, stream, scratch):
    rng = np.random.default_rng(17)
    lens = rng.integers(0, 40, 300)
    step = Step(dev, stream, 19, "f16", "bf16", 1, 4, 64, 8, lens, seq_ids=rng.integers(0, 300, 5000))
    out, lse = step.run(scratch)
    keep = set(range(0, 5000, 37)) | {4999}
    step.check(out, lse, skip=set(range(5000)) - keep)
    # rows of one sequence with one query would be equal: here the statistics depend on the row's own query alone
    assert np.all(np.isfinite(out))
    step.free()


@pytest.mark.parametrize("fmt,dtype", [("f16", "f32"), ("f8", "f32"), ("q8_0", "f32"), ("f32", "f32")])
def test_long_runs_keep_f32(dev, stream, scratch, fmt, dtype):
    """Many tiles in one warp's run: sums of thousands of products stay within f32's rounding (the machine is filled with other
    rows, so that a row is not split)."""
    step = Step(dev, stream, 4, fmt, dtype, 8, 1, 64, 64, [2000, 1500, 1900] + [1700] * 5, seq_ids=list(range(8)) * 60)
    out, lse = step.run(scratch)
    step.check(out, lse, skip=set(range(480)) - {0, 1, 2, 100, 479})
    step.free()


@pytest.mark.parametrize("fmt", list(FORMATS))
@pytest.mark.parametrize("window", [1, 16, 50, 1000])
def test_window(dev, stream, scratch, fmt, window):
    """Keys before the window hold NaN and are not used."""
    step = Step(dev, stream, window, fmt, "f32", 2, 2, 64, 7, [1, 49, 50, 51, 200, 1040], window=window)
    for s, n in enumerate(step.lens):
        if n > window:
            slots = step.paged.slots(s, np.arange(0, n - window))
            step.paged.k[slots] = 255
            step.paged.v[slots] = 255
    step.paged.upload()
    step.check(*step.run(scratch))
    step.free()


@pytest.mark.parametrize("fmt", list(FORMATS))
def test_rows_behind_the_length_are_not_used(dev, stream, scratch, fmt):
    """The rest of the last page holds infinities and NaN (Paged fills every unused row with NaN; here infinities in f16 and f32)."""
    step = Step(dev, stream, 3, fmt, "bf16", 2, 4, 128, 64, [3, 70, 129])
    used = np.concatenate([step.paged.slots(s, np.arange(n)) for s, n in enumerate(step.lens)])
    rest = np.setdiff1d(np.arange(step.paged.k.shape[0]), used)
    inf = {"f32": np.full(step.paged.row // 4, np.inf, np.float32).view(np.uint8), "f16": np.full(step.paged.row // 2, -np.inf, np.float16).view(np.uint8)}
    if fmt in inf:
        step.paged.k[rest] = inf[fmt]
        step.paged.v[rest] = inf[fmt]
        step.paged.upload()
    step.check(*step.run(scratch))
    step.free()


@pytest.mark.parametrize("fmt", list(FORMATS))
def test_rows_that_share_sequences_in_any_order(dev, stream, scratch, fmt):
    step = Step(dev, stream, 8, fmt, "f32", 2, 2, 64, 16, [40, 0, 333, 17], seq_ids=[3, 2, 2, 0, 1, 3, 2])
    out, lse = step.run(scratch)
    step.check(out, lse)
    step.free()


@pytest.mark.parametrize("fmt", list(FORMATS))
def test_ids_out_of_range_become_nan(dev, stream, scratch, fmt):
    """A bad block, length or sequence makes its own row NaN, is reported, and leaves the other rows as they are."""
    step = Step(dev, stream, 12, fmt, "f32", 2, 2, 64, 4, [90, 40, 1200, 13, 30], extra_pages=2)
    good, good_lse = step.run(scratch)
    step.check(good, good_lse)

    def expect(bad_rows, bits):
        step.status.write(np.zeros(4, np.int32))
        out, lse = step.run(scratch)
        assert step.status.read(np.int32, 1)[0] == bits
        for b in range(step.batch):
            if b in bad_rows:
                assert np.all(np.isnan(out[b])) and np.all(np.isnan(lse[b])), b
        step.check(out, lse, skip=bad_rows)

    tables = step.paged.tables.copy()
    for page, block in ((0, step.paged.blocks), (150, -1), (299, 2147483647)):
        step.paged.tables[2, page] = block
        step.paged.tb.write(step.paged.tables)
        expect([2], 1)
        step.paged.tables[:] = tables
    step.paged.tb.write(tables)
    lens = step.nb.read(np.int32, step.batch)
    for value in (-1, step.paged.tables.shape[1] * 4 + 1, 2147483647, -2147483648):
        changed = lens.copy()
        changed[1] = value
        step.nb.write(changed)
        expect([1], 4)
    step.nb.write(lens)
    ids = dev.upload(np.array([0, 1, 2, 5, -1], np.int32))
    step.args.args.seq_ids = ids.h
    expect([3, 4], 2)
    ids.free()
    step.free()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("order", ["head major", "padded"])
def test_strides(dev, stream, scratch, dtype, order):
    """Queries and outputs with all rows of a head behind one another, and with room between heads and rows that stays."""
    step = Step(dev, stream, 21, "f16", dtype, 2, 3, 64, 16, [5, 100, 31])
    B, H, D, size = step.batch, step.heads, 64, step.qg.itemsize
    row, head = (D, B * D) if order == "head major" else (H * 96 + 32, 96)
    n = (B - 1) * row + (H - 1) * head + D
    at = (np.arange(B)[:, None, None] * row + np.arange(H)[None, :, None] * head + np.arange(D)).ravel()
    q = np.zeros(n, storage(dtype))
    q[at] = step.qg.ravel()
    qb, ob = dev.upload(q), dev.upload(np.full(n * size, 0x5A, np.uint8))
    cuda.attention_decode(stream, scratch, step.paged.cache,
                          cuda.DecodeArgs(qb, ob, step.nb, B, H, DTYPES[dtype], q_row_stride=row, q_head_stride=head, out_row_stride=row,
                                          out_head_stride=head, lse=step.lb))
    stream.synchronize()
    got = ob.read(storage(dtype), n)
    step.check(from_dtype(got[at], dtype).reshape(B, H, D), step.lb.read(np.float32, B * H).reshape(B, H))
    between = np.setdiff1d(np.arange(n), at)
    assert np.all(got.view(np.uint8).reshape(n, size)[between] == 0x5A)
    qb.free()
    ob.free()
    step.free()


@pytest.mark.parametrize("fmt,dtype", [("f16", "f32"), ("f16", "f16"), ("q8_0", "f32"), ("f8", "f32"), ("f32", "f32")])
@pytest.mark.parametrize("factor", [1e-3, 30.0])
def test_flat_and_sharp_scores(dev, stream, scratch, fmt, dtype, factor):
    """All keys weigh about the same; one key outweighs all others."""
    step = Step(dev, stream, 5, fmt, dtype, 2, 2, 128, 16, [1500, 40], spread=factor)
    step.check(*step.run(scratch))
    step.free()


@pytest.mark.parametrize("fmt", list(FORMATS))
def test_scale_and_tiny_values(dev, stream, scratch, fmt):
    """A scale of the caller's, queries of 1e-20 or 1e20, and values of 1e-4: nothing is lost to narrow types."""
    for q, scale in ((1e-20, 1e20), (1e20, 1e-20), (1.0, -0.1)):
        step = Step(dev, stream, 5, fmt, "f32", 1, 2, 64, 16, [200], spread=q, scale=scale)
        step.check(*step.run(scratch))
        step.free()
    step = Step(dev, stream, 6, fmt, "f32", 1, 2, 64, 16, [300])
    rng = np.random.default_rng(0)
    x = (rng.standard_normal((300, 1, 64)) * 1e-4).astype(np.float32)
    k = rng.standard_normal((300, 1, 64)).astype(np.float32)
    bufs = [dev.upload(a) for a in (k, x, np.arange(300, dtype=np.int32), np.zeros(300, np.int32))]
    cuda.kv_write(stream, step.paged.cache, cuda.KvRows(bufs[0], bufs[1], bufs[2], 300, seq=bufs[3]))
    stream.synchronize()
    step.paged.k, step.paged.v = step.paged.download()
    step.check(*step.run(scratch))
    for b in bufs:
        b.free()
    step.free()


@pytest.mark.parametrize("dtype,fmt", [("bf16", "f16"), ("f32", "f32")])
@pytest.mark.parametrize("dim", [64, 256])
def test_scores_of_minus_infinity_weigh_nothing(dev, stream, scratch, dtype, fmt, dim):
    """The first 40 keys of each sequence score -infinity (an infinity in an f16 pool, a product beyond f32's range): as if they
    were not there, in whole first tiles and in whole runs of a warp; a sequence of them alone is one without keys."""
    step = Step(dev, stream, 2, fmt, dtype, 1, 2, dim, 16, [300, 57, 41, 40, 5000])
    q = np.abs(from_dtype(step.qg, dtype)) + 0.5
    if fmt == "f32":  # sums of -2^132 and 2^66 * (k of the others), and a scale that brings the others back
        q = np.full(q.shape, 2.0 ** 66)
        step.scale = step.args.args.scale = 2.0 ** -66 / 8
    step.qg = to_dtype(q.astype(np.float32), dtype)
    step.qb.write(step.qg)
    low = {"f32": np.full(step.paged.row // 4, -2.0 ** 66, np.float32).view(np.uint8), "f16": np.full(step.paged.row // 2, -np.inf, np.float16).view(np.uint8)}
    for s in range(5):
        step.paged.k[step.paged.slots(s, np.arange(40))] = low[fmt]
    step.paged.upload()
    out, lse = step.run(scratch)
    assert np.all(out[3] == 0) and np.all(np.isneginf(lse[3]))
    for b in (0, 1, 2, 4):  # the formula without those keys
        step.window = int(step.lens[b]) - 40
        step.check(out, lse, skip=set(range(5)) - {b})
    step.free()


def test_values_of_many_magnitudes(dev, stream, scratch, oracle):
    """Scales of V that grow and shrink along the sequence, zeros among them."""
    for fmt in ("q8_0", "f8"):
        step = Step(dev, stream, 6, fmt, "f32", 1, 2, 128, 16, [640])
        rng = np.random.default_rng(1)
        x = (rng.standard_normal((640, 1, 128)) * np.exp2(np.linspace(-12, 12, 640))[rng.permutation(640), None, None]).astype(np.float32)
        x[:40] = 0.0
        x[300:310] = 0.0
        x[500, 0, 32:] = 0.0
        slots = step.paged.slots(0, np.arange(640))
        step.paged.v[slots] = encode(x, fmt, oracle)
        step.paged.upload()
        step.check(*step.run(scratch))
        step.paged.v[slots] = encode(np.zeros_like(x), fmt, oracle)
        step.paged.upload()
        out, lse = step.run(scratch)
        assert np.all(out == 0) and np.all(np.isfinite(lse))
        step.free()


def test_two_streams_and_scratches_at_once(dev, scratch):
    """Calls that may overlap, each with a scratch of its own."""
    streams = [dev.stream() for _ in range(3)]
    scratches = [cuda.AttentionScratch(dev) for _ in range(3)]
    steps = [Step(dev, s, 40 + i, f, "f32", 2, 4, 128, 16, [2500, 900 + 100 * i]) for i, (s, f) in enumerate(zip(streams, ("f16", "q8_0", "f8")))]
    alone = [s.run(scratch) for s in steps]
    for _ in range(20):
        for s, sc in zip(steps, scratches):
            cuda.attention_decode(s.stream, sc, s.paged.cache, s.args)
    for s in streams:
        s.synchronize()
    for s, (out, lse) in zip(steps, alone):
        got = s.result()
        assert np.array_equal(got[0], out) and np.array_equal(got[1], lse)
        s.free()
    for x in (*scratches,):
        x.destroy()
    for s in streams:
        s.destroy()


def test_captured_steps_follow_the_lengths(dev, oracle):
    """A decode loop in torch's memory and on its stream: write the new token, attend, read it back, captured once and replayed
    as the sequences grow; two graphs with a scratch each, replayed side by side."""
    import torch
    rng = np.random.default_rng(31)
    kv_heads, group, dim, block, cap = 2, 4, 64, 16, 400
    graphs = []
    for g, fmt in enumerate(("q8_0", "f8")):
        lens = [150 + g, 3]
        rb = cuda.kv_row_bytes(FORMATS[fmt], kv_heads, dim)
        pages = cap // block
        pool = [torch.zeros(2 * pages, block, rb, dtype=torch.uint8, device="cuda") for _ in range(2)]
        tables = torch.from_numpy(rng.permutation(2 * pages).astype(np.int32).reshape(2, pages)).cuda()
        view = lambda t: dev.view(t.data_ptr(), t.numel() * t.element_size())  # noqa: E731
        cache = cuda.KvCache(view(pool[0]), view(pool[1]), view(tables), FORMATS[fmt], kv_heads, dim, block, 2 * pages, 2, pages)
        t = {"k": torch.zeros(2, kv_heads, dim, device="cuda"), "v": torch.zeros(2, kv_heads, dim, device="cuda"),
             "q": torch.zeros(2, kv_heads * group, dim, device="cuda"), "out": torch.zeros(2, kv_heads * group, dim, device="cuda"),
             "rk": torch.zeros(2, kv_heads, dim, device="cuda"), "rv": torch.zeros(2, kv_heads, dim, device="cuda"),
             "pos": torch.zeros(2, dtype=torch.int32, device="cuda"), "lens": torch.zeros(2, dtype=torch.int32, device="cuda")}
        scratch, side = cuda.AttentionScratch(dev), torch.cuda.Stream()
        rows, back = (cuda.KvRows(view(t[a]), view(t[b]), view(t["pos"]), 2) for a, b in (("k", "v"), ("rk", "rv")))
        args = cuda.DecodeArgs(view(t["q"]), view(t["out"]), view(t["lens"]), 2, kv_heads * group)
        # history: both sequences up to their lengths
        xs = rng.standard_normal((2, 2, cap, kv_heads, dim)).astype(np.float32)
        s0 = dev.stream_view(torch.cuda.current_stream().cuda_stream)
        for p in range(max(lens)):
            t["k"].copy_(torch.from_numpy(xs[0, :, p]))
            t["v"].copy_(torch.from_numpy(xs[1, :, p]))
            t["pos"].copy_(torch.tensor([p if p < n else -1 for n in lens], dtype=torch.int32))
            cuda.kv_write(s0, cache, rows)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            s = dev.stream_view(torch.cuda.current_stream().cuda_stream)
            cuda.kv_write(s, cache, rows)
            cuda.attention_decode(s, scratch, cache, args)
            cuda.kv_read(s, cache, back)
        graphs.append((fmt, lens, xs, t, graph, side, pool, tables, scratch))
    for step in range(40):
        qs = []
        for fmt, lens, xs, t, graph, side, *_ in graphs:
            at = [n + step for n in lens]
            t["k"].copy_(torch.from_numpy(np.stack([xs[0, s, p] for s, p in enumerate(at)])))
            t["v"].copy_(torch.from_numpy(np.stack([xs[1, s, p] for s, p in enumerate(at)])))
            t["pos"].copy_(torch.tensor(at, dtype=torch.int32))
            t["lens"].copy_(torch.tensor(at, dtype=torch.int32) + 1)
            qs.append(rng.standard_normal((2, kv_heads * group, dim)).astype(np.float32))
            t["q"].copy_(torch.from_numpy(qs[-1]))
        torch.cuda.synchronize()
        for _, _, _, _, graph, side, *_ in graphs:
            with torch.cuda.stream(side):
                graph.replay()
        torch.cuda.synchronize()
        if step % 13:
            continue
        for q, (fmt, lens, xs, t, *_) in zip(qs, graphs):
            out = t["out"].cpu().numpy().astype(np.float64)
            for s, n in enumerate(lens):
                n = n + step + 1
                k, v = (decode(encode(xs[c, s, :n], fmt, oracle), fmt, kv_heads, dim) for c in (0, 1))
                assert np.array_equal(t["rk"][s].cpu().numpy(), k[-1].astype(np.float32))
                assert np.array_equal(t["rv"][s].cpu().numpy(), v[-1].astype(np.float32))
                for h in range(kv_heads * group):
                    want, lse, weight, reach = attend(q[s, h].astype(np.float64), k[:, h // group], v[:, h // group], dim ** -0.5)
                    far, _ = attend_bounds(want, lse, weight, reach, dim, "f32")
                    assert np.all(np.abs(out[s, h] - want) <= far)
    torch.cuda.synchronize()
    for *_, scratch in graphs:
        scratch.destroy()


def test_a_cache_behind_four_gigabytes(dev, stream, scratch, oracle):
    """Row offsets beyond 32 bits, in the last blocks of a large pool."""
    heads, dim, block, blocks = 8, 256, 64, 16500  # f16: 4096 bytes a row, 4.3 GB a pool
    row = cuda.kv_row_bytes(cuda.KV_F16, heads, dim)
    k, v = (dev.alloc(row * block * blocks) for _ in range(2))
    tables = dev.upload(np.array([[blocks - 1, 3, blocks - 2]], np.int32))
    cache = cuda.KvCache(k, v, tables, cuda.KV_F16, heads, dim, block, blocks, 1, 3)
    rng = np.random.default_rng(1)
    n = 150
    x = rng.standard_normal((2, n, heads, dim)).astype(np.float32)
    bufs = [dev.upload(a) for a in (x[0], x[1], np.arange(n, dtype=np.int32), np.zeros(n, np.int32), np.array([n], np.int32))]
    cuda.kv_write(stream, cache, cuda.KvRows(bufs[0], bufs[1], bufs[2], n, seq=bufs[3]))
    q = rng.standard_normal((1, heads, dim)).astype(np.float32)
    qb, ob = dev.upload(q), dev.alloc(q.nbytes)
    cuda.attention_decode(stream, scratch, cache, cuda.DecodeArgs(qb, ob, bufs[4], 1, heads))
    stream.synchronize()
    out = ob.read(np.float32, q.size).reshape(heads, dim)
    kv = [decode(encode(a, "f16", oracle), "f16", heads, dim) for a in x]
    for h in range(heads):
        want, lse, weight, reach = attend(q[0, h].astype(np.float64), kv[0][:, h], kv[1][:, h], dim ** -0.5)
        assert np.all(np.abs(out[h] - want) <= attend_bounds(want, lse, weight, reach, dim, "f32")[0])
    for b in (k, v, tables, qb, ob, *bufs):
        b.free()


def test_one_key_is_its_value(dev, stream, scratch):
    """With a single key the output is the cached value itself, whatever the query."""
    for fmt in FORMATS:
        step = Step(dev, stream, 7, fmt, "f32", 3, 4, 128, 16, [1, 1])
        out, _ = step.run(scratch)
        for b in range(2):
            v = decode(step.paged.v[step.paged.slots(b, np.array([0]))], fmt, 3, 128)[0]
            got = out[b].reshape(3, 4, 128)
            assert np.all(np.abs(got - v[:, None]) <= np.abs(v[:, None]) * 8 * HALF_STEP["f32"] + np.abs(v).max() * 2.0 ** -22)
        step.free()


def test_views_of_memory_that_is_not_the_devices(dev):
    import ctypes
    host = (ctypes.c_uint8 * 4096)()
    with pytest.raises(cuda.YuukaError) as e:
        dev.view(ctypes.addressof(host), 4096)
    assert e.value.status == cuda.ERR_INVALID_ARGUMENT
    b = dev.alloc(1 << 21)
    v = dev.view(cuda.lib().yuuka_buffer_ptr(b.h) + 256, 1024)
    v.write(np.arange(256, dtype=np.int32))
    assert np.array_equal(b.read(np.int32, 256, offset=256), np.arange(256))
    v.free()  # the handle alone
    assert np.array_equal(b.read(np.int32, 256, offset=256), np.arange(256))
    b.free()
