"""attention_decode where numbers leave the ordinary."""
import numpy as np
import pytest

from tests.kv_reference import attend, attend_bounds, decode, from_dtype, to_dtype
from tests.test_attention_decode_gpu import Step, dev, scratch, stream  # noqa: F401  (fixtures)

pytestmark = pytest.mark.gpu


def check_keys(step, out, lse, keep, rows, more=0.0):
    """The formula over the keys `keep(sequence)` alone; `more`: allowed beyond attend_bounds, per output."""
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
            assert np.all(off <= far + more), (b, h, len(slots), float(np.nanmax(off)), float(np.nanmax(off / (far + more))))
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
