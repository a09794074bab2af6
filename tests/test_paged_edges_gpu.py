"""GPU tests of the paged 4-bit cache where its parts meet: a missing page
inside a unit of columns, scores whose fp32 steps are wide, appends whose
workgroups have several heads, calls of more than 64 sequences. Against
paged_oracle; tolerances are counted there or beside the test."""
import numpy as np
import pytest
import torch

from llminfer_amd import _lib, ops
from tests import paged_oracle as po
from tests.test_paged_gpu import Cache, check, dev, filled, ints, rows16

pytestmark = pytest.mark.gpu


# -------------------------------------------------------------- missing pages

def lose_page(cache, s, slot):
    """A sequence's page outside the pool; page 0, whose bytes the kernels may
    have in its place, is a spare one of NaN."""
    table = cache.table.cpu().numpy()
    if (table == 0).any():
        spare = int(np.setdiff1d(np.arange(cache.pool.shape[0]), table)[0])
        cache.pool[spare] = cache.pool[0].clone()
        table[table == 0] = spare
    cache.pool[0] = 0xFF
    table[s, slot] = cache.pool.shape[0] + 5
    cache.table = dev(table)


MISSING = [  # rows, past, Hq, Hkv, dim, page, the page that is missing
    (4, 29, 4, 1, 128, 32, 1),        # 16 columns, some rows before the page
    (9, 61, 4, 1, 64, 64, 1),
    (4, 2046, 4, 1, 128, 32, 64),     # divided keys
    (7, 1275, 2, 1, 256, 64, 20),
    (40, 20, 4, 1, 64, 32, 1),        # 64 columns, whole pages behind
    (12, 2077, 4, 1, 256, 32, 65),    # 32 columns, divided keys
    (11, 90, 10, 2, 128, 32, 3),
    (60, 30, 4, 1, 256, 32, 1),       # tiles, the page in the first unit
    (60, 30, 4, 1, 256, 32, 2),       # and in the second
    (20, 950, 16, 2, 256, 64, 15),
    (100, 5, 4, 1, 128, 32, 1),
    (120, 2030, 4, 1, 128, 32, 64),   # divided
    (120, 2030, 4, 1, 128, 64, 33),
]


@pytest.mark.parametrize("rows, past, hq, hkv, dim, page, slot", MISSING)
def test_rows_before_a_missing_page(gpu, rows, past, hq, hkv, dim, page, slot):
    """Rows whose keys end before the page are answered, those that see it are
    NaN, whatever shares their workgroup; so is the other sequence."""
    rng = np.random.default_rng(31 + rows + past)
    both = [rows, rows]
    cache, kv = filled(rng, both, [past, past], hkv, dim, page)
    lose_page(cache, 0, slot)
    q = rows16(rng, 2 * rows, hq, dim)
    invalid = ints(0)
    out = ops.paged_gqa(dev(q), cache.pool, ints(0, rows, 2 * rows), ints(past, past), cache.table,
                        invalid=invalid).cpu().numpy()
    assert invalid.item() == _lib.PAGED_PLACE
    before = slot * page - past
    assert 0 < before < rows
    check(out[:before], q, [x[:1] for x in kv], [before], [past], dim ** -0.5)
    assert np.isnan(out[before:rows]).all()
    check(out[rows:], q[rows:], [x[1:] for x in kv], [rows], [past], dim ** -0.5)


# ---------------------------------------------- scores with wide fp32 steps

def inside(out, q, kv, past, scale):
    """Outputs are averages of the visible values: between their least and
    most, up to fp32 sums over n keys (twice (n + 64) half steps of the largest)
    and a half step of fp16. Where the best score leads every other by 40 and
    the errors of two scores in fp32 (each half a step of sum |q k| scale for
    every product and sum), the output is its value."""
    rows, heads, dim = out.shape
    k, v = (x.astype(np.float64) for x in kv)
    group = heads // k.shape[1]
    pinned = 0
    for i in range(rows):
        n = past + i + 1
        for h in range(heads):
            kk, vv, o = k[:n, h // group], v[:n, h // group], out[i, h].astype(np.float64)
            qq = q[i, h].astype(np.float64)
            far = 2 * (n + 64) * 2.0 ** -24 * np.abs(vv).max(0) + np.abs(o) * po.U16 + 2.0 ** -25
            assert np.isfinite(o).all(), (i, h)
            assert np.all(o >= vv.min(0) - far) and np.all(o <= vv.max(0) + far), (i, h)
            x = kk @ qq * scale
            wrong = 2 * (dim + 8) * 2.0 ** -24 * (np.abs(kk) @ np.abs(qq)).max() * scale
            best = int(x.argmax())
            if n == 1 or x[best] - np.delete(x, best).max() > 40 + wrong:
                pinned += 1
                rest = n * np.exp(-40.0) * np.abs(vv).max(0)
                assert np.all(np.abs(o - vv[best]) <= far + rest), (i, h)
    return pinned


@pytest.mark.parametrize("rows, past, dim", [(1, 0, 256), (1, 5, 128), (1, 700, 64), (1, 1500, 256),
                                             (9, 3, 128), (20, 40, 64), (50, 0, 256), (45, 900, 256),
                                             (110, 500, 128)])
@pytest.mark.parametrize("size", [50.0, 300.0, 2000.0, 30000.0])
@pytest.mark.parametrize("kind", ["apart", "near", "random", "mixed"])
def test_scores_of_any_size(gpu, rows, past, dim, size, kind):
    """Keys near the format's limit and large queries: scores of up to 2^34, whose
    fp32 steps are wider than the softmax. `apart`: keys of one value each, so
    that one leads by far; `near`: their scores differ by less than a step;
    `mixed`: one head's queries are as large, the others' ordinary."""
    rng = np.random.default_rng(int(size) + rows + past + dim)
    n, hq = rows + past, 4
    q = np.full((rows, hq, dim), size, np.float16)
    if kind in ("random", "mixed"):
        k = rng.uniform(-16384, 16384, (n, 1, dim)).astype(np.float16)
        q = rows16(rng, rows, hq, dim, size=min(size, 8000.0))
        if kind == "mixed":
            q[:, :3] = rows16(rng, rows, 3, dim, size=2.0 ** -12)
    elif kind == "apart":
        k = np.repeat((16384 - 16.0 * rng.permutation(n)).astype(np.float16)[:, None, None], dim, 2)
        q[:, ::2] *= -1
    else:
        k = np.full((n, 1, dim), 16000.0, np.float16)
        k[:, 0, 0] -= 8 * rng.integers(0, 60, n).astype(np.float16)
        q[..., 0] = 1.0
    v = rows16(rng, n, 1, dim)
    cache = Cache(rng, 1, n, 1, dim, 64, fill=0xFF)
    invalid = ints(0)
    cache.append(dev(k), dev(v), ints(0, n), ints(0), invalid=invalid)
    assert invalid.item() == 0
    kv = [x[0] for x in cache.read([n])]
    scale = float(np.float32(dim) ** np.float32(-0.5))
    out = ops.paged_gqa(dev(q), cache.pool, ints(0, rows), ints(past), cache.table)
    pinned = inside(out.cpu().numpy(), q, kv, past, scale)
    if kind == "apart":
        assert pinned == rows * hq  # 16 apart in every channel: a lead of 100 steps and more


# --------------------------------------- appends with several heads a workgroup

MANY = [  # rows of each sequence, past of each, Hkv, dim, page, rotary, layout, an odd element first
    ([500] * 13, [37 * s for s in range(13)], 8, 128, 32, 128, "interleaved", 0),  # 4 heads
    ([700, 1, 0, 2100, 33, 1500], [5, 31, 9, 0, 64, 1001], 3, 128, 64, 64, "half", 0),  # 2, then 1
    ([2100], [17], 3, 256, 128, 64, "half", 0),
    ([2100], [17], 3, 256, 128, 62, "half", 1),
    ([3000, 2600], [3, 70], 5, 64, 32, 64, "half", 0),                # 2, 2 and 1
    ([8300], [11], 5, 64, 64, 64, "interleaved", 1),                  # 4 and 1
    ([1100, 1200], [0, 31], 8, 256, 64, 0, "half", 0),                # 4, not rotated
]


@pytest.mark.parametrize("rows, past, hkv, dim, page, rot, layout, lead", MANY)
def test_append_of_many_rows(gpu, rows, past, hkv, dim, page, rot, layout, lead):
    """Calls in which a workgroup has several heads, a last one with fewer:
    every head's keys and values are the format's, bit for bit."""
    units = min(sum(rows), sum(rows) // 32 + 2 * len(rows))
    assert units * (dim // 64) * -(-hkv // 2) >= 512  # two heads or more
    rng = np.random.default_rng(sum(rows) + dim)
    S, T = len(rows), sum(rows)
    cache = Cache(rng, S, max(r + p for r, p in zip(rows, past)), hkv, dim, page, fill=0xA5)
    wide = dev(rows16(rng, T, 2 * hkv * dim + 8, size=2.0))
    both = wide[:, lead:lead + 2 * hkv * dim].unflatten(1, (2 * hkv, dim))
    k, v = both[:, :hkv], both[:, hkv:]
    freqs, _ = ops.rope_frequencies(rot, 1e4)
    invalid = ints(0)
    starts, lens = ints(0, *np.cumsum(rows)), ints(*past)
    before = cache.pool.clone()
    cache.append(k, v, starts, lens, freqs=freqs if rot else None, layout=layout, invalid=invalid)
    gk, gv = ops.paged_read(cache.pool, starts, lens, cache.table, T, invalid)
    assert invalid.item() == 0
    turned = k
    if rot:
        pos = np.concatenate([np.arange(p, p + r) for r, p in zip(rows, past)]).astype(np.int32)
        turned = ops.rope(k, dev(pos), freqs, layout=layout)
    for got, want in ((gk, turned), (gv, v)):
        got, want = got.cpu().numpy(), po.kept(want.contiguous().cpu().numpy())
        assert np.array_equal(got, want), np.argwhere((got != want).any(-1))[:8]
    # pages that hold none of the rows stay
    held = torch.zeros(before.shape[0], dtype=torch.bool)
    for s in range(S):
        if rows[s]:
            first, last = past[s] // page, (past[s] + rows[s] - 1) // page
            held[cache.table[s, first:last + 1].long().cpu()] = True
    assert torch.equal(before[~held], cache.pool[~held])


# ------------------------------------------------- more than 64 sequences

def late(count, most, small):
    """Pasts of `count` sequences: short, but for some behind the 64th."""
    past = [(37 * s) % small for s in range(count)]
    for s, n in most.items():
        past[s] = n
    return past


CROWDS = [  # rows of each sequence, past of each, Hq, Hkv, dim, page
    ([1] * 70, late(70, {3: 2000, 64: 4100, 69: 3000}, 90), 4, 1, 128, 64),
    ([1] * 130, late(130, {63: 900, 64: 2500, 65: 40, 128: 5000, 129: 1700}, 60), 8, 2, 64, 32),
    ([1] * 66, late(66, {65: 6000}, 50), 16, 4, 256, 64),
    ([5] * 80, late(80, {10: 1500, 66: 3000, 79: 2222}, 70), 8, 1, 256, 32),      # 32 columns
    ([26] * 67, late(67, {64: 2600, 66: 1900}, 40), 4, 1, 64, 64),                # 64
    ([12] * 70, late(70, {0: 1000, 64: 3000, 69: 2500}, 80), 4, 1, 256, 32),      # tiles
    ([24] * 70, late(70, {33: 900, 65: 2400, 69: 2000}, 60), 8, 2, 128, 64),
    ([8, 0, 30] * 44, late(132, {2: 1200, 128: 3100, 131: 2700}, 50), 4, 1, 256, 64),
]


@pytest.mark.parametrize("rows, past, hq, hkv, dim, page", CROWDS)
def test_more_than_64_sequences(gpu, rows, past, hq, hkv, dim, page):
    """Sequences behind the 64th whose keys are divided and joined."""
    rng = np.random.default_rng(len(rows) + dim)
    cache, kv = filled(rng, rows, past, hkv, dim, page)
    T = sum(rows)
    q = rows16(rng, T + 2, hq, dim, size=1.5)
    out = torch.full((T + 2, hq, dim), 9.0, dtype=torch.float16, device="cuda")
    invalid = ints(0)
    ops.paged_gqa(dev(q), cache.pool, ints(0, *np.cumsum(rows)), ints(*past), cache.table, out=out,
                  invalid=invalid)
    assert invalid.item() == 0
    out = out.cpu().numpy()
    assert (out[T:] == 9).all()
    check(out, q, kv, rows, past, dim ** -0.5)
