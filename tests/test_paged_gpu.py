"""GPU tests of rotary rows and the paged 4-bit cache against paged_oracle:
the rotation, appending and reading back, the attention, and a run of them
together. Tolerances are paged_oracle's, counted there."""
import numpy as np
import pytest
import torch

from llminfer_amd import _lib, ops
from tests import paged_oracle as po

pytestmark = pytest.mark.gpu


def dev(a, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(a))
    return (t if dtype is None else t.to(dtype)).cuda()


def ints(*values):
    return torch.tensor(values, dtype=torch.int32).cuda()


def rows16(rng, *shape, size=1.0):
    return (size * rng.standard_normal(shape)).astype(np.float16)


# --------------------------------------------------------------- rotary rows

ROPE = [  # tokens, heads, dim, rotary, layout, first position, step, factor
    (1, 16, 256, 64, "half", 0, 1, 1.0),
    (1, 16, 256, 64, "half", 1_000_003, 1, 1.0),
    (37, 4, 256, 64, "half", 4096, 1, 1.0),
    (5, 3, 128, 128, "interleaved", 70_000, 1, 1.25),
    (9, 2, 64, 64, "half", 2**31 - 10, 1, 1.0),
    (4, 2, 64, 32, "interleaved", -7, 3, 1.0),
    (13, 5, 80, 34, "interleaved", 123_457, -11, 1.0),
    (7, 3, 96, 22, "half", 999, 1, 0.5),
    (6, 2, 7, 4, "half", 1, 1, 1.0),
    (6, 2, 7, 6, "interleaved", 1, 1, 1.0),
    (3, 2, 64, 0, "half", 5, 1, 1.0),
    (2, 1, 2048, 2048, "half", 5, 1, 1.0),
    (65, 1, 2, 2, "interleaved", 11, 1, 1.0),
    (5, 4, 256, 186, "half", 30_000, 1, 1.0),
    (5, 4, 256, 186, "interleaved", 30_000, 1, 1.0),
    (300, 2, 100, 42, "half", 17, 1, 1.0),
]


@pytest.mark.parametrize("T, H, D, rot, layout, first, step, factor", ROPE)
@pytest.mark.parametrize("how", ["out", "in place", "strided", "odd"])
def test_rope(gpu, T, H, D, rot, layout, first, step, factor, how):
    rng = np.random.default_rng(T * 1000 + D)
    x = rows16(rng, T, H, D, size=3.0)
    pos = (first + step * np.arange(T)).astype(np.int32)
    freqs, _ = ops.rope_frequencies(rot, 1e7)
    want, far = po.turned(x, pos, freqs.cpu().numpy(), factor, layout)
    if how == "out":
        got = ops.rope(dev(x), dev(pos), freqs, layout=layout, factor=factor)
    elif how == "in place":
        got = dev(x)
        ops.rope(got, dev(pos), freqs, out=got, layout=layout, factor=factor)
    else:  # heads first, with a gap after each row; `odd` at an odd element
        gap, lead = (8, 0) if how == "strided" else (3, 1)
        wide = torch.zeros(H, T, D + gap, dtype=torch.float16, device="cuda")
        src = wide.transpose(0, 1)[..., lead:D + lead]
        src.copy_(dev(x))
        to = torch.full((T, H, 2 * D + gap), 7.0, dtype=torch.float16, device="cuda")
        got = to[..., lead:D + lead]
        ops.rope(src, dev(pos), freqs, out=got, layout=layout, factor=factor)
        assert (to[..., D + lead:] == 7).all() and (to[..., :lead] == 7).all()
    err = np.abs(got.cpu().numpy().astype(np.float64) - want)
    assert np.all(err <= far), (err - far).max()


def test_rope_refuses(gpu):
    x = torch.zeros(3, 2, 64, dtype=torch.float16, device="cuda")
    f = torch.ones(16, device="cuda")
    good = ints(1, 2, 3)
    for bad in (dict(positions=good.long()), dict(positions=good[:2]), dict(freqs=f.double()),
                dict(freqs=f[None]), dict(x=x.float()), dict(x=x[0]), dict(layout="other"),
                dict(out=torch.zeros(3, 2, 32, dtype=torch.float16, device="cuda")),
                dict(x=x.transpose(1, 2))):
        args = dict(x=x, positions=good, freqs=f) | bad
        args.setdefault("out", torch.zeros_like(args["x"]))
        with pytest.raises(ValueError):
            ops.bind_rope(**args)
    with pytest.raises(_lib.HipError):
        ops.rope(x, good, torch.ones(33, device="cuda"))
    with pytest.raises(_lib.HipError):  # every row of the output the same memory
        ops.rope(x, good, f, out=torch.zeros(1, 1, 64, dtype=torch.float16,
                                             device="cuda").expand(3, 2, 64))
    ops.rope(x[:0], good[:0], f)


# ------------------------------------------------------ the cache of the tests

class Cache:
    """A pool with a table for each sequence, pages in random order."""

    def __init__(self, rng, sequences, capacity, hkv, dim, page, spare=2, fill=None):
        per = -(-capacity // page)
        order = rng.permutation(sequences * per + spare)
        self.table = dev(order[:sequences * per].reshape(sequences, per).astype(np.int32))
        self.pool = ops.paged_pool(order.size, page, hkv, dim)
        if fill is not None:
            self.pool.fill_(fill)

    def append(self, k, v, starts, past, **kwargs):
        ops.paged_append(k, v, self.pool, starts, past, self.table, **kwargs)

    def read(self, lengths):
        """(K, V) of every sequence's first keys."""
        starts = ints(0, *np.cumsum(lengths))
        k, v = ops.paged_read(self.pool, starts, torch.zeros_like(starts[1:]), self.table,
                              int(sum(lengths)))
        cut = lambda t: np.split(t.cpu().numpy(), np.cumsum(lengths)[:-1])
        return cut(k), cut(v)


APPEND = [  # rows of each sequence, past of each, Hkv, dim, page
    ([1], [0], 1, 64, 32),
    ([1], [31], 4, 256, 64),
    ([1, 1, 1, 1], [0, 31, 32, 100], 4, 256, 32),
    ([37], [45], 2, 128, 64),
    ([2, 0, 70, 33], [31, 5, 0, 1], 3, 128, 32),
    ([100, 1, 65], [7, 200, 64], 2, 256, 96),
    ([3, 40], [64, 30], 2, 64, 32),
    ([1] * 70, list(range(70)), 2, 64, 32),
    ([300], [0], 1, 256, 256),
]


@pytest.mark.parametrize("rows, past, hkv, dim, page", APPEND)
@pytest.mark.parametrize("rot, layout", [(0, "half"), (32, "half"), (-1, "interleaved"),
                                         (6, "half"), (-1, "half")])
def test_append_and_read(gpu, rows, past, hkv, dim, page, rot, layout):
    """What is read back is the format's values of the rotated rows, bit for
    bit; what lay before them is kept, and nothing else is written."""
    rng = np.random.default_rng(sum(rows) + dim + rot)
    rot = dim if rot < 0 else rot
    S, T = len(rows), sum(rows)
    cache = Cache(rng, S, max(r + p for r, p in zip(rows, past)), hkv, dim, page, fill=0xA5)
    old_k, old_v = rows16(rng, sum(past), hkv, dim), rows16(rng, sum(past), hkv, dim)
    if sum(past):
        cache.append(dev(old_k), dev(old_v), ints(0, *np.cumsum(past)), ints(*[0] * S))
    before = cache.read(past) if sum(past) else None
    pool = cache.pool.clone()
    k, v = rows16(rng, T + 3, hkv, dim, size=2.0), rows16(rng, T + 3, hkv, dim)
    v[:, :, 32:64] = v[:, :, :1]  # groups of one value: scale 0
    freqs, _ = ops.rope_frequencies(rot, 1e4)
    invalid = ints(0)
    starts, lens = ints(0, *np.cumsum(rows)), ints(*past)
    cache.append(dev(k), dev(v), starts, lens, freqs=freqs if rot else None, layout=layout,
                 factor=1.5, invalid=invalid)
    assert invalid.item() == 0
    pos = np.concatenate([np.arange(p, p + r) for r, p in zip(rows, past)]).astype(np.int32)
    turned = k[:T]
    if rot:
        turned = ops.rope(dev(turned), dev(pos), freqs, layout=layout, factor=1.5).cpu().numpy()
    lengths = [r + p for r, p in zip(rows, past)]
    got = cache.read(lengths)
    at = np.cumsum([0] + rows)
    for s in range(S):
        for x, new, kept_before in ((got[0][s], turned, before and before[0][s]),
                                    (got[1][s], v[:T], before and before[1][s])):
            if past[s]:
                assert np.array_equal(x[:past[s]], kept_before)
            assert np.array_equal(x[past[s]:], po.kept(new[at[s]:at[s + 1]]))
    # the pages' other bytes: a pool whose rows are put back is the pool before
    used = torch.zeros(pool.shape[0], dtype=torch.bool)
    for s in range(S):
        used[cache.table[s, :-(-lengths[s] // page)].long().cpu()] = True
    assert torch.equal(pool[~used], cache.pool[~used])
    # row by row, a part at a time, leaves the same bytes
    if T <= 120:
        parts = Cache(rng, 1, 1, hkv, dim, page)
        parts.table, parts.pool = cache.table, pool
        for i in range(max(rows)):
            one = [j for j in range(S) if i < rows[j]]
            take = np.array([at[j] + i for j in one])
            parts.append(dev(k[take]), dev(v[take]),
                         ints(0, *np.cumsum([int(j in one) for j in range(S)])),
                         ints(*[p + i for p in past]), freqs=freqs if rot else None,
                         layout=layout, factor=1.5)
        assert torch.equal(parts.pool, cache.pool)


def test_append_takes_strided_rows(gpu):
    """Keys and values inside a fused projection's rows, at odd elements too."""
    rng = np.random.default_rng(3)
    T, hkv, dim = 41, 2, 128
    fused = rows16(rng, T, 2 * hkv * dim + 1)
    freqs, _ = ops.rope_frequencies(64, 1e4)
    for lead in (0, 1):
        wide = dev(fused)[:, lead:lead + 2 * hkv * dim].unflatten(1, (2 * hkv, dim))
        k, v = wide[:, :hkv], wide[:, hkv:]
        pools = []
        for a, b in ((k, v), (k.contiguous(), v.contiguous())):
            cache = Cache(np.random.default_rng(0), 1, 60, hkv, dim, 32)
            cache.append(a, b, ints(0, T), ints(11), freqs=freqs)
            pools.append(cache.pool)
        assert torch.equal(*pools)


@pytest.mark.parametrize("value, kept", [(np.nan, 0.0), (np.inf, 16384.0), (-np.inf, -16384.0),
                                         (20000.0, 16384.0), (-65504.0, -16384.0)])
@pytest.mark.parametrize("where", ["k", "v"])
def test_append_flags_values_it_cannot_hold(gpu, value, kept, where):
    rng = np.random.default_rng(4)
    x = {n: rows16(rng, 3, 2, 64) for n in "kv"}
    x[where][1, 1, 40] = value
    cache = Cache(rng, 1, 32, 2, 64, 32)
    invalid = ints(4)  # other bits stay
    cache.append(dev(x["k"]), dev(x["v"]), ints(0, 3), ints(0), invalid=invalid)
    assert invalid.item() == 4 | _lib.PAGED_VALUE
    got = dict(zip("kv", cache.read([3])))
    for n in "kv":
        assert np.isfinite(got[n][0]).all()
        assert np.array_equal(got[n][0], po.kept(x[n]))
    if value == value:  # the group's end, off by its scale's and bias's rounding
        assert abs(got[where][0][1, 1, 40] - kept) <= 3 * po.U16 * 31 * 32768 / 15


def test_rows_with_no_place(gpu):
    """A page outside the pool, a position past the table, a negative one, and
    starts out of order: flagged, never written, NaN where read."""
    rng = np.random.default_rng(5)
    hkv, dim, page, S = 2, 64, 32, 5
    cache = Cache(rng, S, 64, hkv, dim, page, fill=0xA5)
    cache.table[1, 1] = cache.pool.shape[0]
    cache.table[2, 0] = -1
    rows, past = [40, 40, 3, 4, 5], [0, 0, 1, 62, -2]
    T = sum(rows)
    k, v = rows16(rng, T, hkv, dim), rows16(rng, T, hkv, dim)
    starts, lens = ints(0, *np.cumsum(rows)), ints(*past)
    invalid = ints(0)
    before = cache.pool.clone()
    cache.append(dev(k), dev(v), starts, lens, invalid=invalid)
    assert invalid.item() == _lib.PAGED_PLACE
    good = torch.zeros(cache.pool.shape[0], dtype=torch.bool)
    good[[*cache.table[0].tolist(), cache.table[1, 0].item()]] = True
    assert torch.equal(before[~good], cache.pool[~good])
    invalid.zero_()
    gk, gv = (t.cpu().numpy() for t in ops.paged_read(cache.pool, starts, lens, cache.table, T,
                                                       invalid))
    assert invalid.item() == _lib.PAGED_PLACE
    for got, want in ((gk, po.kept(k)), (gv, po.kept(v))):
        assert np.array_equal(got[:72], want[:72])
        assert np.isnan(got[72:]).all()
    # attention: rows that see such a place are NaN, the others are not touched by them
    q = rows16(rng, T, 2 * hkv, dim)
    invalid.zero_()
    out = ops.paged_gqa(dev(q), cache.pool, starts, lens, cache.table, invalid=invalid)
    out = out.cpu().numpy()
    assert invalid.item() == _lib.PAGED_PLACE
    for s, n in ((0, 40), (1, 32)):
        lo = 40 * s
        want, far = po.attention(q[lo:lo + n], gk[lo:lo + n], gv[lo:lo + n], 0, dim ** -0.5)
        assert np.all(np.abs(out[lo:lo + n] - want) <= far)
    assert np.isnan(out[72:]).all()
    # starts that go back, or past the rows: nothing outside is read or written
    # (more of it in test_starts_out_of_order)
    for bad in ([0, 50, 20, 60, 61, 62], [-5, 10, 1000, 3, 2000000000, 2], [92, 92, 92, 92, 92, 92]):
        starts = ints(*bad)
        to = torch.full((T + 8, 2 * hkv, dim), 5.0, dtype=torch.float16, device="cuda")
        ops.paged_gqa(dev(q), cache.pool, starts, lens, cache.table, out=to[:T])
        cache.append(dev(k), dev(v), starts, lens)
        ops.paged_read(cache.pool, starts, lens, cache.table, T)
        assert (to[T:] == 5).all()


@pytest.mark.parametrize("dim, hq, rows", [(64, 4, 2), (128, 4, 2), (256, 8, 2), (128, 8, 40),
                                           (256, 4, 40)])
def test_starts_out_of_order(gpu, dim, hq, rows):
    """Sequences that all claim the same rows, on long histories: more pieces of
    keys than such rows could have; rows of none, and memory behind, stay."""
    rng = np.random.default_rng(6)
    S, T, n = 12, rows, 2000
    cache = Cache(rng, S, n + rows, 1, dim, 64, fill=0)
    q = rows16(rng, T + 4, hq, dim)
    for starts in ([0, rows] * (S // 2) + [0], [rows] + [0] * S, [0] * S + [10 ** 9],
                   [-10 ** 9] + [10 ** 9, 1] * (S // 2)):
        to = torch.full((T + 4, hq, dim), 5.0, dtype=torch.float16, device="cuda")
        k = torch.zeros(T, 1, dim, dtype=torch.float16, device="cuda")
        ops.paged_gqa(dev(q[:T]), cache.pool, ints(*starts), ints(*[n] * S), cache.table, out=to[:T])
        cache.append(k, k, ints(*starts), ints(*[n] * S))
        ops.paged_read(cache.pool, ints(*starts), ints(*[n] * S), cache.table, T)
        torch.cuda.synchronize()
        assert (to[T:] == 5).all()


def test_pages_that_no_row_needs(gpu):
    """Numbers past a sequence's last page may be anything."""
    rng = np.random.default_rng(8)
    for rows, past in (([1, 1], [40, 700]), ([50, 3], [20, 300])):
        cache, kv = filled(rng, rows, past, 2, 128, 32)
        table = cache.table.cpu().numpy()
        for s in range(2):
            table[s, -(-(rows[s] + past[s]) // 32):] = (-1, 2 ** 31 - 1)[s]
        cache.table = dev(table)
        q = rows16(rng, sum(rows), 8, 128)
        invalid = ints(0)
        starts, lens = ints(0, *np.cumsum(rows)), ints(*past)
        out = ops.paged_gqa(dev(q), cache.pool, starts, lens, cache.table, invalid=invalid)
        check(out.cpu().numpy(), q, kv, rows, past, 128 ** -0.5)
        k = rows16(rng, sum(rows), 2, 128)
        cache.append(dev(k), dev(k), starts, lens, invalid=invalid)
        ops.paged_read(cache.pool, starts, lens, cache.table, sum(rows), invalid)
        assert invalid.item() == 0


@pytest.mark.parametrize("rows, past, dim", [(1, 3000, 256), (1, 90, 64), (40, 2000, 256),
                                             (40, 900, 128), (12, 700, 64)])
def test_a_page_outside_the_pool_in_the_middle(gpu, rows, past, dim):
    """Only the rows that see it are NaN, whichever workgroup meets it."""
    rng = np.random.default_rng(9)
    both = [rows, rows]
    cache, kv = filled(rng, both, [past, past], 1, dim, 32)
    at = 2 if past < 100 else 20
    cache.table[0, at] = cache.pool.shape[0] + 5
    q = rows16(rng, 2 * rows, 4, dim)
    invalid = ints(0)
    out = ops.paged_gqa(dev(q), cache.pool, ints(0, rows, 2 * rows), ints(past, past), cache.table,
                        invalid=invalid).cpu().numpy()
    assert invalid.item() == _lib.PAGED_PLACE
    assert np.isnan(out[:rows]).all()
    check(out[rows:], q[rows:], [x[1:] for x in kv], [rows], [past], dim ** -0.5)


# ------------------------------------------------------------------ attention

GQA = [  # rows of each sequence, past of each, Hq, Hkv, dim, page
    ([1], [0], 1, 1, 64, 32),
    ([1], [0], 16, 4, 256, 64),
    ([1], [31], 16, 4, 256, 64),
    ([1], [1000], 16, 4, 256, 32),
    ([1], [5003], 4, 1, 128, 128),
    ([1, 1, 1], [700, 0, 33], 10, 2, 64, 32),
    ([1] * 67, [(37 * s) % 150 for s in range(67)], 4, 2, 128, 32),
    ([1] * 9, [4000, 1, 63, 64, 65, 300, 2, 31, 900], 16, 2, 256, 96),
    ([2], [515], 16, 4, 256, 32),
    ([5, 0, 3], [90, 7, 0], 14, 2, 128, 64),
    ([4, 1], [1029, 31], 32, 1, 128, 32),
    ([17], [0], 16, 4, 256, 64),
    ([33], [47], 8, 8, 64, 32),
    ([61], [611], 16, 4, 256, 128),
    ([130], [0], 4, 4, 128, 32),
    ([129, 40, 1], [31, 0, 500], 16, 4, 256, 32),
    ([70, 33], [5, 260], 6, 2, 64, 64),
    ([50], [2], 16, 1, 256, 32),
    ([150], [100], 8, 1, 128, 32),
    ([1, 1], [9000, 4000], 2, 2, 64, 256),              # eight waves, many pieces
    ([1] * 40, [(411 * s) % 3000 for s in range(40)], 4, 4, 128, 64),  # four waves
    ([6, 2], [2100, 3333], 8, 2, 256, 64),              # two column groups, divided
    ([12], [4100], 4, 1, 128, 32),                      # four
    ([9, 20, 1], [1500, 0, 900], 12, 3, 64, 128),
    ([40], [5000], 4, 1, 256, 64),                      # tiles, divided
    ([70], [2500], 4, 1, 128, 96),
    ([40, 90, 3], [700, 64, 1500], 8, 2, 256, 32),      # tiles, longest first
    ([64], [64], 2, 1, 256, 32),                        # whole units and blocks
    ([33, 65], [31, 63], 4, 1, 128, 32),
    ([1], [2000], 3, 1, 64, 32),                        # a token's heads: 1 to 4,
    ([2], [1500], 4, 2, 128, 32),
    ([1], [40], 7, 1, 64, 32),                          # 5 to 8,
    ([1, 1], [900, 33], 14, 2, 256, 32),
    ([1], [3000], 8, 1, 128, 64),
    ([1], [2500], 8, 1, 64, 64),
    ([1], [70], 9, 1, 128, 32),                         # 9 to 16
    ([100], [2500], 4, 1, 128, 96),                     # tiles, divided
    ([300, 200, 3], [700, 64, 1500], 8, 2, 128, 32),    # longest first
    ([16] * 10, [(97 * s) % 500 for s in range(10)], 16, 4, 256, 32),  # many columns
    ([41], [3000], 4, 1, 128, 32),                      # six units on one round
    ([25], [2000], 4, 1, 64, 64),                       # 64 columns
    ([9], [3900], 4, 1, 256, 64),                       # 33 to 48
]


def filled(rng, rows, past, hkv, dim, page, size=1.0, fill=0xFF):
    """A cache whose sequences hold past + rows keys; a pool of NaN elsewhere."""
    lengths = [r + p for r, p in zip(rows, past)]
    cache = Cache(rng, len(rows), max(lengths), hkv, dim, page, fill=fill)
    k, v = (rows16(rng, sum(lengths), hkv, dim, size=size) for _ in range(2))
    cache.append(dev(k), dev(v), ints(0, *np.cumsum(lengths)), ints(*[0] * len(rows)))
    return cache, cache.read(lengths)


def check(out, q, kv, rows, past, scale):
    at = 0
    for s, (r, p) in enumerate(zip(rows, past)):
        if r:
            want, far = po.attention(q[at:at + r], kv[0][s], kv[1][s], p, scale)
            err = np.abs(out[at:at + r].astype(np.float64) - want)
            assert np.all(err <= far), (s, (err / far).max())
        at += r


@pytest.mark.parametrize("rows, past, hq, hkv, dim, page", GQA)
def test_paged_gqa(gpu, rows, past, hq, hkv, dim, page):
    rng = np.random.default_rng(sum(rows) + sum(past) + dim)
    cache, kv = filled(rng, rows, past, hkv, dim, page)
    T = sum(rows)
    q = rows16(rng, T + 5, hq, dim, size=1.5)
    out = torch.full((T + 5, hq, dim), 9.0, dtype=torch.float16, device="cuda")
    starts, lens, invalid = ints(0, *np.cumsum(rows)), ints(*past), ints(0)
    ops.paged_gqa(dev(q), cache.pool, starts, lens, cache.table, out=out, invalid=invalid)
    assert invalid.item() == 0
    out = out.cpu().numpy()
    assert (out[T:] == 9).all()  # rows behind the last sequence
    check(out, q, kv, rows, past, dim ** -0.5)


@pytest.mark.parametrize("rows, past", [([1], [777]), ([40], [100]), ([3], [0])])
@pytest.mark.parametrize("scale, size", [(0.5, 4.0), (0.0, 1.0), (-0.2, 1.0), (1e-3, 1000.0)])
def test_paged_gqa_scales(gpu, rows, past, scale, size):
    """Steep softmaxes, equal weights, other signs."""
    rng = np.random.default_rng(11)
    cache, kv = filled(rng, rows, past, 2, 128, 64, size=size)
    q = rows16(rng, sum(rows), 8, 128, size=2.0)
    out = ops.paged_gqa(dev(q), cache.pool, ints(0, *np.cumsum(rows)), ints(*past), cache.table,
                        scale=scale)
    check(out.cpu().numpy(), q, kv, rows, past, scale)


@pytest.mark.parametrize("rows, past", [([1], [2000]), ([90], [300])])
def test_scores_that_keep_rising(gpu, rows, past):
    """Each key's score above all before it, by up to 2^10 in all: the running
    maximum moves in every tile; and falling ones: it never moves again."""
    rng = np.random.default_rng(12)
    n, dim = sum(rows) + sum(past), 64
    for ramp in (np.linspace(0, 1, n), np.linspace(1, 0, n)):
        cache = Cache(rng, 1, n, 1, dim, 32, fill=0xFF)
        k = np.zeros((n, 1, dim), np.float16)
        k[:, 0, :] = (64 * ramp)[:, None].astype(np.float16)
        v = rows16(rng, n, 1, dim)
        cache.append(dev(k), dev(v), ints(0, n), ints(0))
        kv = cache.read([n])
        q = np.full((sum(rows), 4, dim), 0.25, np.float16)
        out = ops.paged_gqa(dev(q), cache.pool, ints(0, sum(rows)), ints(*past), cache.table,
                            scale=1.0)
        check(out.cpu().numpy(), q, kv, rows, past, 1.0)


def test_rows_after_a_value_that_was_not_finite(gpu):
    """A later row's NaN and infinities do not reach the rows before it."""
    rng = np.random.default_rng(13)
    n, dim = 50, 128
    k, v = rows16(rng, n, 2, dim), rows16(rng, n, 2, dim)
    k[30, 0, 5], v[30, 1, 7], v[31, 0, 9] = np.nan, np.inf, np.nan
    cache = Cache(rng, 1, n, 2, dim, 32, fill=0xFF)
    cache.append(dev(k), dev(v), ints(0, n), ints(0))
    q = rows16(rng, n, 4, dim)
    out = ops.paged_gqa(dev(q), cache.pool, ints(0, n), ints(0), cache.table).cpu().numpy()
    check(out, q, cache.read([n]), [n], [0], dim ** -0.5)


def test_a_pool_past_4_gib(gpu):
    """Pages whose bytes lie past 2^32."""
    rng = np.random.default_rng(14)
    hkv, dim, page, n = 4, 256, 256, 300
    page_bytes = hkv * page * dim * 5 // 4
    pages = 2 ** 32 // page_bytes + 3
    pool = torch.empty(pages, hkv, page // 32, 40 * dim, dtype=torch.uint8, device="cuda")
    table = ints(pages - 1, pages - 2)[None]
    k, v = rows16(rng, n, hkv, dim), rows16(rng, n, hkv, dim)
    ops.paged_append(dev(k), dev(v), pool, ints(0, n), ints(0), table)
    gk, gv = ops.paged_read(pool, ints(0, n), ints(0), table, n)
    assert np.array_equal(gk.cpu().numpy(), po.kept(k))
    assert np.array_equal(gv.cpu().numpy(), po.kept(v))
    for rows in (1, 40):
        q = rows16(rng, rows, 16, dim)
        out = ops.paged_gqa(dev(q), pool, ints(0, rows), ints(n - rows), table)
        check(out.cpu().numpy(), q, ([gk.cpu().numpy()], [gv.cpu().numpy()]), [rows], [n - rows],
              dim ** -0.5)


def test_paged_refusals(gpu):
    cache = Cache(np.random.default_rng(0), 2, 64, 2, 64, 32)
    x = torch.zeros(3, 2, 64, dtype=torch.float16, device="cuda")
    starts, past = ints(0, 1, 3), ints(0, 0)
    good = dict(pool=cache.pool, starts=starts, past=past, table=cache.table)
    for bad in (dict(starts=starts[:2]), dict(past=past.long()), dict(table=cache.table[:1]),
                dict(table=cache.table[0]), dict(pool=cache.pool[0]), dict(pool=cache.pool[..., :64]),
                dict(pool=cache.pool.half()), dict(invalid=starts)):
        with pytest.raises(ValueError):
            ops.bind_paged_append(x, x, **(good | bad))
        with pytest.raises(ValueError):
            ops.bind_paged_read(k=x, v=x, **(good | bad))
        with pytest.raises(ValueError):
            ops.bind_paged_gqa(x, out=torch.empty_like(x), **(good | bad))
    with pytest.raises(ValueError):
        ops.bind_paged_append(x[:, :1], x[:, :1], **good)
    with pytest.raises(ValueError):
        ops.bind_paged_append(x, x[:2], **good)
    with pytest.raises(ValueError):
        ops.bind_paged_append(x, x, **good, layout="other")
    with pytest.raises(ValueError):
        ops.bind_paged_read(k=x[:, :1].contiguous(), v=x[:, :1].contiguous(), **good)
    with pytest.raises(ValueError):
        ops.bind_paged_gqa(x[:, :1].contiguous(), out=x[:, :1].contiguous(), **good)
    with pytest.raises(_lib.HipError):
        ops.paged_append(x, x, **good, freqs=torch.ones(40, device="cuda"))
    with pytest.raises(_lib.HipError):
        ops.paged_gqa(torch.zeros(3 * 128 + 4, dtype=torch.float16, device="cuda")[4:388].view(3, 2, 64),
                      **good)


# ------------------------------------------------------------- a run together

def test_a_conversation(gpu):
    """Prompts, then tokens, for three sequences: rope, append and attention as
    a layer calls them, against the same rows in numpy, each step."""
    rng = np.random.default_rng(21)
    hq, hkv, dim, page, rot = 8, 2, 128, 32, 64
    cache = Cache(rng, 3, 200, hkv, dim, page, fill=0xFF)
    freqs, factor = ops.rope_frequencies(rot, 1e5, "yarn", 4.0, 64.0)
    held = [[np.zeros((0, hkv, dim), np.float16)] * 2 for _ in range(3)]
    past = [0, 0, 0]
    for rows in ([70, 3, 0], [1, 1, 40], [1, 1, 1], [0, 17, 1], [1, 1, 1]):
        T = sum(rows)
        q, k, v = rows16(rng, T, hq, dim), rows16(rng, T, hkv, dim), rows16(rng, T, hkv, dim)
        pos = dev(np.concatenate([np.arange(p, p + r) for r, p in zip(rows, past)]).astype(np.int32))
        starts, lens = ints(0, *np.cumsum(rows)), ints(*past)
        turned = ops.rope(dev(q), pos, freqs, factor=factor)
        cache.append(dev(k), dev(v), starts, lens, freqs=freqs, factor=factor)
        out = ops.paged_gqa(turned, cache.pool, starts, lens, cache.table).cpu().numpy()
        want_q, far = po.turned(q, pos.cpu().numpy(), freqs.cpu().numpy(), factor, "half")
        turned = turned.cpu().numpy()
        assert np.all(np.abs(turned - want_q) <= far)
        turned_k = ops.rope(dev(k), pos, freqs, factor=factor).cpu().numpy()
        at = np.cumsum([0] + rows)
        for s in range(3):
            part = slice(at[s], at[s + 1])
            held[s] = [np.concatenate((a, po.kept(b[part]))) for a, b in zip(held[s], (turned_k, v))]
        check(out, turned, ([h[0] for h in held], [h[1] for h in held]), rows, past, dim ** -0.5)
        past = [p + r for p, r in zip(past, rows)]


def test_captured_on_new_lengths(gpu):
    """rope, append and attention in one graph, replayed while the lengths in
    device memory grow: every replay gives the eager calls' bits."""
    rng = np.random.default_rng(22)
    S, hq, hkv, dim, page = 3, 8, 2, 128, 32
    caches = [Cache(np.random.default_rng(1), S, 400, hkv, dim, page, fill=0xFF) for _ in range(2)]
    freqs, _ = ops.rope_frequencies(64, 1e5)
    q = torch.zeros(S, hq, dim, dtype=torch.float16, device="cuda")
    k, v = (torch.zeros(S, hkv, dim, dtype=torch.float16, device="cuda") for _ in range(2))
    starts, past = ints(0, 1, 2, 3), ints(0, 0, 0)
    turned, out = torch.empty_like(q), torch.empty_like(q)

    def step(cache, turned, out):
        ops.rope(q, past, freqs, out=turned)
        cache.append(k, v, starts, past, freqs=freqs)
        ops.paged_gqa(turned, cache.pool, starts, past, cache.table, out=out)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step(caches[0], turned, out)  # loads the kernels
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step(caches[0], turned, out)
    lengths = np.array([0, 5, 130])
    for c in caches:
        lead = rows16(np.random.default_rng(2), 135, hkv, dim)
        c.append(dev(lead), dev(lead), ints(0, 0, 5, 135), ints(0, 0, 0))
    for i in range(6):
        past.copy_(dev((lengths + 37 * i).astype(np.int32)))
        for t in (q, k, v):
            t.copy_(dev(rows16(rng, *t.shape)))
        if i:  # keys that the lengths skipped
            gap = rows16(rng, 3 * 36, hkv, dim)
            for c in caches:
                c.append(dev(gap), dev(gap), ints(0, 36, 72, 108), past - 36)
        torch.cuda.synchronize()
        graph.replay()
        a, b = torch.empty_like(q), torch.empty_like(q)
        step(caches[1], a, b)
        torch.cuda.synchronize()
        assert torch.equal(turned, a) and torch.equal(out, b) and not b.isnan().any()
        assert torch.equal(caches[0].pool, caches[1].pool)


def test_two_graphs_at_once(gpu):
    """Graphs captured on one stream and replayed on two at the same time: each
    has a workspace of its own."""
    rng = np.random.default_rng(24)
    made, alone, graphs = [], [], []
    side = torch.cuda.Stream()
    for n in (5000, 3500):
        cache, _ = filled(rng, [1], [n], 4, 128, 64)
        call = (dev(rows16(rng, 1, 16, 128)), cache, ints(0, 1), ints(n))
        q, c, s, p = call
        alone.append(ops.paged_gqa(q, c.pool, s, p, c.table))
        out = torch.zeros_like(q)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            ops.paged_gqa(q, c.pool, s, p, c.table, out=out)
        made.append((call, out))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(5):
        for _, out in made:
            out.zero_()
        torch.cuda.synchronize()
        for _ in range(8):
            for graph, stream in zip(graphs, streams):
                with torch.cuda.stream(stream):
                    graph.replay()
        torch.cuda.synchronize()
        for (_, out), want in zip(made, alone):
            assert torch.equal(out, want)


def test_bound_calls_in_two_graphs(gpu):
    """Calls bound one after the other on one stream, then captured each into a
    graph: replayed at the same time they do not meet."""
    rng = np.random.default_rng(25)
    side = torch.cuda.Stream()
    made, alone = [], []
    for n in (4100, 2700):
        cache, _ = filled(rng, [1], [n], 4, 128, 64)
        q, starts, past = dev(rows16(rng, 1, 16, 128)), ints(0, 1), ints(n)
        alone.append(ops.paged_gqa(q, cache.pool, starts, past, cache.table))
        out = torch.zeros_like(q)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            made.append((ops.bind_paged_gqa(q, cache.pool, starts, past, cache.table, out), out))
    graphs = []
    for bound, _ in made:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=side):
            bound()
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(5):
        for _, out in made:
            out.zero_()
        torch.cuda.synchronize()
        for _ in range(8):
            for graph, stream in zip(graphs, streams):
                with torch.cuda.stream(stream):
                    graph.replay()
        torch.cuda.synchronize()
        for (_, out), want in zip(made, alone):
            assert torch.equal(out, want)


def test_two_streams_at_once(gpu):
    """Two streams' calls, with a workspace each, give what one after the other gives."""
    rng = np.random.default_rng(23)
    made = []
    for n in (4000, 2500):
        cache, _ = filled(rng, [1], [n], 4, 128, 64)
        made.append((dev(rows16(rng, 1, 16, 128)), cache, ints(0, 1), ints(n)))
    alone = [ops.paged_gqa(q, c.pool, s, p, c.table) for q, c, s, p in made]
    streams = [torch.cuda.Stream() for _ in made]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(20):
        for k, (q, c, s, p) in enumerate(made):
            with torch.cuda.stream(streams[k]):
                outs[k].append(ops.paged_gqa(q, c.pool, s, p, c.table))
    torch.cuda.synchronize()
    for k in range(2):
        for o in outs[k]:
            assert torch.equal(o, alone[k])
