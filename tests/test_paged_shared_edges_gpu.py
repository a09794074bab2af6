"""GPU tests of the attention behind a common prefix where its ways of dividing
the work meet their limits. Against paged_oracle, whose tolerances are counted
there."""
import numpy as np
import pytest
import torch

from llminfer_amd import _lib, ops
from tests import paged_oracle as po
from tests.test_paged_shared_gpu import Group, dev, ints, rows16

pytestmark = pytest.mark.gpu

TILES = "pagedGqaTiles+pagedGqaTiles+pagedSharedMerge"


def called(g, q, out=None, scale=None, invalid=None):
    """The call's kernels and its output."""
    q = dev(q)
    out = torch.empty_like(q) if out is None else out
    b = ops.bind_paged_gqa_shared(q, g.pool, g.starts, g.past, g.table, g.groups, g.prefix, out,
                                  scale, invalid)
    b()
    return b.what, out.cpu().numpy()


# ------------------------------------- tiles of shared keys, tiles of own keys

OWN_TILES = [  # groups, heads a KV head, hkv, dim, page, the sequences that are checked
    # 160 columns a sequence and more, some without a row, prefixes cut in a page and a block
    ([(128, [(40 + 5 * i, 128 + 31 * i % 90) for i in range(6)] + [(0, 200), (64, 129)]),
      (90, [(61, 700), (0, 90), (44, 90)])], 4, 1, 256, 32, None),
    # 48 in calls of many columns
    ([(96, [(13, 100 + 40 * i) for i in range(16)] + [(30, 96)] * 2)], 4, 4, 256, 64,
     [0, 1, 7, 15, 16, 17]),
    # 384 and more at head_dim 128, beside sequences of no group
    ([(160, [(100 + 7 * i, 160 + 40 * i) for i in range(4)] + [(0, 170)]), (0, [(120, 50)]),
      (64, [(130, 64), (101, 400)])], 4, 1, 128, 32, None),
    # keys that are divided: few sequences on long pasts
    ([(3000, [(45, 3000), (60, 3700)])], 4, 1, 256, 128, None),
    ([(2016, [(100, 2016), (110, 3500)])], 4, 1, 128, 32, None),
    # more than 64 sequences, and than 256
    ([(64, [(60, 64 + i % 40) for i in range(69)])], 4, 1, 256, 32, [0, 1, 63, 64, 68]),
    ([(64, [(50 + i % 9, 70 + i % 40) for i in range(40)]), (32, [(52, 40 + i) for i in range(40)])],
     8, 1, 128, 32, [0, 39, 40, 63, 64, 79]),
    ([(64, [(41, 64 + i % 40) for i in range(270)])], 4, 1, 256, 32, [0, 64, 255, 256, 269]),
    # and more than 64 groups
    ([(32 * (1 + i % 3), [(42, 96 + i)] * (1 + i % 2)) for i in range(66)], 4, 1, 256, 32,
     [0, 1, 2, 63, 64, 97, 98]),
]


@pytest.mark.parametrize("groups, per, hkv, dim, page, some", OWN_TILES)
@pytest.mark.parametrize("scale", [None, -0.3])
def test_own_keys_in_tiles(gpu, groups, per, hkv, dim, page, some, scale):
    rng = np.random.default_rng(len(groups) * 100 + dim)
    g = Group(rng, groups, hkv, dim, page)
    q = rows16(rng, sum(g.rows), per * hkv, dim)
    word = ints([0])
    what, got = called(g, q, scale=scale, invalid=word)
    assert what == TILES and word.item() == 0 and not np.isnan(got).any()
    g.check(got, q, 1 / np.sqrt(np.float32(dim)) if scale is None else scale,
            set(range(len(g.rows))) - set(some) if some else ())


@pytest.mark.parametrize("members", [5, 66])
@pytest.mark.parametrize("per, dim, rows", [(4, 256, 48), (4, 128, 100)])
def test_own_tiles_without_place(gpu, members, per, dim, rows):
    """A missing page of a sequence's own: NaN in the rows that see it. A missing
    shared one, or a past that does not fit: NaN as a whole. The others are as they
    would be. Page 0, whose bytes the kernels may have in a missing one's place,
    holds NaN."""
    page, prefix = 32, 64
    plain = [(rows, prefix + 9 + i % 7) for i in range(members)]

    def fresh():
        g = Group(np.random.default_rng(8), [(prefix, plain), (32, [(rows, 40)])], 1, dim, page)
        table = g.table.cpu().numpy()
        spare = np.setdiff1d(np.arange(g.pool.shape[0]), table)
        if (table == 0).any():
            spare = int(spare[0])
            g.pool[spare] = g.pool[0].clone()
            table[table == 0] = spare
            g.table = dev(table)
        g.pool[0] = 0xFF
        return g

    q = rows16(np.random.default_rng(members), rows * (members + 1), per, dim)
    at = lambda s: slice(rows * s, rows * (s + 1))
    some = {0, 1, 2, members - 1, members}

    def expect(g, lost):
        """lost: {sequence: its first NaN row}"""
        word = ints([0])
        what, got = called(g, q, invalid=word)
        assert what == TILES and word.item() == 2
        for s in range(members + 1):
            first = lost.get(s, rows)
            assert np.isnan(got[at(s)][first:]).all() and not np.isnan(got[at(s)][:first]).any(), s
            if s in some and first:
                p = g.seqs[s][1]
                want, far = po.attention(q[at(s)][:first], *g.cached(s, p + first), p,
                                         1 / np.sqrt(np.float32(dim)))
                assert np.all(np.abs(got[at(s)][:first].astype(np.float64) - want) <= far), s

    g = fresh()
    g.table[1, 3] = -1  # keys 96 .. 127; the first row is at 74
    expect(g, {1: 96 - 74})
    g = fresh()
    g.table[members, 2] = g.pool.shape[0]  # of the second group: keys 64 .. 95 behind 40
    expect(g, {members: 24})
    g = fresh()
    g.table[0, 1] = 10**6  # shared, but for the first sequence's own keys behind it
    expect(g, {s: 0 for s in range(members)})
    g = fresh()
    g.past[2], g.past[members - 1] = prefix - 1, g.table.shape[1] * page
    expect(g, {2: 0, members - 1: 0})
