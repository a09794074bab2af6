"""GPU tests of the attention behind a common prefix where its ways of dividing
the work meet their limits. Against paged_oracle, whose tolerances are counted
there."""
import numpy as np
import pytest
import torch

from llminfer_amd import _lib, ops
from tests import paged_oracle as po
from tests.test_paged_shared_gpu import Group, dev, free_oracle, ints, rows16

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


# ----------------------------- pieces that take their blocks' places by turns

class Pages:
    """Sequences behind one prefix in a pool of any bytes with finite scales: what
    it holds is what ops.paged_read says."""

    def __init__(self, seed, prefix, seqs, hkv, dim, page, places=0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        common = prefix // page
        owned = [-(-(r + p) // page) - common for r, p in seqs]
        width = max(common + max(owned), places // page)
        order = 1 + torch.randperm(common + sum(owned), generator=g, device="cuda").int()
        pages = order.numel() + 1  # (page 0 is none of the sequences')
        self.pool = torch.randint(0, 256, (pages, hkv, page // 32, 40 * dim), generator=g,
                                  dtype=torch.uint8, device="cuda")
        for at in (16 * dim, 36 * dim):
            scale = 0.05 * torch.randn(pages, hkv, page // 32, 2 * dim, generator=g, device="cuda")
            self.pool[..., at:at + 4 * dim] = scale.half().view(torch.uint8)
        self.table = torch.full((len(seqs), width), -1, dtype=torch.int32, device="cuda")
        self.table[:, :common] = order[:common]
        at = common
        for s, n in enumerate(owned):
            self.table[s, common:common + n] = order[at:at + n]
            at += n
        self.seqs, self.rows = seqs, [r for r, _ in seqs]
        self.starts, self.past = ints(np.cumsum([0] + self.rows)), ints(p for _, p in seqs)
        self.groups, self.prefix = ints([0, len(seqs)]), ints([prefix])

    def check(self, got, q, s, heads):
        """Rows of sequence s, some query heads."""
        at, (r, p) = sum(self.rows[:s]), self.seqs[s]
        k, v = ops.paged_read(self.pool, ints([0, r + p]), ints([0]), self.table[s:s + 1].contiguous(),
                              r + p)
        per = q.shape[1] // k.shape[1]
        for h in heads:
            kv = (x[:, h // per:h // per + 1].cpu().numpy() for x in (k, v))
            want, far = po.attention(q[at:at + r, h:h + 1], *kv, p, 1 / np.sqrt(np.float32(q.shape[2])))
            assert np.all(np.abs(got[at:at + r, h:h + 1].astype(np.float64) - want) <= far), (s, h)


# With 128 KV heads two workgroups have one: the first all shared keys, a unit of 48
# columns, the second's eight waves the own keys, equal runs of them. Places are
# looked up for 64 steps of 512 / dim shared blocks, and for 64 own blocks, at once.
LONG = [  # dim, page, prefix, own keys of the long sequences, how many of 48 they are
    (64, 128, 17408, 3000, 6),   # 544 shared blocks, 68 steps; 594 own, runs of 75
    (128, 64, 9216, 40, 1),      # 288 shared blocks, 72 steps
    (128, 32, 4096, 3001, 6),
    (256, 128, 5120, 2990, 6),   # 160 shared blocks, 80 steps
]


@pytest.mark.parametrize("dim, page, prefix, rest, many", LONG)
def test_long_runs(gpu, dim, page, prefix, rest, many):
    """Runs that look their blocks' places up more than once, and a page that is
    missing behind the first time."""
    hkv, S = 128, 48
    # (the others' columns make one unit; the long ones lie first, so that runs part them)
    seqs = [(1, prefix + rest - 3 * i) for i in range(many)]
    seqs += [(1, prefix + i % 20) for i in range(S - many)]

    def fresh():
        return Pages(dim, prefix, seqs, hkv, dim, page, 16384)

    q = rows16(np.random.default_rng(dim), S, hkv, dim)
    g = fresh()
    word = ints([0])
    what, got = called(g, q, invalid=word)
    assert what == "pagedGqaMixed+pagedSharedMerge" and word.item() == 0 and not np.isnan(got).any()
    for s in (0, many - 1, many, S - 1):
        g.check(got, q, s, (0, 77, 127))
    assert np.array_equal(called(g, q)[1], got)
    # own block 70, of a run from block 0 on, and the last page of another sequence
    for s, key in ((0, min(70 * 32, rest)), (many - 1, rest - 3 * (many - 1))):
        g = fresh()
        g.pool[0] = 0xFF
        g.table[s, (prefix + key) // page] = -1
        word.zero_()
        lost = called(g, q, invalid=word)[1]
        assert word.item() == 2 and np.isnan(lost[s]).all()
        others = np.arange(S) != s
        assert np.array_equal(lost[others], got[others])
    g = fresh()
    g.pool[0] = 0xFF
    g.table[0, (prefix - 32) // page] = g.pool.shape[0]  # the last shared one
    word.zero_()
    assert np.isnan(called(g, q, invalid=word)[1]).all() and word.item() == 2


# -------------------------------------------------- starts and groups in disorder

def claimed(starts, tokens):
    """Rows that a sequence has, of starts in any order."""
    rows = np.zeros(tokens, bool)
    for a, b in zip(starts, starts[1:]):
        lo = min(max(a, 0), tokens)
        rows[lo:min(max(b, lo), tokens)] = True
    return rows


@pytest.mark.parametrize("n, rows, dim, places, what", [
    (20, 2, 256, 0, "pagedGqaSplit+pagedSharedMerge"),
    (100, 2, 256, 0, "pagedGqaSplit+pagedSharedMerge"),
    (30, 2, 256, 16384, "pagedGqaMixed+pagedSharedMerge"),
    (100, 2, 256, 16384, "pagedGqaMixed+pagedSharedMerge"),
    (100, 2, 64, 16384, "pagedGqaMixed+pagedSharedMerge"),
    (9, 48, 256, 0, TILES),
    (70, 48, 256, 0, TILES),
])
def test_disorder_stays_in_its_rows(gpu, n, rows, dim, places, what):
    """Starts and groups out of order, overlapping or out of range change no row
    that no sequence has, and nothing behind the output or a workspace of exactly
    the size that is asked for, whatever it held. In order again, the result is what
    it was."""
    rng = np.random.default_rng(n)
    g = Group(rng, [(64, [(rows, 64 + i) for i in range(n)])], 1, dim, 32)
    g.table = torch.nn.functional.pad(g.table, (0, max(places // 32 - g.table.shape[1], 0)), value=-1)
    T = rows * n + 4
    q = dev(rows16(rng, T, 4, dim))
    lib, guard = _lib.load(), 4096
    around = torch.empty(q.numel() + 2 * guard, dtype=torch.float16, device="cuda")
    out = around[guard:-guard].view(q.shape)
    assert out.data_ptr() % 16 == 0
    kv = _lib.PagedKvParams(g.pool.shape[0], 32, 1, dim, n, g.table.shape[1], T)
    stream = torch.cuda.current_stream().cuda_stream
    ordered = [rows * i for i in range(n + 1)]

    def call(starts, groups, prefix, fill):
        p = _lib.PagedSharedParams(_lib.PagedGqaParams(kv, 4, 0.1), len(prefix))
        need = lib.llmi_hip_paged_gqa_shared_workspace_bytes(p)
        ws = torch.full((need + 2 * guard,), fill, dtype=torch.uint8, device="cuda")
        ws[:guard] = ws[-guard:] = 99
        around.fill_(7)
        arrays = [ints(x) for x in (starts, groups, prefix)]
        _lib.check(lib.llmi_hip_paged_gqa_shared(
            q.data_ptr(), arrays[0].data_ptr(), g.past.data_ptr(), g.table.data_ptr(),
            arrays[1].data_ptr(), arrays[2].data_ptr(), g.pool.data_ptr(), out.data_ptr(), None, p,
            ws.data_ptr() + guard, need, stream))
        torch.cuda.synchronize()
        assert (ws[:guard] == 99).all() and (ws[-guard:] == 99).all()
        assert (around[:guard] == 7).all() and (around[-guard:] == 7).all()
        left = dev(~claimed(starts, T))
        assert (out[left] == 7).all(), (starts[:9], groups, prefix)
        return p, out.clone()

    p, want = call(ordered, [0, n], [64], 0)
    assert "+".join(ops.kernel_names(_lib.OP_PAGED_GQA_SHARED, p)) == what
    assert not (want[:rows * n] == 7).all(-1).any()
    disorders = [ordered, [0, 20 * rows, 3, 10 * rows, 9] + [15 * rows] * (n - 4),
                 list(range(T, T + n + 1)), list(range(n, -1, -1)),
                 [-5] * (n // 2) + [rows * n + 2] * (n + 1 - n // 2),
                 [2**31 - 1] * 2 + [-2**31] * (n - 2) + [T + 9]]
    for starts in disorders:
        for groups, prefix in (([0, n], [64]), ([5, 2], [64]), ([0, n, 0, n, 0, n], [64] * 5),
                               ([-9, 6 * n], [64]), ([n + 10, n + 20], [64]), ([0] * 71, [32] * 70),
                               ([2**31 - 1, -2**31], [2**31 - 1])):
            for fill in (0xFF, 0x01):
                call(starts, groups, prefix, fill)
    assert torch.equal(call(ordered, [0, n], [64], 0xFF)[1], want)


# ------------------------------------------------------------------ free pages

@pytest.mark.parametrize("sequences, width, launches", [
    (96, 256, 1), (97, 256, 3), (48, 513, 1), (49, 513, 3), (96, 1, 1), (97, 1, 3),
    (12, 4096, 1), (12, 4097, 3), (1000, 32, 3), (2100, 7, 3), (2, 20_000, 1),
])
@pytest.mark.parametrize("pages", [33, 8192])
def test_free_by_pieces(gpu, sequences, width, launches, pages):
    """One workgroup for up to 96 pieces of 512 slots of rows, short rows a piece
    each; up to 32 workgroups that mark."""
    rng = np.random.default_rng(width + sequences)
    p = _lib.PagedFreeParams(pages, 32, sequences, width)
    assert len(ops.kernel_names(_lib.OP_PAGED_FREE, p)) == launches
    for most in (width, 3):
        table = rng.integers(0, pages, (sequences, width), dtype=np.int32)
        lengths = rng.integers(0, min(width, most) * 32 + 1, sequences)
        lengths[rng.random(sequences) < 0.6] = 0
        want, count, bad = free_oracle(table, lengths, 32, pages)
        word = ints([0])
        free, n = ops.paged_free(dev(table), ints(lengths), 32, pages, word)
        assert not bad and word.item() == 0 and n.item() == count
        assert np.array_equal(free.cpu().numpy(), want)


# ------------------------------------------- groups and sequences by the hundred

MANY = [  # groups, sequences of each, heads a KV head, hkv, dim, page, launches of how
    (250, 4, 4, 4, 64, 32, "pagedGqaMixed"),
    (130, 5, 4, 8, 128, 32, "pagedGqaMixed"),
    (66, 9, 2, 4, 256, 64, "pagedGqaMixed"),
    (6, 60, 4, 4, 256, 32, "pagedGqaMixed"),
    (130, 2, 4, 2, 64, 32, "pagedGqaSplit"),
    (40, 3, 4, 4, 128, 32, "pagedGqaSplit"),
]


@pytest.mark.parametrize("groups, members, per, hkv, dim, page, how", MANY)
def test_many_groups(gpu, groups, members, per, hkv, dim, page, how):
    """Where the plan of every workgroup, which looks at all groups and sequences,
    is most of the work, the launch with few workgroups is taken."""
    rng = np.random.default_rng(groups + dim)
    each = [(64 + 32 * (i % 3), [(1, 130 + (7 * i + j) % 60) for j in range(members)])
            for i in range(groups)]
    each[groups // 2] = (96, [(0, 99), (2, 96)])
    g = Group(rng, each, hkv, dim, page)
    q = rows16(rng, sum(g.rows), per * hkv, dim)
    word = ints([0])
    what, got = called(g, q, invalid=word)
    assert what == how + "+pagedSharedMerge" and word.item() == 0 and not np.isnan(got).any()
    last = len(g.rows) - 1
    some = {0, 1, members, 63, 64, 127, 128, 191, 192, 255, 256, 257, last - 1, last,
            members * (groups // 2) + 1}
    scale, others = 1 / np.sqrt(np.float32(dim)), set(range(last + 1)) - some
    g.check(got, q, scale, others)
    g.past[last // 2] = -1
    lost = called(g, q, invalid=word)[1]
    at = np.cumsum([0] + g.rows)
    here = np.zeros(len(q), bool)
    here[at[last // 2]:at[last // 2 + 1]] = True
    assert word.item() == 2 and np.isnan(lost[here]).all() and not np.isnan(lost[~here]).any()
    g.check(lost, q, scale, others | {last // 2})
