"""GPU tests of sequences that share pages of the 4-bit cache: forks, the free
pages, moved rows, attention behind a common prefix, and a run of them
together. What moves is compared byte for byte or value for value; the
attention with paged_oracle's, whose tolerances are counted there."""
import numpy as np
import pytest
import torch

from llminfer_amd import _lib, ops
from tests import paged_oracle as po

pytestmark = pytest.mark.gpu


def dev(a, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(a))
    return (t if dtype is None else t.to(dtype)).cuda()


def ints(values):
    return torch.tensor(list(values), dtype=torch.int32).cuda()


def rows16(rng, *shape, size=1.0):
    return (size * rng.standard_normal(shape)).astype(np.float16)


def random_pool(rng, pages, page, hkv, dim):
    """Any bytes, with scales and biases that are finite."""
    pool = ops.paged_pool(pages, page, hkv, dim)
    bytes_ = rng.integers(0, 256, tuple(pool.shape), dtype=np.uint8)
    for at in (16 * dim, 36 * dim):
        n = bytes_[..., at:at + 4 * dim].size // 2
        scale = rows16(rng, n, size=0.05)
        bytes_[..., at:at + 4 * dim] = scale.view(np.uint8).reshape(*bytes_.shape[:-1], 4 * dim)
    pool.copy_(dev(bytes_))
    return pool


def read(pool, table, s, n):
    """K and V of the first n keys of row s of the table."""
    k, v = ops.paged_read(pool, ints([0, n]), ints([0]), table[s:s + 1].contiguous(), n)
    return k.cpu().numpy(), v.cpu().numpy()


# ---------------------------------------------------------------------- fork

def fork_oracle(pool, table, past, parent, spare, page):
    pool, width, bad = pool.copy(), table.shape[1], False
    rows, lengths = [], []
    old = pool.copy()
    for p, t in zip(parent, spare):
        n = past[p] if 0 <= p < len(past) else -1
        if not 0 <= n <= width * page:
            rows.append([-1] * width), lengths.append(-1)
            bad = True
            continue
        lengths.append(n)
        if t < 0:
            rows.append(list(table[p]))
            continue
        whole, rest = divmod(n, page)
        row = list(table[p][:whole]) + [-1] * (width - whole)
        if whole < width:
            source = table[p][whole] if rest else 0
            if t < len(pool) and 0 <= source < len(pool):
                row[whole] = t
                blocks = -(-rest // 32)
                pool[t, :, :blocks] = old[source, :, :blocks]
            else:
                bad = True
        rows.append(row)
    return pool, np.array(rows, np.int32).reshape(-1, width), np.array(lengths, np.int32), bad


FORK = [  # past, width, parent, spare (index behind the tables' pages, or -1), hkv, dim, page
    ([0], 1, [0], [0], 1, 64, 32),
    ([5], 2, [0, 0, 0], [0, 1, -1], 1, 64, 32),
    ([31, 32, 33], 3, [2, 1, 0, 2], [3, 1, 2, 0], 2, 128, 32),
    ([255, 256, 257, 1], 2, [0, 1, 2, 3, 0], [0, 1, 2, 3, 4], 4, 256, 256),
    ([192], 2, [0, 0], [0, 1], 3, 256, 96),       # a full row
    ([700, 13], 9, [1, 0] * 20, list(range(40)), 2, 256, 128),
    ([77], 300, [0] * 3, [0, 1, 2], 1, 128, 64),  # rows longer than a workgroup
    ([2047], 1, [0, 0], [0, 1], 8, 64, 2048),     # blocks of a page by the dozen
]


@pytest.mark.parametrize("past, width, parent, spare, hkv, dim, page", FORK)
def test_fork(gpu, past, width, parent, spare, hkv, dim, page):
    rng = np.random.default_rng(sum(past) + dim)
    held = len(past) * width
    order = rng.permutation(held + len(spare) + 2).astype(np.int32)
    table = order[:held].reshape(len(past), width)
    spare = [int(order[held + i]) if i >= 0 else -1 for i in spare]
    pool = random_pool(rng, order.size, page, hkv, dim)
    want = fork_oracle(pool.cpu().numpy(), table, past, parent, spare, page)
    word = ints([0])
    t, n = ops.paged_fork(pool, dev(table), ints(past), ints(parent), ints(spare), word)
    assert not want[3] and word.item() == 0
    for a, b in zip((pool, t, n), want):
        assert np.array_equal(a.cpu().numpy(), b)


def test_fork_without_place(gpu):
    """Parents that are none or do not fit, and pages outside the pool."""
    rng = np.random.default_rng(5)
    page, pool = 64, random_pool(rng, 12, 64, 2, 128)
    table = np.array([[0, 1, 2], [3, 99, 4], [5, -1, 6], [7, 8, 9], [0, 1, 2]], np.int32)
    past = [100, 70, 128, 193, -1]
    for parent, spare, bad in (([0, 5], [10, 11], True), ([-1], [10], True), ([3], [10], True),
                               ([4], [-1], True), ([1, 0], [10, 11], True), ([0], [12], True),
                               ([2, 2], [10, -1], False), ([0, 2**31 - 1], [10, 11], True)):
        before = pool.clone()
        want = fork_oracle(pool.cpu().numpy(), table, past, parent, spare, page)
        word = ints([0])
        t, n = ops.paged_fork(pool, dev(table), ints(past), ints(parent), ints(spare), word)
        assert want[3] == bad and word.item() == 2 * bad
        for a, b in zip((pool, t, n), want):
            assert np.array_equal(a.cpu().numpy(), b)
        pool.copy_(before)
    ops.paged_fork(pool, dev(table), ints(past), ints([]), ints([]))


# ---------------------------------------------------------------------- free

def free_oracle(table, lengths, page, pages):
    held, bad = np.zeros(pages, bool), False
    for row, n in zip(table, lengths):
        fits = 0 <= n <= len(row) * page
        bad |= not fits
        mine = row[:-(-n // page)] if fits else row
        inside = (mine >= 0) & (mine < pages)
        bad |= not inside.all()
        held[mine[inside]] = True
    free = np.flatnonzero(~held)
    return np.concatenate((free, np.full(pages - free.size, -1))).astype(np.int32), free.size, bad


FREE = [  # sequences, width, page, pages
    (0, 4, 32, 5), (1, 1, 32, 1), (1, 1, 32, 2), (3, 5, 64, 31), (3, 5, 64, 33), (7, 40, 32, 64),
    (5, 1030, 32, 8191), (16, 256, 64, 8192), (16, 256, 64, 8193), (40, 1000, 32, 16383),
    (300, 700, 256, 100_001), (2, 3, 32, 2**19), (2, 3, 32, 2**19 + 1), (90, 2000, 32, 2**20 + 77),
]


@pytest.mark.parametrize("sequences, width, page, pages", FREE)
def test_free(gpu, sequences, width, page, pages):
    rng = np.random.default_rng(width + pages)
    for full in (False, True):
        table = rng.integers(0, pages, (sequences, width), dtype=np.int32)
        lengths = rng.integers(0, width * page + 1, sequences)
        if full:  # every page held, as far as there are entries
            table.reshape(-1)[:pages] = rng.permutation(pages)[:table.size]
            lengths[:] = width * page
        want, count, bad = free_oracle(table, lengths, page, pages)
        word = ints([0])
        free, n = ops.paged_free(dev(table), ints(lengths), page, pages, word)
        assert not bad and word.item() == 0 and n.item() == count
        assert np.array_equal(free.cpu().numpy(), want)


@pytest.mark.parametrize("pages", [50, 20_000])
def test_free_without_place(gpu, pages):
    """Lengths that do not fit hold the whole row; entries outside hold nothing
    and are looked at only where they are held."""
    rng = np.random.default_rng(pages)
    for change, bad in ((None, False), ("short", True), ("long", True), ("below", True),
                        ("above", True), ("behind", False)):
        table = rng.integers(0, pages, (6, 8), dtype=np.int32)
        lengths = np.array([256, 1, 0, 200, 32, 33])
        if change == "short":
            lengths[2] = -1
        elif change == "long":
            lengths[2] = 257
        elif change in ("below", "above"):
            table[3, 6] = -1 if change == "below" else pages
        elif change == "behind":
            table[3, 7], table[2, 0] = -1, pages
        want, count, flag = free_oracle(table, lengths, 32, pages)
        word = ints([0])
        free, n = ops.paged_free(dev(table), ints(lengths), 32, pages, word)
        assert flag == bad and word.item() == 2 * bad and n.item() == count
        assert np.array_equal(free.cpu().numpy(), want)


# ---------------------------------------------------------------------- move

MOVE = [  # (rows, past, span) of each sequence, hkv, dim, page
    ([(1, 0, 1)], 1, 64, 32),
    ([(1, 40, 200)], 4, 256, 64),
    ([(5, 100, 24)] * 6, 4, 256, 64),
    ([(32, 32, 64)], 2, 128, 32),      # a whole block
    ([(33, 31, 90), (0, 9, 9), (70, 1, 70)], 3, 128, 32),
    ([(100, 0, 400)], 2, 256, 96),
    ([(90, 5, 300), (64, 0, 64)], 2, 64, 32),
    ([(3, i, 40) for i in range(70)], 1, 64, 32),
    ([(300, 17, 1000)], 8, 128, 256),
]


@pytest.mark.parametrize("seqs, hkv, dim, page", MOVE)
@pytest.mark.parametrize("apart", [False, True])
@pytest.mark.parametrize("order", ["ascending", "any", "repeated"])
def test_move(gpu, seqs, hkv, dim, page, apart, order):
    """Bit for bit, everything else as it was; within a sequence's own pages and
    between pages apart."""
    rng = np.random.default_rng(len(seqs) * dim + page)
    width = max(-(-max(r + p, n) // page) for r, p, n in seqs) + 1
    S = len(seqs)
    numbers = rng.permutation(2 * S * width + 2).astype(np.int32)
    table = numbers[:S * width].reshape(S, width)
    other = numbers[S * width:2 * S * width].reshape(S, width) if apart else table
    pool = random_pool(rng, numbers.size, page, hkv, dim)
    chosen = []
    for r, _, n in seqs:
        c = rng.permutation(n)[:r] if order != "repeated" else rng.integers(0, n, r)
        chosen.append(np.sort(c) if order == "ascending" else c)
    starts = np.cumsum([0] + [r for r, _, _ in seqs])
    everything = ints([0] + [2 * S * width * page])
    flat = dev(numbers[None, :2 * S * width])

    def values():  # of every page of the tables, in their order
        k, v = ops.paged_read(pool, everything, ints([0]), flat, 2 * S * width * page)
        return [x.cpu().numpy().view(np.uint16).reshape(2 * S, width * page, hkv, dim) for x in (k, v)]

    before, rest = values(), pool[dev(numbers[2 * S * width:]).long()].clone()
    word = ints([0])
    ops.paged_move(pool, ints(starts), ints([p for _, p, _ in seqs]), dev(table),
                   ints(np.concatenate(chosen)), dev(other) if apart else None, word)
    assert word.item() == 0
    for old, new in zip(before, values()):
        want = old.copy()
        for s, (r, p, _) in enumerate(seqs):
            want[s, p:p + r] = old[S + s if apart else s, chosen[s]]
        assert np.array_equal(new, want)
    assert torch.equal(pool[dev(numbers[2 * S * width:]).long()], rest)


def test_move_without_place(gpu):
    """Sources outside, pages outside, a sequence that does not fit: what has a
    place is moved, the rest stays."""
    rng = np.random.default_rng(9)
    page, width = 32, 3
    table = np.arange(9, dtype=np.int32).reshape(3, 3)
    for change in ("none", "below", "behind", "source page", "target page", "sequence", "past"):
        pool = random_pool(rng, 9, page, 2, 128)
        t, past, source = table.copy(), [3, 3, 3], rng.integers(0, 64, 60)
        lost = np.zeros(60, bool)
        if change == "below":
            source[25], lost[25] = -1, True
        if change == "behind":
            source[25], lost[25] = width * page, True
        if change == "source page":
            t[1, 2], source[22:25] = 99, [64, 65, 95]
            lost[22:25] = True
        if change == "target page":
            t[1, 0], source[20:40] = -5, 33  # rows at 3 to 22: all in the page
            lost[20:40] = True
        if change == "sequence":
            past[1] = 90
            lost[20:40] = True
        if change == "past":
            past[1] = -2
            lost[20:40] = True
        whole = np.where((t < 0) | (t > 8), 0, t)
        old = [read(pool, dev(whole), s, width * page) for s in range(3)]
        word = ints([0])
        ops.paged_move(pool, ints([0, 20, 40, 60]), ints(past), dev(t), ints(source), None, word)
        assert word.item() == (0 if change == "none" else 2), change
        for s in range(3):
            if (whole[s] != t[s]).any() and change == "target page":
                continue  # (its pages are read below)
            new = read(pool, dev(whole), s, width * page)
            for a, b in zip(old[s], new):
                want = a.copy()
                for i in range(20):
                    if not lost[20 * s + i]:
                        want[past[s] + i] = a[source[20 * s + i]]
                ok = np.repeat(whole[s] == t[s], page)
                assert np.array_equal(b[ok].view(np.uint16), want[ok].view(np.uint16)), (change, s)


# -------------------------------------------------------------------- shared

class Group:
    """Sequences behind one prefix: a pool and its table, as forks leave them, whose
    rows have place for `places` keys at least."""
    places = 0

    def __init__(self, rng, groups, hkv, dim, page, size=1.0, extra=0):
        """groups: (prefix, [(rows, past) of each sequence]). Whole pages of a
        prefix are shared, its last keys are each sequence's own copy."""
        self.seqs = [s for _, members in groups for s in members]
        width = max([-(-(r + p) // page) for r, p in self.seqs] + [1]) + extra
        need = sum(k // page + len(m) * (width - k // page) for k, m in groups)
        numbers = iter(rng.permutation(need + 2).tolist())
        self.pool = random_pool(rng, need + 2, page, hkv, dim)
        self.table, self.k, self.v = [], [], []
        for keys, members in groups:
            whole = keys // page
            common = [next(numbers) for _ in range(whole)]
            shared = [rows16(rng, keys, hkv, dim, size=size) for _ in range(2)]
            kept = [po.kept(x) for x in shared]
            for i, (r, p) in enumerate(members):
                n = r + p - keys
                own = [rows16(rng, n, hkv, dim, size=size) for _ in range(2)]
                self.table.append(common + [next(numbers) for _ in range(width - whole)])
                self.k.append((kept[0], po.kept(own[0])))
                self.v.append((kept[1], po.kept(own[1])))
                row = dev(np.array(self.table[-1:], np.int32))
                first = whole * page if i else 0  # the shared pages are filled once
                k, v = (np.concatenate((a[first:], b)) for a, b in zip(shared, own))
                if len(k):
                    ops.paged_append(dev(k), dev(v), self.pool, ints([0, len(k)]), ints([first]), row)
        self.table = np.array(self.table, np.int32)
        unused = max(self.places // page - width, 0)
        self.table = dev(np.pad(self.table, ((0, 0), (0, unused)), constant_values=-1))
        self.rows = [r for r, _ in self.seqs]
        self.starts = ints(np.cumsum([0] + self.rows))
        self.past = ints(p for _, p in self.seqs)
        self.groups = ints(np.cumsum([0] + [len(m) for _, m in groups]))
        self.prefix = ints(k for k, _ in groups)

    def call(self, q, **over):
        args = dict(starts=self.starts, past=self.past, table=self.table, groups=self.groups,
                    prefix=self.prefix) | over
        return ops.paged_gqa_shared(dev(q), self.pool, args.pop("starts"), args.pop("past"),
                                    args.pop("table"), args.pop("groups"), args.pop("prefix"), **args)

    def cached(self, s, n):
        return (np.concatenate(x)[:n] for x in (self.k[s], self.v[s]))

    def check(self, got, q, scale, skip=()):
        at = 0
        for s, (r, p) in enumerate(self.seqs):
            if r and s not in skip:
                want, far = po.attention(q[at:at + r], *self.cached(s, r + p), p, scale)
                err = np.abs(got[at:at + r].astype(np.float64) - want)
                assert np.all(err <= far), (s, (err - far).max(), np.isnan(got[at:at + r]).any())
            at += r


@pytest.fixture(params=[0, 16384], ids=["short", "long"])
def room(request, monkeypatch):
    """Tables that are as long as their sequences, and longer: the host divides the
    work by what a table has place for."""
    monkeypatch.setattr(Group, "places", request.param)


SHARED = [  # groups, heads a KV head, hkv, dim, page
    # 160 columns in 640, beside the sequences' own keys: tiles and runs of blocks
    ([(256, [(1, 256 + 9 * i) for i in range(40)])], 4, 4, 256, 32),
    ([(224, [(1, 230 + 31 * i % 97) for i in range(20)]), (96, [(1, 96 + i) for i in range(22)])],
     8, 2, 128, 32),
    ([(320, [(1, 320 + 7 * i) for i in range(50)]), (64, [(2, 70), (0, 80), (1, 64)] * 20)],
     4, 2, 64, 64),
    ([(64, [(1, 64 + i) for i in range(80)]), (0, [(1, 9)] * 9)], 8, 1, 64, 32),
    ([(32, [(1, 3000)] + [(1, 40 + i) for i in range(47)])], 5, 4, 64, 32),
    # more than 256 sequences, and than 64 groups, of each kind
    ([(64, [(1, 64 + i % 40) for i in range(290)])], 4, 1, 64, 32),
    ([(32, [(1, 32 + i)] * 25) for i in range(70)], 4, 1, 64, 32),
    ([(64, [(1, 70), (1, 64)]) for _ in range(140)], 1, 1, 64, 32),
    ([(32, [(1, 32)])], 1, 1, 64, 32),
    ([(64, [(1, 64), (1, 100), (1, 65)])], 4, 2, 256, 64),
    ([(96, [(1, 100), (1, 97)]), (0, [(1, 10), (2, 0)]), (31, [(1, 40)])], 2, 2, 128, 32),
    ([(500, [(1, 500 + i) for i in range(8)])], 4, 2, 256, 64),        # a block cut by the prefix
    ([(640, [(1, 700), (0, 650), (1, 641), (5, 640)])], 5, 1, 128, 64),
    ([(256, [(1, 256 + 7 * i) for i in range(30)])], 4, 1, 64, 32),    # 120 columns
    ([(320, [(4, 320 + 3 * i) for i in range(13)])], 4, 1, 256, 32),   # 208 columns: tiles
    ([(200, [(2, 230 + i) for i in range(50)])], 4, 1, 128, 32),       # 400 columns: tiles
    ([(64, [(1, 64 + i) for i in range(70)])], 2, 1, 64, 32),          # more than 64 sequences
    ([(32 * (1 + i % 3), [(1, 96 + i)] * (1 + i % 2)) for i in range(70)], 2, 1, 128, 32),  # and groups
    ([(1500, [(1, 1500), (1, 2100)]), (700, [(3, 1300), (1, 701)])], 8, 1, 256, 128),
    ([(2048, [(40, 2048), (8, 2100)])], 4, 1, 256, 256),               # chunks of a prompt
    ([(1024, [(60, 1030), (60, 1024)])], 4, 1, 128, 64),               # the same, of 480 columns
    ([(160, [(90, 170), (1, 200)])], 4, 1, 64, 32),
]


@pytest.mark.usefixtures("room")
@pytest.mark.parametrize("groups, per, hkv, dim, page", SHARED)
@pytest.mark.parametrize("scale", [None, -0.3, 0.0])
def test_shared(gpu, groups, per, hkv, dim, page, scale):
    rng = np.random.default_rng(len(groups) * 100 + dim)
    g = Group(rng, groups, hkv, dim, page)
    q = rows16(rng, sum(g.rows), per * hkv, dim)
    word = ints([0])
    got = g.call(q, scale=scale, invalid=word).cpu().numpy()
    assert word.item() == 0
    g.check(got, q, 1 / np.sqrt(np.float32(dim)) if scale is None else scale)


@pytest.mark.usefixtures("room")
@pytest.mark.parametrize("groups, per, hkv, dim, page, some", [
    ([(1280, [(1, 1280 + i % 8) for i in range(288)])], 4, 16, 256, 64, range(0, 288, 31)),
    ([(2048, [(1, 2050)] * 130), (1800, [(1, 1800 + i) for i in range(70)])], 8, 8, 128, 128,
     [0, 1, 99, 129, 130, 160, 199]),
    ([(3968, [(1, 3970 + i % 3) for i in range(300)])], 4, 16, 64, 128, range(0, 300, 43)),
    ([(96, [(1, 96 + i % 60) for i in range(700)])], 4, 32, 64, 32, range(0, 700, 77)),
])
def test_shared_parted_units(gpu, groups, per, hkv, dim, page, some):
    """So many units of shared keys that the workgroups' runs of blocks part them
    anywhere, or that there are more of them than workgroups."""
    rng = np.random.default_rng(hkv + dim)
    g = Group(rng, groups, hkv, dim, page)
    q = rows16(rng, sum(g.rows), per * hkv, dim)
    got = g.call(q)
    g.check(got.cpu().numpy(), q, 1 / np.sqrt(np.float32(dim)), set(range(len(g.rows))) - set(some))
    assert torch.equal(got, g.call(q)) and not got.isnan().any()


def test_shared_reads_the_first_table(gpu):
    """What a group's other sequences have in the places of whole shared blocks
    is not read."""
    rng = np.random.default_rng(2)
    g = Group(rng, [(128, [(1, 130), (2, 128), (1, 150)])], 2, 256, 32)
    q = rows16(rng, 4, 8, 256)
    g.table[1:, :4] = -1
    word = ints([0])
    got = g.call(q, invalid=word).cpu().numpy()
    assert word.item() == 0
    g.check(got, q, 1 / 16)


@pytest.mark.usefixtures("room")
def test_shared_outside_groups(gpu):
    """Sequences before, between and behind the groups share nothing; rows of no
    sequence stay."""
    rng = np.random.default_rng(3)
    g = Group(rng, [(64, [(1, 90)]), (96, [(2, 100), (1, 96)]), (0, [(1, 5)]), (64, [(1, 64)] * 2),
                    (0, [(3, 40)])], 2, 128, 32)
    q = rows16(rng, sum(g.rows) + 3, 8, 128)
    out = torch.full(q.shape, 7.0, dtype=torch.float16, device="cuda")
    got = g.call(q, groups=ints([1, 3, 4, 6]), prefix=ints([96, 0, 64]), out=out).cpu().numpy()
    g.check(got, q, 1 / np.sqrt(128))
    assert (got[-3:] == 7).all()


@pytest.mark.usefixtures("room")
def test_shared_large_scores(gpu):
    """Scores far past the weights' range, in both parts."""
    rng = np.random.default_rng(4)
    g = Group(rng, [(256, [(1, 300), (1, 256), (4, 280)])], 2, 128, 32, size=300.0)
    q = rows16(rng, 6, 8, 128, size=40.0)
    g.check(g.call(q).cpu().numpy(), q, 1 / np.sqrt(128))


@pytest.mark.usefixtures("room")


@pytest.mark.parametrize("members", [3, 60, 90])
def test_shared_without_place(gpu, members):
    """A sequence shorter than its prefix or past its table is NaN as a whole, a
    missing shared page all of the group, a missing own page its rows; the
    others are as they would be."""
    rng = np.random.default_rng(members)
    plain = [(2, 130 + i % 7) for i in range(members)]
    groups = [(128, plain), (64, [(1, 80), (1, 64)])]
    hkv, dim, page = 1, 256, 32
    q = rows16(rng, 2 * members + 2, 4, dim)
    group0 = range(members)

    def lost(g, rows, **over):
        word = ints([0])
        got = g.call(q, invalid=word, **over).cpu().numpy()
        assert word.item() == 2
        seqs = [s for s in range(len(g.seqs)) if s in rows]
        at = np.cumsum([0] + g.rows)
        for s in seqs:
            assert np.isnan(got[at[s]:at[s + 1]]).all(), s
        g.check(got, q, 1 / 16, skip=seqs)

    def fresh():
        return Group(np.random.default_rng(8), groups, hkv, dim, page)

    g = fresh()
    g.past[1] = 127  # shorter than the prefix
    lost(g, [1])
    g = fresh()
    g.past[2] = -1
    lost(g, [2])
    g = fresh()
    g.past[0] = g.table.shape[1] * page  # the first of the group, past its table
    lost(g, [0])
    g = fresh()
    g.table[0, 2] = 10**6  # a shared page
    lost(g, group0)
    g = fresh()
    g.table[members, 1] = -1
    lost(g, [members, members + 1])
    g = fresh()
    g.table[1, 4] = -1  # an own one
    lost(g, [1])
    g = fresh()
    lost(g, group0, prefix=ints([10**6, 64]))  # longer than all of them
    got = g.call(q, prefix=ints([-5, 64])).cpu().numpy()  # none
    g.check(got, q, 1 / 16)


@pytest.mark.usefixtures("room")
@pytest.mark.parametrize("n", [20, 100])
def test_shared_odd_orders(gpu, n):
    """Starts and groups out of order, overlapping or out of range: any values
    in the rows that are claimed twice, no fault, and the rows of no sequence
    as they were."""
    rng = np.random.default_rng(6)
    g = Group(rng, [(64, [(2, 64 + i) for i in range(n)])], 1, 256, 32)
    q = rows16(rng, 2 * n + 4, 4, 256)
    for starts in (g.starts, ints([0, 40, 3, 20, 9] + [30] * (n - 4)), ints(range(5 * n, 6 * n + 1)),
                   ints(range(n, -1, -1)), ints([-5] * 10 + [3 * n] * (n - 9))):
        for groups, prefix in (([0, n], [64]), ([5, 2], [64]), ([0, n, 0, n, 0, n], [64] * 5),
                               ([-9, 6 * n], [64]), ([n + 10, n + 20], [64]), ([0] * 71, [32] * 70)):
            out = torch.full(q.shape, 7.0, dtype=torch.float16, device="cuda")
            g.call(q, starts=starts, groups=ints(groups), prefix=ints(prefix), out=out)
            torch.cuda.synchronize()
            if starts is g.starts:
                assert (out[2 * n:] == 7).all()


@pytest.mark.usefixtures("room")
@pytest.mark.parametrize("n", [6, 90])
def test_shared_rows_are_apart(gpu, n):
    """A query row of infinities or NaN changes no other row."""
    rng = np.random.default_rng(13)
    g = Group(rng, [(96, [(1, 100 + i) for i in range(n)])], 2, 128, 32)
    q = rows16(rng, n, 8, 128)
    bad = q.copy()
    bad[1], bad[4, 3], bad[n - 1, :, 5] = np.nan, np.inf, -np.inf
    got, want = (g.call(x).cpu().numpy() for x in (bad, q))
    same = np.ones((n, 8), bool)
    same[1] = same[4, 3] = same[n - 1] = False
    assert np.array_equal(got[same], want[same]) and np.isnan(got[1]).all()


def test_shared_is_plain_without_groups(gpu):
    rng = np.random.default_rng(7)
    g = Group(rng, [(64, [(1, 70), (3, 64)])], 2, 64, 32)
    q = rows16(rng, 4, 8, 64)
    got = g.call(q, groups=ints([0]), prefix=ints([]))
    assert torch.equal(got, ops.paged_gqa(dev(q), g.pool, g.starts, g.past, g.table))


@pytest.mark.usefixtures("room")
@pytest.mark.parametrize("n", [9, 90])
def test_shared_replayed(gpu, n):
    """A captured call is replayed on other lengths, groups and prefixes, with
    the eager result each time; two graphs bound on one stream run at once."""
    rng = np.random.default_rng(11)
    g = Group(rng, [(512, [(1, 512 + 20 * i) for i in range(n)])], 2, 256, 64, extra=2)
    q = [rows16(rng, n, 8, 256) for _ in range(2)]
    dq = [dev(x) for x in q]
    outs = [torch.zeros_like(x) for x in dq]
    stream = torch.cuda.Stream()
    graphs = []
    with torch.cuda.stream(stream):
        calls = [ops.bind_paged_gqa_shared(x, g.pool, g.starts, g.past, g.table, g.groups, g.prefix, o)
                 for x, o in zip(dq, outs)]
        calls[0]()
    stream.synchronize()
    for call in calls:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            call()
        graphs.append(graph)
    past = g.past.cpu().numpy()
    for prefix, less in ((512, 0), (500, 0), (0, 5), (64, 3), (256, 0)):
        g.past.copy_(dev((past - less).astype(np.int32)))
        g.prefix.fill_(prefix if less == 0 or prefix < 500 else 0)
        want = [g.call(x).cpu() for x in q]
        for s in (0, 1, n // 2, n - 1):
            p = int(past[s]) - less
            exact, far = po.attention(q[0][s:s + 1], *g.cached(s, p + 1), p, 1 / 16)
            assert np.all(np.abs(want[0][s:s + 1].numpy().astype(np.float64) - exact) <= far)
        streams = [torch.cuda.Stream() for _ in graphs]
        torch.cuda.synchronize()
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            assert torch.equal(o.cpu(), w)


def test_pages_replayed(gpu):
    """Forks, free pages and moves captured once and replayed on other lengths."""
    rng = np.random.default_rng(12)
    page, hkv, dim = 32, 2, 128
    pool = random_pool(rng, 9000, page, hkv, dim)
    order = rng.permutation(9000).astype(np.int32)
    table, other = dev(order[:40].reshape(4, 10)), dev(order[40:80].reshape(4, 10))
    spare, parent = dev(order[80:86]), ints([0, 1, 2, 3, 0, 1])
    past, starts, source = ints([0] * 4), ints([0, 5, 5, 9, 12]), ints([0] * 12)
    t, n = torch.zeros(6, 10, dtype=torch.int32, device="cuda"), ints([0] * 6)
    free, count = torch.zeros(9000, dtype=torch.int32, device="cuda"), ints([0])
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        calls = [ops.bind_paged_fork(pool, table, past, parent, spare, t, n),
                 ops.bind_paged_free(table, past, page, free, count),
                 ops.bind_paged_move(pool, starts, past, other, source, table)]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        for call in calls:
            call()
    for i in range(4):
        length = rng.integers(0, 300, 4)
        past.copy_(dev(length.astype(np.int32)))
        source.copy_(dev(rng.integers(0, 320, 12).astype(np.int32)))
        torch.cuda.synchronize()
        first = pool.clone()
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in (pool, t, n, free, count)]
        pool.copy_(first)
        tt, nn = ops.paged_fork(pool, table, past, parent, spare)
        ff, cc = ops.paged_free(table, past, page, 9000)
        ops.paged_move(pool, starts, past, other, source, table)
        for a, b in zip(got, (pool, tt, nn, ff, cc)):
            assert torch.equal(a, b)
        want, number, _ = free_oracle(table.cpu().numpy(), length, page, 9000)
        assert np.array_equal(ff.cpu().numpy(), want) and cc.item() == number


# ------------------------------------------------------- a run of them together

@pytest.mark.parametrize("hq, hkv, dim, page", [(16, 4, 256, 64), (8, 2, 128, 32), (4, 1, 64, 96)])
def test_answers_to_one_prompt(gpu, hq, hkv, dim, page):
    """A prompt, answers forked from it, their tokens, drafts of which some are
    kept, and the pages that are left: each step checked against a cache kept in
    numpy."""
    rng = np.random.default_rng(dim)
    scale, answers, width = 1 / np.sqrt(np.float32(dim)), 5, 16
    pool = ops.paged_pool(64, page, hkv, dim)
    freqs, factor = ops.rope_frequencies(dim // 2)
    free, count = ops.paged_free(ints([]).reshape(0, width), ints([]), page, 64)
    assert count.item() == 64
    length = 3 * page + 37
    table = torch.full((1, width), -1, dtype=torch.int32, device="cuda")
    table[0, :4 + 1] = free[:5]

    def kept_after(kv, s, table, n):
        k, v = read(pool, table, s, n)
        return [np.concatenate((a, b[len(a):])) for a, b in zip(kv, (k, v))]

    def append(table, past, rows):
        k, v = (rows16(rng, sum(rows), hkv, dim) for _ in range(2))
        ops.paged_append(dev(k), dev(v), pool, ints(np.cumsum([0] + rows)), ints(past), table,
                         freqs=freqs, factor=factor)

    append(table, [0], [length])
    prompt = [x for x in read(pool, table, 0, length)]
    free, count = ops.paged_free(table, ints([length]), page, 64)
    assert count.item() == 64 - -(-length // page)
    table, past = ops.paged_fork(pool, table, ints([length]), ints([0] * answers), free[:answers])
    assert past.tolist() == [length] * answers
    caches = [list(prompt) for _ in range(answers)]
    groups, prefix = ints([0, answers]), ints([length // page * page])
    for rows in ([1] * answers, [3, 1, 0, 2, 5], [7] * answers):
        now = past.tolist()
        # pages for the new rows, where the last ones do not hold them
        free, _ = ops.paged_free(table, past, page, 64)
        unused = [x for x in free.tolist() if x >= 0 and x not in table.flatten().tolist()]
        for s in range(answers):
            for j in range(-(-(now[s] + rows[s]) // page)):
                if table[s, j] < 0:
                    table[s, j] = unused.pop(0)
        append(table, now, rows)
        caches = [kept_after(kv, s, table, now[s] + rows[s]) for s, kv in enumerate(caches)]
        q = rows16(rng, sum(rows), hq, dim)
        starts = ints(np.cumsum([0] + rows))
        got = ops.paged_gqa_shared(dev(q), pool, starts, past, table, groups, prefix).cpu().numpy()
        plain = ops.paged_gqa(dev(q), pool, starts, past, table).cpu().numpy()
        at = 0
        for s, r in enumerate(rows):
            if r:
                want, far = po.attention(q[at:at + r], *caches[s], now[s], scale)
                for x in (got, plain):
                    assert np.all(np.abs(x[at:at + r].astype(np.float64) - want) <= far)
            at += r
        past += ints(rows)
    # of the last seven rows of each, the first and two more are kept
    now = [n - 7 for n in past.tolist()]
    picked = [sorted(rng.permutation(np.arange(1, 7))[:2].tolist()) for _ in range(answers)]
    source = [n + i for n, p in zip(now, picked) for i in [0] + p]
    ops.paged_move(pool, ints(range(0, 3 * answers + 1, 3)), ints(now), table, ints(source))
    past = ints(n + 3 for n in now)
    for s, (n, p) in enumerate(zip(now, picked)):
        want = [np.concatenate((x[:n + 1], x[[n + i for i in p]])) for x in caches[s]]
        for a, b in zip(read(pool, table, s, n + 3), want):
            assert np.array_equal(a, b)
    # one answer stays: it takes over its row, the others' pages are free again
    table, past = ops.paged_fork(pool, table, past, ints([3]), ints([-1]))
    free, count = ops.paged_free(table, past, page, 64)
    assert count.item() == 64 - -(-(now[3] + 3) // page)
    for a, b in zip(read(pool, table, 0, length), prompt):
        assert np.array_equal(a, b)


def test_other_stream_and_order(gpu):
    """Bound on a stream of its own, the calls run there."""
    rng = np.random.default_rng(1)
    g = Group(rng, [(256, [(1, 260 + i) for i in range(6)])], 2, 128, 32)
    q = rows16(rng, 6, 8, 128)
    want = g.call(q)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        got = g.call(q)
        free, _ = ops.paged_free(g.table, g.past, 32, g.pool.shape[0])
    stream.synchronize()
    assert torch.equal(got, want)
    assert torch.equal(free, ops.paged_free(g.table, g.past, 32, g.pool.shape[0])[0])


@pytest.mark.usefixtures("room")
def test_two_at_once(gpu):
    """Bound calls in flight on two streams, each with its own workspace."""
    rng = np.random.default_rng(2)
    calls = []
    for groups, per, hkv, dim, page in (SHARED[0], SHARED[1], SHARED[9], SHARED[14]):
        g = Group(rng, groups, hkv, dim, page)
        q = dev(rows16(rng, sum(g.rows), per * hkv, dim))
        out = torch.empty_like(q)
        free, count = ints(range(g.pool.shape[0])), ints([0])
        stream = torch.cuda.Stream()
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            bound = [ops.bind_paged_gqa_shared(q, g.pool, g.starts, g.past, g.table, g.groups,
                                               g.prefix, out),
                     ops.bind_paged_free(g.table, g.past, page, free, count)]
        want = g.call(q.cpu().numpy()), ops.paged_free(g.table, g.past, page, free.numel())[0]
        calls.append((bound, out, free, want))
    torch.cuda.synchronize()
    for _ in range(20):
        for bound, *_ in calls:
            for b in bound:
                b()
    torch.cuda.synchronize()
    for _, out, free, want in calls:
        assert torch.equal(out, want[0]) and torch.equal(free, want[1])


@pytest.mark.usefixtures("room")
@pytest.mark.parametrize("n", [6, 50])
def test_a_pool_past_4_gib(gpu, n):
    """Pages at the end of 6.5 GB hold what those of a small pool do after the same
    calls: offsets in bytes need more than 32 bits."""
    rng = np.random.default_rng(n)
    page, hkv, dim, pages = 32, 4, 256, 160_000
    g = Group(rng, [(256, [(1, 290 + 5 * i) for i in range(n)])], hkv, dim, page, extra=2)
    small = g.pool.shape[0]
    spare = ints(range(small, small + n))
    pool = torch.cat((g.pool, torch.zeros_like(g.pool[:n])))
    far = torch.empty((pages, *pool.shape[1:]), dtype=torch.uint8, device="cuda")
    assert far.nbytes > 1 << 32
    far[-small - n:] = pool
    to = pages - small - n
    q = rows16(rng, n, 4 * hkv, dim)
    want = g.call(q)
    assert not want.isnan().any()
    g.pool, table = far, g.table
    there = torch.where(table >= 0, table + to, table)
    assert torch.equal(g.call(q, table=there), want)
    seen = []
    rows = [20 + i % 14 for i in range(n)]
    source = [int(x) for r in rows for x in np.sort(rng.permutation(280)[:r])]
    for where, add, mine in ((pool, 0, table), (far, to, there)):
        ops.paged_move(where, ints(np.cumsum([0] + rows)), ints([256] * n), mine, ints(source))
        ops.paged_move(where, ints([0, 20]), ints([260]), mine[n - 1:], ints(range(256, 276)),
                       mine[1:2])
        t, past = ops.paged_fork(where, mine, g.past, ints(range(n - 1, -1, -1)), spare + add)
        # (with the pages of their next rows)
        free, count = ops.paged_free(t, past + 1, page, where.shape[0])
        k, v = ops.paged_read(where, ints(range(0, 290 * n + 1, 290)), ints([0] * n), t, 290 * n)
        held = t[t >= 0].unique() - add
        seen.append((t - add * (t >= 0), past, k, v, held, count - where.shape[0]))
        assert not torch.isin(held + add, free).any()
    for a, b in zip(*seen):
        assert torch.equal(a, b)


# ------------------------------------------------------------------- refusals

def test_refuses(gpu):
    i = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")
    pool = ops.paged_pool(4, 32, 2, 64)
    q = torch.zeros(3, 4, 64, dtype=torch.float16, device="cuda")
    good = dict(q=q, pool=pool, starts=i(3), past=i(2), table=i(2, 2), groups=i(2), prefix=i(1),
                out=torch.zeros_like(q))
    ops.bind_paged_gqa_shared(**good)()
    for bad in (dict(q=q.float()), dict(q=q[:, :3].contiguous(), out=q[:, :3].clone()),
                dict(groups=i(3)), dict(prefix=i(1, 1)), dict(groups=i(2).long()),
                dict(prefix=torch.zeros(1, dtype=torch.int32)), dict(starts=i(2)),
                dict(pool=pool[..., 1:]), dict(table=i(3, 2)), dict(invalid=i(2)),
                dict(out=torch.zeros(3, 4, 128, dtype=torch.float16, device="cuda"))):
        with pytest.raises(ValueError):
            ops.bind_paged_gqa_shared(**(good | bad))
    with pytest.raises(_lib.HipError):
        ops.bind_paged_gqa_shared(**(good | dict(out=q)))()
    good = dict(pool=pool, table=i(2, 2), past=i(2), parent=i(3), spare=i(3) - 1, table_out=i(3, 2),
                past_out=i(3))
    ops.bind_paged_fork(**good)()
    for bad in (dict(past=i(3)), dict(spare=i(2)), dict(table_out=i(2, 2)), dict(past_out=i(2)),
                dict(parent=i(3).long()), dict(pool=pool.view(torch.int8)), dict(invalid=i(2))):
        with pytest.raises(ValueError):
            ops.bind_paged_fork(**(good | bad))
    same = i(3, 2)
    for bad in (dict(table=same, past=i(3), table_out=same), dict(past=same[0], past_out=same[1:, 0]),
                dict(table=i(0, 2), past=i(0))):
        with pytest.raises((_lib.HipError, ValueError)):
            ops.bind_paged_fork(**(good | bad))()
    good = dict(table=i(2, 2), lengths=i(2), page_size=32, free=i(4), count=i(1))
    ops.bind_paged_free(**good)()
    for bad in (dict(lengths=i(3)), dict(page_size=33), dict(page_size=0), dict(count=i(2)),
                dict(free=i(2, 2)), dict(free=i(4).float()), dict(invalid=i(0))):
        with pytest.raises(ValueError):
            ops.bind_paged_free(**(good | bad))
    with pytest.raises(_lib.HipError):
        ops.bind_paged_free(**(good | dict(free=i(0))))()
    good = dict(pool=pool, starts=i(3), past=i(2), table=i(2, 2), source=i(3))
    ops.bind_paged_move(**good)()
    for bad in (dict(source=i(3).long()), dict(source=i(3, 1)), dict(source_table=i(2, 3)),
                dict(source_table=i(2, 2).long()), dict(starts=i(2)), dict(invalid=i(2))):
        with pytest.raises(ValueError):
            ops.bind_paged_move(**(good | bad))
    ops.paged_move(pool, i(3), i(2), i(2, 2), i(0))
