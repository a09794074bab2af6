"""GPU tests of the paged 4-bit cache where its parts meet: a missing page
inside a unit of columns. Against paged_oracle; tolerances are counted there or
beside the test."""
import numpy as np
import pytest

from llminfer_amd import _lib, ops
from tests import paged_oracle as po
from tests.test_paged_gpu import check, dev, filled, ints, rows16

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
