"""Forks, free pages, moved rows and attention behind a common prefix on the
host: parameter layouts, the calls refused before any launch, the launches that
a call says it makes (no GPU)."""
import ctypes as C

import pytest

from llminfer_amd import _lib, ops
from tests.test_paged_abi import A16, BAD_KV, FAR, kv_params

MANY = 1 << 40  # bytes of a workspace that is large enough


def shared_params(groups=1, heads=None, **over):
    kv = kv_params(**over)
    return _lib.PagedSharedParams(_lib.PagedGqaParams(kv, kv.kvHeads if heads is None else heads, 1.0),
                                  groups)


def fork_params(**over):
    p = dict(pages=8, pageSize=64, kvHeads=2, headDim=128, sequences=2, tableStride=9, children=5)
    return _lib.PagedForkParams(**(p | over))


def free_params(**over):
    return _lib.PagedFreeParams(**(dict(pages=8, pageSize=64, sequences=2, tableStride=9) | over))


def test_param_structs():
    assert C.sizeof(_lib.PagedSharedParams) == 40
    assert C.sizeof(_lib.PagedForkParams) == 28
    assert C.sizeof(_lib.PagedMoveParams) == 32
    assert C.sizeof(_lib.PagedFreeParams) == 16


@pytest.mark.parametrize("over, status", BAD_KV)
def test_kv_refusals(over, status):
    lib = _lib.load()
    assert lib.llmi_hip_paged_gqa_shared(*[A16] * 7, FAR, A16, shared_params(**over), A16, MANY,
                                         None) == status
    for apart in (0, 1):
        assert lib.llmi_hip_paged_move(*[A16] * 7, _lib.PagedMoveParams(kv_params(**over), apart),
                                       A16, MANY, None) == status
    if status != _lib.OK:
        fork = {k: v for k, v in over.items() if k != "tokens"}
        want = status if fork else _lib.INVALID_ARGUMENT
        p = fork_params(**fork) if fork else fork_params(children=1 << 22)
        assert lib.llmi_hip_paged_fork(*fork_args(), A16, A16, p, None) == want


def fork_args():
    """table, past, parent, spare and the outputs, apart from each other."""
    return [A16 + (i << 32) for i in range(6)]


def test_shared_refusals():
    lib = _lib.load()
    p = shared_params(heads=4)
    need = lib.llmi_hip_paged_gqa_shared_workspace_bytes(p)
    assert need > 0
    args = [A16] * 7 + [FAR, A16]
    for k in range(8):
        bad = list(args)
        bad[k] = None
        assert lib.llmi_hip_paged_gqa_shared(*bad, p, A16, need, None) == _lib.INVALID_ARGUMENT
    for k in (0, 6, 7):
        bad = list(args)
        bad[k] += 8
        assert lib.llmi_hip_paged_gqa_shared(*bad, p, A16, need, None) == _lib.UNSUPPORTED
    for ws, size in ((None, need), (A16, need - 1), (A16 + 8, need)):
        assert lib.llmi_hip_paged_gqa_shared(*args, p, ws, size, None) == _lib.WORKSPACE
    bad = list(args)
    bad[7] = A16 + 16  # inside q
    assert lib.llmi_hip_paged_gqa_shared(*bad, p, A16, need, None) == _lib.INVALID_ARGUMENT
    for over in (dict(groups=1 << 22), dict(heads=3), dict(heads=0), dict(heads=1 << 17),
                 dict(tokens=(1 << 22) - 1, heads=1024)):
        q = shared_params(**over)
        assert lib.llmi_hip_paged_gqa_shared(*args, q, A16, MANY, None) == _lib.INVALID_ARGUMENT
        assert lib.llmi_hip_paged_gqa_shared_workspace_bytes(q) == 0
    # no groups: the call is paged_gqa, with its workspace and errors
    none = shared_params(groups=0, heads=4)
    assert lib.llmi_hip_paged_gqa_shared_workspace_bytes(none) == \
        lib.llmi_hip_paged_gqa_workspace_bytes(none.gqa)
    assert lib.llmi_hip_paged_gqa_shared(A16, A16, A16, A16, None, None, A16, FAR, None, none, None,
                                         0, None) == _lib.WORKSPACE


def test_fork_refusals():
    lib = _lib.load()
    good, pool = fork_args(), [A16, A16]
    for k in range(6):
        bad = list(good)
        bad[k] = None
        assert lib.llmi_hip_paged_fork(*bad, *pool, fork_params(), None) == _lib.INVALID_ARGUMENT
    assert lib.llmi_hip_paged_fork(*good, None, A16, fork_params(), None) == _lib.INVALID_ARGUMENT
    assert lib.llmi_hip_paged_fork(*good, A16 + 8, A16, fork_params(), None) == _lib.UNSUPPORTED
    for k in (4, 5):  # an output inside another buffer
        for other in range(6):
            if other != k:
                bad = list(good)
                bad[k] = good[other] + 4
                assert lib.llmi_hip_paged_fork(*bad, *pool, fork_params(), None) == \
                    _lib.INVALID_ARGUMENT
    assert lib.llmi_hip_paged_fork(*good, *pool, fork_params(children=0), None) == _lib.OK
    for over in (dict(sequences=0), dict(children=1 << 22),
                 dict(children=1 << 20, pageSize=512), dict(kvHeads=65535, children=300)):
        assert lib.llmi_hip_paged_fork(*good, *pool, fork_params(**over), None) == \
            _lib.INVALID_ARGUMENT


def test_free_refusals():
    lib = _lib.load()
    good = [A16 + (i << 34) for i in range(4)]  # table, lengths, free, count
    large = dict(pages=100_000)
    need = lib.llmi_hip_paged_free_workspace_bytes(free_params(**large))
    assert need >= 12_500 and lib.llmi_hip_paged_free_workspace_bytes(free_params()) == 0
    for k in range(4):
        bad = list(good)
        bad[k] = None
        assert lib.llmi_hip_paged_free(*bad, A16, free_params(), None, 0, None) == \
            _lib.INVALID_ARGUMENT
    for k, other in ((2, 0), (2, 1), (3, 0), (3, 1), (3, 2)):
        bad = list(good)
        bad[k] = good[other]
        assert lib.llmi_hip_paged_free(*bad, A16, free_params(), None, 0, None) == \
            _lib.INVALID_ARGUMENT
    for ws, size in ((None, need), (A16, need - 1), (A16 + 4, need)):
        assert lib.llmi_hip_paged_free(*good, A16, free_params(**large), ws, size, None) == \
            _lib.WORKSPACE
    for over, status in ((dict(pageSize=0), _lib.UNSUPPORTED), (dict(pageSize=40), _lib.UNSUPPORTED),
                         (dict(pages=0), _lib.INVALID_ARGUMENT),
                         (dict(tableStride=0), _lib.INVALID_ARGUMENT),
                         (dict(pages=1 << 31), _lib.INVALID_ARGUMENT),
                         (dict(tableStride=1 << 26), _lib.INVALID_ARGUMENT),
                         (dict(sequences=1 << 20, tableStride=1 << 12), _lib.INVALID_ARGUMENT)):
        p = free_params(**over)
        assert lib.llmi_hip_paged_free(*good, A16, p, A16, MANY, None) == status
        assert lib.llmi_hip_paged_free_workspace_bytes(p) == 0


def test_move_refusals():
    lib = _lib.load()
    within, apart = (_lib.PagedMoveParams(kv_params(), x) for x in (0, 1))
    need = lib.llmi_hip_paged_move_workspace_bytes(within)
    assert need > 0 and lib.llmi_hip_paged_move_workspace_bytes(apart) == 0
    for p in (within, apart):
        for k in range(6):  # invalid may be null, the source's table within the pages
            bad = [A16] * 7
            bad[k] = None
            if k != 1 or p is apart:
                assert lib.llmi_hip_paged_move(*bad, p, A16, need, None) == _lib.INVALID_ARGUMENT
    for ws, size in ((None, need), (A16, need - 1), (A16 + 8, need)):
        assert lib.llmi_hip_paged_move(*[A16] * 7, within, ws, size, None) == _lib.WORKSPACE
    wrong = _lib.PagedMoveParams(kv_params(headDim=96), 0)
    assert lib.llmi_hip_paged_move_workspace_bytes(wrong) == 0


def test_launches():
    """A call names one kernel for each launch."""
    assert ops.kernel_names(_lib.OP_PAGED_FORK, fork_params()) == ["pagedFork"]
    assert ops.kernel_names(_lib.OP_PAGED_FORK, fork_params(children=0)) == []
    assert ops.kernel_names(_lib.OP_PAGED_FREE, free_params()) == ["pagedFree"]
    assert ops.kernel_names(_lib.OP_PAGED_FREE, free_params(pages=10**5)) == [
        "pagedFreeMark", "pagedFreeJoin", "pagedFreeList"]
    move = [_lib.PagedMoveParams(kv_params(), x) for x in (0, 1)]
    assert ops.kernel_names(_lib.OP_PAGED_MOVE, move[0]) == ["pagedGather", "pagedPlace"]
    assert ops.kernel_names(_lib.OP_PAGED_MOVE, move[1]) == ["pagedMove"]
    names = ops.kernel_names(_lib.OP_PAGED_GQA_SHARED, shared_params(heads=4))
    assert names[-1] == "pagedSharedMerge" and names[0] == "pagedGqaSplit"
    names = ops.kernel_names(_lib.OP_PAGED_GQA_SHARED,
                             shared_params(heads=16, kvHeads=4, headDim=256, tokens=48, sequences=48,
                                           pages=2000, tableStride=256))
    assert names == ["pagedGqaMixed", "pagedSharedMerge"]
    names = ops.kernel_names(_lib.OP_PAGED_GQA_SHARED,
                             shared_params(heads=16, kvHeads=4, headDim=256, tokens=48, sequences=48,
                                           tableStride=9))
    assert names == ["pagedGqaSplit", "pagedSharedMerge"]
    names = ops.kernel_names(_lib.OP_PAGED_GQA_SHARED,
                             shared_params(heads=16, kvHeads=4, headDim=256, tokens=400, sequences=4))
    assert names == ["pagedGqaTiles", "pagedGqaTiles", "pagedSharedMerge"]
    plain = shared_params(groups=0, heads=4)
    assert ops.kernel_names(_lib.OP_PAGED_GQA_SHARED, plain) == \
        ops.kernel_names(_lib.OP_PAGED_GQA, plain.gqa)
