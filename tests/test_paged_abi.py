"""Rotary rows and the paged 4-bit cache on the host: parameter layouts, the
calls refused before any launch, the scaled frequencies, and the format's
error (no GPU)."""
import ctypes as C

import numpy as np
import pytest
import torch

from llminfer_amd import _lib, ops
from tests import paged_oracle as po

A16 = 4096  # a 16-byte-aligned stand-in pointer; nothing is launched


def test_param_structs():
    assert C.sizeof(_lib.RopeRowsParams) == 40
    assert C.sizeof(_lib.RopeScalingParams) == 28
    assert C.sizeof(_lib.PagedKvParams) == 28
    assert C.sizeof(_lib.PagedAppendParams) == 28
    assert C.sizeof(_lib.PagedGqaParams) == 36


def rope_params(**over):
    p = dict(tokens=3, heads=2, headDim=64, rotaryDim=32, layout=0, inputTokenStride=128,
             inputHeadStride=64, outputTokenStride=128, outputHeadStride=64, factor=1.0)
    p.update(over)
    return _lib.RopeRowsParams(**p)


@pytest.mark.parametrize("over, status", [
    (dict(rotaryDim=31), _lib.INVALID_ARGUMENT),
    (dict(rotaryDim=66), _lib.INVALID_ARGUMENT),
    (dict(layout=2), _lib.INVALID_ARGUMENT),
    (dict(headDim=4096, rotaryDim=4096, outputTokenStride=8192, outputHeadStride=4096),
     _lib.UNSUPPORTED),
    (dict(outputHeadStride=63), _lib.INVALID_ARGUMENT),          # heads overlap
    (dict(outputTokenStride=127), _lib.INVALID_ARGUMENT),        # tokens overlap
    (dict(tokens=1 << 31, heads=64), _lib.INVALID_ARGUMENT),     # 32-bit index range
    (dict(tokens=1 << 24, heads=1, headDim=32), _lib.INVALID_ARGUMENT),
    (dict(tokens=0), _lib.OK),
])
def test_rope_refusals(over, status):
    lib = _lib.load()
    assert lib.llmi_hip_rope(A16, A16, A16, A16, rope_params(**over), None) == status


def test_rope_null_buffers():
    lib = _lib.load()
    for k in range(4):
        args = [A16] * 4
        args[k] = None
        assert lib.llmi_hip_rope(*args, rope_params(), None) == _lib.INVALID_ARGUMENT


def kv_params(**over):
    p = dict(pages=8, pageSize=64, kvHeads=2, headDim=128, sequences=2, tableStride=9, tokens=5)
    p.update(over)
    return _lib.PagedKvParams(**p)


FAR = 1 << 40  # a stand-in pointer apart from A16's buffers


def append_params(**over):
    p = dict(keyTokenStride=256, keyHeadStride=128, valueTokenStride=256, valueHeadStride=128,
             rotaryDim=64, layout=0, factor=1.0)
    p.update(over)
    return _lib.PagedAppendParams(**p)


BAD_KV = [
    (dict(headDim=96), _lib.UNSUPPORTED),
    (dict(pageSize=48), _lib.UNSUPPORTED),
    (dict(pageSize=0), _lib.UNSUPPORTED),
    (dict(pages=0), _lib.INVALID_ARGUMENT),
    (dict(kvHeads=0), _lib.INVALID_ARGUMENT),
    (dict(kvHeads=65536), _lib.INVALID_ARGUMENT),
    (dict(tableStride=0), _lib.INVALID_ARGUMENT),
    (dict(tableStride=1 << 26, pageSize=32), _lib.INVALID_ARGUMENT),  # positions past 2^31
    (dict(tokens=1 << 22), _lib.INVALID_ARGUMENT),
    (dict(pages=1 << 31), _lib.INVALID_ARGUMENT),
    (dict(sequences=1 << 22), _lib.INVALID_ARGUMENT),
    (dict(tokens=0), _lib.OK),
    (dict(sequences=0), _lib.OK),
]


@pytest.mark.parametrize("over, status", BAD_KV)
def test_paged_refusals(over, status):
    lib = _lib.load()
    p = kv_params(**over)
    assert lib.llmi_hip_paged_append(*[A16] * 8, p, append_params(), None) == status
    assert lib.llmi_hip_paged_read(*[A16] * 7, p, None) == status
    assert lib.llmi_hip_paged_gqa(*[A16] * 5, FAR, A16, _lib.PagedGqaParams(p, p.kvHeads, 1.0),
                                  A16, 1 << 40, None) == status


def test_append_refusals():
    lib = _lib.load()
    for over in (dict(rotaryDim=63), dict(rotaryDim=130), dict(layout=2)):
        assert lib.llmi_hip_paged_append(*[A16] * 8, kv_params(), append_params(**over), None) == \
            _lib.INVALID_ARGUMENT
    for k in range(7):  # invalid may be null, the rest not
        args = [A16] * 8
        args[k] = None
        assert lib.llmi_hip_paged_append(*args, kv_params(), append_params(), None) == \
            _lib.INVALID_ARGUMENT
    args = [A16] * 8
    args[6] = A16 + 8
    assert lib.llmi_hip_paged_append(*args, kv_params(), append_params(), None) == _lib.UNSUPPORTED


def test_read_and_gqa_refusals():
    lib = _lib.load()
    gqa = _lib.PagedGqaParams(kv_params(), 4, 1.0)
    for k in range(6):
        args = [A16] * 7
        args[k] = None
        assert lib.llmi_hip_paged_read(*args, kv_params(), None) == _lib.INVALID_ARGUMENT
        assert lib.llmi_hip_paged_gqa(*args, gqa, A16, 1 << 40, None) == _lib.INVALID_ARGUMENT
    for k in (0, 4, 5):
        args = [A16] * 7
        args[k] = A16 + 8
        assert lib.llmi_hip_paged_gqa(*args, gqa, A16, 1 << 40, None) == _lib.UNSUPPORTED
        assert lib.llmi_hip_paged_read(*args, kv_params(), None) == \
            _lib.UNSUPPORTED
    for heads in (0, 3, 65536):
        assert lib.llmi_hip_paged_gqa(*[A16] * 7, _lib.PagedGqaParams(kv_params(), heads, 1.0),
                                      A16, 1 << 40, None) == _lib.INVALID_ARGUMENT
    call = [A16] * 5 + [FAR, A16]
    for ws, size in ((None, 0), (A16, lib.llmi_hip_paged_gqa_workspace_bytes(gqa) - 1),
                     (A16 + 8, 1 << 40)):
        assert lib.llmi_hip_paged_gqa(*call, gqa, ws, size, None) == _lib.WORKSPACE
    # a table whose keys are never divided needs none, and more rows and heads
    # than one call takes are refused
    small = _lib.PagedGqaParams(kv_params(tableStride=2), 4, 1.0)
    assert lib.llmi_hip_paged_gqa_workspace_bytes(small) == 0
    assert ops.kernel_names(_lib.OP_PAGED_GQA, small) == ["pagedGqaSplit"]
    large = _lib.PagedGqaParams(kv_params(tokens=(1 << 22) - 1, kvHeads=512), 512 * 64, 1.0)
    assert lib.llmi_hip_paged_gqa(*call, large, A16, 1 << 60, None) == _lib.INVALID_ARGUMENT
    assert lib.llmi_hip_paged_gqa_workspace_bytes(large) == 0
    # out inside q, and q inside out (5 rows of 4 heads of 128)
    for q, out in ((A16, A16), (A16, A16 + 5104), (A16 + 5104, A16)):
        assert lib.llmi_hip_paged_gqa(q, A16, A16, A16, A16, out, None, gqa, A16, 1 << 40,
                                      None) == _lib.INVALID_ARGUMENT
    assert lib.llmi_hip_paged_gqa_workspace_bytes(_lib.PagedGqaParams(kv_params(), 3, 1.0)) == 0


@pytest.mark.parametrize("dim", [0, 32, 96, 512, 1024, 1 << 31])
def test_plan_of_a_width_without_a_kernel(dim):
    """The calls that plan without buffers refuse what the launch refuses."""
    gqa = _lib.PagedGqaParams(kv_params(headDim=dim, tokens=500), 4, 1.0)
    assert _lib.load().llmi_hip_paged_gqa_workspace_bytes(gqa) == 0
    assert ops.kernel_names(_lib.OP_PAGED_GQA, gqa) == []


def test_plan_names():
    assert ops.kernel_names(_lib.OP_ROPE, rope_params()) == ["ropeRows"]
    assert ops.kernel_names(_lib.OP_ROPE, rope_params(tokens=0)) == []
    assert ops.kernel_names(_lib.OP_PAGED_APPEND, kv_params()) == ["pagedAppend"]
    assert ops.kernel_names(_lib.OP_PAGED_READ, kv_params()) == ["pagedRead"]
    assert ops.kernel_names(_lib.OP_PAGED_GQA, _lib.PagedGqaParams(kv_params(), 4, 1.0)) == \
        ["pagedGqaSplit", "pagedGqaMerge"]
    many = _lib.PagedGqaParams(kv_params(tokens=500, tableStride=64), 4, 1.0)
    assert ops.kernel_names(_lib.OP_PAGED_GQA, many) == ["pagedGqaTiles", "pagedGqaMerge"]
    assert ops.kernel_names(_lib.OP_PAGED_GQA, _lib.PagedGqaParams(kv_params(), 3, 1.0)) == []


@pytest.mark.parametrize("rotary", [2, 4, 64, 128])
@pytest.mark.parametrize("scaling, scale", [(None, 1.0), ("linear", 4.0), ("ntk", 8.0),
                                            ("yarn", 8.0), ("yarn", 0.5), ("bands", 16.0)])
def test_frequencies(rotary, scaling, scale):
    """Within half an fp32 step of the formula (and a few steps of the pow in
    double, far below it)."""
    got, factor = ops.rope_frequencies(rotary, 1e7, scaling, scale, 8192.0, 1.0, 4.0, device="cpu")
    want, want_factor = po.frequencies(rotary, 1e7, scaling, scale, 8192.0, 1.0, 4.0)
    assert got.dtype == torch.float32 and got.shape == (rotary // 2,)
    assert np.all(np.abs(got.numpy() - want) <= want * 2.0 ** -24 * 1.001)
    assert abs(factor - want_factor) <= want_factor * 2.0 ** -24 * 1.001


def test_frequency_refusals():
    for rotary, kwargs in ((64, dict(scaling="twice")), (-2, {})):
        with pytest.raises(ValueError):
            ops.rope_frequencies(rotary, device="cpu", **kwargs)
    for args, kwargs in (((63,), {}), ((2050,), {}), ((64, 0.0), {}), ((64, 1e4, "linear", 0.0), {}),
                         ((64, 1e4, "yarn", 2.0, 0.0), {}),
                         ((64, 1e4, "bands", 2.0, 1024.0, 4.0, 4.0), {})):
        with pytest.raises(_lib.HipError):
            ops.rope_frequencies(*args, device="cpu", **kwargs)
    freqs, factor = ops.rope_frequencies(0, device="cpu")
    assert freqs.numel() == 0 and factor == 1.0


def test_tensors_on_the_host_are_refused():
    x = torch.zeros(2, 2, 64, dtype=torch.float16)
    i = torch.zeros(3, dtype=torch.int32)
    pool = ops.paged_pool(2, 32, 2, 64, device="cpu")
    assert tuple(pool.shape) == (2, 2, 1, 2560)
    with pytest.raises(ValueError):
        ops.bind_rope(x, i[:2], torch.zeros(16), x)
    with pytest.raises(ValueError):
        ops.bind_paged_append(x, x, pool, i, i[:2], i[:2, None])
    with pytest.raises(ValueError):
        ops.bind_paged_read(pool, i, i[:2], i[:2, None], x, x)
    with pytest.raises(ValueError):
        ops.bind_paged_gqa(x, pool, i, i[:2], i[:2, None], x)
    for args in ((2, 48, 2, 64), (2, 0, 2, 64), (2, 32, 2, 96)):
        with pytest.raises(ValueError):
            ops.paged_pool(*args, device="cpu")


@pytest.mark.parametrize("size", [1e-3, 1.0, 100.0, 16000.0])
def test_format_error(size):
    """A kept value is off by at most half a step (range / 15), the roundings
    of scale (31 of them in (16 + code) s at most) and bias, and its own."""
    rng = np.random.default_rng(int(size))
    x = (size / 4 * rng.standard_normal((64, 128))).clip(-size, size).astype(np.float16)
    got = po.kept(x).astype(np.float64).reshape(64, 4, 32)
    g = x.astype(np.float64).reshape(64, 4, 32)
    step = (g.max(-1) - g.min(-1)) / 15
    most = np.abs(g).max(-1) + 31 * step
    far = (step / 2 + 3 * po.U16 * most + 2.0 ** -24 * 33)[..., None]
    assert np.all(np.abs(got - g) <= far)
