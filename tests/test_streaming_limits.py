"""Limits of the streaming operators' launches over the C ABI, no GPU."""
import ctypes

import pytest

from cast_amd import _lib

SHAPE = 2


@pytest.fixture(scope="module")
def lib():
    if not _lib.LIB_PATH.exists():
        from cast_amd import build
        build.build(verbose=False)
    return _lib.load()


def _arr(*v):
    return (ctypes.c_int64 * len(v))(*v)


def _plan(lib, dims, keys):
    n = ctypes.c_int64(-9)
    assert lib.rcsa_window_attn_plan(_arr(*dims), keys, ctypes.byref(n)) == 0
    return n.value


def _launch(lib, dims, n_split, ws=None, ws_bytes=0, scale=0.1):
    """The status of a launch whose pointers lead nowhere: a refusal comes before it."""
    strides = (dims[5],) * 12
    return lib.rcsa_window_attn(4096, 4096, 4096, 4096, None, 0, _arr(*dims), _arr(*strides), None,
                                None, None, 0, 0, 0, 0, 0, 0, 1, scale, n_split, ws, ws_bytes, None)


def test_window_launches_stay_below_2_32_threads(lib):
    """Row blocks of 256 threads, key heads of 512, joined rows of 256."""
    group = (1 << 19, 1, 8, 16, 16, 64)     # 2^23 key heads
    assert _plan(lib, (1 << 19, 1, 8, 15, 15, 64), 8) == -1
    assert _plan(lib, group, 8) >= 1        # (blocks of rows: 2^31 threads)
    assert lib.rcsa_window_attn_workspace_bytes(_arr(*group), -1) == -1
    assert _launch(lib, group, -1) == SHAPE
    units = (512, 1, 1 << 20, 32768, 1024, 64)   # 2^24 rows, a long storage
    assert _plan(lib, (512, 1, 1 << 20, 16384, 512, 64), 1 << 20) == 0
    assert _plan(lib, units, 1 << 20) == -1
    assert lib.rcsa_window_attn_workspace_bytes(_arr(*units), 0) == -1
    assert _launch(lib, units, 0, 4096, 1 << 50) == SHAPE
    blocks = (1 << 19, 1, 8, 32, 32, 64)    # 2^24 blocks of rows
    assert lib.rcsa_window_attn_workspace_bytes(_arr(*blocks), 1) == 0
    assert _launch(lib, blocks, 1) == SHAPE


def test_units_workspace_goes_by_the_storage(lib):
    """Rows of the units that a storage or window can have, never more than for any length;
    a byte less is refused."""
    def size(dims, storage, window=0, sinks=0):
        return lib.rcsa_window_attn_workspace_bytes_for(_arr(*dims), 0, storage, window, sinks)

    dims, row = (2, 4, 64, 16, 4, 128), 4 * 4 * (128 * 4 + 8)
    any_length = lib.rcsa_window_attn_workspace_bytes(_arr(*dims), 0)
    assert any_length == (4 * 8 * 256 + 2 * 4) * row
    assert size(dims, 0) == size(dims, 64) == 2 * 4 * row          # one unit a key head
    assert size(dims, 65) == size(dims, 128) == 2 * 4 * 2 * row    # two tiles a unit
    assert size(dims, 1 << 30) == any_length
    assert size(dims, 1 << 30, 1 << 40, 1 << 40) == any_length     # a window past all
    assert size(dims, 1 << 30, 60, 4) == 2 * 4 * 3 * row           # 5 tiles and the first
    assert all(size(dims, n) <= any_length for n in range(0, 1 << 20, 997))
    assert size(dims, -1) == size(dims, (1 << 30) + 1) == size(dims, 64, -1) == -1
    assert size(dims, 64, 0, -1) == -1
    need = size(dims, 64)
    assert _launch(lib, dims, 0, 4096, need - 1) == SHAPE
    assert _launch(lib, dims, 0, None, need) == SHAPE


@pytest.mark.parametrize("scale", [2.4e38, 3.4e38, 1e-46])
def test_scales_that_leave_fp32_are_refused(lib, scale):
    """The kernels take the scale times log2 e in fp32: infinite there, a logit of 0 would be
    NaN; 0 in fp32, it is no scale."""
    assert _launch(lib, (1, 4, 8, 2, 1, 64), 1, scale=scale) == SHAPE
