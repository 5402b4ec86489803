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


def _launch(lib, dims, n_split, ws=None, ws_bytes=0):
    """The status of a launch whose pointers lead nowhere: a refusal comes before it."""
    strides = (64, 64, 64) * 4
    return lib.rcsa_window_attn(4096, 4096, 4096, 4096, None, 0, _arr(*dims), _arr(*strides), None,
                                None, None, 0, 0, 0, 0, 0, 0, 1, 0.1, n_split, ws, ws_bytes, None)


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
