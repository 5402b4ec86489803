"""Host side of the 8-bit cache and of packed attention, no GPU: refusals of the C ABI before any
launch, plans and workspaces, refusals of the wrappers off the device."""
import ctypes

import pytest
import torch

from cast_amd import _lib, ops

NULL, SHAPE, STRIDE, DTYPE, ALIGN = 1, 2, 3, 4, 6
BF16, F32, I8, E4M3 = 0, 1, 0, 1


@pytest.fixture(scope="module")
def lib():
    if not _lib.LIB_PATH.exists():
        from cast_amd import build
        build.build(verbose=False)
    return _lib.load()


def _arr(*v):
    return (ctypes.c_int64 * len(v))(*v)


TOKENS, CODES, SCALES = (512, 128, 64) * 2, (2048, 128, 64) * 2, (4, 2, 1) * 2


def _append(lib, k=4096, v=4096, dtype=BF16, dims=(2, 4, 2, 64), tokens=TOKENS, codes=CODES,
            scales=SCALES, offsets=None, starts=None, lengths=None, kc=4096, vc=4096, code=I8,
            ks=4096, vs=4096, table=4096, max_pages=4, n_pages=9, page=32, block=16):
    return lib.rcsa_append_cache(k, v, dtype, _arr(*dims), _arr(*tokens, *codes, *scales), offsets,
                                 starts, lengths, kc, vc, code, ks, vs, table, 1, max_pages,
                                 n_pages, page, block, None)


@pytest.mark.parametrize("kw,status", [
    (dict(k=None), NULL), (dict(v=None), NULL), (dict(kc=None), NULL), (dict(vc=None), NULL),
    (dict(ks=None), NULL), (dict(vs=None), NULL), (dict(table=None), NULL), (dict(dtype=7), DTYPE),
    (dict(code=2), DTYPE), (dict(code=-1), DTYPE), (dict(offsets=4096, lengths=4096), SHAPE),
    (dict(dims=(0, 4, 2, 64)), SHAPE), (dict(dims=(2, 0, 2, 64)), SHAPE),
    (dict(dims=(2, 4, 0, 64)), SHAPE), (dict(dims=(2, 4, 5000, 64)), SHAPE),
    (dict(dims=(2, 4, 2, 0)), SHAPE), (dict(dims=(2, 4, 2, 60)), SHAPE),
    (dict(dims=(2, 4, 2, 1032)), SHAPE), (dict(dims=(1 << 20, 4, 2, 64)), SHAPE),
    (dict(dims=(2, 1 << 30, 2, 64)), SHAPE), (dict(dims=(1 << 19, 1 << 19, 2, 64)), SHAPE),
    (dict(dims=(1 << 20, 4, 2, 64), offsets=4096), SHAPE),
    (dict(dims=(1, (1 << 30) - 1, 2, 64)), SHAPE),  # more threads than a launch has
    (dict(max_pages=0), SHAPE), (dict(n_pages=0), SHAPE), (dict(page=0), SHAPE),
    (dict(page=24, block=24), SHAPE), (dict(page=40, block=16), SHAPE), (dict(block=0), SHAPE),
    (dict(block=8), SHAPE), (dict(page=1 << 17, block=1 << 17), SHAPE),
    (dict(page=1 << 12, max_pages=1 << 18), SHAPE), (dict(n_pages=1 << 30), SHAPE),
    (dict(tokens=(512, 128, 60) + TOKENS[3:]), STRIDE),
    (dict(tokens=(-512, 128, 64) + TOKENS[3:]), STRIDE),
    (dict(codes=(2048, 128, 68) + CODES[3:]), STRIDE),
    (dict(codes=(2048, -128, 64) + CODES[3:]), STRIDE),
    (dict(scales=(4, -2, 1) + SCALES[3:]), STRIDE),
    (dict(k=4104), ALIGN), (dict(v=4104), ALIGN), (dict(kc=4100), ALIGN), (dict(vc=4100), ALIGN)])
def test_append_abi_refusals(lib, kw, status):
    """Every refusal comes before a launch: the pointers lead nowhere."""
    assert _append(lib, **kw) == status


def _read(lib, kc=4096, vc=4096, code=I8, ks=4096, vs=4096, ko=4096, vo=4096, dtype=BF16,
          dims=(2, 4, 2, 64), codes=CODES, scales=SCALES, out=TOKENS, lengths=4096, table=4096,
          max_pages=4, n_pages=9, page=32, block=16):
    return lib.rcsa_read_cache(kc, vc, code, ks, vs, ko, vo, dtype, _arr(*dims),
                               _arr(*codes, *scales, *out), None, lengths, table, 1, max_pages,
                               n_pages, page, block, None)


@pytest.mark.parametrize("kw,status", [
    (dict(kc=None), NULL), (dict(vc=None), NULL), (dict(ks=None), NULL), (dict(vs=None), NULL),
    (dict(ko=None), NULL), (dict(vo=None), NULL), (dict(lengths=None), NULL),
    (dict(table=None), NULL), (dict(dtype=7), DTYPE), (dict(code=5), DTYPE),
    (dict(dims=(0, 4, 2, 64)), SHAPE), (dict(dims=(2, 0, 2, 64)), SHAPE),
    (dict(dims=(2, 4, 2, 36)), SHAPE), (dict(dims=(2, 4, 4097, 64)), SHAPE),
    (dict(dims=(1 << 19, 1 << 12, 2, 64)), SHAPE), (dict(dims=(1, (1 << 30) - 1, 2, 1024)), SHAPE),
    (dict(max_pages=0), SHAPE), (dict(n_pages=0), SHAPE), (dict(page=40), SHAPE),
    (dict(block=0), SHAPE), (dict(page=1 << 14, max_pages=1 << 16), SHAPE),
    (dict(codes=(2048, 128, 4) + CODES[3:]), STRIDE),
    (dict(scales=(-4, 2, 1) + SCALES[3:]), STRIDE), (dict(out=(512, 4, 64) + TOKENS[3:]), STRIDE),
    (dict(ko=4104), ALIGN), (dict(vo=4104), ALIGN), (dict(kc=4097), ALIGN), (dict(vc=4097), ALIGN)])
def test_read_abi_refusals(lib, kw, status):
    assert _read(lib, **kw) == status


ROWS = (512, 128, 64)


def _cached(lib, q=4096, k=4096, v=4096, code=I8, ks=4096, vs=4096, out=4096, dtype=BF16,
            dims=(1, 4, 0, 2, 1, 64), q_rows=ROWS, k_rows=(2048, 64, 64), v_rows=(2048, 64, 64),
            o_rows=ROWS, scales=(2, 1, 1) * 2, lengths=4096, table=4096, max_pages=4, n_pages=9,
            page=32, block=16, window=0, sinks=0, order=1, scale=0.1, n_split=1, ws=None,
            ws_bytes=0):
    return lib.rcsa_cached_attn(q, k, v, code, ks, vs, out, None, dtype, _arr(*dims),
                                _arr(*q_rows, *k_rows, *v_rows, *o_rows), _arr(*scales), None,
                                lengths, table, 1, max_pages, n_pages, page, block, window, sinks,
                                order, scale, n_split, ws, ws_bytes, None)


@pytest.mark.parametrize("kw,status", [
    (dict(q=None), NULL), (dict(k=None), NULL), (dict(v=None), NULL), (dict(ks=None), NULL),
    (dict(vs=None), NULL), (dict(out=None), NULL), (dict(table=None), NULL),
    (dict(dtype=F32), DTYPE), (dict(code=2), DTYPE), (dict(dims=(0, 4, 0, 2, 1, 64)), SHAPE),
    (dict(dims=(1, 4, 0, 3, 2, 64)), SHAPE), (dict(dims=(1, 4, 0, 2, 0, 64)), SHAPE),
    (dict(dims=(1, 4, 0, 2, 1, 96)), SHAPE), (dict(dims=(1, 4, 0, 2, 1 << 16, 64)), SHAPE),
    (dict(block=0), SHAPE), (dict(block=24, page=24), SHAPE), (dict(block=64), SHAPE),
    (dict(page=0), SHAPE), (dict(max_pages=0), SHAPE), (dict(n_pages=0), SHAPE),
    (dict(max_pages=1 << 25, page=32), SHAPE), (dict(window=-1), SHAPE), (dict(sinks=-1), SHAPE),
    (dict(order=-1), SHAPE), (dict(order=0, window=4), SHAPE), (dict(scale=0.0), SHAPE),
    (dict(scale=float("nan")), SHAPE), (dict(n_split=65), SHAPE), (dict(n_split=2), SHAPE),
    (dict(n_split=2, ws=4096, ws_bytes=64), SHAPE),
    (dict(n_split=-1, dims=(1, 40, 0, 2, 1, 64)), SHAPE), (dict(n_split=0), SHAPE),
    (dict(k_rows=(2048, 72, 64)), STRIDE), (dict(v_rows=(2048, 64, 72)), STRIDE),
    (dict(k_rows=(2048, 48, 64)), STRIDE), (dict(k_rows=(1 << 31, 64, 64)), STRIDE),
    (dict(q_rows=(512, 128, 68)), STRIDE), (dict(o_rows=(512, 130, 64)), STRIDE),
    (dict(scales=(2, -1, 1) * 2), STRIDE), (dict(scales=(1 << 27, 1, 1) * 2), STRIDE),
    (dict(scales=(2, 1, 1, 1 << 60, 1, 1)), STRIDE),
    (dict(q=4104), ALIGN), (dict(k=4104), ALIGN), (dict(v=4104), ALIGN), (dict(out=4100), ALIGN)])
def test_cached_abi_refusals(lib, kw, status):
    assert _cached(lib, **kw) == status


def _packed(lib, q=4096, k=4096, v=4096, out=4096, dtype=BF16, dims=(2, 9, 9, 2, 1, 64),
            strides=(128, 64, 64, 64, 64, 64, 128, 64), q_offsets=4096, k_offsets=4096, window=0,
            sinks=0, order=1, scale=0.1, n_split=1, ws=None, ws_bytes=0):
    return lib.rcsa_packed_attn(q, k, v, out, None, dtype, _arr(*dims), _arr(*strides), q_offsets,
                                k_offsets, window, sinks, order, scale, n_split, ws, ws_bytes, None)


@pytest.mark.parametrize("kw,status", [
    (dict(q=None), NULL), (dict(k=None), NULL), (dict(v=None), NULL), (dict(out=None), NULL),
    (dict(q_offsets=None), NULL), (dict(k_offsets=None), NULL), (dict(dtype=F32), DTYPE),
    (dict(dims=(0, 9, 9, 2, 1, 64)), SHAPE), (dict(dims=(2, 0, 9, 2, 1, 64)), SHAPE),
    (dict(dims=(2, 9, -1, 2, 1, 64)), SHAPE), (dict(dims=(2, 9, 9, 3, 2, 64)), SHAPE),
    (dict(dims=(2, 9, 9, 1, 2, 64)), SHAPE), (dict(dims=(2, 9, 9, 2, 1, 96)), SHAPE),
    (dict(dims=(1 << 20, 9, 9, 2, 1, 64)), SHAPE), (dict(dims=(2, 1 << 30, 9, 1, 1, 64)), SHAPE),
    (dict(dims=(2, 1 << 29, 9, 4, 1, 64)), SHAPE), (dict(dims=(2, 9, 1 << 30, 2, 1, 64)), SHAPE),
    (dict(dims=(2, 9, 9, 1 << 16, 1, 64)), SHAPE),
    (dict(dims=((1 << 20) - 1, 9, 9, 16, 16, 64)), SHAPE),
    (dict(window=-1), SHAPE), (dict(sinks=-1), SHAPE), (dict(order=-1), SHAPE),
    (dict(order=0, window=4), SHAPE), (dict(order=0, sinks=4), SHAPE), (dict(scale=0.0), SHAPE),
    (dict(scale=float("inf")), SHAPE), (dict(n_split=0), SHAPE), (dict(n_split=65), SHAPE),
    (dict(n_split=2), SHAPE), (dict(n_split=2, ws=4096, ws_bytes=64), SHAPE),
    (dict(strides=(128, 60, 64, 64, 64, 64, 128, 64)), STRIDE),
    (dict(strides=(128, 64, 0, 64, 64, 64, 128, 64)), STRIDE),
    (dict(strides=(128, 64, 64, 64, 1 << 25, 64, 128, 64)), STRIDE),
    (dict(strides=(128, 64, 64, 64, 64, 64, 128, 62)), STRIDE),
    (dict(strides=(-128, 64, 64, 64, 64, 64, 128, 64)), STRIDE),
    (dict(q=4104), ALIGN), (dict(k=4104), ALIGN), (dict(v=4104), ALIGN), (dict(out=4100), ALIGN)])
def test_packed_abi_refusals(lib, kw, status):
    assert _packed(lib, **kw) == status


def test_packed_plan_and_workspace(lib):
    n = ctypes.c_int64(-1)
    plan = lambda dims, most: lib.rcsa_packed_attn_plan(_arr(*dims), most, ctypes.byref(n))
    assert plan((1, 5, 5, 2, 1, 64), 5) == 0 and n.value == 1  # few keys: nothing to share
    assert plan((1, 8000, 8000, 4, 4, 64), 8000) == 0 and n.value > 1  # few blocks of many keys
    assert plan((64, 64000, 64000, 32, 8, 128), 64000) == 0 and n.value == 1
    assert plan((1, 8000, 0, 4, 4, 64), 0) == 0 and n.value == 1
    assert plan((1, 8000, 8000, 4, 3, 64), 8000) == SHAPE
    assert plan((1, 8000, 8000, 4, 4, 64), -1) == SHAPE
    assert lib.rcsa_packed_attn_plan(None, 1, ctypes.byref(n)) == NULL
    assert lib.rcsa_packed_attn_plan(_arr(1, 5, 5, 2, 1, 64), 1, None) == NULL
    dims = _arr(3, 300, 300, 8, 2, 128)
    size = lib.rcsa_packed_attn_workspace_bytes
    assert size(dims, 1) == 0 and size(dims, 0) == -1 and size(dims, 65) == -1
    assert size(None, 1) == -1 and size(_arr(3, 300, 300, 8, 3, 128), 2) == -1
    # every row of every share: 128 rows a block, a block of each request that is not full
    assert size(dims, 4) >= 4 * 2 * 300 * 4 * (128 * 4 + 8)


def test_wrappers_refuse_host_tensors():
    x = torch.zeros(1, 2, 2, 64, dtype=torch.bfloat16)
    codes = torch.zeros(1, 16, 2, 64, dtype=torch.int8)
    scale = torch.zeros(1, 1, 2)
    ints = torch.zeros(1, dtype=torch.int32)
    cache = ops.QuantizedCache(codes, codes.clone(), scale, scale.clone(), ints[:, None])
    for call in (lambda: ops.append_cache(x, x, cache),
                 lambda: ops.read_cache(cache, ints, size=4),
                 lambda: ops.paged_attention(x, cache, ints),
                 lambda: ops.packed_attention(x[0], x[0], x[0], torch.zeros(2, dtype=torch.int32))):
        with pytest.raises(RuntimeError, match="HIP device"):
            call()
    for call in (lambda: ops.packed_attention(x[0], x[0], x[0], ints, window=0),
                 lambda: ops.packed_attention(x[0], x[0], x[0], ints, causal=False, sinks=1),
                 lambda: ops.packed_attention(x[0], x[0], x[0], ints, sm_scale=-1.0),
                 lambda: ops.packed_attention(x[0], x[0], x[0], ints, n_split=0)):
        with pytest.raises(ValueError, match="packed_attention"):
            call()


def test_cached_plan(lib):
    n = ctypes.c_int64(-1)
    plan = lambda dims, most: lib.rcsa_cached_attn_plan(_arr(*dims), most, ctypes.byref(n))
    few = ctypes.c_int64(-1)
    for dims, most in (((1, 1, 4096, 8, 8, 128), 4096), ((1, 1, 4096, 8, 8, 128), 512)):
        assert plan(dims, most) == 0  # few rows: as over 16 bits
        assert lib.rcsa_window_attn_plan(_arr(*dims), most, ctypes.byref(few)) == 0
        assert n.value == few.value <= 0
    assert plan((1, 64, 4096, 8, 8, 128), 64) == 0 and n.value == 1
    assert plan((1, 100, 20000, 8, 8, 128), 20000) == 0 and 8 <= n.value <= 32
    assert lib.rcsa_window_attn_workspace_bytes(_arr(1, 100, 20000, 8, 8, 128), n.value) > 0
    assert plan((256, 100, 20000, 8, 8, 128), 20000) == 0 and n.value == 1  # whole rounds
    assert plan((1, 64, 4096, 8, 3, 128), 4096) == SHAPE
    assert plan((1, 64, 4096, 8, 8, 128), -1) == SHAPE
    assert lib.rcsa_cached_attn_plan(None, 1, ctypes.byref(n)) == NULL
    assert lib.rcsa_cached_attn_plan(_arr(1, 64, 64, 8, 8, 128), 1, None) == NULL
