"""Host side of the streaming operators, no GPU: rotary plans, refusals of the C ABI
before any launch, refusals of the wrappers off the device."""
import ctypes
import math

import pytest
import torch

from cast_amd import _lib, ops
from cast_amd.rotary import rotary_plan
from oracle import streaming_oracle as so

NULL, SHAPE, STRIDE, DTYPE, ALIGN = 1, 2, 3, 4, 6


@pytest.fixture(scope="module")
def lib():
    if not _lib.LIB_PATH.exists():
        from cast_amd import build
        build.build(verbose=False)
    return _lib.load()


@pytest.mark.parametrize("R,kw", [
    (64, {}), (128, dict(axes=(44, 42, 42))), (2, dict(scaling="base", factor=2.0)),
    (96, dict(scaling="linear", factor=4.0, base=500000.0)), (128, dict(scaling="base", factor=8.0)),
    (128, dict(scaling="ramp", factor=16.0, original_length=4096, low=2.0, high=20.0)), (0, {})])
def test_plan_frequencies(R, kw):
    plan = rotary_plan(R, device="cpu", **kw)
    freq, axis = so.frequencies(R, **kw)
    assert plan.rotary_dim == R and plan.turns.dtype == torch.float64
    # pow is off by an ulp or two
    assert torch.allclose(plan.turns * 2 * math.pi, torch.tensor(freq, dtype=torch.float64),
                          rtol=2.0 ** -49, atol=0.0)
    if "axes" in kw:
        assert plan.axis.tolist() == axis and plan.n_axes == 3
    else:
        assert plan.axis is None and plan.n_axes == 1
    assert plan.scale == (0.1 * math.log(16.0) + 1.0 if kw.get("scaling") == "ramp" else 1.0)


def test_plan_limits_of_the_scalings():
    plain = rotary_plan(128, device="cpu").turns
    s = rotary_plan(128, scaling="base", factor=8.0, device="cpu").turns
    assert s[0] == plain[0] and abs(s[-1] * 8.0 / plain[-1] - 1.0) < 1e-12
    r = rotary_plan(128, scaling="ramp", factor=8.0, original_length=4096, device="cpu").turns
    assert r[0] == plain[0] and abs(r[-1] * 8.0 / plain[-1] - 1.0) < 1e-12
    assert bool((r <= plain).all()) and bool((r >= plain / 8 * (1 - 1e-12)).all())
    assert rotary_plan(64, scaling="ramp", factor=8.0, original_length=4096, scale=1.0,
                       device="cpu").scale == 1.0


@pytest.mark.parametrize("R,kw", [
    (63, {}), (64, dict(axes=(32, 16))), (64, dict(axes=(33, 31))), (64, dict(base=0.0)),
    (64, dict(scaling="cubic")), (64, dict(factor=2.0)), (64, dict(scaling="linear", factor=0.0)),
    (64, dict(scaling="ramp", factor=2.0)), (-2, {}),
    (64, dict(scaling="ramp", factor=2.0, original_length=4096, low=4.0, high=4.0))])
def test_plan_refusals(R, kw):
    with pytest.raises(ValueError, match="rotary_plan"):
        rotary_plan(R, device="cpu", **kw)


def _arr(*v):
    return (ctypes.c_int64 * len(v))(*v)


def _rope(lib, x=4096, out=4096, dtype=0, B=1, L=2, H=2, D=64, strides=(256, 128, 64) * 2,
          pos=4096, n_axes=1, turns=4096, n_pairs=32):
    return lib.rcsa_rope(x, out, dtype, B, L, H, D, _arr(*strides), pos, 0, _arr(0, 1, 0), n_axes,
                         turns, None, n_pairs, 0, 1.0, None)


@pytest.mark.parametrize("kw,status", [
    (dict(x=None), NULL), (dict(out=None), NULL), (dict(pos=None), NULL), (dict(turns=None), NULL),
    (dict(dtype=7), DTYPE), (dict(B=0), SHAPE), (dict(L=0), SHAPE), (dict(H=0), SHAPE),
    (dict(D=513), SHAPE), (dict(n_pairs=33), SHAPE), (dict(n_pairs=-1), SHAPE),
    (dict(n_axes=0), SHAPE), (dict(H=5000), SHAPE), (dict(B=1 << 40), SHAPE)])
def test_rope_abi_refusals(lib, kw, status):
    """Every refusal comes before a launch: the pointers lead nowhere."""
    assert _rope(lib, **kw) == status


def _norm(lib, q=4096, k=4096, v=None, q_out=4096, k_out=4096, v_out=None, dtype=0,
          dims=(1, 2, 2, 2, 64), weight=None, w_dtype=0, pos=4096, n_axes=1, turns=4096, n_pairs=32,
          table=None, max_pages=0, n_pages=0, page=0):
    return lib.rcsa_norm_rope(q, k, v, q_out, k_out, v_out, dtype, _arr(*dims),
                              _arr(*(256, 128, 64) * 6), weight, weight, w_dtype, 0, 0, 1e-6, 0,
                              pos, 0, _arr(0, 1, 0), n_axes, turns, None, n_pairs, 0, 1.0, table,
                              1, max_pages, n_pages, page, None, None, None)


PAGES = dict(v=4096, v_out=4096, table=4096, max_pages=4, n_pages=9, page=16)


@pytest.mark.parametrize("kw,status", [
    (dict(q=None), NULL), (dict(k=None), NULL), (dict(q_out=None), NULL), (dict(k_out=None), NULL),
    (dict(pos=None), NULL), (dict(turns=None), NULL), (dict(v=4096), NULL),
    (dict(v_out=4096), NULL), (dict(table=4096), NULL), (dict(PAGES, table=None), NULL),
    (dict(dtype=7), DTYPE), (dict(w_dtype=7), DTYPE), (dict(dims=(0, 2, 2, 2, 64)), SHAPE),
    (dict(dims=(1, 0, 2, 2, 64)), SHAPE), (dict(dims=(1, 2, 0, 2, 64)), SHAPE),
    (dict(dims=(1, 2, 2, 0, 64)), SHAPE), (dict(dims=(1, 2, 2, 5000, 64)), SHAPE),
    (dict(dims=(1, 2, 2, 2, 513)), SHAPE), (dict(dims=(1 << 20, 1 << 20, 2, 2, 64)), SHAPE),
    (dict(n_pairs=33), SHAPE), (dict(n_axes=0), SHAPE), (dict(PAGES, max_pages=0), SHAPE),
    (dict(PAGES, n_pages=0), SHAPE), (dict(PAGES, page=0), SHAPE),
    (dict(PAGES, max_pages=1 << 20, page=1 << 11), SHAPE)])
def test_norm_abi_refusals(lib, kw, status):
    assert _norm(lib, **kw) == status


def _window(lib, q=4096, k=4096, out=4096, dtype=0, dims=(1, 4, 8, 2, 1, 64),
            strides=(512, 128, 64, 512, 64, 64, 512, 64, 64, 512, 128, 64), table=None, ts=1,
            max_pages=0, n_pages=0, page=0, window=0, sinks=0, block=1, n_split=1, ws=None,
            ws_bytes=0, scale=0.1):
    return lib.rcsa_window_attn(q, k, k, out, None, dtype, _arr(*dims), _arr(*strides), None, None,
                                table, ts, max_pages, n_pages, page, window, sinks, block, scale,
                                n_split, ws, ws_bytes, None)


@pytest.mark.parametrize("kw,status", [
    (dict(q=None), NULL), (dict(k=None), NULL), (dict(out=None), NULL), (dict(dtype=1), DTYPE),
    (dict(dims=(0, 4, 8, 2, 1, 64)), SHAPE), (dict(dims=(1, 4, -1, 2, 1, 64)), SHAPE),
    (dict(dims=(1, 4, 8, 3, 2, 64)), SHAPE), (dict(dims=(1, 4, 8, 1, 2, 64)), SHAPE),
    (dict(dims=(1, 4, 8, 2, 1, 96)), SHAPE), (dict(dims=(1, 4, 1 << 30, 2, 1, 64)), SHAPE),
    (dict(window=-1), SHAPE), (dict(sinks=-1), SHAPE), (dict(block=-1), SHAPE),
    (dict(block=0, window=4), SHAPE), (dict(block=0, sinks=4), SHAPE),
    (dict(table=4096, max_pages=4, n_pages=9, page=24), SHAPE),
    (dict(table=4096, max_pages=0, n_pages=9, page=16), SHAPE),
    (dict(table=4096, max_pages=1 << 20, n_pages=9, page=1 << 12), SHAPE),
    (dict(n_split=0), SHAPE), (dict(n_split=-2), SHAPE), (dict(n_split=65), SHAPE),
    (dict(n_split=-1, dims=(1, 40, 8, 2, 1, 64)), SHAPE),
    (dict(n_split=0, dims=(513, 4, 8, 2, 1, 64), ws=4096, ws_bytes=1 << 40), SHAPE), (dict(n_split=2), SHAPE),
    (dict(n_split=2, ws=4096, ws_bytes=64), SHAPE),
    (dict(strides=(512, 128, 63) + (512, 64, 64) * 3), STRIDE),
    (dict(strides=(512, 128, 64, 512, 0, 64, 512, 64, 64, 512, 128, 64)), STRIDE),
    (dict(strides=(512, 128, 64, 512, 64, 64, 512, 56, 64, 512, 128, 64)), STRIDE),
    (dict(strides=(512, 128, 64, 512, 1 << 25, 64, 512, 64, 64, 512, 128, 64)), STRIDE),
    (dict(strides=(512, 128, 64, -512, 64, 64, 512, 64, 64, 512, 128, 64)), STRIDE),
    (dict(scale=0.0), SHAPE), (dict(scale=-1.0), SHAPE), (dict(scale=float('nan')), SHAPE),
    (dict(scale=float('inf')), SHAPE), (dict(q=4098), ALIGN), (dict(k=4104), ALIGN), (dict(out=4100), ALIGN)])
def test_window_abi_refusals(lib, kw, status):
    assert _window(lib, **kw) == status


def test_window_plan_and_workspace(lib):
    n = ctypes.c_int64(-1)
    assert lib.rcsa_window_attn_plan(_arr(1, 1, 4096, 8, 8, 128), 4096, ctypes.byref(n)) == 0
    assert n.value == 0  # few rows, many keys: units of one wavefront
    assert lib.rcsa_window_attn_plan(_arr(1, 1, 4096, 8, 8, 128), 512, ctypes.byref(n)) == 0
    assert n.value == -1  # few keys: a workgroup a key head
    assert lib.rcsa_window_attn_workspace_bytes(_arr(1, 1, 64, 8, 8, 128), -1) == 0
    assert lib.rcsa_window_attn_plan(_arr(1, 64, 4096, 8, 8, 128), 4096, ctypes.byref(n)) == 0
    assert 1 <= n.value <= 64
    assert lib.rcsa_window_attn_workspace_bytes(_arr(1, 64, 64, 8, 8, 128), 0) == -1
    assert lib.rcsa_window_attn_plan(_arr(1, 1, 4096, 8, 3, 128), 4096, ctypes.byref(n)) == SHAPE
    assert lib.rcsa_window_attn_workspace_bytes(_arr(1, 1, 64, 8, 8, 128), 1) == 0
    assert lib.rcsa_window_attn_workspace_bytes(_arr(1, 1, 64, 8, 8, 128), 65) == -1
    assert lib.rcsa_window_attn_workspace_bytes(_arr(2, 100, 64, 8, 8, 128), 3) \
        >= 3 * 2 * 8 * 100 * (128 * 4 + 8)


def test_wrappers_refuse_host_tensors():
    x = torch.zeros(1, 2, 2, 64, dtype=torch.bfloat16)
    plan = rotary_plan(64, device="cpu")
    pos = torch.arange(2)
    for call in (lambda: ops.rope(x, pos, plan), lambda: ops.norm_rope(x, x, pos, plan),
                 lambda: ops.window_attention(x, x, x),
                 lambda: ops.paged_attention(x, ops.PagedCache(x, x, pos), pos)):
        with pytest.raises(RuntimeError, match="HIP device"):
            call()
