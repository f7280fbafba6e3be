"""8-bit KV states on the GPU: rows quantized, read back, kept; refusals
against a real arena; binary16 states' keep."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

from gpu_util import SYN_F16, SYN_F32, Arena, capi, lib
from kv8_cases import refusals
from kv8_util import append8, held, keep, read8, values
from synapse_amd import workloads as wl

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def arena():
    a = Arena(256 << 20)
    yield a
    a.close()


@pytest.fixture
def room(arena):
    """The arena, filled with NaN patterns, its top put back afterwards."""
    mark = arena.top
    arena.fill(mark, 0xff, 64 << 20)
    yield arena
    arena.top = mark


def _rows(g, n, n_kv, hd, dtype=SYN_F32):
    x = g.standard_normal((2, n, n_kv, hd)).astype(np.float32) * np.exp(g.standard_normal((2, n, n_kv, 1))).astype(np.float32)
    return x.astype(np.float16).astype(np.float32) if dtype == SYN_F16 else x


def _want(x, dtype):
    q, step = held(x)
    out = q.astype(np.float32) * step[..., None]  # one f32 rounding of the product
    return out.astype(np.float16) if dtype == SYN_F16 else out


@pytest.mark.parametrize("n_kv,hd", [(8, 128), (2, 64), (1, 2), (3, 40), (5, 18), (2, 96), (4, 256), (7, 34), (2, 160)])
@pytest.mark.parametrize("dtype,out_dtype", [(SYN_F32, SYN_F32), (SYN_F16, SYN_F16), (SYN_F32, SYN_F16)])
def test_append_then_read(room, n_kv, hd, dtype, out_dtype):
    """Runs of odd lengths at odd positions, from one row to several tiles:
    the values are the formula's to the bit, wherever they are read from."""
    g = np.random.default_rng(n_kv * 1000 + hd)
    cache = capi.kv8_state(room, 333, n_kv, hd)
    x = _rows(g, 333, n_kv, hd, dtype)
    at = 0
    for n in (1, 3, 60, 64, 1, 129, 7, 68):
        append8(room, cache, x[0, at:at + n], x[1, at:at + n], at, dtype)
        at += n
    assert at == 333
    want = _want(x, out_dtype)
    for pos, n in ((0, 333), (0, 1), (332, 1), (63, 2), (64, 64), (17, 200)):
        k, v = read8(room, cache, n, pos, out_dtype)
        assert np.array_equal(k.view(np.uint8), want[0, pos:pos + n].view(np.uint8)), (pos, n)
        assert np.array_equal(v.view(np.uint8), want[1, pos:pos + n].view(np.uint8)), (pos, n)


def test_other_positions_stay(room):
    """An append writes its own positions only, byte for byte: the state
    around it holds what another append put there."""
    g = np.random.default_rng(5)
    cache = capi.kv8_state(room, 200, 3, 72)
    x = _rows(g, 200, 3, 72)
    append8(room, cache, x[0], x[1], 0)
    size = capi.kv8_state_bytes(200, 3, 72)
    before = room.download(cache.offset, (size,), np.uint8)
    for pos, n in ((5, 1), (62, 3), (64, 64), (100, 99)):
        y = _rows(g, n, 3, 72)
        append8(room, cache, y[0], y[1], pos)
        x[:, pos:pos + n] = y
        k, v = read8(room, cache, 200, 0)
        want = _want(x, SYN_F32)
        assert np.array_equal(k, want[0]) and np.array_equal(v, want[1]), (pos, n)
        append8(room, cache, x[0, pos:pos + n], x[1, pos:pos + n], pos)
    append8(room, cache, *_rows(np.random.default_rng(5), 200, 3, 72), 0)
    assert np.array_equal(room.download(cache.offset, (size,), np.uint8)[:cache.max_ctx], before[:cache.max_ctx])


@pytest.mark.parametrize("dtype", [SYN_F32, SYN_F16])
def test_borders_and_specials(room, dtype):
    """Values on and next to half a step (ties go to the even number), rows
    of zeros, of the smallest numbers, of one large value, of infinities and
    NaN, which spoil their own row alone."""
    hd, rows = 64, []
    d = np.float32(0.03125)
    ties = (np.arange(hd, dtype=np.float32) - 31 + 0.5) * d  # x / d is k + 1/2 exactly
    ties[0] = 127 * d
    rows += [ties, -ties, np.nextafter(ties, np.float32(np.inf)), np.nextafter(ties, np.float32(-np.inf))]
    third = np.float32(1 / 3)
    rows.append(np.where(np.arange(hd) == 7, third, (np.arange(hd) + np.float32(0.5)) * (third / 127)))
    rows.append(np.zeros(hd))
    tiny = np.zeros(hd)
    tiny[3], tiny[9] = 2.0 ** -24, -(2.0 ** -23)  # binary16's smallest
    rows.append(tiny)
    if dtype == SYN_F32:
        rows += [np.where(np.arange(hd) < 3, 1e-44, 0.0), np.where(np.arange(hd) < 3, 3e38, 1e-3),
                 np.linspace(-1e-40, 1e-40, hd), np.full(hd, 1e-45)]
    else:
        rows.append(np.linspace(-65504, 65504, hd))
    for bad in (np.inf, -np.inf, np.nan):
        r = np.linspace(-1, 1, hd)
        r[13] = bad
        rows.append(r)
    x = np.stack(rows).astype(np.float32)
    if dtype == SYN_F16:
        x = x.astype(np.float16).astype(np.float32)
    x = np.stack([x, x[::-1]])[:, :, None]  # one KV head
    cache = capi.kv8_state(room, 64, 1, hd)
    append8(room, cache, x[0], x[1], 9, dtype)
    k, v = read8(room, cache, x.shape[1], 9)
    want = _want(x, SYN_F32)
    assert np.array_equal(k, want[0], equal_nan=True) and np.array_equal(v, want[1], equal_nan=True)
    assert np.isnan(want).any(-1).sum() == 6


def test_rows_off_sixteen_bytes(room):
    """Rows at offsets that only their type aligns."""
    g = np.random.default_rng(8)
    for hd, dtype, np_t in ((64, SYN_F32, np.float32), (64, SYN_F16, np.float16), (20, SYN_F16, np.float16)):
        cache, L = capi.kv8_state(room, 70, 2, hd), lib()
        x = _rows(g, 66, 2, hd, dtype)
        el = np.dtype(np_t).itemsize
        at = [room.alloc(x[0].size * el + 16) + el for _ in range(4)]
        room.upload(at[0], x[0].astype(np_t))
        room.upload(at[1], x[1].astype(np_t))
        capi.check(L.syn_hip_kv8_append(room.handle, ctypes.byref(cache), at[0], at[1], 66, 3, dtype))
        capi.check(L.syn_hip_kv8_read(room.handle, ctypes.byref(cache), at[2], at[3], 66, 3, dtype))
        for i in range(2):
            got = room.download(at[2 + i], x[i].shape, np_t)
            assert np.array_equal(got, _want(x[i], dtype)), (hd, dtype)


ROWS = [[0], [5], [0, 1, 2], [0, 2, 3, 9], [1, 2, 3, 4], [0, 3, 4, 5, 6, 7, 8, 9, 10, 11, 12, 20],
        list(range(1, 290)), [0, 1, *range(3, 280, 2)]]


@pytest.mark.parametrize("rows", ROWS, ids=lambda r: f"{len(r)}of{r[-1] + 1}")
@pytest.mark.parametrize("n_kv,hd", [(8, 128), (3, 18), (1, 256)])
def test_keep_8bit(room, rows, n_kv, hd):
    n = rows[-1] + 1
    pos = 61
    x = _rows(np.random.default_rng(len(rows)), pos + n + 5, n_kv, hd)
    cache = capi.kv8_state(room, pos + n + 5, n_kv, hd)
    append8(room, cache, x[0], x[1], 0)
    want = values(x).astype(np.float32)
    want[:, pos:pos + len(rows)] = want[:, pos + np.array(rows)].copy()
    keep(room, cache, pos, n, rows)
    k, v = read8(room, cache, pos + n + 5, 0)
    assert np.array_equal(k, want[0]) and np.array_equal(v, want[1])


@pytest.mark.parametrize("rows", ROWS, ids=lambda r: f"{len(r)}of{r[-1] + 1}")
@pytest.mark.parametrize("n_kv,hd", [(8, 128), (3, 18), (1, 256)])
def test_keep_binary16(room, rows, n_kv, hd):
    """Any bit pattern moves as it is, V^T's padding and all other rows stay."""
    g = np.random.default_rng(len(rows))
    n, pos = rows[-1] + 1, 61
    cache = capi.kv_state(room, pos + n + 5, n_kv, hd)
    k = g.integers(0, 1 << 16, (cache.max_ctx, n_kv * hd), dtype=np.uint16)
    vt = g.integers(0, 1 << 16, (n_kv * hd, cache.ctx_stride), dtype=np.uint16)
    room.upload(cache.k_offset, k)
    room.upload(cache.v_offset, vt)
    keep(room, cache, pos, n, rows)
    k[pos:pos + len(rows)] = k[pos + np.array(rows)].copy()
    vt[:, pos:pos + len(rows)] = vt[:, pos + np.array(rows)].copy()
    assert np.array_equal(room.download(cache.k_offset, k.shape, np.uint16), k)
    assert np.array_equal(room.download(cache.v_offset, vt.shape, np.uint16), vt)


def test_refusals_leave_the_arena_alone():
    with Arena(32 << 20) as a:
        a.fill(0, 0x5a, 32 << 20)
        for name, code, call in refusals():
            assert call(a.handle) == code, name
        a.sync()
        assert (a.download(0, (32 << 20,), np.uint8) == 0x5a).all()


def test_append_keep_and_read_captured(room):
    """The three in one HIP graph, replayed between other work on the arena,
    against the same calls made one by one."""
    n_kv, hd, n, pos, rows = 4, 128, 9, 120, [0, 3, 4, 8]
    g = wl.rng(77)
    L, cache, other = lib(), capi.kv8_state(room, 256, n_kv, hd), capi.kv8_state(room, 256, n_kv, hd)
    at = [room.alloc(n * n_kv * hd * 4) for _ in range(4)]
    arr = (ctypes.c_uint32 * 4)(*rows)

    def record():
        capi.check(L.syn_hip_kv8_append(room.handle, ctypes.byref(cache), at[0], at[1], n, pos, SYN_F32))
        capi.check(L.syn_hip_kv8_keep(room.handle, ctypes.byref(cache), pos, n, arr, 4))
        capi.check(L.syn_hip_kv8_read(room.handle, ctypes.byref(cache), at[2], at[3], n, pos, SYN_F32))

    with capi.HipGraph(room, record) as graph:
        assert graph.nodes == 3
        for _ in range(4):
            x = _rows(g, n, n_kv, hd)
            room.upload(at[0], x[0])
            room.upload(at[1], x[1])
            append8(room, other, x[1], x[0], pos)
            graph.launch()
            room.sync()
            want = _want(x, SYN_F32)
            want[:, :4] = want[:, rows].copy()
            for i in range(2):
                assert np.array_equal(room.download(at[2 + i], (n, n_kv, hd), np.float32), want[i])
