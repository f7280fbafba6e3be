"""Attention over 8-bit states (causal runs and drafted trees) and drafted
trees over binary16 states, against the formula in 64 bits."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

from gpu_util import SYN_F16, SYN_F32, Arena, attention, capi, check, lib, scratch_for
from kv8_util import (append8, assert_held, attend8, attend64, attend_tree, causal, keep, random_tree, read8,
                      tree_sees, values)

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def arena():
    a = Arena(512 << 20)
    yield a
    a.close()


@pytest.fixture
def room(arena):
    mark = arena.top
    arena.fill(mark, 0xff, 96 << 20)  # NaN wherever nothing was written
    yield arena
    arena.top = mark


def _state8(arena, g, length, max_ctx, n_kv, hd, scale=1.0):
    x = (g.standard_normal((2, length, n_kv, hd)) * scale).astype(np.float32)
    cache = capi.kv8_state(arena, max_ctx, n_kv, hd)
    append8(arena, cache, x[0], x[1], 0)
    return cache, values(x[0]), values(x[1])


def _state16(arena, g, length, max_ctx, n_kv, hd, fill=0x7e00):
    """A binary16 state, NaN (or another pattern) behind its rows."""
    cache = capi.kv_state(arena, max_ctx, n_kv, hd)
    x = g.standard_normal((2, length, n_kv, hd)).astype(np.float16)
    k = np.full((max_ctx, n_kv * hd), fill, np.uint16)
    vt = np.full((n_kv * hd, cache.ctx_stride), fill, np.uint16)
    k[:length] = x[0].reshape(length, -1).view(np.uint16)
    vt[:, :length] = x[1].reshape(length, -1).view(np.uint16).T
    arena.upload(cache.k_offset, k)
    arena.upload(cache.v_offset, vt)
    return cache, x[0].astype(np.float64), x[1].astype(np.float64)


# (query heads, KV heads, head size): groups of 1, 4, 7, 20 and 33, every
# compiled head size, whole and broken 16s and 32s.
HEADS = [(32, 8, 128), (14, 2, 64), (4, 4, 32), (20, 1, 96), (33, 1, 16), (3, 3, 2), (6, 2, 40), (2, 1, 18),
         (8, 2, 160), (4, 1, 192), (2, 1, 224), (4, 2, 256), (2, 2, 130), (8, 4, 80)]


@pytest.mark.parametrize("n_heads,n_kv,hd", HEADS)
@pytest.mark.parametrize("pos,n", [(0, 1), (5, 1), (63, 1), (64, 1), (300, 1), (1000, 1), (0, 3), (61, 17), (200, 40)])
def test_causal_8bit(room, n_heads, n_kv, hd, pos, n):
    g = np.random.default_rng(pos * 100 + n + hd)
    cache, k, v = _state8(room, g, pos + n, pos + n + 3, n_kv, hd)
    q = g.standard_normal((n, n_heads * hd)).astype(np.float32)
    want, tol = attend64(q, k, v, n_heads, hd ** -0.5, causal(n, pos))
    assert_held(attend8(room, cache, q, pos, n_heads, hd ** -0.5), want, tol)


@pytest.mark.parametrize("n_heads,n_kv,hd,pos,n", [(32, 8, 128, 3000, 1), (8, 8, 64, 5001, 1), (4, 1, 128, 20000, 1),
                                                   (8, 2, 128, 700, 150), (4, 2, 256, 500, 70), (2, 1, 96, 0, 260)])
@pytest.mark.parametrize("q_dtype", [SYN_F32, SYN_F16])
def test_causal_8bit_longer(room, n_heads, n_kv, hd, pos, n, q_dtype):
    g = np.random.default_rng(pos + n)
    cache, k, v = _state8(room, g, pos + n, pos + n, n_kv, hd)
    q = (3 * g.standard_normal((n, n_heads * hd))).astype(np.float32)
    want, tol = attend64(q, k, v, n_heads, hd ** -0.5, causal(n, pos))
    assert_held(attend8(room, cache, q, pos, n_heads, hd ** -0.5, q_dtype=q_dtype), want, tol)


def test_run_is_its_tokens_one_by_one(room):
    """kv8_attention token by token, in uneven runs, and as one run."""
    n_heads, n_kv, hd, n = 8, 2, 64, 150
    g = np.random.default_rng(12)
    q = g.standard_normal((n, n_heads * hd)).astype(np.float32)
    x = g.standard_normal((2, n, n_kv, hd)).astype(np.float32)
    want, tol = attend64(q, values(x[0]), values(x[1]), n_heads, 0.125, causal(n, 0))
    for lengths in ([1] * n, [1, 62, 5, 80, 2], [n]):
        cache = capi.kv8_state(room, n, n_kv, hd)
        at = 0
        for m in lengths:
            part = slice(at, at + m)
            got = attend8(room, cache, q[part], at, n_heads, 0.125, rows=(x[0, part], x[1, part]))
            assert_held(got, want[part], tol[part], f"{m} at {at}")
            at += m


def test_steps_of_any_size(room):
    """V rows whose steps span 60 powers of two, and scores that pick each of
    them: a row's output keeps its own precision down to 2^-17 of the largest
    step, and what is smaller is right to that."""
    n_heads, n_kv, hd, n = 1, 1, 32, 330
    g = np.random.default_rng(4)
    for top in (2.0 ** -100, 1.0, 2.0 ** 100):
        x = g.standard_normal((2, n, 1, hd)).astype(np.float32)
        size = 2.0 ** -g.integers(0, 60, n).astype(np.float64)
        size[5], size[200] = 1.0, 1.0
        x[1] *= (top * size).astype(np.float32)[:, None, None]
        cache = capi.kv8_state(room, n, n_kv, hd)
        append8(room, cache, x[0], x[1], 0)
        q = x[0, :, 0, :] * 8
        for i in (5, 200, int(np.argmin(size)), 77):
            want, tol = attend64(q[i:i + 1], values(x[0]), values(x[1]), 1, 1.0, np.ones((1, n), bool))
            got = attend8(room, cache, q[i:i + 1], n - 1, 1, 1.0)
            # p v in halves against the largest step: 2^-25 of 2^6 p at most 2^14 under it, 127 steps a value
            floor = 2.0 ** -30 * 127 * np.abs(values(x[1])).max() / 127 * n
            assert np.all(np.abs(got - want) <= tol + floor), (top, i)


def test_scores_far_apart(room):
    """Scores of +-300 rising and falling over the tiles: the running maximum
    is followed and everything rescaled, several times a row."""
    n_heads, n_kv, hd, n = 4, 1, 64, 777
    g = np.random.default_rng(9)
    for order in (1, -1):
        x = g.standard_normal((2, n, 1, hd)).astype(np.float32)
        x[0] *= np.linspace(0.1, 5, n)[::order, None, None].astype(np.float32)
        cache = capi.kv8_state(room, n, n_kv, hd)
        append8(room, cache, x[0], x[1], 0)
        q = (6 * g.standard_normal((1, n_heads * hd))).astype(np.float32)
        want, tol = attend64(q, values(x[0]), values(x[1]), n_heads, 1.0, np.ones((1, n), bool))
        got = attend8(room, cache, q, n - 1, n_heads, 1.0)
        assert np.all(np.abs(got - want) <= tol)


TREES = [(32, 8, 128), (14, 2, 64), (20, 1, 96), (3, 3, 2), (6, 2, 40), (2, 1, 18), (8, 2, 160), (4, 2, 256), (3, 1, 12)]


@pytest.mark.parametrize("n_heads,n_kv,hd", TREES)
@pytest.mark.parametrize("pos,n", [(0, 1), (0, 9), (1, 33), (63, 2), (64, 64), (130, 31), (700, 70)])
@pytest.mark.parametrize("eight", [False, True])
def test_tree(room, n_heads, n_kv, hd, pos, n, eight):
    g = np.random.default_rng(pos * 100 + n + hd)
    cache, k, v = (_state8 if eight else _state16)(room, g, pos + n, pos + n + 7, n_kv, hd)
    q = g.standard_normal((n, n_heads * hd)).astype(np.float32)
    mask = random_tree(g, n)
    want, tol = attend64(q, k, v, n_heads, hd ** -0.5, tree_sees(mask, n, pos))
    if eight:
        got = attend8(room, cache, q, pos, n_heads, hd ** -0.5, mask=mask)
    else:
        got = attend_tree(room, cache, q, pos, n_heads, hd ** -0.5, mask)
    assert_held(got, want, tol)


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("pos", [0, 100])
def test_any_mask(room, eight, pos):
    """Patterns that are no trees: empty rows (zeros with no cache before
    them), full ones, tokens that see later ones; bits past the last token."""
    n_heads, n_kv, hd, n = 8, 2, 64, 45
    g = np.random.default_rng(pos)
    cache, k, v = (_state8 if eight else _state16)(room, g, pos + n, pos + n, n_kv, hd)
    q = g.standard_normal((n, n_heads * hd)).astype(np.float32)
    mask = g.integers(0, 1 << 32, (n, 2), dtype=np.uint64).astype(np.uint32)
    mask[3] = mask[17] = 0
    mask[4] = 0xffffffff
    mask[5] = [0, 0xffffe000]  # only bits past token 44
    want, tol = attend64(q, k, v, n_heads, 0.125, tree_sees(mask, n, pos))
    got = attend8(room, cache, q, pos, n_heads, 0.125, mask=mask) if eight else \
        attend_tree(room, cache, q, pos, n_heads, 0.125, mask)
    assert_held(got, want, tol)
    if pos == 0:
        assert not got[3].any() and not got[17].any() and not got[5].any()


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
def test_wild_values_reach_only_who_attends_them(room, eight, bad):
    n_heads, n_kv, hd, pos, n = 8, 2, 64, 70, 40
    g = np.random.default_rng(2)
    x = g.standard_normal((2, pos + n, n_kv, hd)).astype(np.float32)
    x[1, pos + 6, 0, 11] = bad    # V of drafted token 6
    x[0, pos + 33, 1, 3] = np.nan  # K of drafted token 33
    parents = [int(g.integers(max(-1, i - 4), i)) for i in range(n)]
    mask = capi.tree_mask(parents)
    if eight:
        cache = capi.kv8_state(room, pos + n + 9, n_kv, hd)
        append8(room, cache, x[0], x[1], 0)
        k, v = values(x[0]), values(x[1])
    else:
        cache = capi.kv_state(room, pos + n + 9, n_kv, hd)
        h = x.astype(np.float16)
        kc = np.full((cache.max_ctx, n_kv * hd), 0x7e00, np.uint16)
        vt = np.full((n_kv * hd, cache.ctx_stride), 0xfc00, np.uint16)
        kc[:pos + n] = h[0].reshape(pos + n, -1).view(np.uint16)
        vt[:, :pos + n] = h[1].reshape(pos + n, -1).view(np.uint16).T
        room.upload(cache.k_offset, kc)
        room.upload(cache.v_offset, vt)
        k, v = h.astype(np.float64)
    q = g.standard_normal((n, n_heads * hd)).astype(np.float32)
    sees = tree_sees(mask, n, pos)
    assert 0 < sees[:, pos + 6].sum() < n and 0 < sees[:, pos + 33].sum() < n
    want, tol = attend64(q, k, v, n_heads, 0.125, sees)
    got = attend8(room, cache, q, pos, n_heads, 0.125, mask=mask) if eight else \
        attend_tree(room, cache, q, pos, n_heads, 0.125, mask)
    assert_held(got, want, tol)
    assert np.isnan(want).any() or np.isinf(want).any()


def test_causal_run_with_wild_rows_8bit(room):
    """A NaN row of V makes NaN of the tokens from its own on, no earlier one."""
    n_heads, n_kv, hd, n = 4, 2, 32, 90
    g = np.random.default_rng(3)
    x = g.standard_normal((2, n, n_kv, hd)).astype(np.float32)
    x[1, 50, 1, 0] = np.inf
    cache = capi.kv8_state(room, n, n_kv, hd)
    append8(room, cache, x[0], x[1], 0)
    q = g.standard_normal((n, n_heads * hd)).astype(np.float32)
    want, tol = attend64(q, values(x[0]), values(x[1]), n_heads, 0.2, causal(n, 0))
    assert np.isnan(want[50:, 2 * hd:]).all() and np.isfinite(want[:50]).all()
    assert_held(attend8(room, cache, q, 0, n_heads, 0.2), want, tol)


# (query heads, KV heads, head size, tokens): up to 16 rows a KV head, 64, 128, and more.
ROW_COUNTS = [(2, 1, 64, 8), (4, 2, 64, 30), (8, 2, 64, 29), (8, 2, 64, 45), (8, 2, 96, 75), (8, 2, 160, 45), (4, 1, 18, 45)]


@pytest.mark.parametrize("n_heads,n_kv,hd,n", ROW_COUNTS)
@pytest.mark.parametrize("pos,tree", [(0, False), (40, False), (40, True), (100, True)])
def test_larger_steps_of_unseen_keys(room, n_heads, n_kv, hd, n, pos, tree):
    """V rows that grow from token to token, by 2^160 in all: each token's
    output is right to the values it sees itself, however much larger those
    are that it does not see."""
    g = np.random.default_rng(pos + n)
    x = g.standard_normal((2, pos + n, n_kv, hd)).astype(np.float32)
    x[1, pos:] *= (2.0 ** np.linspace(-80, 80, n)).astype(np.float32)[:, None, None]
    x[1, :pos] *= np.float32(2.0 ** -80)
    cache = capi.kv8_state(room, pos + n + 3, n_kv, hd)
    append8(room, cache, x[0], x[1], 0)
    q = g.standard_normal((n, n_heads * hd)).astype(np.float32)
    mask = random_tree(g, n) if tree else None
    sees = tree_sees(mask, n, pos) if tree else causal(n, pos)
    want, tol = attend64(q, values(x[0]), values(x[1]), n_heads, 0.125, sees)
    got = attend8(room, cache, q, pos, n_heads, 0.125, mask=mask)
    for i in range(n):
        assert_held(got[i:i + 1], want[i:i + 1], tol[i:i + 1], f"token {i}")


# Calls whose blocks fill the CUs, so that rows go to the kernels of 32 rows a
# wave: (query heads, KV heads, head size, tokens) behind some 800 keys.
FULL = [(256, 64, 128, 33), (256, 64, 64, 50), (64, 64, 32, 200), (448, 64, 96, 37), (192, 64, 40, 61), (128, 64, 80, 100),
        (128, 64, 128, 40), (128, 64, 160, 50), (128, 64, 256, 37), (64, 64, 224, 90)]


@pytest.mark.parametrize("n_heads,n_kv,hd,n", FULL)
@pytest.mark.parametrize("kind", ["causal8", "tree8", "tree16"])
def test_many_blocks(room, n_heads, n_kv, hd, n, kind):
    """Growing V steps (8-bit), infinities and NaN among the drafted or later
    rows, and NaN behind them; two of the KV heads checked."""
    pos, group = 800 - n // 2, n_heads // n_kv
    g = np.random.default_rng(hd + n)
    eight = kind != "tree16"
    x = g.standard_normal((2, pos + n, n_kv, hd)).astype(np.float32 if eight else np.float16)
    if eight:
        x[1, pos:] *= (2.0 ** np.linspace(-20, 20, n)).astype(np.float32)[:, None, None]
        x[1, :pos] *= np.float32(2.0 ** -20)
    for j, bad in ((n - 9, np.inf), (n - 7, -np.inf), (n - 5, np.nan)):
        x[1, pos + j, n_kv - 1, j % hd] = bad
    x[0, pos + n - 6, 0, 1] = np.nan
    if eight:
        cache = capi.kv8_state(room, pos + n + 70, n_kv, hd)
        append8(room, cache, x[0], x[1], 0)
    else:
        cache = capi.kv_state(room, pos + n + 70, n_kv, hd)
        vt = np.full((n_kv * hd, cache.ctx_stride), 0x7c00, np.uint16)
        vt[:, :pos + n] = x[1].reshape(pos + n, -1).view(np.uint16).T
        room.upload(cache.k_offset, np.ascontiguousarray(x[0]))
        room.upload(cache.v_offset, vt)
    q = g.standard_normal((n, n_heads * hd)).astype(np.float32)
    mask = None if kind == "causal8" else capi.tree_mask([int(g.integers(max(-1, i - 4), i)) for i in range(n)])
    sees = causal(n, pos) if mask is None else tree_sees(mask, n, pos)
    got = attend_tree(room, cache, q, pos, n_heads, 0.125, mask) if not eight else \
        attend8(room, cache, q, pos, n_heads, 0.125, mask=mask)
    heads = [0, n_kv - 1]
    some = [y.reshape(n, n_kv, group * hd)[:, heads].reshape(n, -1) for y in (q, got)]
    k, v = ((values(y[:, heads]) if eight else y[:, heads].astype(np.float64)) for y in x)
    want, tol = attend64(some[0], k, v, 2 * group, 0.125, sees)
    assert np.isfinite(want).any() and not np.isfinite(want).all()
    for i in range(n):
        assert_held(some[1][i:i + 1], want[i:i + 1], tol[i:i + 1], f"token {i}")


@pytest.mark.parametrize("n_heads,n_kv,hd,n", ROW_COUNTS)
@pytest.mark.parametrize("eight", [False, True])
def test_wild_rows_at_every_row_count(room, n_heads, n_kv, hd, n, eight):
    """Infinities and NaN in drafted K and V rows, in a tile that ends inside
    the state and one that does not; what lies behind the rows is NaN too."""
    pos = 57
    g = np.random.default_rng(n + hd)
    x = g.standard_normal((2, pos + n, n_kv, hd)).astype(np.float32)
    for j, bad in ((2, np.inf), (3, -np.inf), (5, np.nan), (n - 1, np.inf)):
        x[1, pos + j, 0, j % hd] = bad
    x[0, pos + 4, n_kv - 1, 1] = np.nan
    if eight:
        cache = capi.kv8_state(room, pos + n + 70, n_kv, hd)
        append8(room, cache, x[0], x[1], 0)
        k, v = values(x[0]), values(x[1])
    else:
        cache, k, v = _state16(room, g, pos + n, pos + n + 70, n_kv, hd)
        rows = x.astype(np.float16)
        kc = np.full((cache.max_ctx, n_kv * hd), 0x7e00, np.uint16)
        vt = np.full((n_kv * hd, cache.ctx_stride), 0x7c00, np.uint16)
        kc[:pos + n] = rows[0].reshape(pos + n, -1).view(np.uint16)
        vt[:, :pos + n] = rows[1].reshape(pos + n, -1).view(np.uint16).T
        room.upload(cache.k_offset, kc)
        room.upload(cache.v_offset, vt)
        k, v = rows.astype(np.float64)
    q = g.standard_normal((n, n_heads * hd)).astype(np.float32)
    mask = capi.tree_mask([int(g.integers(max(-1, i - 4), i)) for i in range(n)])
    want, tol = attend64(q, k, v, n_heads, 0.125, tree_sees(mask, n, pos))
    got = attend8(room, cache, q, pos, n_heads, 0.125, mask=mask) if eight else \
        attend_tree(room, cache, q, pos, n_heads, 0.125, mask)
    assert np.isfinite(want).any() and not np.isfinite(want).all()
    assert_held(got, want, tol)


@pytest.mark.parametrize("n_heads,n_kv,hd,n", ROW_COUNTS)
@pytest.mark.parametrize("eight", [False, True])
def test_tree_of_binary16_queries(room, n_heads, n_kv, hd, n, eight):
    g = np.random.default_rng(n)
    pos = 190
    cache, k, v = (_state8 if eight else _state16)(room, g, pos + n, pos + n, n_kv, hd)
    q = g.standard_normal((n, n_heads * hd)).astype(np.float16)
    mask = random_tree(g, n)
    want, tol = attend64(q, k, v, n_heads, 0.125, tree_sees(mask, n, pos))
    got = attend8(room, cache, q, pos, n_heads, 0.125, mask=mask, q_dtype=SYN_F16) if eight else \
        attend_tree(room, cache, q, pos, n_heads, 0.125, mask, q_dtype=SYN_F16)
    assert_held(got, want, tol)


@pytest.mark.parametrize("pos", [0, 63, 64, 500])
@pytest.mark.parametrize("kv_dtype", [SYN_F32, SYN_F16])
def test_append_and_attend_in_one_call(room, pos, kv_dtype):
    """syn_hip_kv8_attention for one token and for a run, against its two halves."""
    n_heads, n_kv, hd = 8, 2, 128
    g = np.random.default_rng(pos)
    for n in (1, 40):
        x = g.standard_normal((2, pos + n, n_kv, hd)).astype(np.float16 if kv_dtype == SYN_F16 else np.float32)
        one, two = (capi.kv8_state(room, pos + n, n_kv, hd) for _ in range(2))
        q = g.standard_normal((n, n_heads * hd)).astype(np.float32)
        append8(room, two, x[0], x[1], 0, kv_dtype)
        if pos:
            append8(room, one, x[0, :pos], x[1, :pos], 0, kv_dtype)
        got = attend8(room, one, q, pos, n_heads, 0.1, rows=(x[0, pos:], x[1, pos:]), kv_dtype=kv_dtype)
        assert np.array_equal(got, attend8(room, two, q, pos, n_heads, 0.1))
        for a, b in zip(read8(room, one, pos + n, 0), read8(room, two, pos + n, 0)):
            assert np.array_equal(a, b)


def test_a_chain_is_a_causal_run(room):
    """A tree with one branch equals the framework's causal attention to that
    kernel's binary16 probabilities (2^-11 each way), and kv8_attend's own."""
    n_heads, n_kv, hd, pos, n = 16, 4, 128, 300, 20
    g = np.random.default_rng(6)
    chain = capi.tree_mask(list(range(-1, n - 1)))
    q = g.standard_normal((n, n_heads * hd)).astype(np.float32)
    c16, k, v = _state16(room, g, pos + n, pos + n, n_kv, hd)
    got = attend_tree(room, c16, q, pos, n_heads, 0.1, chain)
    zero = np.zeros((n, n_kv * hd), np.float32)
    causal_out = attention(room, c16, scratch_for(room, n_heads, n_kv, hd, pos + n), q, zero, zero, pos, n_heads, 0.1,
                           append=False)
    assert np.abs(got - causal_out).max() <= 2.0 ** -10 * np.abs(v).max()
    c8, _, _ = _state8(room, g, pos + n, pos + n, n_kv, hd)
    a, b = attend8(room, c8, q, pos, n_heads, 0.1, mask=chain), attend8(room, c8, q, pos, n_heads, 0.1)
    assert np.linalg.norm(a - b) <= 1e-6 * np.linalg.norm(b)


def test_a_speculative_step(room):
    """As a serving program runs them, with either state: a prompt, a drafted
    tree appended behind it and attended at once, the accepted path kept, and
    the next token -- each output that of the tokens taken one by one."""
    n_heads, n_kv, hd, prompt, scale = 8, 2, 64, 91, 0.125
    g = np.random.default_rng(21)
    parents = [-1, 0, 0, 1, 1, 2, 3, 3, 4, 6, 6, 9]
    path = [0, 1, 3, 6, 9]
    n, total = len(parents), prompt + len(parents) + 1
    q = g.standard_normal((total, n_heads * hd)).astype(np.float32)
    x = g.standard_normal((2, total, n_kv, hd)).astype(np.float32)
    mask = capi.tree_mask(parents)
    for eight in (False, True):
        if eight:
            cache = capi.kv8_state(room, total, n_kv, hd)
            k, v = values(x[0]), values(x[1])

            def step(rows, pos, mask=None):
                return attend8(room, cache, q[rows], pos, n_heads, scale, mask=mask, rows=(x[0, rows], x[1, rows]))
        else:
            cache = capi.kv_state(room, total, n_kv, hd)
            k, v = x.astype(np.float16).astype(np.float64)
            scratch = scratch_for(room, n_heads, n_kv, hd, total)

            def step(rows, pos, mask=None):
                kr, vr = (a[rows].reshape(len(q[rows]), -1) for a in x)
                if mask is None:
                    return attention(room, cache, scratch, q[rows], kr, vr, pos, n_heads, scale)
                mark = room.top
                at = room.put(kr), room.put(vr)
                check(lib().syn_hip_kv_append(room.handle, ctypes.byref(cache), *at, len(kr), pos, SYN_F32))
                out = attend_tree(room, cache, q[rows], pos, n_heads, scale, mask)
                room.top = mark
                return out
        close = 1e-5 if eight else 1e-3  # the framework's binary16 kernels round probabilities to 2^-12
        step(slice(0, prompt), 0)
        drafted = slice(prompt, prompt + n)
        got = step(drafted, prompt, mask)
        want, tol = attend64(q[drafted], k[:prompt + n], v[:prompt + n], n_heads, scale, tree_sees(mask, n, prompt))
        assert_held(got, want, tol)
        keep(room, cache, prompt, n, path)
        at = prompt + len(path)
        last = total - 1
        got = step(slice(last, last + 1), at)
        order = [*range(prompt), *(prompt + i for i in path), last]
        want, _ = attend64(q[last:], k[order], v[order], n_heads, scale, np.ones((1, len(order)), bool))
        assert np.linalg.norm(got - want) <= close * np.linalg.norm(want), eight


def test_captured_steps_share_their_scratch(room):
    """Two captured steps (a token on an 8-bit state, a tree on a binary16
    one) with one scratch range, replayed in turn between eager work."""
    n_heads, n_kv, hd, L = 8, 2, 128, lib()
    g = np.random.default_rng(31)
    c8, _, _ = _state8(room, g, 3000, 3000, n_kv, hd)
    c16, _, _ = _state16(room, g, 2500, 2500, n_kv, hd)
    mask = random_tree(g, 12)
    need = max(int(L.syn_hip_kv8_attention_scratch_bytes(n_heads, n_kv, hd, 3000, 1)),
               int(L.syn_hip_attend_tree_scratch_bytes(n_heads, n_kv, hd, 2500, 12)))
    scratch = room.alloc(need)
    q8, q16 = (room.put(g.standard_normal((m, n_heads * hd)).astype(np.float32)) for m in (1, 12))
    o8, o16 = room.alloc(n_heads * hd * 4), room.alloc(12 * n_heads * hd * 4)
    d8 = capi.Kv8AttnDesc(cache=c8, q_offset=q8, out_offset=o8, scratch_offset=scratch, scratch_bytes=need,
                          mask_offset=capi.NO_OFFSET, n_heads=n_heads, pos=2999, n=1, scale=0.1)
    d16 = capi.AttnDesc(cache=c16, q_offset=q16, out_offset=o16, scratch_offset=scratch, scratch_bytes=need,
                        n_heads=n_heads, pos=2488, n=12, scale=0.1, q_dtype=SYN_F32, kv_dtype=SYN_F16)
    m_off = room.put(mask, 4)
    calls = [(lambda: check(L.syn_hip_kv8_attend(room.handle, ctypes.byref(d8))), o8, 1),
             (lambda: check(L.syn_hip_attend_tree(room.handle, ctypes.byref(d16), m_off)), o16, 12)]

    def out(i):
        return room.download(calls[i][1], (calls[i][2], n_heads * hd), np.float32)

    eager = []
    for i, (call, *_) in enumerate(calls):
        call()
        eager.append(out(i))
    graphs = [capi.HipGraph(room, call) for call, *_ in calls]
    try:
        for _ in range(4):
            for i in (0, 1):
                room.fill(calls[i][1], 0xff, calls[i][2] * n_heads * hd * 4)
            graphs[0].launch()
            graphs[1].launch()
            calls[1][0]()
            graphs[0].launch()
            room.sync()
            for i in (0, 1):
                assert np.array_equal(out(i), eager[i])
    finally:
        for graph in graphs:
            graph.close()


def test_nothing_outside_is_written(room):
    """Output rows and scratch end where they end; the state is only read."""
    n_heads, n_kv, hd, pos, n = 8, 2, 64, 1000, 5
    g = np.random.default_rng(1)
    cache, k, v = _state8(room, g, pos + n, pos + n + 40, n_kv, hd)
    L, size = lib(), capi.kv8_state_bytes(cache.max_ctx, n_kv, hd)
    need = int(L.syn_hip_kv8_attention_scratch_bytes(n_heads, n_kv, hd, cache.max_ctx, n))
    q = g.standard_normal((n, n_heads * hd)).astype(np.float32)
    at = room.put(q)
    guard = 4096
    base = room.alloc(guard + need + guard + q.nbytes + guard)
    room.fill(base, 0xa5, guard + need + guard + q.nbytes + guard)
    scratch, out = base + guard, base + guard + (need + guard)
    before = room.download(cache.offset, (size,), np.uint8)
    d = capi.Kv8AttnDesc(cache=cache, q_offset=at, out_offset=out, scratch_offset=scratch, scratch_bytes=need,
                         mask_offset=capi.NO_OFFSET, n_heads=n_heads, pos=pos, n=n, scale=0.125)
    check(L.syn_hip_kv8_attend(room.handle, ctypes.byref(d)))
    want, tol = attend64(q, k, v, n_heads, 0.125, causal(n, pos))
    assert_held(room.download(out, q.shape, np.float32), want, tol)
    for lo in (base, scratch + need, out + q.nbytes):
        assert (room.download(lo, (guard,), np.uint8) == 0xa5).all()
    assert np.array_equal(room.download(cache.offset, (size,), np.uint8), before)
    kk, vv = read8(room, cache, pos + n, 0)
    assert np.array_equal(kk, k.astype(np.float32)) and np.array_equal(vv, v.astype(np.float32))
