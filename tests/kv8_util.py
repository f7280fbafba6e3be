"""8-bit KV states and drafted trees: the operators in 64 bits, and helpers
that drive them through the C ABI."""
from __future__ import annotations

import ctypes

import numpy as np

from gpu_util import SYN_F16, SYN_F32, Arena, AttnDesc, capi, check, f16, lib, put_rows


def held(rows: np.ndarray) -> tuple[np.ndarray, np.ndarray]:
    """What a state holds for rows [..., hd] (f32 or f16 values): whole
    numbers and steps. The step is the f32 next to max|x| / 127 (a double
    quotient rounded to f32 is the f32 quotient); the double quotient x / step
    of two f32 numbers is never rounded onto a half, so np.rint of it is the
    nearest whole number of the exact one."""
    x = np.asarray(rows, dtype=np.float64)
    top = np.abs(x).max(-1)
    wild = ~np.isfinite(x).all(-1)
    step = np.where(wild, 0.0, top / 127.0).astype(np.float32)
    by = np.where(step == 0, 1.0, step.astype(np.float64))[..., None]
    q = np.where((step == 0)[..., None], 0.0, np.clip(np.rint(np.where(wild[..., None], 0.0, x) / by), -127, 127))
    return q + 0.0, np.where(wild, np.float32(np.nan), step)  # (whole numbers: no -0)


def values(rows: np.ndarray) -> np.ndarray:
    q, step = held(rows)
    return q * step.astype(np.float64)[..., None]


def attend64(q, k, v, n_heads, scale, sees):
    """q [n][n_heads*hd] as given (rounded to binary16 here), k, v [L][n_kv][hd]
    doubles, sees [n][L]: outputs [n][n_heads*hd], and a bound on an f32
    kernel's error per element.

    The bound. With u = 2^-24: a score is a sum of hd products, each exact in
    f32 (11 + 11 bits), so it is off by at most hd u A, A = scale sum |q k|,
    plus 4 u |s| for the step's, the scale's and the exponent's roundings: d =
    (hd + 4) u A. A weight is off by a factor within 1 +- (d ln... <= 2 d) and
    2 u of exp2, the hi/lo halves leave 2^-21 of it, and the sums of L
    weights and of L weighted values are off by at most L u each, relative to
    the sum of magnitudes. Numerator and denominator together: sum p |v|
    times (4 d + 4 u + 2^-21 + 2 L u), and a few u for the final division,
    scaling and merges (16 u). That is relative to the weights; besides, lo is
    a binary16 number, so a multiple of 2^-24 and off by up to 2^-25, in a
    weight that is 2^6 p (times its key's step over the largest one): 2^-31 of
    the largest |v| for each key, however small p is -- L 2^-31 max |v| in all
    (the sum of the p over the largest one is at least 1). An output that its
    weights make 1e-18 is right to that, not to its own size."""
    n, hd = q.shape[0], q.shape[1] // n_heads
    n_kv, L = k.shape[1], k.shape[0]
    u = 2.0 ** -24
    out = np.zeros((n, n_heads, hd))
    tol = np.zeros_like(out)
    q16 = np.asarray(q, np.float32).astype(np.float16).astype(np.float64).reshape(n, n_heads, hd)
    for h in range(n_heads):
        g = h // (n_heads // n_kv)
        for i in range(n):
            t = np.nonzero(sees[i])[0]
            if t.size == 0:
                continue
            s = scale * (k[t, g] @ q16[i, h])
            if np.isnan(s).any() or s.max() == np.inf:
                out[i, h] = np.nan
                continue
            p = np.exp(s - s.max())
            p /= p.sum()
            with np.errstate(invalid="ignore"):
                out[i, h] = p @ v[t, g]
                d = (hd + 4) * u * scale * (np.abs(k[t, g]) @ np.abs(q16[i, h])).max()
                tol[i, h] = (p @ np.abs(v[t, g])) * (4 * d + 20 * u + 2.0 ** -21 + 2 * L * u) \
                    + L * 2.0 ** -31 * np.abs(v[t, g]).max()
    return out.reshape(n, -1), tol.reshape(n, -1)


def causal(n: int, pos: int) -> np.ndarray:
    return np.arange(pos + n)[None, :] <= pos + np.arange(n)[:, None]


def tree_sees(mask_words: np.ndarray, n: int, pos: int) -> np.ndarray:
    bits = np.unpackbits(mask_words.view(np.uint8), axis=1, bitorder="little")[:, :n].astype(bool)
    return np.concatenate([np.ones((n, pos), bool), bits], 1)


def random_tree(g, n: int) -> np.ndarray:
    return capi.tree_mask([int(g.integers(max(-1, i - 6), i)) for i in range(n)])


def assert_held(got, want, tol, what=""):
    """Every element inside its bound, and the whole within 1e-5 in the
    2-norm: the errors the bound adds up are independent and mostly some u
    each, while a probability rounded to one half would be off by 2^-12."""
    got = np.asarray(got, np.float64)
    assert got.shape == want.shape
    assert np.array_equal(np.isnan(got), np.isnan(want)), (what, "NaN at", np.argwhere(np.isnan(got) != np.isnan(want))[:4])
    ok = np.isfinite(want)
    assert np.array_equal(got[~ok & ~np.isnan(want)], want[~ok & ~np.isnan(want)]), what
    diff = np.abs(got[ok] - want[ok])
    bad = diff > tol[ok]
    assert not bad.any(), (what, float(diff.max()), float(tol[ok][diff.argmax()]), int(bad.sum()))
    norm = np.linalg.norm(want[ok])
    if norm > 0:
        assert np.linalg.norm(diff) <= 1e-5 * norm, (what, np.linalg.norm(diff) / norm)


def append8(arena: Arena, cache, k, v, pos, dtype=SYN_F32):
    mark = arena.top
    check(lib().syn_hip_kv8_append(arena.handle, ctypes.byref(cache), put_rows(arena, k, dtype),
                                   put_rows(arena, v, dtype), len(k), pos, dtype))
    arena.sync()
    arena.top = mark


def read8(arena: Arena, cache, n, pos, dtype=SYN_F32):
    mark = arena.top
    el, np_t = (2, np.float16) if dtype == SYN_F16 else (4, np.float32)
    shape = (n, cache.n_kv_heads, cache.head_dim)
    k, v = (arena.alloc(int(np.prod(shape)) * el) for _ in range(2))
    check(lib().syn_hip_kv8_read(arena.handle, ctypes.byref(cache), k, v, n, pos, dtype))
    out = arena.download(k, shape, np_t), arena.download(v, shape, np_t)
    arena.top = mark
    return out


def attend8(arena: Arena, cache, q, pos, n_heads, scale, mask=None, q_dtype=SYN_F32, rows=None, kv_dtype=SYN_F32,
            scratch=None):
    """syn_hip_kv8_attend, or with rows (k, v) syn_hip_kv8_attention."""
    mark, n = arena.top, len(q)
    need = int(lib().syn_hip_kv8_attention_scratch_bytes(n_heads, cache.n_kv_heads, cache.head_dim, cache.max_ctx, n))
    at = scratch or (arena.alloc(max(need, 16)), need)
    d = capi.Kv8AttnDesc(cache=cache, q_offset=put_rows(arena, q, q_dtype), out_offset=arena.alloc(q.size * 4),
                         scratch_offset=at[0], scratch_bytes=at[1],
                         mask_offset=capi.NO_OFFSET if mask is None else arena.put(mask, 4), n_heads=n_heads, pos=pos,
                         n=n, scale=scale, q_dtype=q_dtype, kv_dtype=kv_dtype)
    if rows is not None:
        d.k_offset, d.v_offset = (put_rows(arena, x, kv_dtype) for x in rows)
    fn = lib().syn_hip_kv8_attend if rows is None else lib().syn_hip_kv8_attention
    check(fn(arena.handle, ctypes.byref(d)))
    out = arena.download(d.out_offset, q.shape, np.float32)
    arena.top = mark
    return out


def attend_tree(arena: Arena, cache, q, pos, n_heads, scale, mask, q_dtype=SYN_F32):
    mark, n = arena.top, len(q)
    need = int(lib().syn_hip_attend_tree_scratch_bytes(n_heads, cache.n_kv_heads, cache.head_dim, cache.max_ctx, n))
    d = AttnDesc(cache=cache, q_offset=put_rows(arena, q, q_dtype), out_offset=arena.alloc(q.size * 4),
                 scratch_offset=arena.alloc(max(need, 16)), scratch_bytes=need, n_heads=n_heads, pos=pos, n=n,
                 scale=scale, q_dtype=q_dtype, kv_dtype=SYN_F16)
    check(lib().syn_hip_attend_tree(arena.handle, ctypes.byref(d), arena.put(mask, 4)))
    out = arena.download(d.out_offset, q.shape, np.float32)
    arena.top = mark
    return out


def keep(arena: Arena, cache, pos, n, rows):
    fn = lib().syn_hip_kv8_keep if isinstance(cache, capi.Kv8Desc) else lib().syn_hip_kv_keep
    arr = (ctypes.c_uint32 * max(1, len(rows)))(*rows)
    check(fn(arena.handle, ctypes.byref(cache), pos, n, arr, len(rows)))


__all__ = ["held", "values", "attend64", "causal", "tree_sees", "random_tree", "assert_held", "append8", "read8",
           "attend8", "attend_tree", "keep", "f16"]
