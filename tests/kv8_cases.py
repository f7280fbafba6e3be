"""Calls on 8-bit KV states and drafted trees that have to be refused, for an
arena of 32 MiB: (name, status, call of the arena's handle)."""
from __future__ import annotations

import ctypes

from synapse_amd import capi

EINVAL, ERANGE = -1, -2
MIB = 1 << 20


def _copy(d, **changes):
    out = type(d).from_buffer_copy(d)
    for name, value in changes.items():
        setattr(out, name, value)
    return out


def refusals() -> list:
    L, ref = capi.lib(), ctypes.byref
    state = capi.Kv8Desc(offset=0, max_ctx=1000, n_kv_heads=2, head_dim=64)  # 279 KB
    state16 = capi.KvDesc(k_offset=0, v_offset=MIB, max_ctx=1000, n_kv_heads=2, head_dim=64, ctx_stride=1024)
    attn = capi.Kv8AttnDesc(cache=state, q_offset=4 * MIB, k_offset=5 * MIB, v_offset=6 * MIB, out_offset=7 * MIB,
                            scratch_offset=8 * MIB, scratch_bytes=8 * MIB, mask_offset=capi.NO_OFFSET, n_heads=8,
                            pos=900, n=5, scale=0.125, q_dtype=0, kv_dtype=0)
    tree = capi.AttnDesc(cache=state16, q_offset=4 * MIB, out_offset=7 * MIB, scratch_offset=8 * MIB,
                         scratch_bytes=8 * MIB, n_heads=8, pos=900, n=5, scale=0.125, q_dtype=0, kv_dtype=1)
    out = []

    def add(name, code, fn, d, *args):
        out.append((name, code, lambda a: fn(a, ref(d) if d is not None else None, *args)))

    for what, fn in (("append", L.syn_hip_kv8_append), ("read", L.syn_hip_kv8_read)):
        add(f"{what}: null", EINVAL, fn, None, 4 * MIB, 5 * MIB, 3, 0, 0)
        for field, value in (("max_ctx", 0), ("max_ctx", 0xffffffff), ("n_kv_heads", 0), ("n_kv_heads", 1 << 20),
                             ("head_dim", 0), ("head_dim", 63), ("head_dim", 258)):
            add(f"{what}: {field} {value}", EINVAL, fn, _copy(state, **{field: value}), 4 * MIB, 5 * MIB, 3, 0, 0)
        add(f"{what}: state off 256", EINVAL, fn, _copy(state, offset=128), 4 * MIB, 5 * MIB, 3, 0, 0)
        add(f"{what}: state past the arena", ERANGE, fn, _copy(state, offset=32 * MIB - 256), 4 * MIB, 5 * MIB, 3, 0, 0)
        add(f"{what}: state wraps", ERANGE, fn, _copy(state, offset=(1 << 64) - 256), 4 * MIB, 5 * MIB, 3, 0, 0)
        add(f"{what}: dtype", EINVAL, fn, state, 4 * MIB, 5 * MIB, 3, 0, 2)
        add(f"{what}: past the cache", EINVAL, fn, state, 4 * MIB, 5 * MIB, 3, 998, 0)
        add(f"{what}: position wraps", EINVAL, fn, state, 4 * MIB, 5 * MIB, 2, 0xffffffff, 0)
        add(f"{what}: k past the arena", ERANGE, fn, state, 32 * MIB - 4, 5 * MIB, 3, 0, 0)
        add(f"{what}: v past the arena", ERANGE, fn, state, 4 * MIB, 32 * MIB - 4, 3, 0, 0)
        add(f"{what}: k off its type", EINVAL, fn, state, 4 * MIB + 2, 5 * MIB, 3, 0, 0)
        add(f"{what}: v off its type", EINVAL, fn, state, 4 * MIB, 5 * MIB + 1, 3, 0, 1)
        add(f"{what}: k in the state", EINVAL, fn, state, 1024, 5 * MIB, 3, 0, 0)
        add(f"{what}: v in the state", EINVAL, fn, state, 4 * MIB, 1024, 3, 0, 0)
    add("read: v in k", EINVAL, L.syn_hip_kv8_read, state, 4 * MIB, 4 * MIB + 512, 3, 0, 0)

    mask = {"mask_offset": 3 * MIB}
    for what, fn, d, args in (("kv8_attention", L.syn_hip_kv8_attention, attn, ()),
                              ("kv8_attend", L.syn_hip_kv8_attend, attn, ()),
                              ("attend_tree", L.syn_hip_attend_tree, tree, (3 * MIB,))):
        eight = d is attn
        add(f"{what}: null", EINVAL, fn, None, *args)
        for field, value in (("n_heads", 0), ("n_heads", 7), ("scale", 0.0), ("scale", -1.0), ("scale", float("inf")),
                             ("scale", float("nan")), ("n", 0), ("n", 101), ("pos", 996), ("pos", 0xffffffff),
                             ("q_dtype", 2), ("kv_dtype", 2), ("q_offset", 4 * MIB + 8), ("out_offset", 7 * MIB + 4),
                             ("scratch_bytes", 0), ("scratch_bytes", 1024), ("scratch_offset", 8 * MIB + 4)):
            add(f"{what}: {field} {value}", EINVAL, fn, _copy(d, **{field: value}), *args)
        for field in ("q_offset", "out_offset", "scratch_offset"):
            add(f"{what}: {field} past the arena", ERANGE, fn, _copy(d, **{field: 32 * MIB - 16}), *args)
        for field, value in (("out_offset", 4 * MIB), ("out_offset", 4 * MIB + 16), ("out_offset", 0),
                             ("out_offset", 8 * MIB), ("scratch_offset", 4 * MIB), ("scratch_offset", 1024),
                             ("scratch_offset", 7 * MIB)):
            add(f"{what}: {field} {value} overlaps", EINVAL, fn, _copy(d, **{field: value}), *args)
        if eight:
            add(f"{what}: mask off 4", EINVAL, fn, _copy(d, mask_offset=3 * MIB + 2))
            add(f"{what}: mask past the arena", ERANGE, fn, _copy(d, mask_offset=32 * MIB - 16))
            if fn is L.syn_hip_kv8_attention:  # (it writes the state before it reads these)
                add(f"{what}: q in the state", EINVAL, fn, _copy(d, q_offset=1024))
                add(f"{what}: mask in the state", EINVAL, fn, _copy(d, mask_offset=1024))
            add(f"{what}: mask in the output", EINVAL, fn, _copy(d, mask_offset=7 * MIB))
            add(f"{what}: state off 256", EINVAL, fn, _copy(d, cache=_copy(state, offset=16)))
            add(f"{what}: state past the arena", ERANGE, fn, _copy(d, cache=_copy(state, offset=32 * MIB - 256)))
        else:
            add(f"{what}: no mask", EINVAL, fn, d, capi.NO_OFFSET)
            add(f"{what}: mask off 4", EINVAL, fn, d, 3 * MIB + 1)
            add(f"{what}: mask past the arena", ERANGE, fn, d, 32 * MIB - 16)
            add(f"{what}: mask in the scratch", EINVAL, fn, d, 8 * MIB + 64)
            add(f"{what}: out in V^T", EINVAL, fn, _copy(d, out_offset=MIB + 256), *args)
    for field, value, code in (("k_offset", 32 * MIB - 4, ERANGE), ("v_offset", 5 * MIB + 2, EINVAL),
                               ("k_offset", 2048, EINVAL)):
        add(f"kv8_attention: {field} {value}", code, L.syn_hip_kv8_attention, _copy(attn, **{field: value, **mask}))

    for what, fn, d in (("keep", L.syn_hip_kv_keep, state16), ("kv8_keep", L.syn_hip_kv8_keep, state)):
        def rows(*r):
            return (ctypes.c_uint32 * len(r))(*r)

        add(f"{what}: null", EINVAL, fn, None, 10, 8, rows(0, 2), 2)
        add(f"{what}: null rows", EINVAL, fn, d, 10, 8, None, 2)
        add(f"{what}: past the cache", EINVAL, fn, d, 995, 8, rows(0, 2), 2)
        add(f"{what}: position wraps", EINVAL, fn, d, 0xfffffffc, 8, rows(0, 2), 2)
        add(f"{what}: more rows than drafted", EINVAL, fn, d, 10, 1, rows(0, 2), 2)
        add(f"{what}: row past the drafted ones", EINVAL, fn, d, 10, 8, rows(0, 8), 2)
        add(f"{what}: the same row twice", EINVAL, fn, d, 10, 8, rows(0, 2, 2), 3)
        add(f"{what}: falling rows", EINVAL, fn, d, 10, 8, rows(3, 2), 2)
        add(f"{what}: too many drafted", EINVAL, fn, _copy(d, max_ctx=70000) if what == "kv8_keep" else d, 0, 65537,
            rows(0, 2), 2)
    add("kv8_keep: state off 256", EINVAL, L.syn_hip_kv8_keep, _copy(state, offset=16), 10, 8, (ctypes.c_uint32 * 1)(2), 1)
    return out
