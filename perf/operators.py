"""Work on 8-bit KV states and drafted tokens, as cases to measure.

A case is one call of a serving program's cache: K, V rows quantized into an
8-bit state as they are written, rows of it read back, attention over it (one
token, a chunk of a prompt), attention of a tree of drafted tokens over a
binary16 or an 8-bit state, and the accepted tokens' rows moved together after
it. `own` picks who computes it: torch's elementary operations, or the
framework's calls on an arena. What an 8-bit state holds is returned as the
values it stands for, so a case that writes one reads the rows back.
"""
from __future__ import annotations

import ctypes
import math

import numpy as np
import torch

own = False

# ---- the cases ---------------------------------------------------------------


def listed() -> list[dict]:
    return [
        # A decode step's append, one layer: nothing but latency.
        dict(name="append8-1-at-4096", kind="append8", dtype="f32", kv_heads=8, head_dim=128, pos=4096, n=1,
             max_ctx=8192),
        # A long prompt's rows behind a short turn; neither end on a tile edge.
        dict(name="append8-2047-at-333", kind="append8", dtype="f16", kv_heads=8, head_dim=128, pos=333, n=2047,
             max_ctx=4096),
        # Part of a small model's cache, for a binary16 state.
        dict(name="read8-700-at-1301", kind="read8", dtype="f16", kv_heads=2, head_dim=64, pos=1301, n=700,
             max_ctx=2048),
        # A whole layer's cache, to be saved or looked at.
        dict(name="read8-16384", kind="read8", dtype="f32", kv_heads=8, head_dim=128, pos=0, n=16384, max_ctx=16384),
        # A small model's early token.
        dict(name="attend8-300", kind="attend8", heads=14, kv_heads=2, head_dim=64, pos=300, n=1, max_ctx=2048),
        # One decode step of one layer in a chat.
        dict(name="attend8-4k", kind="attend8", heads=32, kv_heads=8, head_dim=128, pos=4096, n=1, max_ctx=8192),
        # The same far into a long document.
        dict(name="attend8-100k", kind="attend8", heads=32, kv_heads=8, head_dim=128, pos=100000, n=1,
             max_ctx=131072),
        # A further chunk of a long prompt; neither end on a tile edge.
        dict(name="attend8-509-at-7683", kind="attend8", heads=32, kv_heads=8, head_dim=128, pos=7683, n=509,
             max_ctx=8192),
        # A step that verifies a small draft tree, binary16 state.
        dict(name="tree-26-at-4096", kind="tree", heads=32, kv_heads=8, head_dim=128, pos=4096, n=26, max_ctx=8192),
        # A wide tree far into an 8-bit state.
        dict(name="tree8-61-at-20000", kind="tree8", heads=32, kv_heads=8, head_dim=128, pos=20000, n=61,
             max_ctx=32768),
        # The accepted path of such trees moved to the front of the drafted rows.
        dict(name="keep-6-of-26", kind="keep", kv_heads=8, head_dim=128, pos=4096, n=26, count=6, max_ctx=8192),
        dict(name="keep8-6-of-61", kind="keep8", kv_heads=8, head_dim=128, pos=20000, n=61, count=6, max_ctx=32768),
    ]


# Head layouts (query heads, KV heads, head size): grouped and ungrouped, the
# odd group of 7, sizes that are not powers of two.
LAYOUTS = [(32, 8, 128), (8, 8, 32), (14, 2, 64), (28, 4, 128), (16, 16, 80), (24, 8, 96), (32, 32, 64), (8, 4, 256)]


def _log_int(rng, lo: int, hi: int) -> int:
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5))))))


def draw(rng) -> dict:
    kind = rng.choice(["append8", "read8", "attend8", "attend8", "attend8", "chunk", "chunk", "tree", "tree", "tree8",
                       "tree8", "keep", "keep8"])
    heads, kv_heads, head_dim = rng.choice(LAYOUTS)
    c = dict(kind="attend8" if kind == "chunk" else kind, kv_heads=kv_heads, head_dim=head_dim)
    if kind in ("append8", "read8"):
        c |= dict(dtype=rng.choice(["f32", "f16"]), pos=rng.choice([0, _log_int(rng, 1, 8000)]),
                  n=_log_int(rng, 1, 8000))
    elif kind == "attend8":
        c |= dict(heads=heads, pos=_log_int(rng, 1, 40000), n=1)
    elif kind == "chunk":
        c |= dict(heads=heads, pos=rng.choice([0, _log_int(rng, 1, 6000)]), n=_log_int(rng, 2, 600))
    elif kind in ("tree", "tree8"):
        c |= dict(heads=heads, pos=_log_int(rng, 1, 20000), n=_log_int(rng, 2, 128))
    else:
        c |= dict(pos=_log_int(rng, 1, 20000), n=_log_int(rng, 8, 128))
        c |= dict(count=rng.randint(2, min(12, c["n"] // 2)))
    return c | dict(max_ctx=c["pos"] + c["n"] + rng.randrange(512))


# ---- inputs, from the seed alone ------------------------------------------------

_DTYPE = {"f32": torch.float32, "f16": torch.float16}


def _quantize(x):
    """Rows [t][head][hd] as whole numbers (int8) and a step per row and head
    (f32): the step is the largest magnitude's 127th part, and the quotients
    are rounded from 64 bits, where one next to a half is on its own side."""
    step = (x.abs().amax(-1).double() / 127.0).float()
    div = torch.where(step == 0, torch.ones_like(step), step).double()
    return torch.round(x.double() / div[..., None]).to(torch.int8), step


def _tree(n: int, seed: int) -> np.ndarray:
    """A draft tree's mask: bit j of row i where drafted token i is j or comes after it."""
    r, mask = np.random.default_rng(seed * 31 + 7), np.eye(n, dtype=bool)
    parent = [int(r.integers(max(0, i // 3 - 2), i)) if i else -1 for i in range(n)]
    for i in range(1, n):
        mask[i] |= mask[parent[i]]
    return mask


def _inputs(c, seed) -> dict:
    """What the call takes, as tensors in the order of the tokens: `k`, `v` the
    state's rows (f32 or f16, before any quantization), `q` the queries."""
    g = torch.Generator(device="cuda").manual_seed(seed * 7919 + 12345)
    end, heads, hd = c["pos"] + c["n"], c["kv_heads"], c["head_dim"]
    rows = c["n"] if c["kind"] == "append8" else end
    dt = torch.float16 if c["kind"] in ("tree", "keep") else _DTYPE[c.get("dtype", "f32")]
    x = {name: torch.empty((rows, heads, hd), device="cuda").normal_(generator=g).to(dt) for name in "kv"}
    if "heads" in c:
        x["q"] = torch.empty((c["n"], c["heads"] * hd), device="cuda").normal_(generator=g)
    if c["kind"].startswith("tree"):
        x["mask"] = torch.from_numpy(_tree(c["n"], seed)).cuda()
    if c["kind"].startswith("keep"):
        # The first drafted token, then others behind the kept rows (so that a
        # second pass on the same state finds them as they were).
        late = np.random.default_rng(seed).choice(np.arange(c["count"], c["n"]), c["count"] - 1, replace=False)
        x["rows"] = [0, *sorted(int(i) for i in late)]
    return x


# ---- the plain form ---------------------------------------------------------------


class Plain:
    """The state as torch holds it: the new rows, or whole numbers and steps
    for an 8-bit state and K rows and V^T rows for a binary16 one."""

    def __init__(self, c, x):
        self.c, self.x = c, x
        if c["kind"] == "append8":
            return
        if c["kind"].endswith("8"):
            self.k, self.v = _quantize(x.pop("k")), _quantize(x.pop("v"))
        else:
            self.k, self.vt = _binary16(c, x.pop("k"), x.pop("v"))
        if "rows" in x:
            x["rows"] = torch.tensor(x["rows"], device="cuda")


def _binary16(c, k, v):
    """K [max_ctx][row] and V^T [row][stride], zero past the rows given."""
    row, stride = c["kv_heads"] * c["head_dim"], -(-c["max_ctx"] // 64) * 64
    kc = torch.zeros((c["max_ctx"], row), device="cuda", dtype=torch.float16)
    vt = torch.zeros((row, stride), device="cuda", dtype=torch.float16)
    kc[:len(k)] = k.reshape(len(k), row)
    vt[:, :len(v)] = v.reshape(len(v), row).T
    return kc, vt


def _values(quantized):
    q, step = quantized
    return q.float() * step[..., None]


def _attend(q, k, v, heads: int, scale: float, seen):
    """q [n][heads * hd] f32, k and v [kv head][L][hd] f32; query i sees the
    keys of seen [n][L]."""
    n, (kv_heads, length, hd) = q.shape[0], k.shape
    group = heads // kv_heads
    q = q.half().float().view(n, kv_heads, group, hd).permute(1, 2, 0, 3).reshape(kv_heads, group * n, hd)
    s = torch.matmul(q, k.transpose(1, 2).contiguous()).view(kv_heads, group, n, length) * scale
    s = s.masked_fill(~seen, -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True))
    p = (p / p.sum(-1, keepdim=True)).view(kv_heads, group * n, length)
    return torch.matmul(p, v).view(kv_heads, group, n, hd).permute(2, 0, 1, 3).reshape(n, heads * hd)


def _seen(c, mask):
    pos, n = c["pos"], c["n"]
    if mask is None:
        return torch.arange(pos + n, device="cuda")[None] <= pos + torch.arange(n, device="cuda")[:, None]
    return torch.cat([torch.ones((n, pos), dtype=torch.bool, device="cuda"), mask], 1)


def _run_plain(s: Plain) -> dict:
    c, x = s.c, s.x
    if c["kind"] == "append8":
        return {"k": _values(_quantize(x["k"])).to(x["k"].dtype), "v": _values(_quantize(x["v"])).to(x["v"].dtype)}
    at, new = c["pos"], slice(c["pos"], c["pos"] + c["n"])
    if c["kind"] == "read8":
        return {"k": _values((s.k[0][new], s.k[1][new])).to(_DTYPE[c["dtype"]]),
                "v": _values((s.v[0][new], s.v[1][new])).to(_DTYPE[c["dtype"]])}
    if c["kind"] == "keep":
        kept = slice(at, at + c["count"])
        s.k[kept] = s.k[at + x["rows"]]
        s.vt[:, kept] = s.vt[:, at + x["rows"]]
        return {"k": s.k, "vt": s.vt}
    if c["kind"] == "keep8":
        kept, state = slice(at, at + c["count"]), (*s.k, *s.v)
        moved = [t[at + x["rows"]] for t in state]
        _ = [t[kept].copy_(m) for t, m in zip(state, moved)]
        return {"k": _values((s.k[0][new], s.k[1][new])), "v": _values((s.v[0][new], s.v[1][new]))}
    end, hd = at + c["n"], c["head_dim"]
    if c["kind"] == "tree":
        k = s.k[:end].view(end, c["kv_heads"], hd).permute(1, 0, 2).float()
        v = s.vt[:, :end].reshape(c["kv_heads"], hd, end).transpose(1, 2).float()
    else:
        k, v = (_values(t).permute(1, 0, 2) for t in (s.k, s.v))
    return {"out": _attend(x["q"], k.contiguous(), v.contiguous(), c["heads"], hd ** -0.5, _seen(c, x.get("mask")))}


# ---- the framework's calls ----------------------------------------------------------

ARENA_BYTES = 8 << 30
_TYPESTR = {torch.float32: "<f4", torch.float16: "<f2", torch.uint8: "|u1", torch.int32: "<i4"}


class _View:
    def __init__(self, owner, address, shape, typestr):
        self.owner = owner  # keeps the range while a tensor looks at it
        self.__cuda_array_interface__ = {"shape": shape, "typestr": typestr, "data": (address, False), "version": 3,
                                         "strides": None}


class _Session:
    """The arena that all states share, as the layers of one session do, its
    device address, and the ranges given back, by size."""

    def __init__(self):
        from synapse_amd.capi import Arena

        self.arena = Arena(ARENA_BYTES)
        # The arena object starts with its device address: tensors look at
        # inputs and outputs in place. A round trip shows that it is the address.
        self.base = ctypes.c_void_p.from_address(self.arena.handle.value).value
        self.free = [(0, ARENA_BYTES)]
        tag = np.random.default_rng().integers(0, 255, 64, dtype=np.uint8)
        self.arena.upload(0, tag)
        self.arena.sync()
        if not np.array_equal(self.view(None, 0, (64,), torch.uint8).cpu().numpy(), tag):
            raise RuntimeError("the arena's device address was not found")

    def view(self, owner, offset, shape, dtype) -> torch.Tensor:
        return torch.as_tensor(_View(owner, self.base + offset, tuple(shape), _TYPESTR[dtype]), device="cuda")

    def take(self, nbytes: int) -> int:
        i = next((i for i, (_, size) in enumerate(self.free) if size >= nbytes), None)
        if i is None:
            raise MemoryError(f"out of memory: {nbytes} bytes of the arena")
        at, size = self.free[i]
        self.free[i] = (at + nbytes, size - nbytes)
        return at

    def give(self, at: int, nbytes: int) -> None:
        merged = []
        for lo, size in sorted(self.free + [(at, nbytes)]):
            if merged and merged[-1][0] + merged[-1][1] == lo:
                merged[-1] = (merged[-1][0], merged[-1][1] + size)
            elif size:
                merged.append((lo, size))
        self.free = merged


_session: _Session | None = None


class _Range:
    def __init__(self, session: _Session, nbytes: int):
        self.session, self.nbytes = session, max(256, -(-nbytes // 256) * 256)
        self.at = session.take(self.nbytes)

    def __del__(self):
        self.session.give(self.at, self.nbytes)


class Placed:
    """A case's tensors in the arena, its descriptors and its calls."""

    def __init__(self, c, x):
        global _session
        from synapse_amd import capi

        if _session is None:
            _session = _Session()
        self.kept, self.calls, self.outputs = [], [], {}
        self.L, self.capi, self.handle = capi.lib(), capi, _session.arena.handle
        getattr(self, "_" + c["kind"])(c, x)

    def _room(self, shape, dtype):
        r = _Range(_session, math.prod(shape) * torch.empty((), dtype=dtype).element_size())
        self.kept.append(r)
        return r.at, _session.view(r, r.at, shape, dtype)

    def _put(self, t):
        at, view = self._room(t.shape, t.dtype)
        view.copy_(t)
        return at

    def _call(self, fn, *args):
        self.calls.append((fn, args))

    def _state8(self, c, x):
        """An 8-bit state and, but for an append's case, its rows appended."""
        capi, size = self.capi, int(self.L.syn_hip_kv8_state_bytes(c["max_ctx"], c["kv_heads"], c["head_dim"]))
        d = capi.Kv8Desc(offset=self._room((size,), torch.uint8)[0], max_ctx=c["max_ctx"], n_kv_heads=c["kv_heads"],
                         head_dim=c["head_dim"])
        self.kept.append(d)
        if c["kind"] != "append8":
            k, v = x["k"], x["v"]
            rows = [_Range(_session, t.numel() * t.element_size()) for t in (k, v)]
            _session.view(rows[0], rows[0].at, k.shape, k.dtype).copy_(k)
            _session.view(rows[1], rows[1].at, v.shape, v.dtype).copy_(v)
            torch.cuda.synchronize()
            capi.check(self.L.syn_hip_kv8_append(self.handle, ctypes.byref(d), rows[0].at, rows[1].at, len(k), 0,
                                                 self._type(k)))
            torch.cuda.synchronize()
        return d

    def _type(self, t):
        return self.capi.SYN_F16 if t.dtype == torch.float16 else self.capi.SYN_F32

    def _read(self, c, d, dtype):
        shape = (c["n"], c["kv_heads"], c["head_dim"])
        (k, self.outputs["k"]), (v, self.outputs["v"]) = self._room(shape, dtype), self._room(shape, dtype)
        self._call(self.L.syn_hip_kv8_read, ctypes.byref(d), k, v, c["n"], c["pos"], self._type(self.outputs["k"]))

    def _append8(self, c, x):
        d = self._state8(c, x)
        self._call(self.L.syn_hip_kv8_append, ctypes.byref(d), self._put(x["k"]), self._put(x["v"]), c["n"], c["pos"],
                   self._type(x["k"]))
        self._read(c, d, x["k"].dtype)

    def _read8(self, c, x):
        self._read(c, self._state8(c, x), _DTYPE[c["dtype"]])

    def _mask(self, mask):
        """Bit j of row i: words of 32 bits, rows of whole words."""
        if mask is None:
            return self.capi.NO_OFFSET
        n = len(mask)
        bits = np.zeros((n, -(-n // 32) * 32), dtype=bool)
        bits[:, :n] = mask.cpu().numpy()
        return self._put(torch.from_numpy(np.packbits(bits, axis=1, bitorder="little").view(np.int32)).cuda())

    def _attend8(self, c, x):
        d = self._state8(c, x)
        need = int(self.L.syn_hip_kv8_attention_scratch_bytes(c["heads"], c["kv_heads"], c["head_dim"], c["max_ctx"],
                                                              c["n"]))
        out, self.outputs["out"] = self._room(x["q"].shape, torch.float32)
        a = self.capi.Kv8AttnDesc(cache=d, q_offset=self._put(x["q"]), out_offset=out,
                                  scratch_offset=self._room((need,), torch.uint8)[0], scratch_bytes=need,
                                  mask_offset=self._mask(x.get("mask")), n_heads=c["heads"], pos=c["pos"], n=c["n"],
                                  scale=c["head_dim"] ** -0.5, q_dtype=self.capi.SYN_F32,
                                  kv_dtype=self.capi.SYN_F32)
        self.kept.append(a)
        self._call(self.L.syn_hip_kv8_attend, ctypes.byref(a))

    _tree8 = _attend8

    def _state16(self, c, x):
        kc, vt = _binary16(c, x["k"], x["v"])
        (k, self.k), (v, self.vt) = self._room(kc.shape, kc.dtype), self._room(vt.shape, vt.dtype)
        self.k.copy_(kc)
        self.vt.copy_(vt)
        return self.capi.KvDesc(k_offset=k, v_offset=v, max_ctx=c["max_ctx"], n_kv_heads=c["kv_heads"],
                                head_dim=c["head_dim"], ctx_stride=self.vt.shape[1])

    def _tree(self, c, x):
        need = int(self.L.syn_hip_attend_tree_scratch_bytes(c["heads"], c["kv_heads"], c["head_dim"], c["max_ctx"],
                                                            c["n"]))
        out, self.outputs["out"] = self._room(x["q"].shape, torch.float32)
        a = self.capi.AttnDesc(cache=self._state16(c, x), q_offset=self._put(x["q"]), out_offset=out,
                               scratch_offset=self._room((need,), torch.uint8)[0], scratch_bytes=need,
                               n_heads=c["heads"], pos=c["pos"], n=c["n"], scale=c["head_dim"] ** -0.5,
                               q_dtype=self.capi.SYN_F32, kv_dtype=self.capi.SYN_F16)
        self.kept.append(a)
        self._call(self.L.syn_hip_attend_tree, ctypes.byref(a), self._mask(x["mask"]))

    def _rows(self, x):
        return (ctypes.c_uint32 * len(x["rows"]))(*x["rows"])

    def _keep(self, c, x):
        d = self._state16(c, x)
        self.kept.append(d)
        self._call(self.L.syn_hip_kv_keep, ctypes.byref(d), c["pos"], c["n"], self._rows(x), c["count"])
        self.outputs = {"k": self.k, "vt": self.vt}

    def _keep8(self, c, x):
        d = self._state8(c, x)
        self._call(self.L.syn_hip_kv8_keep, ctypes.byref(d), c["pos"], c["n"], self._rows(x), c["count"])
        self._read(c, d, torch.float32)


# ---- prepare and run ------------------------------------------------------------------


def prepare(case, seed):
    torch.cuda.synchronize()  # ranges given back may still be read by queued passes
    x = _inputs(case, seed)
    s = Placed(case, x) if own else Plain(case, x)
    torch.cuda.synchronize()
    return s


def run(state):
    if own:
        _ = [state.capi.check(fn(state.handle, *args)) for fn, args in state.calls]
        return state.outputs
    return _run_plain(state)


# ---- what a pass cannot do without -------------------------------------------------------


def work(case) -> dict:
    c, n = case, case["n"]
    row, held = c["kv_heads"] * c["head_dim"], c["kv_heads"] * (2 * c["head_dim"] + 8)
    if c["kind"] in ("append8", "read8"):
        el = 2 if c["dtype"] == "f16" else 4
        # An append's case reads the rows back: rows in and out, the state's bytes written and read.
        return {"bytes": n * (2 * row * el + held) * (2 if c["kind"] == "append8" else 1), "flops": 0}
    if c["kind"] == "keep":
        return {"bytes": 8 * row * c["count"], "flops": 0}
    if c["kind"] == "keep8":
        return {"bytes": 2 * held * c["count"] + n * (8 * row + held), "flops": 0}
    end, size = c["pos"] + n, c["heads"] * c["head_dim"]
    mask = c["kind"].startswith("tree")
    seen = int(_tree(n, 0).sum()) if mask else n * (n + 1) // 2
    return {"bytes": end * (4 * row if c["kind"] == "tree" else held) + 8 * n * size + (n * -(-n // 32) * 4 if mask else 0),
            "flops": 4 * size * (n * c["pos"] + seen)}


# ---- the same in 64 bits --------------------------------------------------------------------


def exact(case, seed):
    c, x = case, _inputs(case, seed)
    pos, n, hd = c["pos"], c["n"], c["head_dim"]

    def held(rows):
        """The values an 8-bit state holds: multiples of the step (itself an f32)."""
        rows = rows.double()
        top = rows.abs().max(-1, keepdim=True).values
        step = (top / 127).to(torch.float32).double()
        return torch.where(step > 0, torch.round(rows / step), torch.zeros_like(rows)) * step

    if c["kind"] == "append8":
        return {"k": held(x["k"]), "v": held(x["v"])}
    eight = c["kind"].endswith("8")
    k, v = (held(x[i]) if eight else x[i].double() for i in "kv")
    if c["kind"] == "read8":
        return {"k": k[pos:], "v": v[pos:]}
    if c["kind"].startswith("keep"):
        rows = torch.tensor(x["rows"], device="cuda") + pos
        k[pos:pos + c["count"]], v[pos:pos + c["count"]] = k[rows], v[rows]
        if eight:
            return {"k": k[pos:], "v": v[pos:]}
        kc = torch.zeros((c["max_ctx"], k.shape[1] * hd), device="cuda", dtype=torch.float64)
        vt = torch.zeros((k.shape[1] * hd, (c["max_ctx"] + 63) // 64 * 64), device="cuda", dtype=torch.float64)
        kc[:pos + n], vt[:, :pos + n] = k.flatten(1), v.flatten(1).T
        return {"k": kc, "vt": vt}
    t, i = torch.arange(pos + n, device="cuda")[None], torch.arange(n, device="cuda")[:, None]
    hidden = t > pos + i
    if "mask" in x:
        hidden = torch.zeros_like(hidden)
        hidden[:, pos:] = ~x["mask"]
    out = torch.empty((n, c["heads"], hd), device="cuda", dtype=torch.float64)
    q = x["q"].half().double().view(n, c["heads"], hd)
    for h in range(c["heads"]):
        g = h * c["kv_heads"] // c["heads"]
        s = (q[:, h] @ k[:, g].T.contiguous()) / math.sqrt(hd)
        out[:, h] = torch.softmax(s.masked_fill(hidden, -math.inf), -1) @ v[:, g].contiguous()
    return {"out": out.view(n, -1)}
