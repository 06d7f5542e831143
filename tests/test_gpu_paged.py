"""GPU parity of a serving step's operators over a paged cache against plain float64 restatements (paged_model.py).

Tolerances, from the arithmetic (u = 2^-24 of fp32, half a step of each rounding):
 - rows: about 30 fp32 operations lie between a head's input and its output (the sum of squares over hd values adds hd / 2 u to
   the square root at most): 64 u + hd u of the head's largest magnitude, and half a step of the type that it is stored in
 - lse: q is scaled by a power of two; in f32 it is two fp16 terms (2^-22 of an element, 2^-24 with the rounding of the second).
   A score sums hd products in fp32: hd u sum |q k| at most.  Compared with 2^-22 + hd u of scale sum |q| |k| and 2^-20 for exp2 and log2
 - out: probabilities rounded to fp16 (2^-11 of each) or two terms (2^-22), times |v|, so (eps_p + 2 err_score + n u) sum p |v| / sum p;
   then half a step of out's type.  An fp16 number below 2^-14, the second term of nearly every probability among them, is off by
   2^-25 whatever its size: of p s (s the row scale of v) relative to the row's largest, times |v| / s, so
   2^-25 max(p s) sum(|v| / s) / sum p"""
import ctypes as C
import os
import subprocess
import sys

import numpy as np
import pytest

import paged_model as pm
from helpers import DeviceBuffer
from oxibonsai_amd import GpuError, paged
from paged_model import DevArray

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
HALF_STEP = {"float16": 2.0 ** -11, "bfloat16": 2.0 ** -8, "float32": 2.0 ** -24}


def _i32(a):
    return DevArray(np.asarray(a, dtype=np.int32))


# ---- page tables ------------------------------------------------------------------------------------------------------
class Pages:
    def __init__(self, past, keep, add, page, width, n_pages, n_free=None, n_rows=None, seed=1, alias=False):
        rng = np.random.default_rng(seed)
        b = len(past)
        self.past, self.keep, self.add, self.page = np.array(past), keep, np.array(add), page
        order = rng.permutation(n_pages).astype(np.int32)
        self.tables, at = np.full((b, width), -1, np.int32), 0
        for r in range(b):
            n = min(width, -(-max(0, int(past[r])) // page))
            self.tables[r, :n] = order[at:at + n]
            at += n
        self.n_free = n_pages - at if n_free is None else n_free
        self.free = np.full(n_pages, -7, np.int32)
        self.free[:n_pages - at] = order[at:]
        self.n_rows = int(max(0, sum(add))) + 5 if n_rows is None else n_rows
        d = self.d = dict(past=_i32(past), add=_i32(add), tables=_i32(self.tables), free_pages=_i32(self.free), n_free=_i32([self.n_free]),
                          cu_tokens=_i32(np.full(b + 1, 99)), cu_pages=_i32(np.full(b + 1, 99)), slots=_i32(np.full(self.n_rows, 99)),
                          positions=_i32(np.full(self.n_rows, 99)), status=_i32([99, 99]))
        d["lens"] = d["past"] if alias else _i32(np.full(b, 99))
        d["n_free_out"] = None if alias else _i32([99])
        d["keep"] = None if keep is None else _i32(keep)
        self.call = paged.PageAssign(page_size=page, **d)

    def check(self):
        want = pm.assign(self.past, self.keep, self.add, self.tables, self.free, self.n_free, self.page, self.n_rows)
        got = {n: self.d[m].get() for n, m in (("tables", "tables"), ("free", "free_pages"), ("lens", "lens"), ("cu_tokens", "cu_tokens"),
                                               ("cu_pages", "cu_pages"), ("slots", "slots"), ("positions", "positions"), ("status", "status"))}
        got["n_free"] = (self.d["n_free_out"] or self.d["n_free"]).get()[0]
        for n in got:
            assert np.array_equal(got[n], want[n]), (n, got[n], want[n])
        return want


@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("b,most_past,most_add", [(1, 0, 1), (1, 40, 300), (5, 100, 1), (63, 200, 70), (300, 90, 40), (1300, 60, 9), (4096, 30, 3)])
@pytest.mark.parametrize("alias", [False, True])
def test_pages_ragged(backend, page, b, most_past, most_add, alias):
    rng = np.random.default_rng(b + page)
    past = rng.integers(0, most_past + 1, b)
    add = rng.integers(0, most_add + 1, b)
    keep = np.where(rng.random(b) < 0.3, rng.integers(0, most_past + 5, b), past) if b > 1 else None
    width = -(-(most_past + most_add + 5) // page)
    p = Pages(past, keep, add, page, width, b * width + 3, alias=alias)
    p.call()
    p.check()


@pytest.mark.parametrize("case", ["short", "just", "width", "rows", "negative", "count", "freed", "bad_page"])
def test_pages_that_do_not_fit(backend, case):
    past, add, keep = [17, 0, 64, 33], [15, 40, 1, 0], [17, 0, 3, 33]
    kw = dict(page=16, width=8, n_pages=40)
    if case == "short":
        kw["n_free"], add[1] = 0, 60       # three pages come back, four are needed
    if case == "just":
        kw["n_free"], add[1] = 1, 60
    if case == "width":
        add[1] = 129
    if case == "rows":
        kw["n_rows"] = 55
    if case == "negative":
        add[3] = -1
    if case == "count":
        kw["n_free"] = 41
    if case == "freed":
        kw["n_free"] = 38
    p = Pages(past, keep, add, **kw)
    if case == "bad_page":                 # a free page that is none: no slot lies in it
        p.free[p.n_free + 2] = p.free[p.n_free - 1] = 40
        p.tables[2, 3] = -3
        p.d["free_pages"].put(p.free)
        p.d["tables"].put(p.tables)
    p.call()
    want = p.check()
    assert want["status"][0] == dict(short=1, just=0, width=2, rows=2, negative=3, count=3, freed=3, bad_page=0)[case]


def test_pages_of_many_steps(backend):
    # a server's loop: the calls' own outputs are the next step's inputs, requests end and others take their places
    rng = np.random.default_rng(3)
    p = Pages([0] * 37, [0] * 37, [0] * 37, 16, 20, 37 * 12, n_rows=900, alias=True)
    past, free, n_free, tables = p.past, p.free, p.n_free, p.tables
    for _ in range(40):
        add = np.where(rng.random(37) < 0.2, rng.integers(0, 60, 37), 1)
        keep = np.where((rng.random(37) < 0.1) | (past + add > 300), 0, past)
        p.d["add"].put(add)
        p.d["keep"].put(keep)
        p.past, p.keep, p.add, p.tables, p.free, p.n_free = past, keep, add, tables, free, n_free
        p.call()
        want = p.check()
        past, free, n_free, tables = np.array(want["lens"]), want["free"], want["n_free"], want["tables"]
        held = [int(x) for r in range(37) for x in tables[r, :-(-past[r] // 16)]] + [int(x) for x in free[:n_free]]
        assert sorted(held) == sorted(set(held)) and len(held) == 37 * 12


# ---- rows -------------------------------------------------------------------------------------------------------------
KV_KIND = {"f16": "float16", "i8": "int8", "fp8": "float8_e4m3fn"}


def make_pool(rng, kv, nkv, n_pages, page, hd, spread=1.0):
    shape = (nkv, n_pages, page, hd)
    if kv == "f16":
        rows = [(rng.standard_normal(shape) * spread).astype(np.float16) for _ in "kv"]
        return rows, [None, None]
    codes = [rng.integers(-127, 128, shape).astype(np.int8) if kv == "i8" else
             np.where(rng.integers(0, 256, shape) & 0x7f == 0x7f, 0x3a, rng.integers(0, 256, shape)).astype(np.uint8) for _ in "kv"]
    if kv == "fp8":
        codes = [np.where(c & 0x7f == 0x7f, 0x3a, c).astype(np.uint8) for c in codes]
    scales = [((0.5 + rng.random(shape[:3])) * spread / (60 if kv == "i8" else 200)).astype(np.float32) for _ in "kv"]
    return codes, scales


def dev_pool(rows, scales, kv):
    d = [DevArray(r, KV_KIND[kv]) for r in rows] + [None if s is None else DevArray(s) for s in scales]
    return paged.PagePool(*d), d


@pytest.mark.parametrize("hd,nq,nkv", [(32, 4, 1), (64, 6, 2), (128, 8, 8), (128, 5, 1), (256, 3, 3)])
@pytest.mark.parametrize("kv", ["f16", "i8", "fp8"])
@pytest.mark.parametrize("x,q", [("float32", "float16"), ("float16", "float32"), ("bfloat16", "bfloat16")])
@pytest.mark.parametrize("norm,rope", [(True, True), (False, False), (True, False), (False, True)])
def test_rows(backend, hd, nq, nkv, kv, x, q, norm, rope):
    rng = np.random.default_rng(hd + nq)
    n, page, n_pages, angles = 23, 16, 4, 300
    wide = (nq + 2 * nkv) * hd
    pad = 24
    data = pm.to_type(rng.standard_normal((n, wide + pad)) * np.exp(rng.uniform(-3, 3, (n, 1))), x)
    slots = rng.permutation(n_pages * page)[:n].astype(np.int32)
    pos = rng.integers(0, angles, n).astype(np.int32)
    slots[[4, 9]] = [-1, n_pages * page]
    pos[[6, 11]] = [-1, angles]            # (position 300: no angles)
    pos[0], pos[1] = 0, angles - 1
    angle = np.outer(np.arange(angles), 1e6 ** (-np.arange(0, hd, 2) / hd))
    cos, sin = np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32)
    qn, kn = (1 + 0.2 * rng.standard_normal((2, hd))).astype(np.float32)
    rows, scales = make_pool(rng, kv, nkv, n_pages, page, hd)
    pool, d = dev_pool(rows, scales, kv)
    q_old = pm.to_type(np.full((n, nq * hd + 8), 7.5), q)
    dx, dq = DevArray(data, x), DevArray(q_old, q)
    store = paged.RowStore(pool, nq=nq, slots=_i32(slots), positions=_i32(pos), **(dict(q_norm=DevArray(qn), k_norm=DevArray(kn), eps=1e-5) if norm else {}),
                           **(dict(cos=DevArray(cos), sin=DevArray(sin)) if rope else {}))
    store(dx.view(0, (n, wide), (wide + pad, 1)), dq.view(0, (n, nq, hd), (nq * hd + 8, hd, 1)))
    v64 = pm.from_type(data[:, :wide], x).reshape(n, nq + 2 * nkv, hd)
    at = np.clip(pos, 0, angles - 1)
    c, s = (cos[at], sin[at]) if rope else (None, None)
    want_q, want_k = pm.turned(v64[:, :nq], qn if norm else None, c, s, 1e-5), pm.turned(v64[:, nq:nq + nkv], kn if norm else None, c, s, 1e-5)
    want_v = v64[:, nq + nkv:]
    live = (pos >= 0) & (pos < (angles if rope else 1 << 30))
    rel = (64 + hd) * U
    got = pm.from_type(dq.get(), q)
    for t in range(n):
        if not live[t]:
            assert np.all(got[t] == 7.5)
            continue
        big = np.abs(want_q[t]).max(-1, keepdims=True)
        err = np.abs(got[t, :nq * hd].reshape(nq, hd) - want_q[t])
        assert np.all(err <= rel * big + HALF_STEP[q] * np.abs(want_q[t]) * (1 + 2 * rel) + 2.0 ** -25), (t, err.max())
        assert np.all(got[t, nq * hd:] == 7.5)
    stored = {int(sl): t for t, sl in enumerate(slots) if live[t] and 0 <= sl < n_pages * page}
    for name, want, i in (("k", want_k, 0), ("v", want_v, 1)):
        now = d[i].get().reshape(nkv, -1, hd)
        was = rows[i].reshape(nkv, -1, hd)
        sc = None if kv == "f16" else d[2 + i].get().reshape(nkv, -1)
        for sl in range(n_pages * page):
            if sl not in stored:
                assert np.array_equal(now[:, sl], was[:, sl]), (name, sl)
                assert sc is None or np.array_equal(sc[:, sl], scales[i].reshape(nkv, -1)[:, sl])
                continue
            w = want[stored[sl]]
            big = np.abs(w).max(-1, keepdims=True)
            if kv == "f16":
                assert np.all(np.abs(now[:, sl].astype(np.float64) - w) <= rel * big + 2.0 ** -11 * np.abs(w) * (1 + 2 * rel) + 2.0 ** -25)
                continue
            full = 127 if kv == "i8" else 448
            assert np.all(np.abs(sc[:, sl] - big[:, 0] / full) <= (rel + 4 * U) * big[:, 0] / full)
            val = pm.pool_values(now[:, sl][:, None, None], sc[:, sl][:, None, None], kv)[:, 0, 0]
            # half a step of the code (an INT8 code is one part in 127 of the largest, an E4M3 one 2^-4 of the value, at least 2^-10 of scale)
            step = 0.5 * sc[:, sl][:, None] if kv == "i8" else np.maximum(2.0 ** -4 * np.abs(w), 2.0 ** -10 * sc[:, sl][:, None])
            assert np.all(np.abs(val - w) <= step * (1 + 1e-5) + 2 * rel * big)


@pytest.mark.parametrize("kv", ["i8", "fp8"])
def test_rows_codes_bit_for_bit(backend, kv):
    # the scale's and the codes' definition in fp32, and what the row quantiser makes of the same rows
    from oxibonsai_amd.model import kv_quantize_rows
    rng = np.random.default_rng(8)
    n, nkv, hd = 40, 2, 64
    data = (rng.standard_normal((n, 2 * nkv * hd)) * np.exp(rng.uniform(-20, 5, (n, 1)))).astype(np.float32)
    data[3] = 0
    rows, scales = make_pool(rng, kv, nkv, 5, 16, hd)
    pool, d = dev_pool(rows, scales, kv)
    slots = rng.permutation(80)[:n]
    paged.RowStore(pool, nq=0, slots=_i32(slots))(DevArray(data))
    full = np.float32(127 if kv == "i8" else 448)
    for i in (0, 1):
        part = data.reshape(n, 2, nkv, hd)[:, i]
        scale = np.maximum(np.abs(part).max(-1) * (np.float32(1) / full), np.float32(2.0 ** -23))
        quotient = (part / scale[..., None]).astype(np.float64)
        codes, sc = kv_quantize_rows(1 if kv == "i8" else 2, part.reshape(-1, hd))
        now, nsc = d[i].get().reshape(nkv, -1, hd)[:, slots].transpose(1, 0, 2), d[2 + i].get().reshape(nkv, -1)[:, slots].T
        assert np.array_equal(nsc, scale)
        assert np.all(np.abs(nsc - sc.reshape(n, nkv)) <= np.spacing(scale))
        if kv == "i8":
            assert np.array_equal(now, np.clip(np.sign(quotient) * np.floor(np.abs(quotient) + 0.5), -127, 127))
            assert np.max(np.abs(now.astype(int) - codes.view(np.int8).reshape(n, nkv, hd))) <= 1
        else:
            step = 2.0 ** (np.clip(np.floor(np.log2(np.maximum(np.abs(quotient), 2.0 ** -30))), -6, 8) - 3)
            assert np.array_equal(pm.E4M3[now], np.clip(np.round(quotient / step) * step, -448, 448))


# ---- attention ----------------------------------------------------------------------------------------------------------
class Attention:
    """A batch: groups = [(prefix, [(rest, new), ..]), ..] or [(0, ..)] of requests on their own."""

    def __init__(self, groups, *, nq, nkv, hd, page, dtype, kv, seed=0, share=True, pad_rows=0, spread=1.0, scale=0.0, tail=0, poison=True):
        rng = self.rng = np.random.default_rng(seed)
        self.nq, self.nkv, self.hd, self.page, self.dtype, self.kv = nq, nkv, hd, page, dtype, kv
        self.scale = scale or hd ** -0.5
        lens, new, self.cu_g, self.prefix = [], [], [0], []
        for prefix, reqs in groups:
            lens += [prefix + r for r, _ in reqs]
            new += [n for _, n in reqs]
            self.cu_g.append(len(lens))
            self.prefix.append(prefix)
        b = len(lens)
        width = max(1, max(-(-n // page) for n in lens)) + tail
        own = [[-(-lens[r] // page) - self.prefix[g] // page for r in range(self.cu_g[g], self.cu_g[g + 1])] for g in range(len(groups))]
        n_pages = sum(p // page for p in self.prefix) + sum(map(sum, own)) + 3
        order = rng.permutation(n_pages)
        tables, at = np.full((b, width), -1, np.int32), 0
        for g in range(len(groups)):
            whole = self.prefix[g] // page
            tables[self.cu_g[g]:self.cu_g[g + 1], :whole] = order[at:at + whole]
            at += whole
            for i, r in enumerate(range(self.cu_g[g], self.cu_g[g + 1])):
                tables[r, whole:whole + own[g][i]] = order[at:at + own[g][i]]
                at += own[g][i]
        if not share:          # the same keys without sharing: a partly filled page of the prefix has to be everybody's own
            assert all(p % page == 0 for p in self.prefix)
        self.tables, self.lens = tables, np.array(lens)
        self.cu = np.concatenate([[0], np.cumsum(new)])
        self.t = int(self.cu[-1]) + pad_rows
        self.pos = np.concatenate([np.arange(lens[r] - new[r], lens[r]) for r in range(b)] + [np.full(pad_rows, -1)]).astype(np.int32)
        self.rows, self.scales = make_pool(rng, kv, nkv, n_pages, page, hd, spread)
        self.used = np.zeros((n_pages, page), bool)      # rows that some request owns
        for r in range(b):
            g = int(np.searchsorted(self.cu_g, r, side="right")) - 1
            at_ = np.arange(0 if r == self.cu_g[g] else self.prefix[g], lens[r])
            self.used[tables[r][at_ // page], at_ % page] = True
        if poison:             # whatever no request owns holds no numbers
            self._poison()
        self.q = pm.to_type(rng.standard_normal((self.t, nq, hd)) * spread, dtype)
        self.share, self.n_groups = share, len(groups)
        self.make()

    def _poison(self):
        for i in (0, 1):
            if self.kv == "f16":
                self.rows[i][:, ~self.used] = np.nan if i else np.inf
            else:
                if self.kv == "fp8":
                    self.rows[i][:, ~self.used] = 0x7f
                self.scales[i][:, ~self.used] = np.nan

    def make(self):
        self.pool, self.dpool = dev_pool(self.rows, self.scales, self.kv)
        self.dq, self.dout = DevArray(self.q, self.dtype), DevArray(pm.to_type(np.full((self.t, self.nq, self.hd), 9.0), self.dtype), self.dtype)
        self.dlse = DevArray(np.full((self.t, self.nq), 9.0, np.float32))
        self.dev = dict(tables=_i32(self.tables), cu_tokens=_i32(self.cu), positions=_i32(self.pos), lens=_i32(self.lens))
        if self.share:
            self.dev |= dict(cu_groups=_i32(self.cu_g), prefix_lens=_i32(self.prefix))
        self.call = paged.PagedAttention(self.pool, nq=self.nq, scale=0.0 if self.scale == self.hd ** -0.5 else self.scale, **self.dev)
        self.ws = DevArray(np.full(self.call.workspace_bytes // 4, np.nan, np.float32))

    def run(self):
        self.call(self.dq, self.dout, lse=self.dlse, workspace=self.ws)
        return self

    def expect(self):
        k, v = (pm.pool_values(r, s, self.kv) for r, s in zip(self.rows, self.scales))
        q = pm.from_type(self.q, self.dtype)
        self.want = pm.attention(q, k, v, self.scales[1], self.tables, self.cu, self.pos, self.lens, self.cu_g if self.share else None, self.prefix, self.page, self.scale)
        fine = np.where(np.isfinite(k), np.abs(k), 0)
        self.size = self.scale * np.abs(q).sum(-1) * fine.max() if self.t else np.zeros((0, self.nq))
        return self

    def check(self):
        out, lse, mag, low = self.want
        got, got_lse = pm.from_type(self.dout.get(), self.dtype), self.dlse.get()
        none = np.isnan(lse)
        assert np.all(got[none] == 9.0) and np.all(got_lse[none] == 9.0)       # rows of no request
        score = (2.0 ** -22 + self.hd * U) * self.size
        empty = np.isneginf(lse)
        assert np.array_equal(empty, np.isneginf(got_lse) & ~none)
        ok = ~none & ~empty
        err = np.abs(got_lse[ok] - lse[ok])
        assert np.all(err <= score[ok] + 2.0 ** -20 + 2.0 ** -22 * np.abs(lse[ok])), err.max()
        p_err = (2.0 ** -11 if self.dtype != "float32" else 2.0 ** -22) + 2 * score[..., None] + max(64, int(self.lens.max())) ** 0.5 * 8 * U + 2.0 ** -20
        limit = p_err * mag + 2.0 ** -25 * low + HALF_STEP[self.dtype] * np.abs(out) + 2.0 ** -24
        assert np.all(got[empty] == 0)
        bad = np.abs(got[ok] - out[ok]) > limit[ok]
        assert not bad.any(), (int(bad.sum()), np.max(np.abs(got[ok] - out[ok]) / limit[ok]))


TYPES = [("float16", "f16"), ("bfloat16", "f16"), ("float32", "f16"), ("float16", "i8"), ("float32", "i8"), ("bfloat16", "fp8"), ("float32", "fp8")]
HEADS = [(4, 1, 32), (6, 2, 64), (8, 8, 64), (8, 2, 128), (16, 1, 128), (6, 2, 256)]
BATCHES = {
    "one_token": [(0, [(1, 1)])],
    "lengths": [(0, [(n, 1) for n in (1, 15, 16, 17, 31, 32, 33, 127, 128, 129, 300)])],
    "empty": [(0, [(0, 0), (20, 0), (5, 1), (0, 0)])],
    "prefix": [(100, [(1, 1), (40, 1), (7, 1), (64, 1)])],
    "prefix_page_end": [(96, [(1, 1), (33, 1), (17, 2)])],
    "groups": [(33, [(9, 1)] * 3), (0, [(50, 1), (3, 1)]), (200, [(12, 1)]), (47, [(0, 0), (6, 1), (29, 3)])],
    "many_rows": [(70, [(11, 1)] * 45)],
    "chunk": [(0, [(50, 50), (90, 13), (3, 3)])],
    "chunk_prefix": [(75, [(40, 40), (33, 5), (70, 70)]), (20, [(20, 20), (9, 2)])],
    "long": [(700, [(30, 1), (400, 1)]), (0, [(1500, 1)])],
}


@pytest.mark.parametrize("name", BATCHES)
@pytest.mark.parametrize("dtype,kv", TYPES)
@pytest.mark.parametrize("heads", HEADS[3:4] + HEADS[1:2], ids=str)
def test_attention(backend, name, dtype, kv, heads):
    nq, nkv, hd = heads
    Attention(BATCHES[name], nq=nq, nkv=nkv, hd=hd, page=16, dtype=dtype, kv=kv, seed=len(name)).run().expect().check()


@pytest.mark.parametrize("heads", HEADS, ids=str)
@pytest.mark.parametrize("dtype,kv", TYPES)
@pytest.mark.parametrize("page", [32, 64, 128])
def test_attention_heads_and_pages(backend, heads, dtype, kv, page):
    nq, nkv, hd = heads
    Attention([(150, [(40, 1), (5, 1), (77, 9)]), (0, [(260, 1)])], nq=nq, nkv=nkv, hd=hd, page=page, dtype=dtype, kv=kv, seed=page + hd, pad_rows=3,
              tail=2).run().expect().check()


@pytest.mark.parametrize("dtype,kv", TYPES)
@pytest.mark.parametrize("heads", [(8, 2, 128), (6, 2, 64), (3, 3, 256)], ids=str)
@pytest.mark.parametrize("what", [np.nan, np.inf, -np.inf])
def test_attention_values_that_only_later_rows_see(backend, heads, dtype, kv, what):
    """A key's value that is no number, or infinite, reaches the rows that see the key and no others."""
    nq, nkv, hd = heads
    a = Attention([(0, [(50, 50), (90, 13), (3, 3)]), (20, [(9, 2), (9, 3), (30, 1)]), (70, [(40, 40), (33, 35)]), (0, [(1500, 5)])], nq=nq, nkv=nkv, hd=hd, page=16,
                  dtype=dtype, kv=kv, seed=hd)
    for r in range(len(a.lens)):
        n = int(a.cu[r + 1] - a.cu[r])
        for at in {int(a.lens[r]) - 1, int(a.lens[r]) - (n + 1) // 2}:
            page, row = a.tables[r, at // 16], at % 16
            if kv == "f16":
                a.rows[1][:, page, row, at % hd] = what
            elif kv == "fp8" and np.isnan(what):
                a.rows[1][:, page, row, at % hd] = 0x7f
            else:
                a.scales[1][:, page, row] = what
    a.make()
    with np.errstate(invalid="ignore"):
        a.run().expect().check()
        out, got = a.want[0], pm.from_type(a.dout.get(), dtype)
        odd = ~np.isfinite(out)
        assert odd.any() and np.isfinite(out).any()
        assert np.array_equal(np.isfinite(got), ~odd)
        assert np.array_equal(got[odd], out[odd], equal_nan=True)


SMALL = dict(nq=8, nkv=2, hd=64, page=16)
MIXED = [(40, [(3, 1), (20, 5), (17, 1)]), (0, [(60, 41)])]


@pytest.mark.parametrize("page", [-1, None, 1 << 30, -(1 << 31)])
@pytest.mark.parametrize("dtype,kv", TYPES[::2])
def test_attention_page_numbers_that_are_none(backend, page, dtype, kv):
    """They stay inside the pool, and other requests' answers are right."""
    a = Attention([(0, [(60, 1)]), (0, [(50, 1), (70, 30)]), (33, [(20, 2), (9, 1)])], **SMALL, dtype=dtype, kv=kv, seed=3)
    n_pages = a.rows[0].shape[1]
    a.expect()
    a.tables[1:3, 1::2] = n_pages if page is None else page
    a.make()
    a.run()
    bad = np.zeros(a.t, bool)
    bad[a.cu[1]:a.cu[3]] = True
    out, lse, mag, low = a.want
    got, got_lse = a.dout.get(), a.dlse.get()
    got[bad], got_lse[bad] = pm.to_type(out[bad], dtype), lse[bad]
    a.dout.put(got)
    a.dlse.put(got_lse)
    a.check()


@pytest.mark.parametrize("what", ["tokens", "groups"])
def test_attention_sums_that_do_not_ascend_do_nothing(backend, what):
    a = Attention(MIXED, **SMALL, dtype="float16", kv="f16")
    if what == "tokens":
        a.cu = np.array([0, 6, 1, 7, a.t])
    else:
        a.cu_g = [0, 5, 4]
    a.make()
    a.run()
    assert np.all(a.dout.get() == 9.0) and np.all(a.dlse.get() == 9.0)


@pytest.mark.parametrize("dtype,kv", TYPES)
def test_attention_positions_and_lengths_at_their_ends(backend, dtype, kv):
    a = Attention([(0, [(60, 4)]), (0, [(50, 3), (70, 30)]), (33, [(20, 2), (9, 1)])], **SMALL, dtype=dtype, kv=kv, seed=3)
    a.pos = a.pos.astype(np.int64)
    a.pos[[1, 5, 20]] = 2 ** 31 - 1, -(2 ** 31), 0
    a.lens[1] = -5
    a.make()
    a.run().expect().check()


@pytest.mark.parametrize("scale", [-0.2, 0.01, 1.0])
@pytest.mark.parametrize("dtype,kv", TYPES)
def test_attention_scales(backend, scale, dtype, kv):
    a = Attention(MIXED, **SMALL, dtype=dtype, kv=kv, seed=4, scale=scale, spread=0.5)
    a.run().expect()
    a.size = np.abs(a.size)
    a.check()


@pytest.mark.parametrize("dtype,kv", TYPES)
def test_attention_strided_rows(backend, dtype, kv):
    """q as a slice of a product's rows, out as a slice of something wider: what lies beside them stays."""
    a = Attention(MIXED, **SMALL, dtype=dtype, kv=kv, seed=5, pad_rows=2)
    wide, own = a.nq * a.hd, a.nq * a.hd
    q = np.full((a.t, wide + 256), np.nan)
    q[:, 128:128 + own] = pm.from_type(a.q, dtype).reshape(a.t, -1)
    base, out = DevArray(pm.to_type(q, dtype), dtype), DevArray(pm.to_type(np.full((a.t, wide + 72), 9.0), dtype), dtype)
    a.call(base.view(128, (a.t, a.nq, a.hd), (wide + 256, a.hd, 1)), out.view(64, (a.t, a.nq, a.hd), (wide + 72, a.hd, 1)), lse=None, workspace=a.ws)
    got = out.get()
    beside = pm.from_type(got, dtype)
    assert np.all(beside[:, :64] == 9.0) and np.all(beside[:, 64 + own:] == 9.0)
    assert np.all(a.dlse.get() == 9.0)
    a.run()
    whole = a.dout.get()
    assert np.array_equal(whole.reshape(a.t, -1), got[:, 64:64 + own])       # the same bits, with lse and without
    a.expect().check()


@pytest.mark.parametrize("kv", ["i8", "fp8"])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("how", ["wide", "ends", "huge"])
def test_attention_value_scales_far_apart(backend, kv, dtype, how):
    a = Attention([(100, [(30, 1), (9, 3)]), (0, [(260, 60), (40, 40)])], **SMALL, dtype=dtype, kv=kv, seed=6)
    s = a.scales[1]
    keys = a.rng.random(s.shape)
    if how == "wide":
        s[:] = np.where(np.isnan(s), s, 2.0 ** (40 * keys - 20)).astype(np.float32)
    elif how == "ends":
        s[:] = np.where(np.isnan(s), s, np.where(keys < 0.1, 2e-38, np.where(keys > 0.97, 1e30, s)))
    else:
        for r in range(4):       # one key of each request, which all its rows see
            s[:, a.tables[r, 0], 7] = 1e35
    a.make()
    a.run().expect().check()


@pytest.mark.parametrize("how", ["alone", "groups", "most"])
@pytest.mark.parametrize("dtype,kv", [("float16", "f16"), ("float32", "i8")])
def test_attention_of_many_requests(backend, how, dtype, kv):
    rng = np.random.default_rng(8)
    if how == "alone":
        groups = [(0, [(int(rng.integers(1, 60)), 1)]) for _ in range(700)]
    else:
        groups, left = [], 4096 if how == "most" else 400
        while left:
            n = min(left, int(rng.integers(1, 8)))
            groups.append((int(rng.integers(0, 40)), [(int(rng.integers(4, 30)), int(rng.choice([0, 1, 1, 1, 1, 3]))) for _ in range(n)]))
            left -= n
    a = Attention(groups, nq=4, nkv=1, hd=32, page=16, dtype=dtype, kv=kv, seed=9, share=how != "alone", poison=False)
    a.run().expect().check()


def test_rows_and_attention_far_into_a_large_pool(backend):
    """Rows past 2^31 elements and 2^32 bytes of the pool."""
    a = Attention([(140, [(3, 1), (200, 1)]), (0, [(300, 70)])], nq=8, nkv=2, hd=128, page=128, dtype="float16", kv="f16", poison=False)
    n_pages, page, hd = 100000, 128, 128
    small = a.rows[0].shape[1]

    def big():
        d = object.__new__(DevArray)
        d.host, d.dtype, d.first, d.shape = np.empty(1, np.float16), "x.float16", 0, (2, n_pages, page, hd)
        d._stride, d.buf = (n_pages * page * hd, page * hd, hd, 1), DeviceBuffer(2 * n_pages * page * hd * 2)
        return d

    far = {p: n_pages - 1 - 37 * p for p in range(small)}
    pools = [big(), big()]
    try:
        hip = DeviceBuffer.hip()
        for d, rows in zip(pools, a.rows):
            for h in range(2):
                for p in range(small):
                    block = np.ascontiguousarray(rows[h, p])
                    assert hip.hipMemcpy(d.buf.ptr + (h * n_pages + far[p]) * page * hd * 2, block.ctypes.data, block.nbytes, 1) == 0
        tables = np.vectorize(lambda p: far.get(p, -1))(a.tables).astype(np.int32)
        pool = paged.PagePool(*pools)
        a.dev["tables"] = _i32(tables)
        call = paged.PagedAttention(pool, nq=8, **a.dev)
        call(a.dq, a.dout, lse=a.dlse, workspace=a.ws)
        a.expect().check()
        slots = [far[0] * page + 5, far[1] * page + 127]
        x = a.rng.standard_normal((2, 12 * hd)).astype(np.float16)
        paged.RowStore(pool, nq=8, slots=_i32(slots))(DevArray(x))
        for i, s in enumerate(slots):
            for h in range(2):
                for d, at in ((pools[0], 8 + h), (pools[1], 10 + h)):
                    row = np.empty(hd, np.float16)
                    assert hip.hipDeviceSynchronize() == 0
                    assert hip.hipMemcpy(row.ctypes.data, d.buf.ptr + (h * n_pages * page + s) * hd * 2, hd * 2, 2) == 0
                    assert np.array_equal(row, x[i, at * hd:(at + 1) * hd])
    finally:
        for d in pools:
            d.buf.free()


def _graphs():
    hip = DeviceBuffer.hip()
    for f, args in (("hipStreamCreate", [C.POINTER(C.c_void_p)]), ("hipStreamDestroy", [C.c_void_p]), ("hipStreamBeginCapture", [C.c_void_p, C.c_int]),
                    ("hipStreamEndCapture", [C.c_void_p, C.POINTER(C.c_void_p)]), ("hipStreamSynchronize", [C.c_void_p]),
                    ("hipGraphInstantiate", [C.POINTER(C.c_void_p), C.c_void_p, C.c_void_p, C.c_void_p, C.c_size_t]),
                    ("hipGraphLaunch", [C.c_void_p, C.c_void_p]), ("hipGraphExecDestroy", [C.c_void_p]), ("hipGraphDestroy", [C.c_void_p])):
        getattr(hip, f).argtypes = args
    return hip


def test_attention_on_two_streams_at_once(backend):
    hip = _graphs()
    calls = [Attention([(400, [(30, 1)] * 9)], nq=8, nkv=2, hd=128, page=16, dtype="float16", kv="f16", seed=1),
             Attention([(70, [(90, 60), (20, 1)])], nq=8, nkv=2, hd=128, page=16, dtype="float32", kv="i8", seed=2)]
    streams = [C.c_void_p(0), C.c_void_p(0)]
    for s in streams:
        assert hip.hipStreamCreate(C.byref(s)) == 0
    try:
        for _ in range(20):
            for a, s in zip(calls, streams):
                backend.set_stream(s.value)
                a.run()
        for s in streams:
            assert hip.hipStreamSynchronize(s) == 0
    finally:
        backend.set_stream(0)
        for s in streams:
            assert hip.hipStreamDestroy(s) == 0
    for a in calls:
        a.expect().check()


class Step(Attention):
    """A server's step as it is used: pages, rows, attention, on buffers that stay."""

    def __init__(self, groups, *, nq, nkv, hd, page, dtype, kv, n_rows, seed=0):
        rng = self.rng = np.random.default_rng(seed)
        self.nq, self.nkv, self.hd, self.page, self.dtype, self.kv, self.t, self.share = nq, nkv, hd, page, dtype, kv, n_rows, True
        self.scale = hd ** -0.5
        b, width, n_pages, most = sum(n for _, n in groups), 24, 300, 400
        self.prefix, self.cu_g = [p for p, _ in groups], np.concatenate([[0], np.cumsum([n for _, n in groups])])
        order, at = rng.permutation(n_pages).astype(np.int32), 0
        self.tables = np.full((b, width), -1, np.int32)
        for g, (p, _) in enumerate(groups):
            assert p % page == 0
            self.tables[self.cu_g[g]:self.cu_g[g + 1], :p // page] = order[at:at + p // page]
            at += p // page
        self.free, self.n_free = np.full(n_pages, -7, np.int32), n_pages - at
        self.free[:self.n_free] = order[at:]
        self.lens = np.repeat(self.prefix, [n for _, n in groups])
        self.rows, self.scales = make_pool(rng, kv, nkv, n_pages, page, hd)
        self.pool, self.dpool = dev_pool(self.rows, self.scales, kv)
        angle = rng.random((most, hd // 2)) * 6
        self.cos, self.sin = np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32)
        self.w = (0.5 + rng.random((2, hd))).astype(np.float32)
        self.d = d = dict(past=_i32(self.lens), keep=_i32(self.lens), add=_i32(np.zeros(b)), tables=_i32(self.tables), free_pages=_i32(self.free), n_free=_i32([self.n_free]),
                          cu_tokens=_i32(np.zeros(b + 1)), cu_pages=_i32(np.zeros(b + 1)), slots=_i32(np.zeros(n_rows)), positions=_i32(np.zeros(n_rows)), status=_i32([9, 9]))
        self.assign = paged.PageAssign(page_size=page, lens=d["past"], **d)
        self.store = paged.RowStore(self.pool, nq=nq, slots=d["slots"], positions=d["positions"], q_norm=DevArray(self.w[0]), k_norm=DevArray(self.w[1]), cos=DevArray(self.cos),
                                    sin=DevArray(self.sin), eps=1e-6)
        self.call = paged.PagedAttention(self.pool, nq=nq, tables=d["tables"], cu_tokens=d["cu_tokens"], positions=d["positions"], lens=d["past"], cu_groups=_i32(self.cu_g),
                                         prefix_lens=_i32(self.prefix))
        self.ws = DevArray(np.full(self.call.workspace_bytes // 4, np.nan, np.float32))
        self.dqkv = DevArray(np.zeros((n_rows, (nq + 2 * nkv) * hd), np.float32))
        self.dq, self.dout = (DevArray(pm.to_type(np.full((n_rows, nq, hd), 9.0), dtype), dtype) for _ in range(2))
        self.dlse = DevArray(np.full((n_rows, nq), 9.0, np.float32))

    def launch(self):
        self.assign()
        self.store(self.dqkv, self.dq)
        self.call(self.dq, self.dout, lse=self.dlse, workspace=self.ws)

    def step(self, keep, add, run):
        """New lengths and rows, the step by run(), and everything against the plain forms."""
        self.d["keep"].put(keep)
        self.d["add"].put(add)
        x = self.rng.standard_normal((self.t, self.nq + 2 * self.nkv, self.hd)).astype(np.float32)
        self.dqkv.put(x.reshape(self.t, -1))
        self.dout.put(pm.to_type(np.full(self.dout.shape, 9.0), self.dtype))
        self.dlse.put(np.full(self.dlse.shape, 9.0))
        run()
        w = pm.assign(self.lens, keep, add, self.tables, self.free, self.n_free, self.page, self.t)
        self.tables, self.free, self.n_free, self.lens, self.cu, self.pos = (w[n] for n in ("tables", "free", "n_free", "lens", "cu_tokens", "positions"))
        for n in ("tables", "cu_tokens", "positions", "slots", "status"):
            assert np.array_equal(self.d[n].get(), w[n]), n
        assert np.array_equal(self.d["past"].get(), w["lens"]) and self.d["n_free"].get()[0] == w["n_free"]
        n = int(self.cu[-1])
        at = self.pos[:n]
        turned = [pm.turned(x[:n, lo:hi], wt, self.cos[at], self.sin[at], 1e-6)
                  for lo, hi, wt in ((0, self.nq, self.w[0]), (self.nq, self.nq + self.nkv, self.w[1]))]
        self.q = self.dq.get()
        err = np.abs(pm.from_type(self.q, self.dtype)[:n] - turned[0])
        assert np.all(err <= HALF_STEP[self.dtype] * np.abs(turned[0]) + (64 + self.hd) * U * np.abs(turned[0]).max(-1, keepdims=True) + 2.0 ** -25)
        k = [d.get() for d in self.dpool if d is not None]
        self.rows, self.scales = k[:2], k[2:] or [None, None]
        stored = pm.pool_values(self.rows[0], self.scales[0], self.kv)[:, w["slots"][:n] // self.page, w["slots"][:n] % self.page].transpose(1, 0, 2)
        top = np.abs(turned[1]).max(-1, keepdims=True)
        step = {"f16": 2.0 ** -11 * np.abs(turned[1]) + 2.0 ** -25, "i8": top / 127 / 2 * 1.001, "fp8": 2.0 ** -4 * np.abs(turned[1]) + top / 448 * 2.0 ** -10}[self.kv]
        assert np.all(np.abs(stored - turned[1]) <= step + 2 * (64 + self.hd) * U * top)
        self.expect().check()


PLAN = [("add", [37, 5, 12, 0, 50, 3]), ("one", None), ("one", None), ("draft", 4), ("reject", 1), ("end", [2, 4]), ("add", [1, 1, 30, 1, 21, 1]), ("one", None)]


@pytest.mark.parametrize("dtype,kv", TYPES)
@pytest.mark.parametrize("graph", [False, True])
def test_steps_of_a_server(backend, dtype, kv, graph):
    """Chunks, single tokens, drafts, requests that end and others in their place: every step the same three calls, eagerly or as
    one captured graph that reads the lengths of its replay."""
    hip = _graphs()
    s = Step([(32, 2), (0, 1), (64, 3)], nq=8, nkv=2, hd=64, page=16, dtype=dtype, kv=kv, n_rows=130, seed=11)
    other = Attention(MIXED, **SMALL, dtype=dtype, kv=kv, seed=5)
    prefix = np.repeat(s.prefix, np.diff(s.cu_g))
    stream, graph_, gexec = C.c_void_p(0), C.c_void_p(0), C.c_void_p(0)
    run = s.launch
    try:
        if graph:
            assert hip.hipStreamCreate(C.byref(stream)) == 0
            backend.set_stream(stream.value)
            assert hip.hipStreamBeginCapture(stream, 0) == 0
            s.launch()
            assert hip.hipStreamEndCapture(stream, C.byref(graph_)) == 0
            assert hip.hipGraphInstantiate(C.byref(gexec), graph_, None, None, 0) == 0

            def run():
                assert hip.hipGraphLaunch(gexec, stream) == 0
                assert hip.hipStreamSynchronize(stream) == 0
        for what, arg in PLAN:
            keep, add = s.lens.copy(), np.ones(6, np.int32)
            if what == "add":
                add = np.array(arg)
            elif what == "draft":
                add[:] = arg
            elif what == "reject":
                keep -= 3
                add[:] = arg
            elif what == "end":
                keep[arg], add[arg] = prefix[arg], 0
            s.step(keep, add, run)
            other.run()
        other.expect().check()
    finally:
        backend.set_stream(0)
        if gexec:
            hip.hipGraphExecDestroy(gexec)
        if graph_:
            hip.hipGraphDestroy(graph_)
        if stream:
            hip.hipStreamDestroy(stream)


@pytest.mark.parametrize("kind", ["float32", "float16", "bfloat16"])
def test_rows_in_place(backend, kind):
    """q back into the product's rows: the same bits as into a buffer of its own, k and v beside it as they were."""
    rng = np.random.default_rng(2)
    n, nq, nkv, hd = 9, 6, 2, 64
    wide = (nq + 2 * nkv) * hd
    x = pm.to_type(rng.standard_normal((n, wide)), kind)
    angle = rng.random((20, hd // 2)) * 6
    kw = dict(nq=nq, slots=_i32(np.arange(n) + 3), positions=_i32(np.arange(n) * 2), q_norm=DevArray(np.ones(hd, np.float32) * 1.5), k_norm=DevArray(np.ones(hd, np.float32)),
              cos=DevArray(np.cos(angle).astype(np.float32)), sin=DevArray(np.sin(angle).astype(np.float32)))
    rows, scales = make_pool(rng, "f16", nkv, 2, 16, hd)
    got = []
    for own in (True, False):
        pool, d = dev_pool(rows, scales, "f16")
        qkv, q = DevArray(x, kind), DevArray(pm.to_type(np.zeros((n, nq, hd)), kind), kind)
        paged.RowStore(pool, **kw)(qkv, q if own else qkv.view(0, (n, nq, hd), (wide, hd, 1)))
        after = qkv.get()
        assert np.array_equal(after[:, nq * hd:], x[:, nq * hd:])
        got.append((q.get().reshape(n, -1) if own else after[:, :nq * hd], d[0].get(), d[1].get()))
    for a, b in zip(*got):
        assert np.array_equal(a, b)


def test_calls_between_torch_operations(backend):
    """The three calls on torch's default stream and on another of its streams, without a wait between them and torch's work."""
    here = os.path.dirname(os.path.abspath(__file__))
    env = dict(os.environ, PYTHONPATH=os.path.dirname(here))
    r = subprocess.run([sys.executable, os.path.join(here, "paged_torch.py")], env=env, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr
    assert r.stdout.split("\n")[:2] == ["the default stream ok", "a side stream ok"]


# Rows of one kv head: 4 (a wave to 16 rows), 40 (one tile of 16 rows to a wave), 280 (two of them).
DOMINATED = {"single": [(0, [(6000, 1)]), (3000, [(50, 1), (700, 1)])], "some": [(0, [(4000, 10)])], "chunk": [(0, [(3000, 70)])]}


@pytest.mark.parametrize("gap", [12.0, 17.5])
@pytest.mark.parametrize("name", DOMINATED)
@pytest.mark.parametrize("dtype,kv", TYPES)
def test_attention_one_key_over_thousands(backend, dtype, kv, name, gap):
    """The first key's score lies `gap` above all others': what the thousands have together is not lost beside it.

    Probabilities are rounded relative to 2^14 times the largest, so fp16 numbers below 2^-14 are off by 2^-25 = 2^-39 times the
    largest (p s) each, and all others by half a step, 2^-11, or 2^-22 for two terms."""
    a = Attention(DOMINATED[name], **SMALL, dtype=dtype, kv=kv, seed=7, poison=False, scale=1.0)
    rng, hd = a.rng, a.hd
    q = rng.uniform(-0.01, 0.01, (a.t, a.nq, hd))
    q[..., 0] = 1
    a.q = pm.to_type(q, dtype)
    shape = a.rows[0].shape
    first = np.zeros(shape[1:3], bool)
    for g in range(len(a.prefix)):
        first[a.tables[a.cu_g[g], 0], 0] = True
    small = rng.uniform(-0.01, 0.01, shape)
    small[..., 0] = 0
    if kv == "f16":
        small[:, first] = 0
        small[:, first, 0] = gap
        a.rows = [small.astype(np.float16), rng.uniform(0.5, 1.5, shape).astype(np.float16)]
    else:
        code = {"i8": lambda x: np.round(x * 12700).astype(np.int8), "fp8": lambda x: rng.integers(0x38, 0x40, shape).astype(np.uint8)}[kv](small)
        code[..., 0] = 0
        code[:, first] = 0
        code[:, first, 0] = 127 if kv == "i8" else 0x7e          # (448)
        full = 127 if kv == "i8" else 448
        a.rows = [code, (rng.integers(60, 128, shape).astype(np.int8) if kv == "i8" else rng.integers(0x30, 0x40, shape).astype(np.uint8))]
        a.scales = [np.where(first, gap / full, 0.01 / 128)[None].repeat(shape[0], 0).astype(np.float32),
                    rng.uniform(0.5, 1.5, shape[:3]).astype(np.float32) / (64 if kv == "i8" else 1)]
    a.rows[1][:, first, ::2] = 0                                 # (the others alone make up these dimensions)
    a.make()
    a.run().expect()
    out, lse, mag, low = a.want
    score = (2.0 ** -22 + hd * U) * a.size
    got, got_lse = pm.from_type(a.dout.get(), dtype), a.dlse.get()
    assert np.all(np.abs(got_lse - lse) <= score + 2.0 ** -20 + 2.0 ** -22 * np.abs(lse))
    p_err = (2.0 ** -11 if dtype != "float32" else 2.0 ** -22) + 2 * score[..., None] + int(a.lens.max()) ** 0.5 * 8 * U + 2.0 ** -20
    limit = p_err * mag + 2.0 ** -39 * low + HALF_STEP[dtype] * np.abs(out) + (2.0 ** -25 if dtype == "float16" else 0)
    assert np.max(np.abs(got - out) / limit) <= 1


@pytest.mark.parametrize("how", ["scale", "queries"])
@pytest.mark.parametrize("dtype,kv", TYPES)
def test_attention_scores_too_small_for_numbers(backend, dtype, kv, how):
    """scale times a query's largest value lies below all fp32 numbers: every key that is seen counts the same."""
    if how == "queries" and dtype == "float16":
        pytest.skip("a float16 query's smallest value times the scale is a number")
    a = Attention(MIXED + [(0, [(30, 12)])], **SMALL, dtype=dtype, kv=kv, seed=4, scale=1e-45 if how == "scale" else 2.0 ** -24)
    a.q = pm.to_type(pm.from_type(a.q, dtype) * (2.0 ** -12 if how == "scale" else 2.0 ** -131), dtype)
    a.make()
    a.run().expect().check()
    assert np.isfinite(a.dlse.get()).all()


def test_rows_that_overlap_are_refused(backend):
    """Through the C entries too, which see addresses alone; rows that lie side by side in one buffer are taken."""
    a = Attention(MIXED, **SMALL, dtype="float16", kv="f16", seed=5)
    t, wide, hd = a.t, a.nq * a.hd, a.hd
    both = DevArray(pm.to_type(np.concatenate([pm.from_type(a.q, "float16").reshape(t, -1), np.full((t, wide + 64), 9.0)], 1), "float16"), "float16")
    at = lambda first, stride=2 * wide + 64: both.view(first, (t, a.nq, hd), (stride, hd, 1))  # noqa: E731
    for out in (at(wide - 8), at(8), at(2 * wide + 64), at(16, wide)):
        with pytest.raises(GpuError, match="overlap"):
            a.call(at(0), out, workspace=a.ws)
    a.call(at(0), at(wide), workspace=a.ws)
    assert np.array_equal(both.get()[:, wide:2 * wide].reshape(t, a.nq, hd), a.run().dout.get())
    n, nq, nkv = 6, 4, 2
    full = (nq + 2 * nkv) * hd
    x = DevArray(np.zeros((n, 2 * full), np.float32))
    store = paged.RowStore(a.pool, nq=nq, slots=_i32(np.full(n, -1)), positions=_i32(np.zeros(n)))
    half = DevArray(None, view=(x, 0, (n, nq, hd), (2 * full, hd, 1)))
    half.dtype = "x.float16"                                     # (the same addresses as another type)
    qkv = x.view(0, (n, full), (2 * full, 1))
    for q in (half, x.view(8, (n, nq, hd), (2 * full, hd, 1)), x.view(0, (n, nq, hd), (full, hd, 1)), x.view(full - 8, (n, nq, hd), (2 * full, hd, 1))):
        with pytest.raises(GpuError, match="overlap"):
            store(qkv, q)
    for q in (x.view(0, (n, nq, hd), (2 * full, hd, 1)), x.view(full, (n, nq, hd), (2 * full, hd, 1))):
        store(qkv, q)
