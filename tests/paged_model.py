"""Plain float64 / integer restatements of a serving step's operators over a paged cache, and device arrays for their tests."""
import numpy as np

from helpers import DeviceBuffer

E4M3 = np.array([(-1.0) ** (c >> 7) * ((c & 7) * 2.0 ** -9 if not (c >> 3) & 15 else (1 + (c & 7) / 8) * 2.0 ** (((c >> 3) & 15) - 7)) if c & 0x7f != 0x7f else np.nan
                 for c in range(256)])


def bf16_bits(x):
    """float32 -> bfloat16 bits, to nearest even."""
    u = np.ascontiguousarray(x, dtype=np.float32).view(np.uint32).astype(np.uint64)
    nan = (u & 0x7fffffff) > 0x7f800000
    return np.where(nan, (u >> 16) | 0x40, (u + 0x7fff + ((u >> 16) & 1)) >> 16).astype(np.uint16)


def bf16_values(b):
    return (np.ascontiguousarray(b).astype(np.uint32) << 16).view(np.float32)


def to_type(x, kind):
    """Values as the array that a buffer of this type holds."""
    if kind == "bfloat16":
        return bf16_bits(x)
    return np.ascontiguousarray(x, dtype={"float16": np.float16, "float32": np.float32, "int32": np.int32}[kind])


def from_type(a, kind):
    return bf16_values(a).astype(np.float64) if kind == "bfloat16" else a.astype(np.float64)


class _Device:
    type = "cuda"

    def __eq__(self, other):
        return getattr(other, "type", None) == "cuda"


class DevArray:
    """What the package asks of a buffer (data_ptr, shape, stride, dtype, device), on the HIP runtime that the library links."""
    device = _Device()

    def __init__(self, a, kind=None, view=None):
        if view is not None:     # (DevArray, first element, shape, strides)
            base, first, self.shape, self._stride = view
            self.buf, self.host, self.dtype, self.first = base.buf, base.host, base.dtype, base.first + first
            return
        self.host = np.ascontiguousarray(a)
        self.dtype = "x." + (kind or str(self.host.dtype))
        self.shape, self._stride = tuple(self.host.shape), tuple(s // self.host.itemsize for s in self.host.strides)
        self.first = 0
        self.buf = DeviceBuffer.from_numpy(self.host) if self.host.nbytes else DeviceBuffer(16)

    def data_ptr(self):
        return self.buf.ptr + self.first * self.host.itemsize

    def stride(self):
        return self._stride

    def is_contiguous(self):
        want, n = [], 1
        for s in reversed(self.shape):
            want.insert(0, n)
            n *= s
        return all(a == b or s == 1 for a, b, s in zip(self._stride, want, self.shape))

    def numel(self):
        return int(np.prod(self.shape))

    def element_size(self):
        return self.host.itemsize

    def view(self, first, shape, strides):
        return DevArray(None, view=(self, first, tuple(shape), tuple(strides)))

    def get(self):
        """The whole allocation as it is now."""
        return self.buf.to_numpy(self.host.dtype, self.host.shape)

    def put(self, a):
        a = np.ascontiguousarray(a, dtype=self.host.dtype)
        assert a.shape == self.host.shape
        assert DeviceBuffer.hip().hipDeviceSynchronize() == 0
        assert DeviceBuffer.hip().hipMemcpy(self.buf.ptr, a.ctypes.data, a.nbytes, 1) == 0


def assign(past, keep, add, tables, free, n_free, page, n_rows):
    """The step's tables, slots and positions, one request after the other."""
    past, add = [int(x) for x in past], [int(x) for x in add]
    keep = past if keep is None else [min(int(k), p) for k, p in zip(keep, past)]
    pages = lambda n: -(-n // page)  # noqa: E731
    tables, free, b, w = tables.copy(), free.copy(), len(past), tables.shape[1]
    none = np.full(n_rows, -1, np.int32)
    zeros = np.zeros(b + 1, np.int32)

    def failed(code, need):
        return dict(tables=tables, free=free, n_free=n_free, lens=np.array(past), cu_tokens=zeros, cu_pages=zeros, slots=none, positions=none, status=[code, need])

    fits = [k + a <= w * page and p <= w * page for k, a, p in zip(keep, add, past)]
    freed = sum(pages(p) - pages(k) for k, p, f in zip(keep, past, fits) if f and min(k, p) >= 0)
    need = sum(pages(k + a) - pages(k) for k, a, p, f in zip(keep, add, past, fits) if f and min(k, a, p) >= 0)
    if min(past + keep + add) < 0 or n_free < 0 or n_free + freed > len(free):
        return failed(3, need)
    if need > n_free + freed:
        return failed(1, need)
    if not all(fits) or sum(add) > n_rows:
        return failed(2, need)
    for r in range(b):
        for j in range(pages(keep[r]), pages(past[r])):
            free[n_free] = tables[r, j]
            n_free += 1
    slots, positions, cu, cup = [], [], [0], [0]
    for r in range(b):
        for j in range(pages(keep[r]), pages(keep[r] + add[r])):
            n_free -= 1
            tables[r, j] = free[n_free]
        for i in range(add[r]):
            p = keep[r] + i
            positions.append(p)
            slots.append(tables[r, p // page] * page + p % page if 0 <= tables[r, p // page] < len(free) else -1)
        cu.append(cu[-1] + add[r])
        cup.append(cup[-1] + pages(keep[r] + add[r]) - pages(keep[r]))
    s, q = none.copy(), none.copy()
    s[:len(slots)], q[:len(slots)] = slots, positions
    return dict(tables=tables, free=free, n_free=n_free, lens=np.array(keep) + np.array(add), cu_tokens=cu, cu_pages=cup, slots=s, positions=q, status=[0, need])


def turned(x, w, cos, sin, eps):
    """RMSNorm with weights w (None: not) and RoPE by the rows cos, sin (None: not) of heads [n, heads, hd], in float64."""
    x = x.astype(np.float64)
    if w is not None:
        x = w.astype(np.float64) * x / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    if cos is not None:
        h = x.shape[-1] // 2
        c, s = cos.astype(np.float64)[:, None], sin.astype(np.float64)[:, None]
        x = np.concatenate([x[..., :h] * c - x[..., h:] * s, x[..., :h] * s + x[..., h:] * c], -1)
    return x


def pool_values(rows, scales, kv):
    """Cache rows [nkv, n_pages, page, hd] as the numbers they stand for."""
    v = rows.astype(np.float64) if kv == "f16" else rows.view(np.int8).astype(np.float64) if kv == "i8" else E4M3[rows.view(np.uint8)]
    return v if scales is None else v * scales.astype(np.float64)[..., None]


def attention(q, k, v, v_scale, tables, cu_tokens, positions, lens, cu_groups, prefix_lens, page, scale):
    """out [n_tokens, nq, hd], lse [n_tokens, nq] of the definition, and what bounds the roundings of the probabilities, both
    [n_tokens, nq, hd]: sum p |v| / sum p, and max(p s) sum(|v| / s) / sum p with the row scales s of v (None: 1).
    q [n_tokens, nq, hd], k and v [nkv, n_pages, page, hd] float64.  Rows of no request stay NaN."""
    t, nq, hd = q.shape
    nkv = k.shape[0]
    out, mag, low, lse = np.full((t, nq, hd), np.nan), np.zeros((t, nq, hd)), np.zeros((t, nq, hd)), np.full((t, nq), np.nan)
    for r in range(len(lens)):
        g0, shared = r, 0
        for a, b, n in zip(cu_groups[:-1], cu_groups[1:], prefix_lens) if cu_groups is not None else ():
            if a <= r < b:
                g0, shared = a, n
        for i in range(cu_tokens[r], cu_tokens[r + 1]):
            n = max(0, min(positions[i] + 1, lens[r]))
            at = np.arange(n)
            pages = np.where(at < shared, tables[g0][at // page], tables[r][at // page])
            for h in range(nq):
                if n == 0:
                    out[i, h], lse[i, h] = 0, -np.inf
                    continue
                kk, vv = k[h // (nq // nkv)][pages, at % page], v[h // (nq // nkv)][pages, at % page]
                s = kk @ q[i, h] * scale
                top = s.max()
                e = np.exp(s - top)
                out[i, h], mag[i, h], lse[i, h] = e @ vv / e.sum(), e @ np.abs(vv) / e.sum(), top + np.log(e.sum())
                size = np.ones(n) if v_scale is None else v_scale[h // (nq // nkv)][pages, at % page].astype(np.float64)
                low[i, h] = (e * size).max() * (np.abs(vv) / size[:, None]).sum(0) / e.sum()
    return out, lse, mag, low
