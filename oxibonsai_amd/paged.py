"""A serving step over a paged cache, on device buffers: requests of different lengths, prefixes that several of them share.

Three operators, each an object that is made once for a program's buffers and called once per step (``PageAssign``) or per
step and layer (``RowStore``, ``PagedAttention``):

    assign = PageAssign(past=..., add=..., tables=..., ...)       # lengths -> page tables, slots, positions
    store = RowStore(pool, nq=32, slots=..., positions=..., q_norm=..., k_norm=..., cos=..., sin=...)
    attend = PagedAttention(pool, nq=32, tables=..., cu_tokens=..., positions=..., lens=..., cu_groups=..., prefix_lens=...)
    assign(); store(qkv, q); attend(q, out, workspace=ws)

The reference keeps its tables on the host and its rows one token at a time (``PagedKvCache``,
crates/oxibonsai-model/src/paged_kv_cache.rs:294-470).  Buffers are anything with ``data_ptr()``, ``shape``, ``stride()``,
``dtype`` and ``device`` (torch tensors); they stay the caller's and have to live as long as the object.  Calls run on
the library's stream (``NativeHipBackend.set_stream``) and wait for nothing; they may be captured into a graph.  An object takes calls of one thread at a time.  What the
fields mean stands at the C structs of the same names, include/oxb_hip.h."""
from __future__ import annotations

import ctypes as C

from . import _lib
from .backend import GpuError, _check

DTYPES = {"float32": 0, "float16": 1, "bfloat16": 2}                               # OXB_DTYPE_*
KV_DTYPES = {"float16": 0, "int8": 1, "float8_e4m3fn": 2}                          # OXB_KV_DTYPE_*


class _PagePool(C.Structure):
    _fields_ = [(n, C.c_void_p) for n in ("d_k", "d_v", "d_k_scale", "d_v_scale")] + \
               [(n, C.c_uint32) for n in ("kv_dtype", "nkv", "hd", "page_size", "n_pages")]


class _PageAssign(C.Structure):
    _fields_ = [(n, C.c_uint32) for n in ("n_requests", "page_size", "n_pages", "table_width", "n_rows")] + \
               [(n, C.c_void_p) for n in ("d_past", "d_keep", "d_add", "d_tables", "d_free_pages", "d_n_free", "d_n_free_out", "d_lens",
                                          "d_cu_tokens", "d_cu_pages", "d_slots", "d_positions", "d_status")]


class _PagedRows(C.Structure):
    _fields_ = [("n_rows", C.c_uint32), ("nq", C.c_uint32), ("d_qkv", C.c_void_p), ("qkv_dtype", C.c_uint32), ("qkv_stride", C.c_uint32)] + \
               [(n, C.c_void_p) for n in ("d_positions", "d_slots", "d_q_norm", "d_k_norm", "d_cos", "d_sin")] + \
               [("n_angles", C.c_uint32), ("eps", C.c_float), ("d_q_out", C.c_void_p), ("q_dtype", C.c_uint32), ("q_stride", C.c_uint32),
                ("pool", _PagePool)]


class _PagedAttention(C.Structure):
    _fields_ = [(n, C.c_uint32) for n in ("n_tokens", "n_requests", "n_groups", "nq", "dtype", "q_stride", "out_stride", "table_width")] + \
               [(n, C.c_void_p) for n in ("d_q", "d_out", "d_lse", "d_tables", "d_cu_tokens", "d_positions", "d_lens", "d_cu_groups",
                                          "d_prefix_lens")] + \
               [("scale", C.c_float), ("d_workspace", C.c_void_p), ("workspace_bytes", C.c_size_t), ("pool", _PagePool)]


def _bad(text: str) -> GpuError:
    return GpuError(5, f"invalid argument: {text}")


def _kind(t) -> str:
    return str(t.dtype).rpartition(".")[2]


def _at(t, name: str, device):
    """A tensor's address, on the GPU that the other tensors are on."""
    if t.device.type != "cuda" or (device is not None and t.device != device):
        raise _bad(f"{name} is on {t.device}" + (f", not on {device}" if device is not None else ", not on a GPU"))
    return t.data_ptr()


_one_runtime = False


def _runtimes() -> list[str]:
    """The HIP runtimes in this process: torch ships one of its own, which a library that is loaded later uses too."""
    with open("/proc/self/maps") as maps:
        return sorted({line.split()[-1] for line in maps if "/libamdhip64.so" in line})


def _home(t) -> None:
    """The library runs on one GPU, this one if it has not started yet; tensors of another are refused, and so are those of a torch that
    brought a second runtime, whose streams and graphs are none to the library."""
    global _one_runtime
    device = t.device
    if not _one_runtime and type(t).__module__.partition(".")[0] == "torch":
        _lib.lib()
        found = _runtimes()
        if len(found) > 1:
            raise _bad(f"two HIP runtimes are loaded ({', '.join(found)}): import torch before the library is")
        _one_runtime = True
    if device.type == "cuda" and getattr(device, "index", None) is not None:
        _check(_lib.lib().oxb_hip_init(device.index))


def _flat(t, name: str, kind: str, shape, device):
    """Address of a contiguous tensor of this type and shape; None stays None."""
    if t is None:
        return None
    if _kind(t) != kind or tuple(t.shape) != tuple(shape) or not t.is_contiguous():
        raise _bad(f"{name} is {_kind(t)} {tuple(t.shape)} with strides {tuple(t.stride())}, not contiguous {kind} {tuple(shape)}")
    return _at(t, name, device)


def _rows(t, name: str, n: int, wide: int, device):
    """Address, type and row stride of n rows of `wide` values each, given as [n, wide] or [n, heads, head_dim]."""
    if _kind(t) not in DTYPES:
        raise _bad(f"{name} is {_kind(t)}, not one of {', '.join(DTYPES)}")
    shape, stride = tuple(t.shape), tuple(t.stride())
    packed = (len(shape) == 2 and stride[1] == 1) or (len(shape) == 3 and stride[2] == 1 and (stride[1] == shape[2] or shape[1] == 1))
    if not packed or shape[0] != n or wide != (shape[1] if len(shape) == 2 else shape[1] * shape[2]):
        raise _bad(f"{name} has shape {shape} and strides {stride}, not {n} rows of {wide} values side by side")
    return _at(t, name, device), DTYPES[_kind(t)], stride[0] if n > 1 else max(stride[0], wide)


class PagePool:
    """One layer's cache rows, ``oxb_page_pool``: k and v [nkv, n_pages, page_size, hd] as float16, int8 or float8_e4m3fn, the
    one-byte types with float32 row scales [nkv, n_pages, page_size]."""

    def __init__(self, k, v, k_scale=None, v_scale=None):
        kind = _kind(k)
        if len(k.shape) != 4 or KV_DTYPES.get(kind) is None:
            raise _bad(f"k is {kind} {tuple(k.shape)}, not float16, int8 or float8_e4m3fn [nkv, n_pages, page_size, hd]")
        _home(k)
        self.device, self.kv_dtype = k.device, KV_DTYPES[kind]
        self.nkv, self.n_pages, self.page_size, self.hd = (int(n) for n in k.shape)
        scales = [None, None]
        if self.kv_dtype:
            if k_scale is None or v_scale is None:
                raise _bad(f"{kind} rows need row scales")
            scales = [_flat(t, n, "float32", k.shape[:3], k.device) for t, n in ((k_scale, "k_scale"), (v_scale, "v_scale"))]
        self._keep = (k, v, k_scale, v_scale)
        self.c = _PagePool(_flat(k, "k", kind, k.shape, None), _flat(v, "v", kind, k.shape, k.device), *scales, self.kv_dtype, self.nkv, self.hd,
                           self.page_size, self.n_pages)


class _Bound:
    """A descriptor with the buffers that it points into."""

    def _bind(self, desc, keep):
        self._lib, self.c, self._keep = _lib.lib(), desc, keep
        self._ref = C.byref(desc)


class PageAssign(_Bound):
    """``oxb_page_assign``: page tables, slot map and positions of a step from the requests' lengths.  All buffers int32."""

    def __init__(self, *, past, add, tables, free_pages, n_free, lens, cu_tokens, cu_pages, slots, positions, status, page_size: int,
                 n_free_out=None, keep=None):
        if len(tables.shape) != 2 or len(slots.shape) != 1 or len(free_pages.shape) != 1:
            raise _bad("tables is [n_requests, width], slots [n_rows], free_pages [n_pages]")
        _home(tables)
        b, width = (int(n) for n in tables.shape)
        rows, pages, dev = int(slots.shape[0]), int(free_pages.shape[0]), tables.device
        n_free_out = n_free if n_free_out is None else n_free_out
        sizes = dict(past=(past, b), keep=(keep, b), add=(add, b), tables=(tables, None), free_pages=(free_pages, pages), n_free=(n_free, 1),
                     n_free_out=(n_free_out, 1), lens=(lens, b), cu_tokens=(cu_tokens, b + 1), cu_pages=(cu_pages, b + 1), slots=(slots, rows),
                     positions=(positions, rows), status=(status, 2))
        at = {n: _flat(t, n, "int32", (b, width) if k is None else (k,), dev) for n, (t, k) in sizes.items()}
        self._bind(_PageAssign(b, page_size, pages, width, rows, *at.values()), [t for t, _ in sizes.values()])

    def __call__(self) -> None:
        _check(self._lib.oxb_hip_paged_assign_dev(self._ref))


class RowStore(_Bound):
    """``oxb_paged_rows``: QK-norm, RoPE and the store of a step's new rows.  ``positions`` may be None where nothing is rotated."""

    def __init__(self, pool: PagePool, *, nq: int, slots, positions=None, q_norm=None, k_norm=None, cos=None, sin=None, eps: float = 1e-6):
        if len(slots.shape) != 1:
            raise _bad("slots is [n_rows]")
        n, hd, dev = int(slots.shape[0]), pool.hd, pool.device
        angles = int(cos.shape[0]) if cos is not None else 0
        at = [_flat(t, name, kind, shape, dev) for t, name, kind, shape in
              ((positions, "positions", "int32", (n,)), (slots, "slots", "int32", (n,)), (q_norm, "q_norm", "float32", (hd,)), (k_norm, "k_norm", "float32", (hd,)),
               (cos, "cos", "float32", (angles, hd // 2)), (sin, "sin", "float32", (angles, hd // 2)))]
        self.n, self.nq, self.wide, self._q_wide, self._dev = n, nq, (nq + 2 * pool.nkv) * hd, nq * hd, dev
        self._bind(_PagedRows(n, nq, None, 0, 0, *at, angles, eps, None, 0, 0, pool.c), (pool, slots, positions, q_norm, k_norm, cos, sin))

    def __call__(self, qkv, q_out=None) -> None:
        """qkv [n_rows, (nq + 2 nkv) hd]; q_out [n_rows, nq, hd] receives the q heads (None: they are not looked at)."""
        c = self.c
        c.d_qkv, c.qkv_dtype, c.qkv_stride = _rows(qkv, "qkv", self.n, self.wide, self._dev)
        c.d_q_out, c.q_dtype, c.q_stride = _rows(q_out, "q_out", self.n, self._q_wide, self._dev) if q_out is not None else (None, 0, 0)
        _check(self._lib.oxb_hip_paged_rows_dev(self._ref))


class PagedAttention(_Bound):
    """``oxb_paged_attention``: attention of a step's queries over the pool, prefixes that groups of requests share read once."""

    def __init__(self, pool: PagePool, *, nq: int, tables, cu_tokens, positions, lens, cu_groups=None, prefix_lens=None, scale: float = 0.0):
        if len(tables.shape) != 2 or len(positions.shape) != 1 or (cu_groups is None) != (prefix_lens is None):
            raise _bad("tables is [n_requests, width], positions [n_tokens]; cu_groups and prefix_lens come together")
        (b, width), t, dev = (int(n) for n in tables.shape), int(positions.shape[0]), pool.device
        groups = int(prefix_lens.shape[0]) if prefix_lens is not None else 0
        at = [_flat(x, name, "int32", shape, dev) for x, name, shape in
              ((tables, "tables", (b, width)), (cu_tokens, "cu_tokens", (b + 1,)), (positions, "positions", (t,)), (lens, "lens", (b,)),
               (cu_groups, "cu_groups", (groups + 1,)), (prefix_lens, "prefix_lens", (groups,)))]
        self.n, self.nq, self._wide, self._dev = t, nq, nq * pool.hd, dev
        self._bind(_PagedAttention(t, b, groups, nq, 0, 0, 0, width, None, None, None, *at, scale, None, 0, pool.c),
                   (pool, tables, cu_tokens, positions, lens, cu_groups, prefix_lens))
        n = C.c_size_t(0)
        _check(self._lib.oxb_hip_paged_attention_workspace(self._ref, C.byref(n)))
        self.workspace_bytes = int(n.value)

    def __call__(self, q, out, *, workspace, lse=None) -> None:
        """q, out [n_tokens, nq, hd] of one type, lse float32 [n_tokens, nq]; workspace: workspace_bytes of GPU memory, which calls
        on one stream may share."""
        c, dev = self.c, self._dev
        c.d_q, c.dtype, c.q_stride = _rows(q, "q", self.n, self._wide, dev)
        c.d_out, kind, c.out_stride = _rows(out, "out", self.n, self._wide, dev)
        if kind != c.dtype:
            raise _bad(f"q is {_kind(q)}, out {_kind(out)}")
        if c.d_q == c.d_out:
            raise _bad("out is q, which is still read while rows of out are written")
        c.d_lse = _flat(lse, "lse", "float32", (self.n, self.nq), dev)
        if not workspace.is_contiguous():
            raise _bad("the workspace is not contiguous")
        c.d_workspace, c.workspace_bytes = _at(workspace, "workspace", dev), workspace.numel() * workspace.element_size()
        _check(self._lib.oxb_hip_paged_attention_dev(self._ref))
