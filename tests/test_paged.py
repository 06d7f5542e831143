"""A serving step's operators over a paged cache, without a GPU: structs, refusals, workspaces, and the plain restatements that the
GPU tests compare with."""
import ctypes as C
import os
import shutil
import subprocess
import sys
from types import SimpleNamespace

import numpy as np
import pytest

import paged_model as pm
from oxibonsai_amd import GpuError, NativeHipBackend, _lib, paged

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
INVALID, NOT_AVAILABLE = 5, 1


def test_structs_match_the_header_layout(tmp_path):
    mirrors = {"oxb_page_pool": paged._PagePool, "oxb_page_assign": paged._PageAssign, "oxb_paged_rows": paged._PagedRows,
               "oxb_paged_attention": paged._PagedAttention}
    cc = shutil.which("gcc") or shutil.which("cc")
    if not cc:
        pytest.skip("no C compiler")
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "oxb_hip.h"', 'int main(void) {']
    for name, cls in mirrors.items():
        lines.append(f'  printf("{name} %zu\\n", sizeof({name}));')
        lines += [f'  printf("{name}.{f} %zu\\n", offsetof({name}, {f}));' for f, _ in cls._fields_]
    (tmp_path / "layout.c").write_text("\n".join(lines + ['  return 0;', '}']))
    subprocess.run([cc, "-std=c99", "-I", os.path.join(ROOT, "include"), str(tmp_path / "layout.c"), "-o", str(tmp_path / "layout")], check=True)
    seen = dict(l.split() for l in subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True, text=True).stdout.splitlines())
    for name, cls in mirrors.items():
        assert int(seen[name]) == C.sizeof(cls), name
        for f, _ in cls._fields_:
            assert int(seen[f"{name}.{f}"]) == getattr(cls, f).offset, (name, f)


P = 1 << 20     # an address that no call of this file follows


def pool(**kw):
    f = dict(d_k=P, d_v=P, d_k_scale=P, d_v_scale=P, kv_dtype=0, nkv=2, hd=64, page_size=16, n_pages=10) | kw
    return paged._PagePool(*f.values())


def assign(**kw):
    f = dict(n_requests=3, page_size=16, n_pages=10, table_width=4, n_rows=7, d_past=P, d_keep=0, d_add=P, d_tables=P, d_free_pages=P, d_n_free=P,
             d_n_free_out=P, d_lens=P, d_cu_tokens=P, d_cu_pages=P, d_slots=P, d_positions=P, d_status=P) | kw
    return _lib.lib().oxb_hip_paged_assign_dev(C.byref(paged._PageAssign(*f.values())))


def rows(pool_kw=(), **kw):
    f = dict(n_rows=5, nq=4, d_qkv=P, qkv_dtype=0, qkv_stride=512, d_positions=P, d_slots=P, d_q_norm=P, d_k_norm=P, d_cos=P, d_sin=P, n_angles=9,
             eps=1e-6, d_q_out=P, q_dtype=1, q_stride=256) | kw
    return _lib.lib().oxb_hip_paged_rows_dev(C.byref(paged._PagedRows(*f.values(), pool(**dict(pool_kw)))))


def attention(pool_kw=(), **kw):
    f = dict(n_tokens=5, n_requests=3, n_groups=1, nq=4, dtype=1, q_stride=256, out_stride=256, table_width=4, d_q=P, d_out=P, d_lse=P, d_tables=P,
             d_cu_tokens=P, d_positions=P, d_lens=P, d_cu_groups=P, d_prefix_lens=P, scale=0.0, d_workspace=P, workspace_bytes=1 << 40) | kw
    return _lib.lib().oxb_hip_paged_attention_dev(C.byref(paged._PagedAttention(*f.values(), pool(**dict(pool_kw)))))


# (without a GPU a call that is in order ends at the library's start; with one it is not made)
@pytest.mark.skipif(_lib.lib().oxb_hip_device_count() > 0, reason="the addresses are none")
@pytest.mark.parametrize("call", [assign, rows, attention])
def test_calls_in_order_need_a_gpu(call):
    assert call() == NOT_AVAILABLE


BAD_POOLS = [dict(d_k=0), dict(d_v=0), dict(d_k=P + 8), dict(kv_dtype=3), dict(kv_dtype=1, d_k_scale=0), dict(kv_dtype=2, d_v_scale=P + 4), dict(nkv=0),
             dict(nkv=2000), dict(hd=48), dict(hd=0), dict(hd=512), dict(page_size=8), dict(page_size=24), dict(page_size=256), dict(n_pages=0),
             dict(n_pages=1 << 27)]


@pytest.mark.parametrize("kw", [dict(n_requests=0), dict(n_requests=4097), dict(page_size=0), dict(page_size=17), dict(n_pages=0), dict(n_pages=1 << 28),
                                dict(table_width=0), dict(table_width=1 << 28), dict(n_rows=(1 << 30) + 1)] +
                         [{n: 0} for n in ("d_past", "d_add", "d_tables", "d_free_pages", "d_n_free", "d_n_free_out", "d_lens", "d_cu_tokens", "d_cu_pages",
                                           "d_slots", "d_positions", "d_status")], ids=str)
def test_assign_refusals(kw):
    assert assign(**kw) == INVALID
    assert "invalid argument" in _lib.last_error()


@pytest.mark.parametrize("kw", [dict(n_rows=0), dict(n_rows=(1 << 30) + 1), dict(nq=1 << 20), dict(d_qkv=0), dict(d_qkv=P + 8), dict(qkv_dtype=3), dict(q_dtype=7),
                                dict(qkv_stride=504), dict(qkv_stride=516), dict(q_stride=248), dict(q_stride=260), dict(d_slots=0), dict(d_cos=0), dict(d_sin=0),
                                dict(d_positions=0), dict(n_angles=0), dict(d_q_out=P + 4), dict(nq=0), dict(d_cos=P + 4), dict(d_q_norm=P + 8)] +
                         [dict(pool_kw=tuple(p.items())) for p in BAD_POOLS], ids=str)
def test_rows_refusals(kw):
    assert rows(**kw) == INVALID
    assert "invalid argument" in _lib.last_error()


@pytest.mark.parametrize("kw", [dict(n_tokens=0), dict(n_tokens=1 << 29), dict(n_requests=0), dict(n_requests=4097), dict(n_groups=4), dict(nq=0), dict(nq=5), dict(nq=34),
                                dict(dtype=3), dict(q_stride=248), dict(out_stride=252), dict(q_stride=260), dict(table_width=0), dict(table_width=1 << 27),
                                dict(scale=float("nan")), dict(scale=float("inf")), dict(workspace_bytes=100), dict(d_workspace=P + 16), dict(d_q=P + 8),
                                dict(d_out=P + 2)] +
                         [{n: 0} for n in ("d_q", "d_out", "d_tables", "d_cu_tokens", "d_positions", "d_lens", "d_cu_groups", "d_prefix_lens", "d_workspace")] +
                         [dict(pool_kw=tuple(p.items())) for p in BAD_POOLS], ids=str)
def test_attention_refusals(kw):
    assert attention(**kw) == INVALID
    assert "invalid argument" in _lib.last_error()


def test_null_descriptors():
    L, n = _lib.lib(), C.c_size_t(0)
    for f in (L.oxb_hip_paged_assign_dev, L.oxb_hip_paged_rows_dev, L.oxb_hip_paged_attention_dev):
        assert f(None) == INVALID
    assert L.oxb_hip_paged_attention_workspace(None, C.byref(n)) == INVALID


class Host:
    """A buffer of the binding's interface that is nowhere."""

    def __init__(self, shape, kind, device="cuda", stride=None):
        self.shape, self.dtype, self._stride = shape, "x." + kind, stride or tuple(int(np.prod(shape[i + 1:])) for i in range(len(shape)))
        self.device = type("D", (), {"type": device, "__eq__": lambda a, b: a.type == b.type, "__str__": lambda a: a.type})()

    def data_ptr(self):
        return P

    def stride(self):
        return self._stride

    def is_contiguous(self):
        return self._stride == tuple(int(np.prod(self.shape[i + 1:])) for i in range(len(self.shape)))


def ints(*shape, **kw):
    return Host(shape, "int32", **kw)


def test_binding_refuses_other_types_shapes_and_devices():
    k = Host((2, 10, 16, 64), "float16")
    p = paged.PagePool(k, k)
    assert (p.nkv, p.n_pages, p.page_size, p.hd, p.kv_dtype) == (2, 10, 16, 64, 0)
    for bad in (lambda: paged.PagePool(Host((2, 10, 16, 64), "bfloat16"), k), lambda: paged.PagePool(k, Host((2, 10, 16, 32), "float16")),
                lambda: paged.PagePool(k, Host((2, 10, 16, 64), "float16", device="cpu")), lambda: paged.PagePool(Host((2, 10, 16, 64), "int8"), k),
                lambda: paged.PagePool(Host((2, 10, 64), "float16"), k), lambda: paged.PagePool(k, Host((2, 10, 16, 64), "float16", stride=(1, 1, 1, 1)))):
        with pytest.raises(GpuError):
            bad()
    ok = dict(nq=4, tables=ints(3, 4), cu_tokens=ints(4), positions=ints(5), lens=ints(3))
    assert paged.PagedAttention(p, **ok).workspace_bytes > 0
    for kw in (dict(tables=ints(3, 4, device="cpu")), dict(tables=Host((3, 4), "int64")), dict(cu_tokens=ints(3)), dict(lens=ints(4)), dict(cu_groups=ints(2)),
               dict(cu_groups=ints(2), prefix_lens=ints(2)), dict(nq=3), dict(tables=ints(3, 4, stride=(8, 1))), dict(positions=ints(0))):
        with pytest.raises(GpuError):
            paged.PagedAttention(p, **(ok | kw))
    store = dict(nq=4, slots=ints(5), positions=ints(5), cos=Host((9, 32), "float32"), sin=Host((9, 32), "float32"))
    paged.RowStore(p, **store)
    for kw in (dict(sin=None), dict(sin=Host((8, 32), "float32")), dict(q_norm=Host((32,), "float32")), dict(slots=ints(4)), dict(positions=None)):
        with pytest.raises(GpuError):
            paged.RowStore(p, **(store | kw))(Host((5, 512), "float32"), Host((5, 4, 64), "float16"))
    s = paged.RowStore(p, **store)
    for x, q in ((Host((5, 500), "float32"), None), (Host((4, 512), "float32"), None), (Host((5, 512), "float64"), None), (Host((5, 512), "float32", stride=(512, 2)), None),
                 (Host((5, 512), "float32"), Host((5, 4, 32), "float16")), (Host((5, 512), "float32"), Host((5, 4, 64), "float16", stride=(512, 128, 1)))):
        with pytest.raises(GpuError):
            s(x, q)
    a = paged.PagedAttention(p, **ok)
    ws = Host((a.workspace_bytes,), "uint8")
    for q, out, lse in ((Host((5, 4, 64), "float16"), Host((5, 4, 64), "float32"), None), (Host((5, 4, 64), "float16"), Host((5, 4, 64), "float16"), Host((5, 3), "float32"))):
        with pytest.raises(GpuError):
            a(q, out, lse=lse, workspace=ws)
    with pytest.raises(GpuError):
        paged.PageAssign(past=ints(3), add=ints(3), tables=ints(3, 4), free_pages=ints(9), n_free=ints(1), lens=ints(3), cu_tokens=ints(3), cu_pages=ints(4),
                         slots=ints(7), positions=ints(7), status=ints(2), page_size=16)


def test_plain_attention_in_two_parts_is_one_softmax():
    # the restatement itself: without sharing it is softmax(q k^T) v over the request's rows
    rng = np.random.default_rng(0)
    k, v = rng.standard_normal((2, 1, 4, 16, 32))
    q = rng.standard_normal((3, 2, 32))
    tables = np.array([[2, 0, -1], [2, 3, 1]])
    out, lse, _, _ = pm.attention(q, k, v, None, tables, [0, 1, 3], [20, 30, 31], [21, 32], [0, 2], [16], 16, 0.3)
    for t, r, n in ((0, 0, 21), (1, 1, 31), (2, 1, 32)):
        kk, vv = (np.concatenate([x[0][p] for p in tables[r] if p >= 0])[:n] for x in (k, v))
        for h in range(2):
            e = np.exp(kk @ q[t, h] * 0.3)
            assert np.allclose(out[t, h], e @ vv / e.sum()) and np.isclose(lse[t, h], np.log(e.sum()))


@pytest.mark.parametrize("n_rows", [(1 << 26) - 3, 1 << 26, 1 << 27, 1 << 30])
def test_rows_of_more_threads_than_a_launch_has(n_rows):
    assert rows(n_rows=n_rows) == INVALID
    assert "too many" in _lib.last_error()


def test_attention_into_its_own_queries_is_refused():
    k = Host((2, 10, 16, 64), "float16")
    a = paged.PagedAttention(paged.PagePool(k, k), nq=4, tables=ints(3, 4), cu_tokens=ints(4), positions=ints(5), lens=ints(3))
    q = Host((5, 4, 64), "float16")
    with pytest.raises(GpuError, match="out is q"):
        a(q, q, workspace=Host((a.workspace_bytes,), "uint8"))


def test_the_null_stream_has_a_name_of_its_own():
    seen = []
    be = object.__new__(NativeHipBackend)
    be._lib = SimpleNamespace(oxb_hip_set_stream=lambda handle: seen.append(handle) or 0)
    for handle in (None, 0, 0x7f00):
        be.set_stream(handle)
    be.set_stream()
    assert seen == [None, 1, 0x7f00, None]      # null restores the library's stream, 1 is OXB_HIP_NULL_STREAM
    header = open(os.path.join(ROOT, "include", "oxb_hip.h")).read()
    assert f"#define OXB_HIP_NULL_STREAM ((void*){_lib.NULL_STREAM})" in header


def test_row_overlap_against_all_bytes(tmp_path):
    """The check behind the refusals of overlapping rows, on small spans whose bytes are marked one by one."""
    cxx = shutil.which("g++")
    if not cxx:
        pytest.skip("no C++ compiler")
    (tmp_path / "overlap.cpp").write_text("""
#include <cstdio>
#include <vector>
#include "row_overlap.h"
using oxb::RowSpan;
static bool plain(const RowSpan& a, const RowSpan& b) {
    std::vector<char> in(400, 0);
    for (unsigned i = 0; i < a.n; i++) for (unsigned x = 0; x < a.wide; x++) in[a.at + i * a.stride + x] = 1;
    for (unsigned i = 0; i < b.n; i++) for (unsigned x = 0; x < b.wide; x++) if (in[b.at + i * b.stride + x]) return true;
    return false;
}
int main() {
    long n = 0, yes = 0;
    for (unsigned na = 1; na <= 4; na++) for (unsigned nb = 1; nb <= 4; nb++)
    for (unsigned wa = 1; wa <= 5; wa += 2) for (unsigned wb = 1; wb <= 5; wb++)
    for (unsigned sa = wa; sa <= 11; sa += 1) for (unsigned sb = wb; sb <= 11; sb++)
    for (unsigned at = 0; at <= 100; at += 3) {
        const RowSpan a = {50, na, wa, sa}, b = {at, nb, wb, sb};
        const bool want = plain(a, b);
        if (oxb::rows_overlap(a, b) != want || oxb::rows_overlap(b, a) != want) {
            printf("%u %u %u %u %u %u %u: %d\\n", na, nb, wa, wb, sa, sb, at, want);
            return 1;
        }
        n++, yes += want;
    }
    const RowSpan far = {1ull << 40, 1ull << 30, 64, 1ull << 34}, near = {4096, 8, 64, 64};
    if (oxb::rows_overlap(far, near) || !oxb::rows_overlap(far, {(1ull << 40) + (5ull << 34) + 63, 3, 64, 1ull << 34})) return 2;
    printf("%ld %ld\\n", n, yes);
    return yes > 1000 ? 0 : 3;
}
""".replace("\\\\n", "\\n"))
    subprocess.run([cxx, "-std=c++17", "-O1", "-I", os.path.join(ROOT, "oxibonsai_amd", "csrc"), str(tmp_path / "overlap.cpp"), "-o", str(tmp_path / "overlap")], check=True)
    r = subprocess.run([str(tmp_path / "overlap")], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout


def test_binding_refuses_the_tensors_of_another_gpu(monkeypatch):
    """The library has started on GPU 0: nothing is made for tensors of GPU 1."""
    real, asked = _lib.lib(), []

    class Started:
        def __getattr__(self, name):
            return getattr(real, name)

        def oxb_hip_init(self, index):
            asked.append(index)
            return 0 if index == 0 else INVALID

    monkeypatch.setattr(_lib, "lib", Started)

    def on(index, shape, kind):
        t = Host(shape, kind)
        t.device.index = index
        return t

    def pool_on(index):
        return paged.PagePool(*(on(index, (2, 10, 16, 64), "float16") for _ in "kv"))

    def assign_on(index):
        i = lambda *shape: on(index, shape, "int32")  # noqa: E731
        return paged.PageAssign(past=i(3), add=i(3), tables=i(3, 4), free_pages=i(9), n_free=i(1), lens=i(3), cu_tokens=i(4), cu_pages=i(4), slots=i(7),
                                positions=i(7), status=i(2), page_size=16)

    for make in (pool_on, assign_on):
        make(0)
        with pytest.raises(GpuError):
            make(1)
    assert asked == [0, 1, 0, 1]


@pytest.mark.parametrize("first", ["torch", "library"])
def test_torch_after_the_library_is_refused(first):
    """Loaded the other way round, torch brings a HIP runtime that knows nothing of the library's streams."""
    load = {"torch": "import torch", "library": "from oxibonsai_amd import _lib; _lib.lib()"}
    program = "\n".join([load[first], *load.values(), "from oxibonsai_amd import paged", "k = torch.zeros((1, 1, 16, 32), dtype=torch.float16)", "paged.PagePool(k, k)"])
    r = subprocess.run([sys.executable, "-c", program], cwd=ROOT, capture_output=True, text=True, timeout=300)
    wanted = "not on a GPU" if first == "torch" else "two HIP runtimes"     # (here on the CPU both end with an error)
    assert r.returncode != 0 and wanted in r.stderr, r.stderr
