"""A torch program that makes a serving step's calls between its own operations and waits for nothing: what a user of the package writes.

Run by test_gpu_paged.py as a process of its own (torch brings its HIP runtime, which the library then uses too).  A step's inputs
come from a chain of operations, long enough that calls that ran ahead of them would read what the step before left, and are
overwritten right behind the calls; outputs are copied by torch.  The same steps with a wait at every turn have to give the
same bits."""
import sys

import torch

from oxibonsai_amd import NativeHipBackend
from oxibonsai_amd.paged import PageAssign, PagePool, PagedAttention, RowStore

NQ, NKV, HD, PAGE, B, STEPS = 8, 2, 128, 16, 6, 12


def ints(*shape):
    return torch.zeros(shape, dtype=torch.int32, device="cuda")


def steps(be, wait):
    be.set_stream(None if wait else torch.cuda.current_stream().cuda_stream)
    rest = torch.cuda.synchronize if wait else lambda: None
    g = torch.Generator(device="cuda")
    g.manual_seed(5)
    width, n_pages, n_rows = 8, 64, 24
    k, v = (torch.zeros((NKV, n_pages, PAGE, HD), dtype=torch.float16, device="cuda") for _ in "kv")
    pool = PagePool(k, v)
    lens, add, tables, n_free, cu, cu_pages = ints(B), ints(B), ints(B, width), ints(1) + n_pages, ints(B + 1), ints(B + 1)
    slots, positions, status = ints(n_rows), ints(n_rows), ints(2)
    free = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32)
    angle = torch.rand((width * PAGE, HD // 2), generator=g, device="cuda") * 6
    w = torch.rand(HD, generator=g, device="cuda") + 0.5
    rest()
    assign = PageAssign(past=lens, lens=lens, add=add, tables=tables, free_pages=free, n_free=n_free, cu_tokens=cu, cu_pages=cu_pages, slots=slots,
                        positions=positions, status=status, page_size=PAGE)
    cos, sin = angle.cos(), angle.sin()
    store = RowStore(pool, nq=NQ, slots=slots, positions=positions, q_norm=w, k_norm=w, cos=cos, sin=sin)
    attend = PagedAttention(pool, nq=NQ, tables=tables, cu_tokens=cu, positions=positions, lens=lens)
    ws = torch.empty(attend.workspace_bytes, dtype=torch.uint8, device="cuda")
    wide = (NQ + 2 * NKV) * HD
    x, q, out = torch.randn((4096, 4096), generator=g, device="cuda"), torch.zeros((n_rows, NQ, HD), device="cuda"), torch.zeros((n_rows, NQ, HD), device="cuda")
    got = []
    for i in range(STEPS):
        for _ in range(20):
            x = torch.sin(5 * x + x.roll(1, 1))
        qkv = x[:n_rows, :wide].contiguous()
        add.copy_((x[0, :B] > 0).to(torch.int32) + 1)        # (lengths come late, too)
        rest()
        assign()
        rest()
        store(qkv, q)
        rest()
        attend(q, out, workspace=ws)
        rest()
        got += [out.clone(), positions.clone(), status.clone()]
        for t in (qkv, q, out):
            t.fill_(float("nan"))
    rest()
    return [t.cpu() for t in got] + [k.cpu(), v.cpu()]       # (these wait for the stream that made them)


def main():
    be = NativeHipBackend(0)
    want = steps(be, True)
    for i in range(0, 3 * STEPS, 3):
        n = int((want[i + 1] >= 0).sum())
        assert want[i + 2][0] == 0 and B <= n <= 2 * B and bool(torch.isfinite(want[i][:n]).all())
        assert i == 0 or not torch.equal(want[i][:n], want[i - 3][:n])
    side = torch.cuda.Stream()
    for name, stream in (("the default stream", torch.cuda.default_stream()), ("a side stream", side)):
        with torch.cuda.stream(stream):
            got = steps(be, False)
        for a, b in zip(want, got):
            assert torch.equal(a.view(-1).view(torch.uint8), b.view(-1).view(torch.uint8)), name
        print(name, "ok", flush=True)
    be.set_stream(None)


if __name__ == "__main__":
    sys.exit(main())
