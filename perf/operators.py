"""The operators of a serving step over a paged KV cache, as cases that can be timed and compared.

A step of a server that batches requests of different lengths goes through three operators, the last two once per layer:

  pages      page tables, slot map and positions of the step, built on the GPU from the requests' lengths: cached rows that are
             given up return their pages to the pool, new tokens take pages from it (``oxibonsai_amd.paged.PageAssign``)
  rows       the step's new q, k and v rows: RMSNorm per head and RoPE for q and k, k and v rows into the cache's slots as fp16
             numbers or as one-byte codes with a scale per row (``oxibonsai_amd.paged.RowStore``)
  attention  the step's queries over the cache: requests of a group begin with the same prefix, which is read once for all
             of them, then each has its own rest (``oxibonsai_amd.paged.PagedAttention``)

``own`` says who computes: False, the plain form in elementary torch operations; True, the package's kernels.
"""
import math

import torch

own = False

#: Head layouts: the package's 8B and 1.7B benchmark models, and smaller heads of its tests.
H8B = dict(nq=32, nkv=8, hd=128)
H1P7B = dict(nq=16, nkv=8, hd=128)
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
CACHE = {"f16": torch.float16, "i8": torch.int8, "fp8": torch.float8_e4m3fn}
EPS = 1e-6


def listed():
    return [
        # One decode step of a small batch: every request has one new token, a few need a new page.  Latency is everything.
        dict(name="pages_decode", op="pages", B=24, past=3000, add=1, page=16, rows=32),
        # A batch of prompts is admitted at once, where others have ended: hundreds of thousands of slots.
        dict(name="pages_prompts", op="pages", B=500, past=900, add=1100, page=16, rows=280000),
        # The rows of one decode step, as the QKV product leaves them.
        dict(name="rows_decode", op="rows", T=17, **H8B, page=16, x="f32", q="f16", kv="f16", norm=True, rope=True),
        # The rows of a prompt chunk, bf16 activations.
        dict(name="rows_prompt", op="rows", T=8192, **H8B, page=64, x="bf16", q="bf16", kv="f16", norm=True, rope=True),
        # Rows that the model has already rotated go to an INT8 cache.
        dict(name="rows_int8", op="rows", T=2999, **H8B, page=32, x="f16", q="f16", kv="i8", norm=False, rope=False),
        # A chunk of a small model with an FP8 cache, fp32 in and out.
        dict(name="rows_fp8", op="rows", T=700, nq=16, nkv=4, hd=64, page=16, x="f32", q="f32", kv="fp8", norm=True, rope=True),
        # A few chat requests behind a short system prompt: the smallest attention.
        dict(name="attn_chat", op="attention", groups=1, B=5, prefix=300, rest=60, new=1, **H1P7B, page=16, q="f16", kv="f16"),
        # The ordinary serving batch: sixty-odd requests behind a long instruction.
        dict(name="attn_batch", op="attention", groups=1, B=62, prefix=4100, rest=700, new=1, **H8B, page=16, q="bf16", kv="f16"),
        # Several tenants, each with a prompt of its own; INT8 cache, fp32 queries straight from the product.
        dict(name="attn_tenants", op="attention", groups=5, B=90, prefix=2000, rest=400, new=1, **H8B, page=32, q="f32", kv="i8"),
        # A handful of questions about one very long document, FP8 cache.
        dict(name="attn_document", op="attention", groups=1, B=9, prefix=60000, rest=250, new=1, **H8B, page=64, q="f16", kv="fp8"),
        # Follow-up prompts of several requests in one chunk, ragged, behind the shared prefix.
        dict(name="attn_chunk", op="attention", groups=2, B=14, prefix=3500, rest=500, new=300, **H8B, page=16, q="f16", kv="f16"),
        # A full batch behind a long prefix: the largest case.
        dict(name="attn_full", op="attention", groups=1, B=256, prefix=16000, rest=900, new=1, **H8B, page=16, q="bf16", kv="f16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("pages", "rows", "attention", "attention"))
    page = rng.choice((16, 32, 64, 128))
    if op == "pages":
        B, add = _log(rng, 1, 500), _log(rng, 1, 1100)
        return dict(op=op, B=B, past=_log(rng, 1, 4000), add=add, page=page, rows=sum(_spread(B, add, 0.7548776662)) + rng.randrange(40))
    heads = rng.choice((H8B, H1P7B, dict(nq=16, nkv=4, hd=64), dict(nq=12, nkv=4, hd=128), dict(nq=8, nkv=8, hd=64),
                        dict(nq=10, nkv=2, hd=256), dict(nq=4, nkv=1, hd=32)))
    q, kv = rng.choice(("f16", "bf16", "f32")), rng.choice(("f16", "i8", "fp8"))
    if op == "rows":
        # (codes are whole numbers and have to be equal: an INT8 cache takes rows that are stored as they are)
        fused = kv != "i8"
        return dict(op=op, T=_log(rng, 1, 8000), **heads, page=page, x=rng.choice(("f16", "bf16", "f32")), q=q, kv=kv, norm=fused, rope=fused)
    new = rng.choice((1, 1, 1, _log(rng, 2, 300)))
    B = _log(rng, 1, 256 if new == 1 else 14)
    prefix = _log(rng, 16, min(60000, 4000000 // B)) if new == 1 else _log(rng, 16, 3500)
    return dict(op=op, groups=rng.choice((1, 1, 2, 5)) if B >= 5 else 1, B=B, prefix=prefix, rest=max(new, _log(rng, 1, 900 if new == 1 else 500)), new=new,
                **heads, page=page, q=q, kv=kv)


# ---- lengths: those of a case are fixed, the seed deals them out --------------------------------------------------------
def _spread(n, most, by):
    """n lengths between 1 and most, ragged, the last one the longest."""
    got = [1 + int((most - 1) * ((i * by) % 1.0)) for i in range(n)]
    got[-1] = most
    return got


def _lengths(c):
    """Requests of every group, prefix of every group, rest and new tokens of every request (the new tokens are the rest's last)."""
    g, b = c["groups"], c["B"]
    sizes = [b // g + (i < b % g) for i in range(g)]
    for i in range(0, g - 1, 2):     # groups of different sizes
        k = sizes[i + 1] // 2
        sizes[i], sizes[i + 1] = sizes[i] + k, sizes[i + 1] - k
    prefix = [max(1, c["prefix"] - 37 * i) for i in range(g)]
    rest = _spread(b, c["rest"], 0.6180339887)
    new = [min(r, n) for r, n in zip(rest, _spread(b, c["new"], 0.7548776662))]
    return sizes, prefix, rest, new


def _ints(v, dev="cuda"):
    return torch.tensor(v, dtype=torch.int32, device=dev)


def _cum(v):
    out = [0]
    for x in v:
        out.append(out[-1] + x)
    return out


def _pool(c, n_pages, g):
    """K and V pages of one layer, [kv head][page][position][head_dim], and their row scales (one-byte rows)."""
    shape, one_byte = (c["nkv"], n_pages, c["page"], c["hd"]), c["kv"] != "f16"
    parts = []
    for _ in "kv":
        if c["kv"] == "i8":
            parts.append(torch.randint(-127, 128, shape, generator=g, device="cuda", dtype=torch.int8))
        else:
            t = torch.empty(shape, dtype=torch.float16, device="cuda").normal_(generator=g)
            parts.append((t * 60).to(CACHE["fp8"]) if one_byte else t)
    full = {"i8": 55.0, "fp8": 60.0, "f16": 1.0}[c["kv"]]
    scales = [(0.6 + 0.8 * torch.rand(shape[:3], generator=g, device="cuda")) / full if one_byte else None for _ in "kv"]
    return parts + scales


def prepare(case, seed):
    c = dict(case)
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    h = torch.Generator()
    h.manual_seed(seed)
    s = {"c": c}
    if c["op"] == "pages":
        b, p, w = c["B"], c["page"], -(-(c["past"] + c["add"]) // c["page"]) + 2
        turn = torch.randperm(b, generator=h)
        past = torch.tensor(_spread(b, c["past"], 0.6180339887), dtype=torch.int32)[turn]
        add = torch.tensor(_spread(b, c["add"], 0.7548776662), dtype=torch.int32)[torch.randperm(b, generator=h)]
        # one request in eight has ended (a new one takes its place), one in eight gives up its last three tokens
        keep = past.clone()
        keep[turn % 8 == 3] = 0
        keep[turn % 8 == 5] = (past[turn % 8 == 5] - 3).clamp(min=0)
        taken = (past + p - 1) // p
        n_pages = b * w + 7
        order = torch.randperm(n_pages, generator=h).to(torch.int32)
        at = torch.cumsum(taken, 0) - taken
        j = torch.arange(w)
        tables = torch.where(j < taken[:, None], order[(at[:, None] + j).clamp(max=n_pages - 1)], torch.full((), -1, dtype=torch.int32))
        used = int(taken.sum())
        free = torch.full((n_pages,), -1, dtype=torch.int32)
        free[:n_pages - used] = order[used:]
        s |= dict(past=past.cuda(), keep=keep.cuda(), add=add.cuda(), tables=tables.contiguous().cuda(), free=free.cuda(), n_free=_ints([n_pages - used]))
        for name, n in (("n_free_out", 1), ("lens", b), ("cu_tokens", b + 1), ("cu_pages", b + 1), ("slots", c["rows"]), ("positions", c["rows"]), ("status", 2)):
            s[name] = torch.zeros(n, dtype=torch.int32, device="cuda")
    elif c["op"] == "rows":
        t, hd = c["T"], c["hd"]
        n_pages = -(-t // c["page"]) + 3
        slots = torch.randperm(n_pages * c["page"], generator=g, device="cuda")[:t].to(torch.int32)
        slots[t - t // 20:] = -1     # (a batch padded to a fixed number of rows)
        positions = torch.randint(0, 8192, (t,), generator=g, device="cuda", dtype=torch.int32)
        positions[t - t // 20:] = -1
        x = torch.randn((t, (c["nq"] + 2 * c["nkv"]) * hd), generator=g, device="cuda").to(TYPES[c["x"]])
        angle = torch.arange(8192, dtype=torch.float64, device="cuda")[:, None] * 1e6 ** (-torch.arange(0, hd, 2, dtype=torch.float64, device="cuda") / hd)
        s |= dict(x=x, slots=slots, positions=positions, cos=angle.cos().float(), sin=angle.sin().float(), pool=_pool(c, n_pages, g),
                  q_norm=1 + 0.1 * torch.randn(hd, generator=g, device="cuda"), k_norm=1 + 0.1 * torch.randn(hd, generator=g, device="cuda"),
                  q=torch.zeros((t, c["nq"], hd), dtype=TYPES[c["q"]], device="cuda"))
    else:
        sizes, prefix, rest, new = _lengths(c)
        turn = torch.randperm(c["B"], generator=h).tolist()
        rest, new = [rest[i] for i in turn], [new[i] for i in turn]
        cu_g, p = _cum(sizes), c["page"]
        of = [k for k, n in enumerate(sizes) for _ in range(n)]
        lens = [prefix[of[r]] + rest[r] for r in range(c["B"])]
        # tables: the prefix's whole pages are the group's, from there on every request has its own; a page that the prefix fills
        # in part is copied by each (here: its rows of the prefix are read through the first request's)
        w = -(-max(lens) // p) + 1
        own_pages = [-(-lens[r] // p) - prefix[of[r]] // p for r in range(c["B"])]
        n_pages = sum(prefix[k] // p for k in range(c["groups"])) + sum(own_pages) + 5
        order = torch.randperm(n_pages, generator=h).to(torch.int32)
        tables, at, shared = torch.full((c["B"], w), -1, dtype=torch.int32), 0, []
        for k in range(c["groups"]):
            shared.append(order[at:at + prefix[k] // p])
            at += prefix[k] // p
        for r in range(c["B"]):
            n = len(shared[of[r]])
            tables[r, :n] = shared[of[r]]
            tables[r, n:n + own_pages[r]] = order[at:at + own_pages[r]]
            at += own_pages[r]
        positions = [lens[r] - new[r] + i for r in range(c["B"]) for i in range(new[r])]
        t = len(positions)
        s |= dict(tables=tables.cuda(), cu_tokens=_ints(_cum(new)), positions=_ints(positions), lens=_ints(lens), cu_groups=_ints(cu_g), prefix_lens=_ints(prefix),
                  pool=_pool(c, n_pages, g), q=torch.randn((t, c["nq"], c["hd"]), generator=g, device="cuda").to(TYPES[c["q"]]),
                  out=torch.zeros((t, c["nq"], c["hd"]), dtype=TYPES[c["q"]], device="cuda"), lse=torch.zeros((t, c["nq"]), device="cuda"),
                  # what a program knows about its batch on the host
                  most=dict(prefix=max(prefix), rest=max(rest), new=max(new),
                            group_tokens=max(sum(new[cu_g[k]:cu_g[k + 1]]) for k in range(c["groups"]))))
    if own:
        _bind(s)
    return s


# ---- the package's kernels: descriptors that a program makes once for its buffers ---------------------------------------
def _bind(s):
    from oxibonsai_amd import NativeHipBackend, paged
    NativeHipBackend(0).set_stream(torch.cuda.current_stream().cuda_stream)
    c = s["c"]
    if c["op"] == "pages":
        s["call"] = paged.PageAssign(past=s["past"], keep=s["keep"], add=s["add"], tables=s["tables"], free_pages=s["free"], n_free=s["n_free"],
                                     n_free_out=s["n_free_out"], lens=s["lens"], cu_tokens=s["cu_tokens"], cu_pages=s["cu_pages"], slots=s["slots"],
                                     positions=s["positions"], status=s["status"], page_size=c["page"])
        return
    pool = paged.PagePool(*s["pool"])
    if c["op"] == "rows":
        norm = dict(q_norm=s["q_norm"], k_norm=s["k_norm"], eps=EPS) if c["norm"] else {}
        rope = dict(cos=s["cos"], sin=s["sin"]) if c["rope"] else {}
        s["call"] = paged.RowStore(pool, nq=c["nq"], slots=s["slots"], positions=s["positions"], **norm, **rope)
    else:
        s["call"] = paged.PagedAttention(pool, nq=c["nq"], tables=s["tables"], cu_tokens=s["cu_tokens"], positions=s["positions"], lens=s["lens"],
                                         cu_groups=s["cu_groups"], prefix_lens=s["prefix_lens"])
        s["workspace"] = torch.empty(s["call"].workspace_bytes, dtype=torch.uint8, device="cuda")


# ---- the plain form ---------------------------------------------------------------------------------------------------
def _plain_pages(s):
    p, past, add, free = s["c"]["page"], s["past"], s["add"], s["free"]
    keep = torch.minimum(s["keep"], past)
    lens, w, rows = keep + add, s["tables"].shape[1], s["slots"].shape[0]
    had, held, has = (past + p - 1) // p, (keep + p - 1) // p, (lens + p - 1) // p
    freed, need = torch.cumsum(had - held, 0, dtype=torch.int32), torch.cumsum(has - held, 0, dtype=torch.int32)
    n = s["n_free"] + freed[-1]
    cu = torch.cumsum(add, 0, dtype=torch.int32)
    short = need[-1] > n
    ok = ~(short | (lens > w * p).any() | (cu[-1] > rows))
    j = torch.arange(w, device="cuda", dtype=torch.int32)[None]
    # pages given up go on top of the free ones, in the order of requests and positions ...
    at = (s["n_free"] + freed - (had - held))[:, None] + j - held[:, None]
    goes = (j >= held[:, None]) & (j < had[:, None]) & ok
    m = free.shape[0]
    pushed = torch.cat([free, free.new_zeros(1)]).index_put((torch.where(goes, at, m).long(),), s["tables"])[:m]
    # ... and new pages come from the top
    take = (n - 1 - (need - (has - held)))[:, None] - (j - held[:, None])
    comes = (j >= held[:, None]) & (j < has[:, None]) & ok
    free.copy_(pushed)
    s["tables"].copy_(torch.where(comes, pushed[take.clamp(0, m - 1).long()], s["tables"]))
    s["n_free_out"].copy_(torch.where(ok, n - need[-1], s["n_free"]))
    s["lens"].copy_(torch.where(ok, lens, past))
    s["cu_tokens"][1:] = torch.where(ok, cu, torch.zeros_like(cu))
    s["cu_pages"][1:] = torch.where(ok, need, torch.zeros_like(need))
    i = torch.arange(rows, device="cuda", dtype=torch.int32)
    r = torch.searchsorted(cu, i, right=True).clamp(max=len(past) - 1)
    pos = keep[r] + i - (cu - add)[r]
    live = (i < cu[-1]) & ok
    page = s["tables"][r, (pos // p).clamp(0, w - 1).long()]
    s["slots"].copy_(torch.where(live, page * p + pos % p, -1))
    s["positions"].copy_(torch.where(live, pos, -1))
    s["status"][0] = torch.where(ok, 0, torch.where(short, 1, 2))
    s["status"][1] = need[-1]


def _rms(x, w):
    return w * x * (1 / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS))


def _turn(x, cos, sin):
    a, b = x.chunk(2, -1)
    return torch.cat([a * cos - b * sin, a * sin + b * cos], -1)


def _encode(x, kv):
    """Rows as one-byte codes and their scales."""
    if kv == "f16":
        return x.half(), None
    scale = (x.abs().amax(-1) / (127.0 if kv == "i8" else 448.0)).clamp(min=1.1920929e-07)
    t = x / scale[..., None]
    if kv == "fp8":
        return t.clamp(-448, 448).to(CACHE["fp8"]), scale
    t = t.double()
    return (t.sign() * torch.floor(t.abs() + 0.5)).clamp(-127, 127).to(torch.int8), scale


def _plain_rows(s):
    c = s["c"]
    x = s["x"].float().view(c["T"], c["nq"] + 2 * c["nkv"], c["hd"])
    q, k, v = x.split([c["nq"], c["nkv"], c["nkv"]], 1)
    if c["norm"]:
        q, k = _rms(q, s["q_norm"]), _rms(k, s["k_norm"])
    if c["rope"]:
        at = s["positions"].clamp(min=0).long()
        cos, sin = s["cos"][at][:, None], s["sin"][at][:, None]
        q, k = _turn(q, cos, sin), _turn(k, cos, sin)
    there = s["positions"] >= 0
    s["q"].copy_(torch.where(there[:, None, None], q.to(s["q"].dtype), s["q"]))
    # (rows without a slot rewrite the row that the first one goes to with what goes there)
    live = s["slots"] >= 0
    pick = torch.where(live, torch.arange(c["T"], device="cuda"), torch.zeros_like(s["slots"], dtype=torch.int64))
    slots = s["slots"].long()[pick]
    for rows, pool, scales in ((k, s["pool"][0], s["pool"][2]), (v, s["pool"][1], s["pool"][3])):
        code, scale = _encode(rows[pick], c["kv"])
        bits = torch.int16 if c["kv"] == "f16" else torch.int8
        pool.view(bits).view(c["nkv"], -1, c["hd"])[:, slots] = code.view(bits).transpose(0, 1)
        if scales is not None:
            scales.view(c["nkv"], -1)[:, slots] = scale.transpose(0, 1)


def _gather(pool, scales, tables, keys, page):
    """Rows of the positions `keys` [n, m] of the requests of `tables` [n, w], in fp32: [kv head, n, m, head_dim]."""
    at = torch.gather(tables, 1, (keys // page).clamp(0, tables.shape[1] - 1).long()).clamp(min=0).long() * page + keys % page
    rows = pool.view(pool.shape[0], -1, pool.shape[3])
    rows = rows.view(torch.int8)[:, at].view(pool.dtype) if pool.element_size() == 1 else rows[:, at]
    return rows.float() * scales.view(pool.shape[0], -1)[:, at][..., None] if scales is not None else rows.float()


def _part(s, q, sees, tables, keys):
    """Softmax parts of queries [n, m, nq, hd] over keys [n, k]: largest score, sum and un-normalised output, [n, m, nq (, hd)]."""
    c, pool = s["c"], s["pool"]
    n, m, heads = q.shape[0], q.shape[1], c["nq"] // c["nkv"]
    rows = q.view(n, m, c["nkv"], heads, c["hd"]).permute(2, 0, 1, 3, 4).reshape(c["nkv"], n, m * heads, c["hd"])
    k = _gather(pool[0], pool[2], tables, keys, c["page"])
    score = torch.matmul(rows, k.transpose(-1, -2).contiguous()) * c["hd"] ** -0.5
    del k
    seen = (keys[:, None] < sees[:, :, None])[:, :, None].expand(-1, -1, heads, -1).reshape(n, m * heads, -1)
    score = score.masked_fill(~seen, -math.inf)
    top = score.amax(-1)
    weight = torch.exp(score - torch.where(top == -math.inf, 0.0, top)[..., None])
    del score
    out = torch.matmul(weight, _gather(pool[1], pool[3], tables, keys, c["page"]))
    back = lambda t: t.view(c["nkv"], n, m, heads, -1).permute(1, 2, 0, 3, 4).reshape(n, m, c["nq"], -1)  # noqa: E731
    return back(top)[..., 0], back(weight.sum(-1))[..., 0], back(out)


def _plain_attention(s):
    c, most = s["c"], s["most"]
    cu, cu_g, lens, prefix = s["cu_tokens"], s["cu_groups"], s["lens"], s["prefix_lens"]
    t, b, q = s["q"].shape[0], c["B"], s["q"].float()
    count = lambda n: torch.arange(n, device="cuda", dtype=torch.int32)  # noqa: E731
    request = torch.searchsorted(cu[1:].contiguous(), count(t), right=True)
    group = torch.searchsorted(cu_g[1:].contiguous(), count(b), right=True)
    sees = torch.minimum(s["positions"] + 1, lens[request])
    first = cu[cu_g.long()]
    # the prefixes: all queries of a group over its first request's rows
    at = (first[:-1, None] + count(most["group_tokens"])).clamp(max=t - 1).long()
    keys = count(most["prefix"]).expand(c["groups"], -1)
    parts = _part(s, q[at], torch.minimum(sees[at], prefix[:, None]), s["tables"][cu_g[:-1].long()], keys)
    mine = group[request], (count(t) - first[group[request]]).long()
    a = [x[mine] for x in parts]
    # the rests, request by request
    at = (cu[:-1, None] + count(most["new"])).clamp(max=t - 1).long()
    parts = _part(s, q[at], sees[at], s["tables"], prefix[group][:, None] + count(most["rest"]))
    mine = request, (count(t) - cu[request]).long()
    z = [x[mine] for x in parts]
    top = torch.maximum(a[0], z[0])
    low = torch.where(top == -math.inf, 0.0, top)
    wa, wz = torch.exp(a[0] - low), torch.exp(z[0] - low)
    total = a[1] * wa + z[1] * wz
    out = (a[2] * wa[..., None] + z[2] * wz[..., None]) / torch.where(total > 0, total, 1.0)[..., None]
    s["out"].copy_(out.to(s["out"].dtype))
    s["lse"].copy_(low + torch.log(total))


def run(s):
    op = s["c"]["op"]
    if own:
        if op == "pages":
            s["call"]()
        elif op == "rows":
            s["call"](s["x"], s["q"])
        else:
            s["call"](s["q"], s["out"], lse=s["lse"], workspace=s["workspace"])
    else:
        {"pages": _plain_pages, "rows": _plain_rows, "attention": _plain_attention}[op](s)
    if op == "pages":
        return {n: s[n] for n in ("tables", "free", "n_free_out", "lens", "cu_tokens", "cu_pages", "slots", "positions", "status")}
    if op == "rows":
        return {"q": s["q"], "k": s["pool"][0], "v": s["pool"][1], "k_scale": s["pool"][2], "v_scale": s["pool"][3]}
    return {"out": s["out"], "lse": s["lse"]}


# ---- what a pass costs at least ---------------------------------------------------------------------------------------
def work(case):
    c = case
    if c["op"] == "pages":
        past, add = _spread(c["B"], c["past"], 0.6180339887), _spread(c["B"], c["add"], 0.7548776662)
        pages = sum(-(-a // c["page"]) for a in add) + sum(-(-p // c["page"]) for p in past) // 8
        # lengths in and out, a free page read and a table entry written for each new page, slot and position of each row
        return {"bytes": 4 * (6 * c["B"] + 2 * pages + 2 * c["rows"]), "flops": 0}
    size = {"f16": 2, "bf16": 2, "f32": 4}
    row = c["hd"] * (2 if c["kv"] == "f16" else 1) + (0 if c["kv"] == "f16" else 4)
    if c["op"] == "rows":
        live = c["T"] - c["T"] // 20
        wide = (c["nq"] + 2 * c["nkv"]) * c["hd"]
        return {"bytes": live * (wide * size[c["x"]] + c["nq"] * c["hd"] * size[c["q"]] + 2 * c["nkv"] * row + 8 + (4 * c["hd"] if c["rope"] else 0)),
                "flops": live * wide * (7 if c["norm"] else 1)}
    sizes, prefix, rest, new = _lengths(c)
    of = [k for k, n in enumerate(sizes) for _ in range(n)]
    pairs = sum(n * (prefix[of[r]] + rest[r]) - n * (n - 1) // 2 for r, n in enumerate(new))
    t = sum(new)
    return {"bytes": 2 * c["nkv"] * row * (sum(prefix) + sum(rest)) + t * c["nq"] * (2 * c["hd"] * size[c["q"]] + 4), "flops": 4 * c["nq"] * c["hd"] * pairs}


# ---- the definition in 64 bits ----------------------------------------------------------------------------------------
def exact(case, seed):
    c = dict(case)
    if c["op"] == "pages":
        return None      # whole numbers
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    kd, vd = ((s["pool"][i].view(torch.int8).view(s["pool"][i].dtype) if c["kv"] != "i8" else s["pool"][i]) for i in (0, 1))
    if c["op"] == "rows":
        x = s["x"].double().view(c["T"], -1, c["hd"])
        half, out = c["hd"] // 2, {}
        pieces = {"q": x[:, :c["nq"]], "k": x[:, c["nq"]:c["nq"] + c["nkv"]], "v": x[:, c["nq"] + c["nkv"]:]}
        for n in "qk":
            y = pieces[n]
            if c["norm"]:
                y = y / (y.square().sum(-1, keepdim=True) / c["hd"] + EPS).sqrt() * s[n + "_norm"].double()
            if c["rope"]:
                # a pair of dimensions as a complex number, turned by the position's angle
                z = torch.complex(y[..., :half].contiguous(), y[..., half:].contiguous())
                p = s["positions"].long().clamp(min=0)
                z = z * torch.complex(s["cos"].double()[p], s["sin"].double()[p])[:, None]
                y = torch.cat([z.real, z.imag], -1)
            pieces[n] = y
        live = (s["slots"] >= 0).nonzero()[:, 0]
        out["q"] = s["q"].double()
        out["q"][s["positions"] >= 0] = pieces["q"][s["positions"] >= 0]
        for n, old, scales in (("k", kd, s["pool"][2]), ("v", vd, s["pool"][3])):
            rows = pieces[n][live]
            page, off = s["slots"][live].long() // c["page"], s["slots"][live].long() % c["page"]
            out[n] = out[n + "_scale"] = None
            if c["kv"] == "f16":
                out[n] = old.double()
                out[n][:, page, off] = rows.transpose(0, 1)
                continue
            size = rows.abs().max(-1).values / {"i8": 127, "fp8": 448}[c["kv"]]
            out[n + "_scale"] = scales.double()
            out[n + "_scale"][:, page, off] = size.transpose(0, 1)
            if c["kv"] == "fp8":
                # the nearest of the eight values of a binade (those below 2^-6 lie as far apart as those above)
                y = rows / size[..., None]
                step = 2.0 ** (torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -30))).clamp(min=-6) - 3)
                out[n] = old.double()
                out[n][:, page, off] = (torch.round(y / step) * step).transpose(0, 1)
        return out
    cu, lens, tables = s["cu_tokens"].tolist(), s["lens"].tolist(), s["tables"].long()
    heads, t = c["nq"] // c["nkv"], s["q"].shape[0]
    out, lse = torch.zeros((t, c["nq"], c["hd"]), dtype=torch.float64, device="cuda"), torch.zeros((t, c["nq"]), dtype=torch.float64, device="cuda")
    # a request's rows lie where its table says, but for those that its group shares: the first request's
    first = {r: a for a, b in zip(s["cu_groups"].tolist(), s["cu_groups"].tolist()[1:]) for r in range(a, b)}
    shared = {r: n for a, b, n in zip(s["cu_groups"].tolist(), s["cu_groups"].tolist()[1:], s["prefix_lens"].tolist()) for r in range(a, b)}
    for r in range(c["B"]):
        at = torch.arange(lens[r], device="cuda")
        page = torch.where(at < shared[r], tables[first[r]][at // c["page"]], tables[r][at // c["page"]])
        rows = []
        for x, scales in ((kd, s["pool"][2]), (vd, s["pool"][3])):
            y = (x.view(torch.int8)[:, page, at % c["page"]].view(x.dtype) if x.element_size() == 1 else x[:, page, at % c["page"]]).double()
            rows.append(y if scales is None else y * scales[:, page, at % c["page"]].double()[..., None])
        span = slice(cu[r], cu[r + 1])
        q = s["q"][span].double()
        for k in range(c["nkv"]):
            mine = slice(k * heads, (k + 1) * heads)
            score = (q[:, mine].reshape(-1, c["hd"]) @ rows[0][k].T).view(-1, heads, lens[r]) / math.sqrt(c["hd"])
            score.masked_fill_((at[None] > s["positions"][span].long()[:, None])[:, None], -math.inf)
            lse[span, mine] = torch.logsumexp(score, -1)
            out[span, mine] = (torch.softmax(score, -1).view(-1, lens[r]) @ rows[1][k]).view(-1, heads, c["hd"])
    return {"out": out, "lse": lse}
