"""Paged append and paged attention (C ABI) against plain 64-bit forms.

Tolerances, with u = 2^-24 (half an fp32 step):

append.  A normed value is x * scale * w: the mean of squares is off by u (the
sum is exact enough to round like the sequential one), eps adds u, the root
halves that and adds u, the reciprocal u, the two products u each: 6u at most.
The rotation a c - b s multiplies (u each) and adds (u): 8u (|a c| + |b s|),
taken as 9u for the second-order terms.  K and V are then rounded to the cache's
type: half a step, eps/2 of the value, or half the smallest fp16 subnormal.

attention.  q enters as two fp16 or three bf16 parts that leave at most 2^-22 of
it; a score is a chain of D/16 matrix steps per part (each rounds by at most
2^-23 of the running sum of |q||k|), the scale and the exponent's argument three
roundings more: with S = scale sum |q||k|, d = (4 + 2 * 16 + 4) u S at D = 128.
A probability is off by d, the exponential's 2^-22 and the split's 2^-22; sums of
n cells add in some order, at most n/4 + 64 terms in one thread's chain, u each.
With A = sum p|v| / sum p:  |out - exact| <= (2 max d + 2^-20 + 2 (n/4 + 64) u) A
and |lse - exact| <= max d + 2^-21 + (n/4 + 64) u + 4u |lse|.
"""
import ctypes as C
import math

import numpy as np
import pytest

import arclight_b200 as A

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
U = 2.0 ** -24
DT = {A.ALB_KV_F16: torch.float16, A.ALB_KV_BF16: torch.bfloat16}
L = None


def setup_module():
    global L
    L = A.lib()


def st():
    return torch.cuda.current_stream().cuda_stream


def ptr(t):
    return None if t is None else t.data_ptr()


class Cache:
    """A paged cache whose pool holds NaN wherever nothing was put."""

    def __init__(self, n_pages, page, hkv, dim, typ, table, layout="dense", device="cuda"):
        self.page, self.hkv, self.dim, self.typ = page, hkv, dim, typ
        self.n_pages = n_pages
        nan = float("nan")
        kw = dict(device=device, dtype=DT[typ])
        strides = {}
        if layout == "dense":          # [pages][cells][heads][dim]
            self.k = torch.full((n_pages, page, hkv, dim), nan, **kw)
            self.v = torch.full((n_pages, page, hkv, dim), nan, **kw)
        elif layout == "heads":        # [pages][heads][cells][dim]
            self.k = torch.full((n_pages, hkv, page, dim), nan, **kw).transpose(1, 2)
            self.v = torch.full((n_pages, hkv, page, dim), nan, **kw).transpose(1, 2)
        elif layout == "joined":       # [pages][k, v][cells][heads][dim], cells 8 values apart
            self.pool = torch.full((n_pages, 2, page, hkv * dim + 8), nan, **kw)
            self.k = self.pool[:, 0, :, :hkv * dim].unflatten(-1, (hkv, dim))
            self.v = self.pool[:, 1, :, :hkv * dim].unflatten(-1, (hkv, dim))
        elif layout == "head_major":   # [heads][pages][cells][dim]
            self.k = torch.full((hkv, n_pages, page, dim), nan, **kw).permute(1, 2, 0, 3)
            self.v = torch.full((hkv, n_pages, page, dim), nan, **kw).permute(1, 2, 0, 3)
        if layout != "dense":
            strides = dict(page_stride=self.k.stride(0), cell_stride=self.k.stride(1), head_stride=self.k.stride(2))
        self.table = table.to(device, torch.int32)
        self.c = A.PagedKV(k=self.k.data_ptr(), v=self.v.data_ptr(), page_table=self.table.data_ptr(),
                           table_stride=self.table.stride(0), n_pages=n_pages, n_seqs=table.shape[0],
                           max_pages=table.shape[1], page_size=page, n_head_kv=hkv, head_dim=dim, type=typ, **strides)

    def ref(self):
        return C.byref(self.c)

    def where(self, seq, pos):
        return int(self.table[seq, pos // self.page]), pos % self.page

    def rows(self, seq, lo, hi):
        """K and V of positions [lo, hi) as float64 on the CPU [n][hkv][dim]."""
        p = torch.arange(lo, hi, device=self.k.device)
        pg = self.table[seq, p // self.page].long().clamp(0, self.n_pages - 1)
        return self.k[pg, p % self.page].double().cpu(), self.v[pg, p % self.page].double().cpu()

    def fill(self, seq, n, gen, scale=1.0):
        p = torch.arange(n, device=self.k.device)
        pg = self.table[seq, p // self.page].long()
        for pool in (self.k, self.v):
            pool[pg, p % self.page] = (torch.randn(n, self.hkv, self.dim, generator=gen, device=pool.device) * scale).to(pool.dtype)


def make_table(lens, page, gen, spare=3, pad_columns=0):
    """Distinct pages in no order, -1 where a sequence has none."""
    held = [(n + page - 1) // page for n in lens]
    most, total = max(1, max(held)), sum(held)
    order = torch.randperm(total + spare, generator=gen)[:total]
    wide = torch.full((len(lens), most + pad_columns), -1, dtype=torch.int32)
    at = 0
    for s, h in enumerate(held):
        wide[s, :h] = order[at:at + h]
        at += h
    return wide[:, :most] if pad_columns else wide, total + spare


def attend(cache, q, lengths, seqs=None, window=0, scale=None, out=None, lse=None, ws=None):
    rows, heads, dim = q.shape
    out = torch.full_like(q, 7.0) if out is None else out
    lse = torch.full((rows, heads), 7.0, device=q.device) if lse is None else lse
    need = L.alb_paged_attn_workspace_bytes(cache.ref(), rows, heads)
    assert need > 0
    ws = torch.full((need,), 0xFF, dtype=torch.uint8, device=q.device) if ws is None else ws   # no state is expected in it
    A.check(L.alb_paged_attn(q.data_ptr(), rows, heads, cache.ref(), ptr(seqs), lengths.data_ptr(), window,
                             dim ** -0.5 if scale is None else scale, ws.data_ptr(), out.data_ptr(), lse.data_ptr(),
                             st()), "alb_paged_attn")
    torch.cuda.synchronize()
    return out, lse


def check_rows(cache, q, lens, out, lse, seqs=None, window=0, scale=None, hidden=()):
    """Every row against the 64-bit form; `hidden`: (seq, position) of cells that are not seen."""
    rows, heads, dim = q.shape
    scale = dim ** -0.5 if scale is None else scale
    out, lse, q = out.double().cpu(), lse.double().cpu(), q.double().cpu()
    g = heads // cache.hkv
    for r in range(rows):
        s, n = (r if seqs is None else seqs[r]), lens[r]
        if n < 0:
            assert torch.all(out[r] == 7.0) and torch.all(lse[r] == 7.0)
            continue
        lo = max(0, n - window) if window else 0
        seen = [p for p in range(lo, n) if (s, p) not in hidden] if hidden else None
        if n == lo or seen == []:
            assert torch.all(out[r] == 0) and torch.all(lse[r] == -math.inf)
            continue
        k, v = cache.rows(s, lo, n)
        if seen is not None:
            k, v = k[[p - lo for p in seen]], v[[p - lo for p in seen]]
        qr = q[r].view(cache.hkv, g, dim)
        x = torch.einsum("hgd,nhd->hgn", qr, k) * scale
        S = torch.einsum("hgd,nhd->hgn", qr.abs(), k.abs()) * scale
        d = (8 + 2 * dim / 8) * U * S.amax(-1)
        p = torch.softmax(x, -1)
        want = torch.einsum("hgn,nhd->hgd", p, v)
        spread = torch.einsum("hgn,nhd->hgd", p, v.abs())
        m = len(k) / 4 + 64
        tol = (2 * d + 2.0 ** -20 + 2 * m * U)[..., None] * spread + 1e-37
        err = (out[r].view_as(want) - want).abs()
        assert torch.all(err <= tol), (r, n, float((err / tol).max()))
        z = torch.logsumexp(x, -1)
        err = (lse[r].view_as(z) - z).abs()
        tol = d + 2.0 ** -21 + m * U + 4 * U * z.abs()
        assert torch.all(err <= tol), (r, n, float((err / tol).max()))


LENGTHS = [1, 0, 15, 16, 17, 64, 129, 300, 2, 1000, 63, 65]


@pytest.mark.parametrize("typ", [A.ALB_KV_F16, A.ALB_KV_BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("heads,hkv,dim,page,layout", [
    (32, 8, 128, 16, "dense"),
    (8, 8, 128, 1, "dense"),        # one query head per K/V head, cells as pages
    (14, 2, 64, 7, "dense"),        # seven query heads each, an odd page
    (32, 2, 128, 64, "heads"),      # sixteen: two groups of eight
    (5, 1, 64, 256, "joined"),      # a page longer than most sequences
    (40, 8, 128, 48, "joined"),
    (12, 1, 64, 16, "head_major"),  # twelve: a group of eight and one of four
])
def test_attention(heads, hkv, dim, page, layout, typ):
    gen = torch.Generator().manual_seed(heads * dim + page)
    dg = torch.Generator(device="cuda").manual_seed(heads + typ)
    table, pool = make_table(LENGTHS, page, gen, pad_columns=3)
    cache = Cache(pool, page, hkv, dim, typ, table, layout)
    for s, n in enumerate(LENGTHS):
        cache.fill(s, n, dg)
    q = torch.randn(len(LENGTHS), heads, dim, generator=dg, device="cuda") * 2
    lens = torch.tensor(LENGTHS, dtype=torch.int32, device="cuda")
    L.alb_device_error(1)
    out, lse = attend(cache, q, lens)
    assert L.alb_device_error(0) == 0
    check_rows(cache, q, LENGTHS, out, lse)
    again, lse2 = attend(cache, q, lens)
    assert torch.equal(out, again) and torch.equal(lse, lse2)
    # one row alone, without lse, gives a row within the same bounds
    o1 = torch.empty(1, heads, dim, device="cuda")
    ws = torch.empty(L.alb_paged_attn_workspace_bytes(cache.ref(), 1, heads), dtype=torch.uint8, device="cuda")
    nine = torch.tensor([9], dtype=torch.int32, device="cuda")
    A.check(L.alb_paged_attn(q[9].data_ptr(), 1, heads, cache.ref(), nine.data_ptr(), lens[9:].data_ptr(), 0,
                             dim ** -0.5, ws.data_ptr(), o1.data_ptr(), None, st()))
    torch.cuda.synchronize()
    check_rows(cache, q[9:10], [1000], o1, lse[9:10], seqs=[9])


@pytest.mark.parametrize("window", [1, 5, 16, 100, 299, 300, 5000])
@pytest.mark.parametrize("dim,page", [(128, 16), (64, 5)])
def test_window(dim, page, window):
    gen = torch.Generator().manual_seed(window)
    dg = torch.Generator(device="cuda").manual_seed(window)
    lens = [300, 0, 1, 16, 33, 299]
    table, pool = make_table(lens, page, gen)
    cache = Cache(pool, page, 2, dim, A.ALB_KV_F16, table)
    for s, n in enumerate(lens):
        cache.fill(s, n, dg)
        if n > window:   # what the window hides is not read: NaN there and in the other free cells changes nothing
            p = torch.arange(n - window, device="cuda")
            pg = cache.table[s, p // page].long()
            cache.k[pg, p % page] = float("nan")
            cache.v[pg, p % page] = float("inf")
    q = torch.randn(len(lens), 8, dim, generator=dg, device="cuda")
    out, lse = attend(cache, q, torch.tensor(lens, dtype=torch.int32, device="cuda"), window=window)
    check_rows(cache, q, lens, out, lse, window=window)


def test_rows_name_their_sequences_and_padding_is_left():
    """Several tokens of one sequence as rows (a prompt's causal rows), rows of other
    sequences, and padding rows whose sequence and length mean nothing."""
    gen = torch.Generator().manual_seed(3)
    dg = torch.Generator(device="cuda").manual_seed(3)
    held = [40, 7, 200]
    table, pool = make_table(held, 16, gen)
    cache = Cache(pool, 16, 4, 128, A.ALB_KV_F16, table)
    for s, n in enumerate(held):
        cache.fill(s, n, dg)
    seqs = [2] * 20 + [0, 1, 0, 77, -5]
    lens = list(range(181, 201)) + [40, 7, 0, -1, -3]
    q = torch.randn(len(lens), 16, 128, generator=dg, device="cuda")
    i32 = dict(dtype=torch.int32, device="cuda")
    L.alb_device_error(1)
    out, lse = attend(cache, q, torch.tensor(lens, **i32), torch.tensor(seqs, **i32))
    assert L.alb_device_error(0) == 0
    check_rows(cache, q, lens, out, lse, seqs=seqs)


def test_bad_tables_are_reported_and_their_cells_unseen():
    gen = torch.Generator().manual_seed(4)
    dg = torch.Generator(device="cuda").manual_seed(4)
    held = [100, 50, 16, 33]
    table, pool = make_table(held, 16, gen)
    cache = Cache(pool, 16, 2, 128, A.ALB_KV_F16, table)
    for s, n in enumerate(held):
        cache.fill(s, n, dg)
    q = torch.randn(4, 8, 128, generator=dg, device="cuda")
    i32 = dict(dtype=torch.int32, device="cuda")
    # pages outside the pool: their cells are not seen, a row of nothing else is empty
    cache.table[0, 2], cache.table[0, 5], cache.table[2, 0] = pool, -1, 1 << 30
    hidden = {(0, p) for p in list(range(32, 48)) + list(range(80, 96))} | {(2, p) for p in range(16)}
    L.alb_device_error(1)
    out, lse = attend(cache, q, torch.tensor(held, **i32))
    assert L.alb_device_error(1) == 4
    check_rows(cache, q, held, out, lse, hidden=hidden)
    # a length beyond the table is cut to it (seven pages); a sequence that is none has no cells
    cache.table[0] = torch.arange(7)
    cache.fill(0, 112, dg)
    out, lse = attend(cache, q[:1], torch.tensor([2 ** 31 - 1], **i32))
    assert L.alb_device_error(1) == 4
    check_rows(cache, q[:1], [112], out, lse)
    out, lse = attend(cache, q, torch.tensor([20, 20, 20, 112], **i32), torch.tensor([4, -1, 2 ** 31 - 1, 0], **i32))
    assert L.alb_device_error(1) == 4
    assert torch.all(out[:3] == 0) and torch.all(lse[:3] == -math.inf)
    check_rows(cache, q[3:], [112], out[3:], lse[3:], seqs=[0])
    # more rows than sequences, none named
    out, lse = attend(cache, torch.cat([q, q]), torch.tensor([112, 0, 0, 0, 5, 0, 0, 0], **i32))
    assert L.alb_device_error(1) == 4
    assert torch.all(out[4:] == 0)
    check_rows(cache, q[:1], [112], out[:1], lse[:1])


@pytest.mark.parametrize("typ", [A.ALB_KV_F16, A.ALB_KV_BF16], ids=["f16", "bf16"])
def test_extreme_scores(typ):
    """One cell far above all others, scores of thousands, tiny and huge queries, equal scores."""
    gen = torch.Generator().manual_seed(5)
    dg = torch.Generator(device="cuda").manual_seed(5)
    held = [500] * 6
    table, pool = make_table(held, 16, gen)
    cache = Cache(pool, 16, 1, 128, typ, table)
    for s in range(6):
        cache.fill(s, 500, dg)
    q = torch.randn(6, 4, 128, generator=dg, device="cuda")
    q[0] *= 1e3
    q[1] *= 1e-30
    q[2] *= 1e30
    q[3] = 0
    q[4, :, 1:] = 0                                   # one component alone
    q[5, 0] = torch.tensor([1e-9, 1.0, 1e4, -3e-5] * 32, device="cuda")   # spread over many binades
    lens = torch.tensor(held, dtype=torch.int32, device="cuda")
    keep = [0, 1, 3, 4, 5]
    out, lse = attend(cache, q, lens)
    assert torch.isfinite(out).all()
    check_rows(cache, q[keep], [500] * 5, out[keep], lse[keep], seqs=keep)
    # scores of 1e30: the largest one alone counts
    k, v = cache.rows(2, 0, 500)
    x = torch.einsum("gd,nd->gn", q[2].double().cpu(), k[:, 0])
    torch.testing.assert_close(out[2].double().cpu(), v[x.argmax(-1), 0], rtol=2.0 ** -22, atol=0)
    # a NaN in a query stays in its row and head group's own head
    q[0, 2, 7] = float("nan")
    bad, _ = attend(cache, q, lens)
    assert torch.isnan(bad[0, 2]).all()
    assert torch.equal(bad[0, [0, 1, 3]], out[0, [0, 1, 3]]) and torch.equal(bad[1:], out[1:])


@pytest.mark.parametrize("rows,longest", [(1, 40000), (3, 20000), (700, 90), (2500, 9)])
def test_splits_and_many_rows(rows, longest):
    gen = torch.Generator().manual_seed(rows)
    dg = torch.Generator(device="cuda").manual_seed(rows)
    lens = torch.randint(0, longest + 1, (rows,), generator=gen).tolist()
    lens[0] = longest
    if rows > 1:
        lens[-1] = -1
    table, pool = make_table([max(0, n) for n in lens], 16, gen)
    cache = Cache(pool, 16, 2, 64, A.ALB_KV_F16, table)
    # the cells of all sequences at once
    for pool_t in (cache.k, cache.v):
        pool_t.copy_(torch.randn(pool_t.shape, generator=dg, device="cuda"))
    q = torch.randn(rows, 6, 64, generator=dg, device="cuda")
    out, lse = attend(cache, q, torch.tensor(lens, dtype=torch.int32, device="cuda"))
    some = sorted(set(list(range(min(rows, 40))) + list(range(max(0, rows - 5), rows))))
    check_rows(cache, q[some], [lens[r] for r in some], out[some], lse[some], seqs=some)


def test_batches_of_nothing():
    """All rows empty or padding, one empty row, one row among many empty ones."""
    gen = torch.Generator().manual_seed(1)
    dg = torch.Generator(device="cuda").manual_seed(1)
    table, pool = make_table([70] + [0] * 599, 16, gen)
    cache = Cache(pool, 16, 2, 64, A.ALB_KV_BF16, table)
    cache.fill(0, 70, dg)
    for lens in ([0], [-1], [0] * 600, [-1, 0] * 300, [70] + [0, -1] * 299 + [0]):
        q = torch.randn(len(lens), 4, 64, generator=dg, device="cuda")
        out, lse = attend(cache, q, torch.tensor(lens, dtype=torch.int32, device="cuda"))
        check_rows(cache, q, lens, out, lse)


def test_first_call_inside_a_capture():
    """A process whose first call of the library is captured into a graph."""
    import subprocess
    import sys
    code = """
import ctypes as C, torch, arclight_b200 as A
L = A.lib()
k = torch.zeros(4, 16, 1, 64, dtype=torch.float16, device="cuda"); v = torch.ones_like(k)
t = torch.zeros(1, 1, dtype=torch.int32, device="cuda"); n = torch.full((1,), 3, dtype=torch.int32, device="cuda")
q = torch.ones(1, 2, 64, device="cuda"); o = torch.zeros_like(q); x = torch.ones(1, 9, device="cuda"); y = torch.zeros_like(x)
c = A.PagedKV(k=k.data_ptr(), v=v.data_ptr(), page_table=t.data_ptr(), n_pages=4, n_seqs=1, max_pages=1, page_size=16,
              n_head_kv=1, head_dim=64, type=A.ALB_KV_F16)
ws = torch.empty(L.alb_paged_attn_workspace_bytes(C.byref(c), 1, 2), dtype=torch.uint8, device="cuda")
r = A.LogitsRules(temperature=x.data_ptr())
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    s = torch.cuda.current_stream().cuda_stream
    A.check(L.alb_paged_attn(q.data_ptr(), 1, 2, C.byref(c), None, n.data_ptr(), 0, 0.1, ws.data_ptr(), o.data_ptr(), None, s))
    A.check(L.alb_logits_process(x.data_ptr(), 1, 9, 0, C.byref(r), y.data_ptr(), 0, None, s))
g.replay(); torch.cuda.synchronize()
assert torch.all(o == 1) and torch.all(y == 1) and L.alb_device_error(0) == 0
print("captured")
"""
    import os
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300, cwd=root)
    assert r.returncode == 0 and "captured" in r.stdout, r.stderr[-2000:]


def test_rope_table_of_64_dimensions():
    """alb_rope_table for head_dim 64, as the append reads it: angles by repeated fp32 products, each off by
    half a step, so position p's angle i is off by (i + 1) u p and its cosine by that and the rounding."""
    t = torch.empty(300, 32, 2, device="cuda")
    A.check(L.alb_rope_table(t.data_ptr(), 300, 64, 1e6))
    # theta_scale = powf(base, -2/64): its own rounding enters every product (one step at most)
    tol = 300 * (3 * torch.arange(32)[None, :, None] + 4) * U + 2 * U
    assert torch.all((t.double().cpu() - angles(300, 64).double().cpu()).abs() <= tol)


def test_offsets_beyond_32_bits():
    """A pool of 2.2e9 elements whose used pages lie at its end."""
    page, hkv, dim = 64, 8, 128
    n_pages = (1 << 31) // (page * hkv * dim) + 200
    table = torch.arange(n_pages - 1, n_pages - 9, -1).view(2, 4)
    cache = Cache.__new__(Cache)
    cache.page, cache.hkv, cache.dim, cache.typ, cache.n_pages = page, hkv, dim, A.ALB_KV_F16, n_pages
    cache.k = torch.empty(n_pages, page, hkv, dim, dtype=torch.float16, device="cuda")
    cache.v = torch.empty(n_pages, page, hkv, dim, dtype=torch.float16, device="cuda")
    cache.table = table.to("cuda", torch.int32)
    cache.c = A.PagedKV(k=cache.k.data_ptr(), v=cache.v.data_ptr(), page_table=cache.table.data_ptr(), n_pages=n_pages,
                        n_seqs=2, max_pages=4, page_size=page, n_head_kv=hkv, head_dim=dim, type=A.ALB_KV_F16)
    dg = torch.Generator(device="cuda").manual_seed(1)
    for s in range(2):
        cache.fill(s, 256, dg)
    q = torch.randn(2, 32, dim, generator=dg, device="cuda")
    out, lse = attend(cache, q, torch.tensor([256, 200], dtype=torch.int32, device="cuda"))
    check_rows(cache, q, [256, 200], out, lse)
    # and the append writes there
    qkv = torch.randn(2, (32 + 16) * dim, generator=dg, device="cuda")
    rope = angles(512, dim)
    pos = torch.tensor([255, 201], dtype=torch.int32, device="cuda")
    append(cache, qkv, 32, None, None, rope, pos)
    want = qkv.view(2, 48, dim)[:, 40:].half()
    for s, p in ((0, 255), (1, 201)):
        g, c = cache.where(s, p)
        assert torch.equal(cache.v[g, c], want[s])


def test_graph_replays_with_new_lengths_and_streams_do_not_meet():
    gen = torch.Generator().manual_seed(8)
    dg = torch.Generator(device="cuda").manual_seed(8)
    held = [700, 300, 64]
    table, pool = make_table(held, 16, gen)
    cache = Cache(pool, 16, 8, 128, A.ALB_KV_F16, table)
    for s, n in enumerate(held):
        cache.fill(s, n, dg)
    q = torch.randn(3, 32, 128, generator=dg, device="cuda")
    lens = torch.tensor([1, 1, 1], dtype=torch.int32, device="cuda")
    out, lse = torch.full_like(q, 7.0), torch.full((3, 32), 7.0, device="cuda")
    ws = torch.empty(L.alb_paged_attn_workspace_bytes(cache.ref(), 3, 32), dtype=torch.uint8, device="cuda")
    g = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    with torch.cuda.graph(g, stream=side):
        for _ in range(2):   # two calls in a row in one graph, the second over the first's workspace
            A.check(L.alb_paged_attn(q.data_ptr(), 3, 32, cache.ref(), None, lens.data_ptr(), 0, 128 ** -0.5,
                                     ws.data_ptr(), out.data_ptr(), lse.data_ptr(), st()))
    for now in ([700, 300, 64], [1, 0, 64], [699, -1, 1], [64, 64, 64]):
        lens.copy_(torch.tensor(now, dtype=torch.int32))
        out.fill_(7.0)
        lse.fill_(7.0)
        g.replay()
        torch.cuda.synchronize()
        check_rows(cache, q, now, out, lse)
    # two streams at once, a workspace each
    lens.copy_(torch.tensor(held, dtype=torch.int32))
    want, _ = attend(cache, q, lens)
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [torch.empty_like(q) for _ in streams]
    wss = [torch.empty_like(ws) for _ in streams]
    torch.cuda.synchronize()
    for _ in range(20):
        for s, o, w in zip(streams, outs, wss):
            A.check(L.alb_paged_attn(q.data_ptr(), 3, 32, cache.ref(), None, lens.data_ptr(), 0, 128 ** -0.5,
                                     w.data_ptr(), o.data_ptr(), None, s.cuda_stream))
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want) and torch.equal(outs[1], want)


# ------------------------------------------------------------------------------------------------------- append
def angles(n, dim):
    inv = 1e6 ** (-torch.arange(0, dim, 2, dtype=torch.float64) / dim)
    a = torch.arange(n, dtype=torch.float64)[:, None] * inv
    return torch.stack([a.cos(), a.sin()], -1).float().contiguous().cuda()


def append(cache, qkv, heads, qn, kn, rope, pos, seqs=None, q=None, stride=0, eps=1e-6):
    T = len(pos)
    q = torch.full((T, heads, cache.dim), 7.0, device="cuda") if q is None else q
    A.check(L.alb_qk_norm_rope_kv_paged(qkv.data_ptr(), stride, T, heads, ptr(qn), ptr(kn), eps, rope.data_ptr(),
                                        rope.shape[0], pos.data_ptr(), ptr(seqs), cache.ref(), q.data_ptr(), st()),
            "alb_qk_norm_rope_kv_paged")
    torch.cuda.synchronize()
    return q


def rotated(x, w, rope, pos, eps=1e-6):
    """(value, bound) in 64 bits of norm and rotation of x [T][heads][dim]."""
    x, half = x.double().cpu(), x.shape[-1] // 2
    if w is not None:
        x = x / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + eps) * w.double().cpu()
    cs = rope.double().cpu()[pos][:, None]
    a, b, c, s = x[..., :half], x[..., half:], cs[..., 0], cs[..., 1]
    y = torch.cat([a * c - b * s, a * s + b * c], -1)
    size = torch.cat([(a * c).abs() + (b * s).abs(), (a * s).abs() + (b * c).abs()], -1)
    return y, 9 * U * size


@pytest.mark.parametrize("typ", [A.ALB_KV_F16, A.ALB_KV_BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("norms", ["both", "none", "k"])
@pytest.mark.parametrize("heads,hkv,dim,page,layout,T,wide", [
    (32, 8, 128, 16, "dense", 1, 0),
    (16, 4, 128, 7, "heads", 37, 4),
    (14, 2, 64, 1, "joined", 101, 0),
    (3, 1, 64, 64, "head_major", 5, 12),
])
def test_append(heads, hkv, dim, page, layout, T, wide, norms, typ):
    gen = torch.Generator().manual_seed(T + dim)
    dg = torch.Generator(device="cuda").manual_seed(T + typ)
    seq_of = torch.arange(T) % 3
    pos = 11 + torch.arange(T) // 3 * 2                 # every second position
    held = [int(pos[seq_of == s].max()) + 1 if (seq_of == s).any() else 0 for s in range(3)]
    table, pool = make_table(held, page, gen)
    cache = Cache(pool, page, hkv, dim, typ, table, layout)
    wait_k, wait_v = cache.k.clone(), cache.v.clone()
    H = heads + 2 * hkv
    buf = torch.full((T, H * dim + wide), float("nan"), device="cuda")
    buf[:, :H * dim] = torch.randn(T, H * dim, generator=dg, device="cuda") * 3
    x = buf[:, :H * dim].view(T, H, dim) if not wide else buf[:, :H * dim].reshape(T, H, dim)
    qn = 1 + 0.3 * torch.randn(dim, generator=dg, device="cuda") if norms == "both" else None
    kn = 1 + 0.3 * torch.randn(dim, generator=dg, device="cuda") if norms != "none" else None
    rope = angles(200, dim)
    i32 = dict(dtype=torch.int32, device="cuda")
    L.alb_device_error(1)
    q = append(cache, buf, heads, qn, kn, rope, pos.to(**i32), seq_of.to(**i32), stride=H * dim + wide if wide else 0)
    assert L.alb_device_error(0) == 0
    want, tol = rotated(x[:, :heads], qn, rope, pos)
    assert torch.all((q.double().cpu() - want).abs() <= tol)
    kw, tol = rotated(x[:, heads:heads + hkv], kn, rope, pos)
    half = torch.finfo(DT[typ]).eps / 2
    tol = tol + half * kw.abs() * (1 + 2 ** -10) + (2.0 ** -25 if typ == A.ALB_KV_F16 else 0)
    vw = x[:, heads + hkv:].to(DT[typ])
    for t in range(T):
        g, c = cache.where(int(seq_of[t]), int(pos[t]))
        assert torch.all((cache.k[g, c].double().cpu() - kw[t]).abs() <= tol[t])
        assert torch.equal(cache.v[g, c], vw[t])
        wait_k[g, c], wait_v[g, c] = cache.k[g, c], cache.v[g, c]
    # no other cell changed
    assert torch.equal(torch.nan_to_num(wait_k, 5.0), torch.nan_to_num(cache.k, 5.0))
    assert torch.equal(torch.nan_to_num(wait_v, 5.0), torch.nan_to_num(cache.v, 5.0))


def test_append_equals_the_cell_form():
    """With page size 1 and the manager's cells as table, the rows and queries are
    alb_qk_norm_rope_kv_cells' bit for bit."""
    from arclight_b200.kvcache import KVCache
    heads, hkv, T = 32, 8, 60
    kv = KVCache(256, 2, True, 32)
    seq = (np.arange(T) % 2).astype(np.int32)
    tpos = (np.arange(T) // 2).astype(np.int32)
    (slot,) = kv.prepare([(tpos, seq)])
    n_kv = kv.apply(tpos, seq, slot)
    table = torch.stack([torch.from_numpy(kv.visible_cells(s, T // 2 - 1, n_kv)) for s in (0, 1)])
    cache = Cache(256, 1, hkv, 128, A.ALB_KV_F16, table)
    dg = torch.Generator(device="cuda").manual_seed(2)
    qkv = torch.randn(T, (heads + 2 * hkv) * 128, generator=dg, device="cuda") * 2
    qn = 1 + 0.1 * torch.randn(128, generator=dg, device="cuda")
    kn = 1 + 0.1 * torch.randn(128, generator=dg, device="cuda")
    rope = angles(64, 128)
    i32 = dict(dtype=torch.int32, device="cuda")
    P, S = torch.from_numpy(tpos).cuda(), torch.from_numpy(seq).cuda()
    q = append(cache, qkv, heads, qn, kn, rope, P, S)
    K, V, Q = torch.zeros_like(cache.k), torch.zeros_like(cache.v), torch.empty_like(q)
    cells = torch.from_numpy(np.asarray(slot, np.int64)).cuda()
    A.check(L.alb_qk_norm_rope_kv_cells(qkv.data_ptr(), T, heads, hkv, qn.data_ptr(), kn.data_ptr(), 1e-6,
                                        rope.data_ptr(), 64, P.data_ptr(), cells.data_ptr(), 256, Q.data_ptr(),
                                        K.data_ptr(), V.data_ptr(), st()))
    torch.cuda.synchronize()
    assert torch.equal(q, Q)
    assert torch.equal(cache.k[cells], K[cells]) and torch.equal(cache.v[cells], V[cells])
    # and the attention of each sequence's last token over the manager's cells
    lens = torch.full((2,), T // 2, **i32)
    out, lse = attend(cache, q[-2:].contiguous(), lens)
    check_rows(cache, q[-2:], [T // 2] * 2, out, lse)


def test_append_skips_padding_and_reports_bad_tokens():
    gen = torch.Generator().manual_seed(6)
    dg = torch.Generator(device="cuda").manual_seed(6)
    table, pool = make_table([32, 32, 32], 16, gen)
    cache = Cache(pool, 16, 2, 128, A.ALB_KV_F16, table)
    qkv = torch.randn(9, 8 * 128, generator=dg, device="cuda")
    rope = angles(40, 128)
    i32 = dict(dtype=torch.int32, device="cuda")
    # 0 good, 1 padding (sequence), 2 padding (position), then with an error: past the rope table, past the pages,
    # no such sequence, a page outside the pool
    cache.table[2, 1] = pool
    L.alb_device_error(1)
    q = append(cache, qkv[:3], 4, None, None, rope, torch.tensor([3, 5, -1], **i32), torch.tensor([0, -1, 1], **i32))
    assert L.alb_device_error(0) == 0
    assert not torch.any(q[0] == 7.0) and torch.all(q[1:] == 7.0)
    assert int(torch.isfinite(cache.v).sum()) == 2 * 128
    for p, s in ((40, 0), (33, 0), (2 ** 31 - 1, 1), (3, 3), (3, 2 ** 31 - 1), (17, 2)):
        q = append(cache, qkv[:2], 4, None, None, rope, torch.tensor([p, 4], **i32), torch.tensor([s, 1], **i32))
        assert L.alb_device_error(1) == 4, (p, s)
        assert torch.all(q[0] == 7.0) and not torch.any(q[1] == 7.0)
        assert int(torch.isfinite(cache.v).sum()) == 4 * 128
    # sequences not named: token t is sequence t; the fourth has no table row
    q = append(cache, qkv[:4], 4, None, None, rope, torch.tensor([1, 1, 1, 1], **i32))
    assert L.alb_device_error(1) == 4
    assert torch.all(q[3] == 7.0) and not torch.any(q[:3] == 7.0)


# ------------------------------------------------------------------------------------------------- a run of them
@pytest.mark.parametrize("dim,typ", [(128, A.ALB_KV_F16), (64, A.ALB_KV_BF16)])
def test_decode_steps_of_a_batch(dim, typ):
    """Prompts appended at once, then steps of append, attend and choose for a batch with a
    padding row, captured once and replayed: every step against the 64-bit forms on its own inputs."""
    heads, hkv, page, vocab, B, steps = 8, 2, 16, 999, 4, 6
    gen = torch.Generator().manual_seed(dim)
    dg = torch.Generator(device="cuda").manual_seed(dim)
    prompts = [33, 1, 15]                                     # row 3 is padding
    table, pool = make_table([n + steps for n in prompts] + [0], page, gen)
    cache = Cache(pool, page, hkv, dim, typ, table)
    rope = angles(64, dim)
    i32 = dict(dtype=torch.int32, device="cuda")
    H = heads + 2 * hkv
    T = sum(prompts)
    seqs = torch.tensor(sum(([s] * n for s, n in enumerate(prompts)), []), **i32)
    pos = torch.tensor(sum((list(range(n)) for n in prompts), []), **i32)
    append(cache, torch.randn(T, H * dim, generator=dg, device="cuda"), heads, None, None, rope, pos, seqs)
    wout = torch.randn(heads * dim, vocab, generator=dg, device="cuda")
    embed = torch.randn(vocab, H * dim, generator=dg, device="cuda")
    positions = torch.tensor(prompts + [-1], **i32)
    lengths = torch.tensor([n + 1 for n in prompts] + [-1], **i32)
    history = torch.zeros(B, 32, **i32)
    hist_len = torch.tensor([1, 1, 1, -1], **i32)
    history[:, 0] = torch.arange(B)
    rep = torch.full((B,), 1.3, device="cuda")
    rules = A.LogitsRules(history=history.data_ptr(), history_stride=32, history_len=hist_len.data_ptr(),
                          repetition=rep.data_ptr())
    token = torch.arange(B, **i32)
    q = torch.full((B, heads, dim), 7.0, device="cuda")
    out, lse = torch.zeros_like(q), torch.zeros(B, heads, device="cuda")
    ws = torch.empty(L.alb_paged_attn_workspace_bytes(cache.ref(), B, heads), dtype=torch.uint8, device="cuda")
    qkv, logits = torch.empty(B, H * dim, device="cuda"), torch.empty(B, vocab, device="cuda")
    final = torch.full((B, vocab), 7.0, device="cuda")

    def step():
        qkv.copy_(embed[token.clamp(0, vocab - 1).long()])
        A.check(L.alb_qk_norm_rope_kv_paged(qkv.data_ptr(), 0, B, heads, None, None, 1e-6, rope.data_ptr(), 64,
                                            positions.data_ptr(), None, cache.ref(), q.data_ptr(), st()))
        A.check(L.alb_paged_attn(q.data_ptr(), B, heads, cache.ref(), None, lengths.data_ptr(), 0, dim ** -0.5,
                                 ws.data_ptr(), out.data_ptr(), lse.data_ptr(), st()))
        torch.mm(out.view(B, -1), wout, out=logits)
        A.check(L.alb_logits_process(logits.data_ptr(), B, vocab, 0, C.byref(rules), final.data_ptr(), 0,
                                     token.data_ptr(), st()))

    torch.mm(out.view(B, -1), wout, out=logits)   # cuBLAS starts up outside the capture
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        step()
    L.alb_device_error(1)
    for n in range(steps):
        fed = token.clone()
        g.replay()
        torch.cuda.synchronize()
        assert L.alb_device_error(0) == 0
        x = embed[fed[:3].clamp(0, vocab - 1).long()].view(3, H, dim)
        p = torch.tensor([a + n for a in prompts])
        want, tol = rotated(x[:, :heads], None, rope, p)
        assert torch.all((q[:3].double().cpu() - want).abs() <= tol)
        check_rows(cache, q[:3], [a + n + 1 for a in prompts], out[:3], lse[:3])
        z = logits[:3].cpu().numpy()
        for b in range(3):
            ids = history[b, :int(hist_len[b])].unique().cpu().numpy()
            hit = np.zeros(vocab, bool)
            hit[ids] = True
            f = np.float32(1.3)
            want = np.where(hit, np.where(z[b] > 0, z[b] / f, z[b] * f), z[b])
            np.testing.assert_array_equal(final[b].cpu().numpy(), want)
            assert int(token[b]) == int(want.argmax())
        assert torch.all(final[3] == 7.0) and int(token[3]) == 3 and torch.all(q[3] == 7.0)
        for b in range(3):
            history[b, n + 1] = token[b]
        hist_len[:3] += 1
        positions[:3] += 1
        lengths[:3] += 1
