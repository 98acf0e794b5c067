"""Paged append and attention where test_gpu_paged.py does not reach: tables of
the cell manager, values at the ends of their types, each part of the split
queries and probabilities by itself, every way to deal heads out to units.
Tolerances are test_gpu_paged.py's unless a test derives its own."""
import ctypes as C
import math

import numpy as np
import pytest

import arclight_b200 as A
from arclight_b200.kvcache import KVCache
from tests import test_gpu_paged as P

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
U = 2.0 ** -24
F16, BF16 = A.ALB_KV_F16, A.ALB_KV_BF16
L = None


def setup_module():
    global L
    P.setup_module()
    L = P.L


def i32(a):
    return torch.as_tensor(a, dtype=torch.int32, device="cuda")


# ----------------------------------------------------------------------------------- tables of the cell manager
@pytest.mark.parametrize("typ", [F16, BF16], ids=["f16", "bf16"])
def test_tables_of_a_manager_whose_slots_wrapped(typ):
    """Freed cells are taken again, so cells and positions are in different orders:
    appends, a sliding window and a prompt's causal rows by position."""
    heads, hkv, dim, n = 8, 2, 128, 20
    kv = KVCache(32, 2, True, 32)
    dg = torch.Generator(device="cuda").manual_seed(7 + typ)
    x = torch.randn(n, heads + 2 * hkv, dim, generator=dg, device="cuda")
    rope = P.angles(64, dim)
    (slot,) = kv.prepare([(np.arange(16), np.zeros(16))])
    kv.apply(np.arange(16), np.zeros(16), slot)          # sequence 0 holds cells 0 .. 15, then leaves
    cache = P.Cache(32, 1, hkv, dim, typ, torch.full((2, n), -1))
    L.alb_device_error(1)
    q = torch.empty(n, heads, dim, device="cuda")
    for first, last in [(0, 10)] + [(p, p + 1) for p in range(10, n)]:
        if first == 10:
            kv.seq_rm(0, -1, -1)
        pos = np.arange(first, last)
        (slot,) = kv.prepare([(pos, np.ones(len(pos)))])
        kv.apply(pos, np.ones(len(pos)), slot)
        cache.table[1].copy_(i32(kv.position_cells(1, n)))
        P.append(cache, x[first:last].reshape(last - first, -1), heads, None, None, rope, i32(pos),
                 i32(np.ones(len(pos))), q=q[first:last])
        assert all(int(cache.table[1, p]) == int(c) for p, c in zip(pos, slot))
    cells = cache.table[1].tolist()
    assert sorted(cells) == sorted(kv.visible_cells(1, n - 1, 32)) and cells != sorted(cells)
    # position p's rows lie in its cell
    k, v = cache.rows(1, 0, n)
    assert torch.equal(v, x[:, heads + hkv:].to(P.DT[typ]).double().cpu())
    want, tol = P.rotated(x[:, heads:heads + hkv], None, rope, torch.arange(n))
    half = torch.finfo(P.DT[typ]).eps / 2
    assert torch.all((k - want).abs() <= tol + half * want.abs() * (1 + 2 ** -10) + 2.0 ** -25)
    for window in (0, 5):
        out, lse = P.attend(cache, q, i32(range(1, n + 1)), i32([1] * n), window=window)
        P.check_rows(cache, q, list(range(1, n + 1)), out, lse, seqs=[1] * n, window=window)
    # the front goes and the rest closes up: rows are read by their new positions
    kv.seq_rm(1, 0, 6)
    kv.seq_add(1, 6, -1, -6)
    cache.table[1].copy_(i32(kv.position_cells(1, n)))
    out, lse = P.attend(cache, q[:1], i32([n - 6]), i32([1]), window=4)
    P.check_rows(cache, q[:1], [n - 6], out, lse, seqs=[1], window=4)
    assert torch.equal(cache.rows(1, 0, n - 6)[1], v[6:])
    assert L.alb_device_error(0) == 0


# --------------------------------------------------------------------------------------- values at the types' ends
@pytest.mark.parametrize("lens", [[1, 2, 15, 33, 300, 5000], [40000]], ids=["batch", "one"])
@pytest.mark.parametrize("heads,hkv,dim", [(4, 1, 128), (8, 1, 128), (2, 2, 64), (6, 1, 64), (16, 1, 128), (17, 1, 64)])
def test_bf16_values_over_the_whole_type(heads, hkv, dim, lens):
    """Finite K and V give finite results up to the type's end: a mean of values lies
    among them, and scores that fit are made of large and small factors."""
    top = torch.finfo(torch.bfloat16).max
    gen = torch.Generator().manual_seed(heads + dim)
    dg = torch.Generator(device="cuda").manual_seed(heads + dim + len(lens))
    table, pool = P.make_table(lens, 16, gen)
    cache = P.Cache(pool, 16, hkv, dim, BF16, table)
    q = torch.randn(len(lens), heads, dim, generator=dg, device="cuda")
    n = i32(lens)
    for k_size, q_size in ((1.0, 1.0), (1e36, 1e-36), (7e37, 1e-37), (1e-36, 1e36)):
        for s, m in enumerate(lens):
            cache.fill(s, m, dg)
        cache.k.copy_((cache.k.float() * k_size).clamp(-top, top))
        v = cache.v.float()
        v[..., 0::4] = torch.where(v[..., 0::4].isnan(), v[..., 0::4], top)               # the end itself
        v[..., 1::4] = torch.copysign(torch.where(v[..., 1::4].isnan(), v[..., 1::4], top), v[..., 1::4])
        v[..., 2::4] *= 1e35
        v[..., 3::4] *= 1e-30
        cache.v.copy_(v)
        out, lse = P.attend(cache, q * q_size, n)
        assert torch.isfinite(out).all() and torch.isfinite(lse).all()
        P.check_rows(cache, q * q_size, lens, out, lse)
        assert torch.allclose(out[..., 0::4], torch.tensor(top, device="cuda"), rtol=2.0 ** -18)


# ----------------------------------------------------------------------------------------- the parts one by one
KINDS = [(1, 1), (4, 1), (6, 2), (5, 1), (8, 1), (12, 1), (16, 1), (17, 1)]


def parts(x, typ, n):
    """x as the sum of its n leading parts in the cache's type."""
    got = torch.zeros_like(x)
    for _ in range(n):
        got = got + (x - got).to(P.DT[typ]).to(x.dtype)
    return got


@pytest.mark.parametrize("typ", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads,hkv", KINDS)
def test_every_part_of_the_query_counts(heads, hkv, dim, typ):
    """Rows of one cell whose K is 1 in one place d: lse is q_d itself (scale 1, 1 <= |q_d| < 2).

    The score's parts add up without rounding (bf16: three hold all 24 bits; fp16: two leave 2^-23 at most).
    x log2(e): the constant is 2^-26.2 off, 4e-8; the exponent 2^-25 (between -1 and 0; fp16: 2^-21, between 14
    and 15); ex2 2^-22; ln 2 times those, the logarithm 2^-24 and the last sum 2^-24: 4.2e-7 < 2^-21 with bf16;
    fp16 has 3.1e-7 + 2^-23 more: 8.5e-7 < 2^-20.
    """
    g = torch.Generator().manual_seed(heads * dim + typ)
    q = (2 ** 23 + 2 * torch.randint(0, 2 ** 22, (dim, heads, dim), generator=g) + 1).double() / 2 ** 23
    q = q * (1 - 2 * torch.randint(0, 2, q.shape, generator=g))
    table = torch.arange(dim)[:, None]
    cache = P.Cache(dim, 1, hkv, dim, typ, table)
    cache.v.zero_()
    cache.k.zero_()
    at = torch.arange(dim)
    cache.k[at, 0, :, at] = 1.0
    _, lse = P.attend(cache, q.float().cuda(), i32([1] * dim), scale=1.0)
    want = q[at, :, at]
    tol = 2.0 ** -20 if typ == F16 else 2.0 ** -21
    assert float((lse.double().cpu() - want).abs().max()) <= tol
    # one part fewer lies outside
    assert float((parts(want, typ, 1 if typ == F16 else 2) - want).abs().max()) > 4 * tol


@pytest.mark.parametrize("typ", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads,hkv", KINDS)
def test_every_part_of_the_probabilities_counts(heads, hkv, dim, typ):
    """Cell j's V is 1 in one place, so that value is its probability; its K is a_j in the first place and q_0 is
    1, so its score a_j (-2 to 2) is exact.

    A weight is off by the constant (4e-8), the exponent's rounding (-7 to 0: 2^-22; fp16 8 to 16: 2^-21), both
    times ln 2, and ex2's 2^-22: 4.4e-7, fp16 6e-7.  Their sum adds eight roundings (2 in a tile, 2 among lanes, 4
    warps) of 2^-24: 4.8e-7.  Three bf16 parts hold the weight, two fp16 parts leave 2^-23; the sum of the parts,
    the rescaled sum and the quotient round: 1.8e-7.  Twice the weight's, then: 1.6e-6, fp16 2e-6 at most.
    """
    n = 40
    g = torch.Generator().manual_seed(heads * dim + typ)
    rows = 6
    a = (torch.rand(rows, n, hkv, generator=g) * 4 - 2).to(P.DT[typ])
    table = torch.arange(rows * 3).view(rows, 3)
    cache = P.Cache(rows * 3, 16, hkv, dim, typ, table)
    k = torch.zeros(rows, 48, hkv, dim, dtype=P.DT[typ])
    v = torch.zeros_like(k)
    k[:, :n, :, 0] = a
    place = (torch.arange(n)[None] + 11 * torch.arange(rows)[:, None]) % dim
    v[torch.arange(rows)[:, None], torch.arange(n)[None], :, place] = 1.0
    cache.k.copy_(k.view(rows * 3, 16, hkv, dim))
    cache.v.copy_(v.view(rows * 3, 16, hkv, dim))
    q = torch.randn(rows, heads, dim, generator=g)
    q[..., 0] = 1.0
    out, _ = P.attend(cache, q.cuda(), i32([n] * rows), scale=1.0)
    p = torch.softmax(a.double(), 1).repeat_interleave(heads // hkv, 2)            # [rows][n][heads]
    want = torch.zeros(rows, heads, dim, dtype=torch.float64)
    want[torch.arange(rows)[:, None], :, place] = p
    tol = 2e-6 if typ == F16 else 1.6e-6
    assert torch.all((out.double().cpu() - want).abs() <= tol * want)
    # one part fewer lies outside (weights as the kernel has them, largest 1 or a power of two below)
    w = torch.exp2(a.double() / math.log(2) - (a.double() / math.log(2)).amax(1, keepdim=True).ceil())
    assert float(((parts(w, typ, 1 if typ == F16 else 2) - w).abs() / w).max()) > 2 * tol


# -------------------------------------------------------------------------------------- heads dealt out to units
@pytest.mark.parametrize("typ", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("heads,hkv,dim,page,layout,window", [
    (17, 1, 128, 16, "dense", 0),        # a unit of 16 heads and one of a single head
    (17, 1, 64, 5, "heads", 100),
    (40, 1, 64, 7, "head_major", 0),     # 16, 16 and 8
    (40, 1, 128, 64, "joined", 17),
    (48, 2, 128, 32, "dense", 0),        # 16 and 8 for each K/V head
    (66, 2, 64, 1, "dense", 63),         # 16, 16 and 1
    (24, 2, 128, 16, "dense", 129),      # one unit of 12
    (16, 2, 64, 16, "heads", 16),        # eight
    (12, 2, 128, 16, "dense", 65),       # six
    (6, 2, 128, 1, "joined", 300),       # three
])
def test_units_and_windows(heads, hkv, dim, page, layout, window, typ):
    gen = torch.Generator().manual_seed(heads * dim + page)
    dg = torch.Generator(device="cuda").manual_seed(heads + typ)
    lens = P.LENGTHS + [-1]
    table, pool = P.make_table([max(0, n) for n in lens], page, gen)
    cache = P.Cache(pool, page, hkv, dim, typ, table, layout)
    for s, n in enumerate(lens):
        if n > 0:
            cache.fill(s, n, dg)
    q = torch.randn(len(lens), heads, dim, generator=dg, device="cuda") * 2
    L.alb_device_error(1)
    out, lse = P.attend(cache, q, i32(lens), window=window)
    assert L.alb_device_error(0) == 0
    P.check_rows(cache, q, lens, out, lse, window=window)


@pytest.mark.parametrize("heads,hkv,dim,typ", [
    (4, 1, 128, BF16), (6, 1, 128, BF16), (8, 1, 128, F16), (16, 1, 128, F16), (16, 1, 64, BF16),
    (17, 1, 128, BF16), (33, 1, 64, F16), (40, 2, 128, BF16),
])
def test_one_long_row_in_many_pieces(heads, hkv, dim, typ):
    """Units cut into more pieces than a round of the join takes, then beside short rows."""
    gen = torch.Generator().manual_seed(heads)
    dg = torch.Generator(device="cuda").manual_seed(heads)
    lens = [40000, 1, 700, 0]
    table, pool = P.make_table(lens, 16, gen)
    cache = P.Cache(pool, 16, hkv, dim, typ, table)
    for s, n in enumerate(lens):
        cache.fill(s, n, dg)
    q = torch.randn(len(lens), heads, dim, generator=dg, device="cuda")
    for rows in (1, 4):
        out, lse = P.attend(cache, q[:rows], i32(lens[:rows]))
        P.check_rows(cache, q[:rows], lens[:rows], out, lse)
        out, lse = P.attend(cache, q[:rows], i32(lens[:rows]), window=30000)
        P.check_rows(cache, q[:rows], lens[:rows], out, lse, window=30000)


# ------------------------------------------------------------------------------------------- calls behind calls
def test_a_call_reads_what_the_call_before_it_writes():
    """Each kernel may start while the one before it still runs: the append's input comes from
    the logits operator, the attention's cache from the append, without a wait between."""
    T, heads, hkv, dim = 600, 8, 2, 128
    wide = (heads + 2 * hkv) * dim
    dg = torch.Generator(device="cuda").manual_seed(1)
    cache = P.Cache(T, 1, hkv, dim, F16, torch.arange(T)[None])
    rope, pos, seqs = P.angles(T, dim), i32(range(T)), i32([0] * T)
    hist = torch.randint(0, wide, (T, 3000), generator=dg, device="cuda", dtype=torch.int32)
    rep, temp = torch.full((T,), 1.2, device="cuda"), torch.full((T,), 0.7, device="cuda")
    r = A.LogitsRules(history=hist.data_ptr(), history_stride=3000, repetition=rep.data_ptr(), temperature=temp.data_ptr())
    qkv = torch.empty(T, wide, device="cuda")
    lens = i32(range(1, T + 1))
    bufs = [dict(q=torch.empty(T, heads, dim, device="cuda"), out=torch.empty(T, heads, dim, device="cuda"),
                 lse=torch.empty(T, heads, device="cuda")) for _ in range(2)]
    ws = torch.empty(L.alb_paged_attn_workspace_bytes(cache.ref(), T, heads), dtype=torch.uint8, device="cuda")
    for _ in range(10):
        x = torch.randn(T, wide, generator=dg, device="cuda")
        kept = []
        for wait, b in zip((False, True), bufs):
            for t in (qkv, cache.k, cache.v, b["q"]):
                t.fill_(100.0)               # a stale read shows
            torch.cuda.synchronize()
            A.check(L.alb_logits_process(x.data_ptr(), T, wide, 0, C.byref(r), qkv.data_ptr(), 0, None, P.st()))
            if wait:
                torch.cuda.synchronize()
            A.check(L.alb_qk_norm_rope_kv_paged(qkv.data_ptr(), 0, T, heads, None, None, 1e-6, rope.data_ptr(), T,
                                                pos.data_ptr(), seqs.data_ptr(), cache.ref(), b["q"].data_ptr(), P.st()))
            if wait:
                torch.cuda.synchronize()
            A.check(L.alb_paged_attn(b["q"].data_ptr(), T, heads, cache.ref(), seqs.data_ptr(), lens.data_ptr(), 0,
                                     dim ** -0.5, ws.data_ptr(), b["out"].data_ptr(), b["lse"].data_ptr(), P.st()))
            torch.cuda.synchronize()
            kept.append([t.clone() for t in (cache.k, cache.v, b["q"], b["out"], b["lse"])])
        for a, b in zip(*kept):
            assert torch.equal(a, b)


def test_captured_calls_on_streams_that_fork_and_join():
    """Two branches of one graph: append and logits side by side, the attention behind both."""
    B, heads, hkv, dim, vocab = 5, 8, 2, 64, 5000
    lens = [40, 1, 300, 17, 64]
    gen = torch.Generator().manual_seed(2)
    dg = torch.Generator(device="cuda").manual_seed(2)
    table, pool = P.make_table(lens, 16, gen)
    cache = P.Cache(pool, 16, hkv, dim, BF16, table)
    for s, n in enumerate(lens):
        cache.fill(s, n, dg)
    qkv = torch.randn(B, (heads + 2 * hkv) * dim, generator=dg, device="cuda")
    src = torch.empty_like(qkv)
    x, y = torch.randn(B, vocab, generator=dg, device="cuda"), torch.empty(B, vocab, device="cuda")
    temp, nxt = torch.full((B,), 0.5, device="cuda"), i32([-7] * B)
    r = A.LogitsRules(temperature=temp.data_ptr())
    rope, pos, n = P.angles(512, dim), i32([m - 1 for m in lens]), i32(lens)
    q, out, lse = torch.empty(B, heads, dim, device="cuda"), torch.empty(B, heads, dim, device="cuda"), torch.empty(B, heads, device="cuda")
    ws = torch.empty(L.alb_paged_attn_workspace_bytes(cache.ref(), B, heads), dtype=torch.uint8, device="cuda")
    side = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        main = torch.cuda.current_stream()
        src.copy_(qkv)                                    # a copy node
        side.wait_stream(main)
        A.check(L.alb_qk_norm_rope_kv_paged(src.data_ptr(), 0, B, heads, None, None, 1e-6, rope.data_ptr(), 512,
                                            pos.data_ptr(), None, cache.ref(), q.data_ptr(), main.cuda_stream))
        with torch.cuda.stream(side):
            A.check(L.alb_logits_process(x.data_ptr(), B, vocab, 0, C.byref(r), y.data_ptr(), 0, nxt.data_ptr(),
                                         side.cuda_stream))
        main.wait_stream(side)
        A.check(L.alb_paged_attn(q.data_ptr(), B, heads, cache.ref(), None, n.data_ptr(), 0, dim ** -0.5,
                                 ws.data_ptr(), out.data_ptr(), lse.data_ptr(), main.cuda_stream))
    for _ in range(3):
        qkv.copy_(torch.randn(qkv.shape, generator=dg, device="cuda"))
        x.copy_(torch.randn(x.shape, generator=dg, device="cuda"))
        for t in (src, q, out, lse, y):
            t.fill_(100.0)
        g.replay()
        torch.cuda.synchronize()
        want, tol = P.rotated(qkv.view(B, -1, dim)[:, :heads], None, rope, torch.tensor(lens) - 1)
        assert torch.all((q.double().cpu() - want).abs() <= tol)
        P.check_rows(cache, q, lens, out, lse)
        assert torch.equal(y, x / temp[:, None]) and torch.equal(nxt, x.argmax(1).int())


# --------------------------------------------------------------------------------------------------- in place
@pytest.mark.parametrize("heads,hkv,dim,typ", [(8, 2, 128, F16), (14, 2, 64, BF16), (17, 1, 128, BF16)])
def test_outputs_in_the_place_of_the_queries(heads, hkv, dim, typ):
    """Whole units, units cut into pieces, empty rows and padding."""
    lens = [30000, 0, 5, 300, -1, 1]
    gen = torch.Generator().manual_seed(dim)
    dg = torch.Generator(device="cuda").manual_seed(heads)
    table, pool = P.make_table([max(n, 0) for n in lens], 16, gen)
    cache = P.Cache(pool, 16, hkv, dim, typ, table)
    for s, n in enumerate(lens):
        if n > 0:
            cache.fill(s, n, dg)
    q = torch.randn(len(lens), heads, dim, generator=dg, device="cuda")
    want, lse = P.attend(cache, q, i32(lens))
    want[4] = q[4]                                        # padding keeps what is there
    for _ in range(5):
        both = q.clone()
        _, l2 = P.attend(cache, both, i32(lens), out=both)
        assert torch.equal(both, want) and torch.equal(l2, lse)


def test_one_token_appended_in_place():
    heads, hkv, dim = 8, 2, 128
    dg = torch.Generator(device="cuda").manual_seed(3)
    cache = P.Cache(4, 16, hkv, dim, F16, torch.arange(2)[None])
    x = torch.randn(1, (heads + 2 * hkv) * dim, generator=dg, device="cuda")
    w, rope, pos = 1 + 0.1 * torch.randn(dim, generator=dg, device="cuda"), P.angles(32, dim), i32([17])
    want = P.append(cache, x, heads, w, w, rope, pos)
    kept = x.clone()
    P.append(cache, x, heads, w, w, rope, pos, q=x)
    assert torch.equal(x[:, :heads * dim], want.view(1, -1)) and torch.equal(x[:, heads * dim:], kept[:, heads * dim:])
