"""alb_logits_process against numpy: every step is one fp32 operation rounded to
nearest, so the logits are equal bit for bit, and the tokens equal."""
import ctypes as C

import numpy as np
import pytest

import arclight_b200 as A

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
L = None
F = np.float32


def setup_module():
    global L
    L = A.lib()


def st():
    return torch.cuda.current_stream().cuda_stream


def cu(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def plain(x, history=None, lens=None, prompt=None, last_n=0, rep=None, freq=None, pres=None, temp=None, bias=None,
          allow=None, allow_row=None):
    """(logits, tokens); bias: per row a list of (id, value); allow: bool [masks][vocab]."""
    rows, vocab = x.shape
    out, nxt = x.astype(F).copy(), np.full(rows, -1, np.int32)
    with np.errstate(all="ignore"):
        for b in range(rows):
            z = out[b]
            for i, v in (dict(e for e in bias[b] if 0 <= e[0] < vocab).items() if bias else ()):
                z[i] = z[i] + F(v)
            if history is not None and not (rep is None and freq is None and pres is None):
                n = min(history.shape[1] if lens is None else int(lens[b]), history.shape[1])
                lo = max(0, n - last_n) if last_n else 0
                pr = 0 if prompt is None else int(prompt[b])
                ids = history[b, lo:n]
                late = history[b, max(lo, pr):n] if pr < n else ids[:0]
                ids, late = ids[(ids >= 0) & (ids < vocab)], late[(late >= 0) & (late < vocab)]
                seen = np.bincount(ids, minlength=vocab) > 0
                n_out = np.bincount(late, minlength=vocab)
                r = F(1) if rep is None else rep[b]
                z[:] = np.where(seen, np.where(z > 0, z / r, z * r), z)
                hit = n_out > 0
                z[hit] = z[hit] - (F(0) if freq is None else freq[b]) * n_out[hit].astype(F)
                z[hit] = z[hit] - (F(0) if pres is None else pres[b])
            if temp is not None and temp[b] > 0:
                z[:] = z / temp[b]
            if allow is not None:
                m = b if allow_row is None else int(allow_row[b])
                if 0 <= m < len(allow):
                    z[~allow[m]] = -np.inf
            fine = z > -np.inf
            if fine.any():
                nxt[b] = int(np.argmax(np.where(fine, z, -np.inf)))
    return out, nxt


def pack(allow):
    m, vocab = allow.shape
    words = np.zeros((m, (vocab + 31) // 32 * 32), bool)
    words[:, :vocab] = allow
    return np.packbits(words, axis=1, bitorder="little").view(np.uint32)


def call(x, history=None, lens=None, prompt=None, last_n=0, rep=None, freq=None, pres=None, temp=None, bias=None,
         allow=None, allow_row=None, stride=0, out_stride=0, inplace=False, offset=0, out_offset=0, want_next=True,
         runs=1):
    rows, vocab = x.shape
    xs, ys = stride or vocab, out_stride or vocab
    hold = torch.full((offset + rows * xs + 8,), 3.5, device="cuda")
    X = hold[offset:offset + rows * xs].view(rows, xs)
    X[:, :vocab] = cu(x)
    hold_y = hold if inplace else torch.full((out_offset + rows * ys + 8,), 7.5, device="cuda")
    Y = X if inplace else hold_y[out_offset:out_offset + rows * ys].view(rows, ys)
    keep, r = [], A.LogitsRules(last_n=last_n)

    def give(name, a, dtype):
        if a is not None:
            keep.append(cu(np.asarray(a).astype(dtype)))
            setattr(r, name, keep[-1].data_ptr())

    give("history", history, np.int32)
    if history is not None:
        r.history_stride = history.shape[1]
    give("history_len", lens, np.int32)
    give("prompt_len", prompt, np.int32)
    for name, a in (("repetition", rep), ("frequency", freq), ("presence", pres), ("temperature", temp)):
        give(name, a, F)
    if bias is not None:
        give("bias_offsets", np.cumsum([0] + [len(b) for b in bias]), np.int32)
        give("bias_ids", [i for b in bias for i, _ in b] or [0], np.int32)
        give("bias_values", [v for b in bias for _, v in b] or [0], F)
        r.n_bias = sum(len(b) for b in bias)
    if allow is not None:
        packed = pack(allow)
        keep.append(cu(packed.view(np.int32)))
        r.allow, r.n_allow, r.allow_stride = keep[-1].data_ptr(), len(allow), packed.shape[1]
    give("allow_row", allow_row, np.int32)
    nxt = torch.full((rows + 1,), -7, dtype=torch.int32, device="cuda")
    for _ in range(runs):
        A.check(L.alb_logits_process(X.data_ptr(), rows, vocab, stride, C.byref(r), Y.data_ptr(), out_stride,
                                     nxt.data_ptr() if want_next else None, st()), "alb_logits_process")
    torch.cuda.synchronize()
    if not inplace:                     # what lies between the rows and around them is left, x too
        mask = torch.zeros_like(hold_y, dtype=torch.bool)
        mask[out_offset:out_offset + rows * ys].view(rows, ys)[:, :vocab] = True
        assert torch.all(hold_y[~mask] == 7.5)
        np.testing.assert_array_equal(X[:, :vocab].cpu().numpy(), x)
    assert int(nxt[rows]) == -7
    return Y[:, :vocab].cpu().numpy(), nxt[:rows].cpu().numpy()


def case(rng, rows, vocab, hist, bias=0, mask=False):
    ids = (vocab * rng.random((rows, hist)) ** 3).astype(np.int32).clip(0, vocab - 1) if hist else None
    kw = dict(rep=(1 + rng.random(rows) * 0.4).astype(F), freq=rng.random(rows).astype(F), pres=rng.random(rows).astype(F),
              temp=(0.4 + rng.random(rows)).astype(F))
    if hist:
        lens = rng.integers(0, hist + 1, rows).astype(np.int32)
        lens[0] = hist
        kw.update(history=ids, lens=lens, prompt=(lens * rng.random(rows)).astype(np.int32))
    if bias:
        kw["bias"] = [[(int(rng.integers(0, vocab)), F(rng.standard_normal() * 5)) for _ in range(int(rng.integers(0, bias + 1)))]
                      for _ in range(rows)]
    if mask:
        kw["allow"] = rng.random((max(1, rows - 1), vocab)) < 0.3
        kw["allow_row"] = rng.integers(-1, max(1, rows - 1), rows).astype(np.int32)
    return (rng.standard_normal((rows, vocab)) * 4).astype(F), kw


def same(x, kw, **more):
    L.alb_device_error(1)
    y, n = call(x, **kw, **more)
    assert L.alb_device_error(0) == 0
    wy, wn = plain(x, **kw)
    np.testing.assert_array_equal(y, wy)
    np.testing.assert_array_equal(n, wn)


@pytest.mark.parametrize("rows,vocab,hist,bias,mask", [
    (1, 1, 3, 1, False), (2, 2, 1, 3, True), (3, 31, 50, 4, True), (5, 33, 0, 0, True), (1, 1000, 200, 0, False),
    (7, 1001, 100, 20, True), (4, 32003, 5000, 40, False), (3, 151936, 300, 0, False), (2, 151936, 9000, 300, True),
    (2, 262144, 700, 3, True), (1, 400001, 50, 2, True), (300, 257, 20, 2, True),
    (9, 185000, 40, 2, True), (9, 96000, 20000, 2, False), (1, 450000, 20000, 2, False),   # shared memory around its limits
    (1000, 300, 20, 2, True), (120, 151936, 50, 3, True),   # many rows
])
def test_rules(rows, vocab, hist, bias, mask):
    same(*case(np.random.default_rng(rows * vocab), rows, vocab, hist, bias, mask))


@pytest.mark.parametrize("inplace", [False, True])
@pytest.mark.parametrize("vocab,stride,out_stride,offset,out_offset", [
    (1003, 1003, 1003, 0, 0), (1003, 1004, 1007, 0, 0), (1004, 1004, 1004, 1, 1), (1001, 1010, 1010, 3, 2),
    (2, 5, 5, 2, 1), (35, 36, 36, 1, 3),
])
def test_strides_alignment_and_in_place(vocab, stride, out_stride, offset, out_offset, inplace):
    x, kw = case(np.random.default_rng(vocab + offset), 5, vocab, 60, 9, True)
    if inplace:
        out_stride, out_offset = stride, offset
    same(x, kw, stride=stride, out_stride=out_stride, offset=offset, out_offset=out_offset, inplace=inplace)


@pytest.mark.parametrize("last_n", [1, 7, 59, 60, 61, 1000])
def test_last_n(last_n):
    x, kw = case(np.random.default_rng(last_n), 4, 500, 60)
    same(x, dict(kw, last_n=last_n))


def test_each_rule_alone_and_none():
    x, kw = case(np.random.default_rng(9), 3, 700, 40, 5, True)
    hist = {k: kw[k] for k in ("history", "lens", "prompt")}
    same(x, {})
    same(x, hist)
    for k in ("rep", "freq", "pres"):
        same(x, dict(hist, **{k: kw[k]}))
    same(x, dict(history=kw["history"], rep=kw["rep"]))           # every id counts, all of it output
    same(x, dict(history=kw["history"], freq=kw["freq"], prompt=np.array([0, 40, 99], np.int32)))
    for k in ("temp", "bias"):
        same(x, {k: kw[k]})
    same(x, dict(allow=kw["allow"], allow_row=kw["allow_row"]))
    same(x, dict(allow=np.concatenate([kw["allow"], kw["allow"]])))   # mask r for row r
    same(x, dict(temp=np.array([0.0, -1.0, 2.0], F)))                 # no division by 0 or less
    y, n = call(x, **kw, want_next=False)
    assert (n == -7).all()
    np.testing.assert_array_equal(y, plain(x, **kw)[0])


def test_the_same_id_many_times():
    """Counts of one id add up, a bias entry that comes later replaces an earlier one, and the
    result does not depend on which thread came first."""
    rng = np.random.default_rng(1)
    x = rng.standard_normal((2, 300)).astype(F)
    h = np.full((2, 70000), 7, np.int32)
    h[1, ::2] = 299
    bias = [[(5, F(k)) for k in range(1500)] + [(6, F(1)), (5, F(-0.25))], [(299, F(2)), (299, F(3))] * 40]
    kw = dict(history=h, freq=np.full(2, 1e-3, F), pres=np.ones(2, F), rep=np.full(2, 1.5, F), bias=bias,
              prompt=np.array([0, 30000], np.int32))
    same(x, kw)
    same(x, kw, inplace=True)


def test_values_that_are_not_finite():
    x, kw = case(np.random.default_rng(4), 6, 64, 30, 4, True)
    x[0, :] = -np.inf                       # nothing is left: no token
    x[1, 3], x[1, 9], x[1, 10] = np.nan, np.inf, np.inf
    x[2, :] = np.nan
    x[3, ::2] = -np.inf
    x[4, :] = 0.0                           # all equal: the lowest index
    x[4, 5] = -0.0
    x[5, 11] = np.finfo(F).max
    same(x, {})
    del kw["allow"], kw["allow_row"]
    same(x, kw)
    same(x, dict(allow=np.zeros((1, 64), bool), allow_row=np.zeros(6, np.int32)))   # a mask that leaves nothing
    one = np.zeros((6, 64), bool)
    one[:, 63] = True
    same(x, dict(allow=one))


def test_padding_rows_are_left():
    x, kw = case(np.random.default_rng(6), 5, 4000, 50, 6, True)
    kw["lens"][[1, 4]] = -1
    y, n = call(x, **kw)
    assert (y[[1, 4]] == 7.5).all() and (n[[1, 4]] == -7).all()
    kw["lens"][[1, 4]] = 0
    wy, wn = plain(x, **kw)
    np.testing.assert_array_equal(y[[0, 2, 3]], wy[[0, 2, 3]])
    np.testing.assert_array_equal(n[[0, 2, 3]], wn[[0, 2, 3]])
    # padding rows between others, many rows
    x9, kw9 = case(np.random.default_rng(9), 900, 700, 30, 3, True)
    pad = np.arange(900) % 7 == 2
    kw9["lens"][pad] = -1
    y, n = call(x9, **kw9)
    assert (y[pad] == 7.5).all() and (n[pad] == -7).all()
    kw9["lens"][pad] = 0
    wy, wn = plain(x9, **kw9)
    np.testing.assert_array_equal(y[~pad], wy[~pad])
    np.testing.assert_array_equal(n[~pad], wn[~pad])
    kw["lens"][:] = -1
    y, n = call(x, **kw)
    assert (y == 7.5).all() and (n == -7).all()
    # padding is marked by history_len alone too, when no history counts
    y, n = call(x, lens=np.array([0, -1, 5, -1, 0]), temp=kw["temp"])
    assert (y[[1, 3]] == 7.5).all() and (n[[1, 3]] == -7).all() and (y[[0, 2, 4]] != 7.5).all()


def test_ids_out_of_range_are_reported_and_left_out():
    x, kw = case(np.random.default_rng(7), 3, 200, 30, 0, False)
    kw["lens"][:] = 30
    kw["history"][1, :10] = -1              # negative: no entry, no error
    same(x, kw)
    for where, value in (((0, 0), 200), ((2, 29), 2 ** 31 - 1)):
        bad = dict(kw, history=kw["history"].copy())
        bad["history"][where] = value
        L.alb_device_error(1)
        y, n = call(x, **bad)
        assert L.alb_device_error(1) == 4
        np.testing.assert_array_equal(y, plain(x, **bad)[0])
    bad = dict(kw, lens=np.array([30, 31, 2 ** 31 - 1], np.int32))       # cut to the row
    y, n = call(x, **bad)
    assert L.alb_device_error(1) == 4
    np.testing.assert_array_equal(y, plain(x, **bad)[0])
    same(x, dict(bias=[[(-1, F(3)), (4, F(1))], [], [(-2 ** 31, F(3))]]))
    bias = dict(bias=[[(200, F(3)), (4, F(1))], [(2 ** 31 - 1, F(1))], []])
    y, n = call(x, **bias)
    assert L.alb_device_error(1) == 4
    np.testing.assert_array_equal(y, plain(x, **bias)[0])
    masks = np.random.default_rng(0).random((2, 200)) < 0.5
    rows = dict(allow=masks, allow_row=np.array([1, 2, 2 ** 31 - 1], np.int32))   # no such mask: none
    y, n = call(x, **rows)
    assert L.alb_device_error(1) == 4
    np.testing.assert_array_equal(y, plain(x, **rows)[0])


def test_bias_offsets_outside_the_list_are_cut():
    x = np.zeros((2, 50), F)
    X, Y = cu(x), torch.zeros(2, 50, device="cuda")
    off, ids, val = cu(np.array([-3, 2, 900], np.int32)), cu(np.arange(4, dtype=np.int32)), cu(np.ones(4, F))
    r = A.LogitsRules(bias_offsets=off.data_ptr(), bias_ids=ids.data_ptr(), bias_values=val.data_ptr(), n_bias=4)
    L.alb_device_error(1)
    A.check(L.alb_logits_process(X.data_ptr(), 2, 50, 0, C.byref(r), Y.data_ptr(), 0, None, st()))
    torch.cuda.synchronize()
    assert L.alb_device_error(1) == 4
    want = x.copy()
    want[0, :2], want[1, 2:4] = 1, 1
    np.testing.assert_array_equal(Y.cpu().numpy(), want)


def test_two_streams_and_a_replayed_graph():
    x, kw = case(np.random.default_rng(12), 8, 30000, 400, 0, False)
    wy, wn = plain(x, **kw)
    X = cu(x)
    d = {k: cu(v) for k, v in kw.items()}
    r = A.LogitsRules(history=d["history"].data_ptr(), history_stride=400, history_len=d["lens"].data_ptr(),
                      prompt_len=d["prompt"].data_ptr(), repetition=d["rep"].data_ptr(),
                      frequency=d["freq"].data_ptr(), presence=d["pres"].data_ptr(), temperature=d["temp"].data_ptr())
    ys = [torch.zeros_like(X) for _ in range(3)]
    ns = [torch.zeros(8, dtype=torch.int32, device="cuda") for _ in range(3)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(10):
        for s, y, n in zip(streams, ys, ns):
            A.check(L.alb_logits_process(X.data_ptr(), 8, 30000, 0, C.byref(r), y.data_ptr(), 0, n.data_ptr(), s.cuda_stream))
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        A.check(L.alb_logits_process(X.data_ptr(), 8, 30000, 0, C.byref(r), ys[2].data_ptr(), 0, ns[2].data_ptr(), st()))
    g.replay()
    torch.cuda.synchronize()
    for y, n in zip(ys, ns):
        np.testing.assert_array_equal(y.cpu().numpy(), wy)
        np.testing.assert_array_equal(n.cpu().numpy(), wn)
    # the graph reads the arrays anew: other lengths, other logits
    kw["lens"] = np.arange(8, dtype=np.int32)
    d["lens"].copy_(cu(kw["lens"]))
    x2 = (x * F(0.5)).astype(F)
    X.copy_(cu(x2))
    g.replay()
    torch.cuda.synchronize()
    wy, wn = plain(x2, **kw)
    np.testing.assert_array_equal(ys[2].cpu().numpy(), wy)
    np.testing.assert_array_equal(ns[2].cpu().numpy(), wn)


@pytest.mark.parametrize("vocab,hist", [(16000, 9000), (9000, 20000)])   # 16-bit and 32-bit counts
def test_more_distinct_ids_than_a_cta_lists(vocab, hist):
    rng = np.random.default_rng(hist)
    x, kw = case(rng, 500, vocab, hist, 20, True)
    kw["history"] = rng.integers(0, vocab, (500, hist)).astype(np.int32)
    kw["lens"][:] = rng.integers(0, hist + 1, 500)
    kw["lens"][:3] = (hist, hist, 0)
    same(x, kw)
    same(x, kw, inplace=True)


def test_division_by_the_temperature_rounds_as_the_quotient():
    """Values over all exponents, temperatures inside and outside the range of the short division."""
    rng = np.random.default_rng(3)
    temps = np.concatenate([rng.uniform(0.01, 3.0, 40), 2.0 ** rng.uniform(-19.9, 19.9, 20),
                            [2.0 ** -20, 2.0 ** 20, np.nextafter(F(2.0 ** -20), F(1)), 1e-25, 1e25, 1e-42, 3e38, 1.0, 0.7, 1.9999999]]).astype(F)
    bits = rng.integers(0, 2 ** 32, (len(temps), 30000), dtype=np.uint64).astype(np.uint32)
    x = bits.view(F).copy()
    x[np.isnan(x)] = 0
    x[:, ::3] = (rng.standard_normal(x[:, ::3].shape) * 5).astype(F)
    x[:, :6] = [0.0, -0.0, np.inf, -np.inf, np.finfo(F).max, 1e-45]
    y, n = call(x, temp=temps)
    with np.errstate(all="ignore"):
        want = x / temps[:, None]
    np.testing.assert_array_equal(y.view(np.uint32), want.view(np.uint32))
    np.testing.assert_array_equal(n, want.argmax(1))


@pytest.mark.parametrize("offsets", [(900, 4, 4), (0, -5, 0), (-9, -5, -1), (5, 9, 900), (2, 1, 4), (0, 2 ** 31 - 1, -2 ** 31)])
def test_bias_offsets_outside_the_list_or_falling_are_reported(offsets):
    """Starts and ends on either side of the list, and ranges that run backwards: what lies in the list counts."""
    X, Y = torch.zeros(2, 50, device="cuda"), torch.zeros(2, 50, device="cuda")
    off, ids, val = cu(np.array(offsets, np.int32)), cu(np.arange(4, dtype=np.int32)), cu(np.ones(4, F))
    r = A.LogitsRules(bias_offsets=off.data_ptr(), bias_ids=ids.data_ptr(), bias_values=val.data_ptr(), n_bias=4)
    for row in range(2):                     # each row alone, so that each reports
        r.bias_offsets = off[row:].data_ptr()
        L.alb_device_error(1)
        A.check(L.alb_logits_process(X.data_ptr(), 1, 50, 0, C.byref(r), Y[row].data_ptr(), 0, None, st()))
        torch.cuda.synchronize()
        b0, b1 = offsets[row], offsets[row + 1]
        assert L.alb_device_error(1) == (0 if 0 <= b0 <= b1 <= 4 else 4), (b0, b1)
        want = np.zeros(50, F)
        want[max(b0, 0):max(min(b1, 4), 0)] = 1
        np.testing.assert_array_equal(Y[row].cpu().numpy(), want)
