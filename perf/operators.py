"""The operators of a batch-serving step, as a user calls them, beside their plain forms in torch.

Three operators that follow one another when many sequences decode together:

  append   ``alb_qk_norm_rope_kv_paged``: QK-norm and RoPE of the new tokens, their K/V rows into a paged cache
  attend   ``alb_paged_attn``: each query token over its sequence's pages
  choose   ``alb_logits_process``: bias, repetition penalties, temperature and grammar mask on the logits, and the
           greedy token

``run`` computes a case in plain torch operations, or through the library when ``own`` is true; ``exact`` computes
the same from the definition in 64 bits.
"""
import math

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-6
FREQ_BASE = 1e6


def listed():
    return [
        # one user, a 4B-shaped model (32 / 8 heads) shortly after its prompt: latency is all
        dict(name="attend_one_640", op="attend", rows=1, heads=32, heads_kv=8, dim=128, page=16, longest=640,
             shortest=640, window=0, kv="f16"),
        # a handful of chats on one card: uneven lengths, one slot of the batch still empty
        dict(name="attend_chats_37", op="attend", rows=37, heads=32, heads_kv=8, dim=128, page=16, longest=8191,
             shortest=0, window=0, kv="bf16"),
        # one long document, the cache split over the whole card
        dict(name="attend_document_32768", op="attend", rows=1, heads=32, heads_kv=8, dim=128, page=64, longest=32768,
             shortest=32768, window=0, kv="f16"),
        # cells instead of pages (page of one, as the cell manager hands them out), small heads, a sliding window
        dict(name="attend_cells_window", op="attend", rows=200, heads=15, heads_kv=3, dim=64, page=1, longest=1500,
             shortest=0, window=512, kv="f16"),
        # a full card: 48 long sequences
        dict(name="attend_full_48", op="attend", rows=48, heads=32, heads_kv=8, dim=128, page=32, longest=32768,
             shortest=8192, window=0, kv="f16"),
        # one decode step of a few sequences
        dict(name="append_decode_5", op="append", tokens=5, sequences=5, heads=32, heads_kv=8, dim=128, page=16,
             furthest=4000, kv="f16"),
        # one decode step of a wide batch of a small model
        dict(name="append_decode_251", op="append", tokens=251, sequences=251, heads=14, heads_kv=2, dim=64, page=16,
             furthest=2000, kv="bf16"),
        # prompts of several sequences entering the cache together
        dict(name="append_prompts_8192", op="append", tokens=8192, sequences=7, heads=32, heads_kv=8, dim=128, page=32,
             furthest=30000, kv="f16"),
        # one user's next token under the usual penalties
        dict(name="choose_one", op="choose", rows=1, vocab=151936, history=512, bias=0, mask=False, last_n=0),
        # structured output for a batch: grammar masks, logit biases, short histories, an odd vocabulary
        dict(name="choose_grammar_48", op="choose", rows=48, vocab=151669, history=2000, bias=60, mask=True, last_n=0),
        # penalties over the last tokens of long chats
        dict(name="choose_long_64", op="choose", rows=64, vocab=32003, history=32768, bias=0, mask=False, last_n=8192),
        # a wide batch with long outputs
        dict(name="choose_wide_256", op="choose", rows=256, vocab=151936, history=4096, bias=0, mask=True, last_n=0),
    ]


def _log(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["attend", "attend", "append", "choose"])
    if op == "choose":
        vocab = _log(rng, 1000, 262144)
        rows = min(_log(rng, 1, 256), max(1, 256 * 151936 // vocab))
        history = _log(rng, 1, 32768)
        return dict(op=op, rows=rows, vocab=vocab, history=history, bias=rng.choice([0, 0, _log(rng, 1, 300)]),
                    mask=rng.random() < 0.5, last_n=rng.choice([0, 0, _log(rng, 1, 32768)]))
    heads, heads_kv = rng.choice([(32, 8), (16, 8), (8, 8), (14, 2), (15, 3), (32, 2), (5, 1), (40, 8)])
    dim, page = rng.choice([64, 128, 128]), rng.choice([1, 7, 16, 16, 32, 64, 128, 256])
    kv = rng.choice(["f16", "bf16"])
    if op == "append":
        tokens = _log(rng, 1, 8192)
        sequences = rng.choice([tokens, min(tokens, _log(rng, 1, 64))])
        return dict(op=op, tokens=tokens, sequences=sequences, heads=heads, heads_kv=heads_kv, dim=dim, page=page,
                    furthest=_log(rng, tokens // sequences + 1, 32768), kv=kv)
    longest = _log(rng, 1, 32768)
    rows = min(_log(rng, 1, 256), max(1, 48 * 20480 // longest))
    return dict(op=op, rows=rows, heads=heads, heads_kv=heads_kv, dim=dim, page=page, longest=longest,
                shortest=rng.randint(0, longest), window=rng.choice([0, 0, _log(rng, 1, 8192)]), kv=kv)


# ------------------------------------------------------------------------------------------------------- inputs
def _lengths(case, seed):
    """Lengths of the rows, on the host: the longest first, the rest spread between shortest and longest."""
    g = torch.Generator().manual_seed(seed)
    n = torch.randint(case["shortest"], case["longest"] + 1, (case["rows"],), generator=g)
    n[0] = case["longest"]
    return n


def _pages(counts, gen, device):
    """A page table [sequences][most pages] of distinct pages in no order, and the pages in the pool."""
    most, total = max(1, int(counts.max())), int(counts.sum())
    pool = max(1, total + total // 16)
    table = torch.full((len(counts), most), -1, dtype=torch.int32, device=device)
    order = torch.randperm(pool, generator=gen, device=device)[:total].to(torch.int32)
    column = torch.arange(most, device=device)[None, :]
    table[column < counts.to(device)[:, None]] = order
    return table, pool


def _angles(positions, dim, device):
    inv = FREQ_BASE ** (-torch.arange(0, dim, 2, dtype=torch.float64, device=device) / dim)
    a = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * inv
    return torch.stack([a.cos(), a.sin()], -1).float().contiguous()


def prepare(case, seed):
    device = torch.device("cuda")
    gen = torch.Generator(device=device).manual_seed(seed)

    def normal(*shape, dtype=torch.float32):
        return torch.randn(shape, generator=gen, device=device, dtype=dtype)

    if case["op"] == "choose":
        rows, vocab, history = case["rows"], case["vocab"], case["history"]
        words = (vocab + 31) // 32

        def uniform(low, high):
            return low + (high - low) * torch.rand(rows, generator=gen, device=device)

        # few tokens make up most of a text
        ids = (vocab * torch.rand(rows, history, generator=gen, device=device) ** 4).to(torch.int32).clamp_(max=vocab - 1)
        lens = torch.randint(0, history + 1, (rows,), generator=gen, device=device, dtype=torch.int32)
        lens[0] = history
        s = dict(case=case, logits=normal(rows, vocab) * 3, ids=ids, lens=lens,
                 prompt=(lens * torch.rand(rows, generator=gen, device=device)).to(torch.int32),
                 repetition=uniform(1.0, 1.3), frequency=uniform(0.0, 0.5), presence=uniform(0.0, 0.5),
                 temperature=uniform(0.5, 1.3), out=torch.empty(rows, vocab, device=device),
                 next=torch.empty(rows, dtype=torch.int32, device=device),
                 allow=None, allow_row=None, bias_ids=None)
        if case["bias"]:
            n = torch.randint(0, case["bias"] + 1, (rows,), generator=gen, device=device)
            n[0] = case["bias"]
            s["bias_offsets"] = torch.cat([torch.zeros(1, dtype=torch.int64, device=device), n.cumsum(0)]).to(torch.int32)
            total = int(n.sum())
            s["bias_ids"] = torch.randint(0, vocab, (total,), generator=gen, device=device, dtype=torch.int32)
            s["bias_values"] = normal(total) * 5
        if case["mask"]:   # a few grammar states shared by the rows; every fourth row writes freely
            states = (rows + 3) // 4
            s["allow"] = torch.randint(-2**31, 2**31, (states, words), generator=gen, device=device).to(torch.int32)
            row = torch.randint(0, states, (rows,), generator=gen, device=device, dtype=torch.int32)
            s["allow_row"] = torch.where(torch.arange(rows, device=device) % 4 == 3, -1, row).to(torch.int32)
    elif case["op"] == "attend":
        lens = _lengths(case, seed)
        table, pool = _pages((lens + case["page"] - 1) // case["page"], gen, device)
        shape = (pool, case["page"], case["heads_kv"], case["dim"])
        s = dict(case=case, table=table, k=normal(*shape, dtype=DTYPES[case["kv"]]),
                 v=normal(*shape, dtype=DTYPES[case["kv"]]), q=normal(case["rows"], case["heads"], case["dim"]) * 1.5,
                 lens=lens.to(device, torch.int32), longest=int(lens.max()), scale=case["dim"] ** -0.5,
                 out=torch.empty(case["rows"], case["heads"], case["dim"], device=device),
                 lse=torch.empty(case["rows"], case["heads"], device=device))
    else:
        g = torch.Generator().manual_seed(seed)
        n = torch.full((case["sequences"],), case["tokens"] // case["sequences"])
        n[: case["tokens"] - int(n.sum())] += 1
        first = (torch.rand(len(n), generator=g) * (case["furthest"] - n + 1).clamp_(min=1)).to(torch.int64)
        most = case["furthest"] + int(n.max())
        # the pages that the tokens go to are their own; earlier ones may be a prefix that sequences share
        page, pool = case["page"], case["tokens"] // case["page"] + 2 * case["sequences"]
        columns = torch.arange((most + page - 1) // page, device=device)[None, :]
        table = torch.randint(0, pool, (len(n), columns.shape[1]), generator=gen, device=device, dtype=torch.int32)
        fresh = (columns >= (first // page).to(device)[:, None]) & (columns <= ((first + n - 1) // page).to(device)[:, None])
        order = torch.randperm(pool, generator=gen, device=device).to(torch.int32)
        table[fresh] = order[: int(fresh.sum())]
        seqs = torch.repeat_interleave(torch.arange(len(n)), n)
        within = torch.arange(case["tokens"]) - torch.repeat_interleave(n.cumsum(0) - n, n)
        shape = (pool, case["page"], case["heads_kv"], case["dim"])
        wide = (case["heads"] + 2 * case["heads_kv"]) * case["dim"]
        s = dict(case=case, table=table, k=normal(*shape, dtype=DTYPES[case["kv"]]),
                 v=normal(*shape, dtype=DTYPES[case["kv"]]), qkv=normal(case["tokens"], wide) * 2,
                 q_norm=1 + 0.1 * normal(case["dim"]), k_norm=1 + 0.1 * normal(case["dim"]),
                 angles=_angles(most, case["dim"], device), most=most,
                 seqs=seqs.to(device, torch.int32), positions=(first[seqs] + within).to(device, torch.int32),
                 q=torch.empty(case["tokens"], case["heads"], case["dim"], device=device))
    if own:
        _handle(s)
    return s


# ----------------------------------------------------------------------------------------- the library's own calls
def _handle(s):
    """What a program keeps between its calls: the descriptors, the workspace and the pointers."""
    import ctypes

    import arclight_b200 as A

    case, lib = s["case"], A.lib()
    p = {k: v.data_ptr() for k, v in s.items() if isinstance(v, torch.Tensor)}
    if case["op"] == "choose":
        r = A.LogitsRules(history=p["ids"], history_stride=case["history"], history_len=p["lens"],
                          prompt_len=p["prompt"], last_n=case["last_n"], repetition=p["repetition"],
                          frequency=p["frequency"], presence=p["presence"], temperature=p["temperature"])
        if s["bias_ids"] is not None:
            r.bias_ids, r.bias_values, r.bias_offsets = p["bias_ids"], p["bias_values"], p["bias_offsets"]
            r.n_bias = len(s["bias_ids"])
        if s["allow"] is not None:
            r.allow, r.allow_row = p["allow"], p["allow_row"]
            r.allow_stride, r.n_allow = s["allow"].shape[1], s["allow"].shape[0]
        s["call"] = lib.alb_logits_process, (p["logits"], case["rows"], case["vocab"], 0, ctypes.byref(r), p["out"], 0,
                                             p["next"])
        s["keep"] = r
        return
    kv = A.PagedKV(k=p["k"], v=p["v"], page_table=p["table"], n_pages=s["k"].shape[0], n_seqs=s["table"].shape[0],
                   max_pages=s["table"].shape[1], page_size=case["page"], n_head_kv=case["heads_kv"],
                   head_dim=case["dim"], type=A.ALB_KV_BF16 if case["kv"] == "bf16" else A.ALB_KV_F16)
    s["keep"] = kv
    if case["op"] == "attend":
        need = lib.alb_paged_attn_workspace_bytes(ctypes.byref(kv), case["rows"], case["heads"])
        s["workspace"] = torch.empty(max(1, need), dtype=torch.uint8, device="cuda")
        s["call"] = lib.alb_paged_attn, (p["q"], case["rows"], case["heads"], ctypes.byref(kv), None, p["lens"],
                                         case["window"], s["scale"], s["workspace"].data_ptr(), p["out"], p["lse"])
    else:
        s["call"] = lib.alb_qk_norm_rope_kv_paged, (p["qkv"], 0, case["tokens"], case["heads"], p["q_norm"],
                                                    p["k_norm"], EPS, p["angles"], s["most"], p["positions"],
                                                    p["seqs"], ctypes.byref(kv), p["q"])


def _own(s):
    f, a = s["call"]
    rc = f(*a, torch.cuda.current_stream().cuda_stream)
    if rc != 0:
        import arclight_b200 as A
        A.check(rc, f.__name__)
    op = s["case"]["op"]
    if op == "append":
        return {"q": s["q"], "k": s["k"], "v": s["v"]}
    return {"out": s["out"], "lse": s["lse"]} if op == "attend" else {"out": s["out"], "next": s["next"]}


# ------------------------------------------------------------------------------------------------ the plain forms
def _append(s):
    case, dim, hq, hkv = s["case"], s["case"]["dim"], s["case"]["heads"], s["case"]["heads_kv"]
    x = s["qkv"].view(case["tokens"], -1, dim)
    cs = s["angles"][s["positions"].long()][:, None]

    def turned(x, w):
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + EPS) * w
        a, b = x[..., : dim // 2], x[..., dim // 2:]
        return torch.cat([a * cs[..., 0] - b * cs[..., 1], a * cs[..., 1] + b * cs[..., 0]], -1)

    q, k, v = turned(x[:, :hq], s["q_norm"]), turned(x[:, hq:hq + hkv], s["k_norm"]), x[:, hq + hkv:]
    pos = s["positions"].long()
    page = s["table"][s["seqs"].long(), pos // case["page"]].long()
    s["k"][page, pos % case["page"]] = k.to(s["k"].dtype)
    s["v"][page, pos % case["page"]] = v.to(s["v"].dtype)
    return {"q": q, "k": s["k"], "v": s["v"]}


def _attend(s):
    case, rows, hkv, dim = s["case"], s["case"]["rows"], s["case"]["heads_kv"], s["case"]["dim"]
    pos = torch.arange(max(1, s["longest"]), device="cuda")
    page = s["table"][:, pos // case["page"]].clamp(min=0).long()
    at = page * case["page"] + pos % case["page"]
    k = s["k"].view(-1, hkv, dim)[at].float().permute(0, 2, 3, 1)
    x = torch.matmul(s["q"].view(rows, hkv, -1, dim), k) * s["scale"]
    del k
    seen = pos[None] < s["lens"][:, None]
    if case["window"]:
        seen &= pos[None] >= s["lens"][:, None] - case["window"]
    x = x.masked_fill(~seen[:, None, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    e = torch.exp(x - torch.where(top.isfinite(), top, 0.0))
    total = e.sum(-1, keepdim=True)
    v = s["v"].view(-1, hkv, dim)[at].float().transpose(1, 2)
    out = torch.matmul(e, v) / torch.where(total > 0, total, 1.0)
    return {"out": out.view(rows, -1, dim), "lse": (top + torch.log(total)).view(rows, -1)}


def _choose(s):
    case, rows, vocab = s["case"], s["case"]["rows"], s["case"]["vocab"]
    x = s["logits"]
    if s["bias_ids"] is not None:   # the last entry of an id counts
        n = torch.arange(len(s["bias_ids"]), device="cuda")
        row = torch.searchsorted(s["bias_offsets"][1:].long(), n, right=True)
        last = torch.full((rows * vocab,), -1, device="cuda")
        last = last.scatter_reduce(0, row * vocab + s["bias_ids"], n, "amax").view(rows, vocab)
        x = torch.where(last >= 0, x + s["bias_values"][last.clamp(min=0)], x)
    at = torch.arange(case["history"], device="cuda")[None]
    used = at < s["lens"][:, None]
    if case["last_n"]:
        used &= at >= s["lens"][:, None] - case["last_n"]
    seen = torch.zeros(rows, vocab, device="cuda").scatter_add(1, s["ids"].long(), used.float())
    n_out = torch.zeros(rows, vocab, device="cuda").scatter_add(1, s["ids"].long(),
                                                               (used & (at >= s["prompt"][:, None])).float())
    r = s["repetition"][:, None]
    x = torch.where(seen > 0, torch.where(x > 0, x / r, x * r), x)
    x = x - s["frequency"][:, None] * n_out
    x = x - s["presence"][:, None] * (n_out > 0)
    x = x / s["temperature"][:, None]
    if s["allow"] is not None:
        i = torch.arange(vocab, device="cuda")
        bit = (s["allow"][s["allow_row"].clamp(min=0).long()][:, i >> 5] >> (i & 31).int()) & 1
        x = x.masked_fill((bit == 0) & (s["allow_row"] >= 0)[:, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    first = torch.where(x == top, torch.arange(vocab, device="cuda"), vocab).amin(-1)
    return {"out": x, "next": torch.where(top[:, 0] > -math.inf, first, -1).to(torch.int32)}


def run(state):
    if own:
        return _own(state)
    return {"append": _append, "attend": _attend, "choose": _choose}[state["case"]["op"]](state)


# --------------------------------------------------------------------------------------------------------- work
def work(case):
    if case["op"] == "choose":
        rows, vocab = case["rows"], case["vocab"]
        used = min(case["history"], case["last_n"] or case["history"])
        tokens = used + (rows - 1) * used / 2   # lengths are spread evenly, the first row's is the longest
        b = rows * vocab * 8 + tokens * 4 + rows * 24
        b += rows * case["bias"] * 4 if case["bias"] else 0
        b += (rows + 3) // 4 * ((vocab + 31) // 32) * 4 if case["mask"] else 0
        return {"bytes": b, "flops": 4 * rows * vocab}
    hq, hkv, dim = case["heads"], case["heads_kv"], case["dim"]
    if case["op"] == "append":
        t = case["tokens"]
        return {"bytes": t * ((hq + 2 * hkv) * dim * 4 + hq * dim * 4 + 2 * hkv * dim * 2 + dim * 4 + 12),
                "flops": t * (hq + hkv) * dim * 8}
    cells = 0
    for seed in range(4):   # the mean over a few of the draws of lengths
        n = _lengths(case, seed)
        cells += int((n.clamp(max=case["window"]) if case["window"] else n).sum()) / 4
    return {"bytes": cells * hkv * dim * 4 + case["rows"] * hq * (dim * 8 + 4) + cells / case["page"] * 4,
            "flops": cells * hq * dim * 4}


# ------------------------------------------------------------------------------------- the definition in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "choose":
        vocab = case["vocab"]
        out, chosen = s["logits"].double(), []
        index = torch.arange(vocab, device="cuda")
        lens, prompt = s["lens"].tolist(), s["prompt"].tolist()
        for b, z in enumerate(out):
            if s["bias_ids"] is not None:
                lo, hi = s["bias_offsets"][b:b + 2].tolist()
                table = dict(zip(s["bias_ids"][lo:hi].tolist(), s["bias_values"][lo:hi].tolist()))
                if table:
                    z[torch.tensor(list(table), device="cuda")] += torch.tensor(list(table.values()),
                                                                                dtype=torch.float64, device="cuda")
            start = max(0, lens[b] - case["last_n"]) if case["last_n"] else 0
            ids = s["ids"][b].long()
            every = torch.bincount(ids[start:lens[b]], minlength=vocab)
            written = torch.bincount(ids[max(start, prompt[b]):lens[b]], minlength=vocab)
            r = s["repetition"][b].double()
            hit = every > 0
            z[hit] = torch.where(z[hit] > 0, z[hit] / r, z[hit] * r)
            z -= s["frequency"][b].double() * written + s["presence"][b].double() * written.clamp(max=1)
            z /= s["temperature"][b].double()
            if s["allow"] is not None and int(s["allow_row"][b]) >= 0:
                word = s["allow"][int(s["allow_row"][b])].long() & 0xFFFFFFFF
                z[(word[index // 32] // 2 ** (index % 32)) % 2 == 0] = -math.inf
            best = z.max()
            chosen.append(int((z == best).nonzero()[0]) if float(best) > -math.inf else -1)
        return {"out": out, "next": torch.tensor(chosen, dtype=torch.int32, device="cuda")}
    dim, hq, hkv, page = case["dim"], case["heads"], case["heads_kv"], case["page"]
    if case["op"] == "append":
        heads = s["qkv"].double().view(case["tokens"], -1, dim)
        norm = (heads / (heads.pow(2).sum(-1, keepdim=True) / dim + EPS).sqrt())
        weight = torch.cat([s["q_norm"].double().expand(hq, dim), s["k_norm"].double().expand(hkv, dim)])
        turn = torch.view_as_complex(s["angles"].double())[s["positions"].long()][:, None]
        pair = (norm[:, :hq + hkv] * weight).unflatten(-1, (2, dim // 2))
        z = torch.complex(pair[..., 0, :].contiguous(), pair[..., 1, :].contiguous()) * turn
        z = torch.cat([z.real, z.imag], -1)
        k, v = s["k"].double(), s["v"].double()
        cell = s["table"].long()[s["seqs"].long(), (s["positions"] // page).long()] * page + s["positions"] % page
        k.view(-1, hkv, dim)[cell] = z[:, hq:]
        v.view(-1, hkv, dim)[cell] = heads[:, hq + hkv:]
        return {"q": z[:, :hq].contiguous(), "k": k, "v": v}
    out = torch.zeros(case["rows"], hq, dim, dtype=torch.float64, device="cuda")
    lse = torch.full((case["rows"], hq), -math.inf, dtype=torch.float64, device="cuda")
    for b, n in enumerate(s["lens"].tolist()):
        low = max(0, n - case["window"]) if case["window"] else 0
        if n == low:
            continue
        held = (n + page - 1) // page
        took = s["table"][b, :held].long()
        k = s["k"][took].view(-1, hkv, dim)[low:n].double().permute(1, 2, 0)
        v = s["v"][took].view(-1, hkv, dim)[low:n].double().permute(1, 0, 2)
        x = s["q"][b].double().view(hkv, -1, dim) @ k * s["scale"]
        lse[b] = torch.logsumexp(x, -1).view(-1)
        out[b] = (torch.softmax(x, -1) @ v).view(hq, dim)
    return {"out": out, "lse": lse}
