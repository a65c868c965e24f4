"""Measured cases of the bounded-cache operators: attention over a sliding window with sinks (decode
and prefill), decode attention that accumulates each cached key's weight, and the eviction of the
keys with the smallest accumulated weight.

A model that runs past its cache's budget keeps a few first tokens, a recent window, and either
nothing else (window with sinks) or the tokens that the queries so far have attended to most
(eviction by accumulated weight). All cases work on the paged cache of this framework: pages of 32
cells, K and V [n_cells][n_head_kv][128] f16 or q8_0 planes, int32 block tables.

`own = False` computes every operator in elementary torch operations in f32; `own = True` makes the
framework's calls. `exact` restates each operator in f64.
"""
import math

import torch

own = False

D = 128
PAGE = 32
SCALE = 1.0 / math.sqrt(D)


# ---- cases -----------------------------------------------------------------------------------------
# lo, hi: the sequences' lengths are spread evenly over [lo, hi] (the seed shuffles them).


def listed():
    return [
        # One sequence of a short chat with a small window: the smallest call, bound by its latency.
        dict(name="window 1x513", op="window", kind="f16", B=1, Hq=16, Hkv=8, lo=513, hi=513, W=256, sink=4, empty=0),
        # A serving batch of mixed contexts up to 32 k, each held to a window of 4096 and 4 sinks.
        dict(name="window 64x1k-32k", op="window", kind="f16", B=64, Hq=32, Hkv=4, lo=1024, hi=32768, W=4096, sink=4,
             empty=0),
        # The same service on a q8_0 cache with ragged lengths, a finished (empty) slot, a window and a
        # sink count that end inside pages.
        dict(name="window q8 37x1-16k", op="window", kind="q8", B=37, Hq=16, Hkv=8, lo=1, hi=16001, W=1999, sink=33,
             empty=1),
        # One prompt of the smaller model shape, window shorter than the prompt.
        dict(name="prefill 1x2048", op="prefill", kind="f16", qd="f16", B=1, Hq=16, Hkv=8, T=2048, lo=2048, hi=2048,
             W=512, sink=4),
        # A continuous-batching step: eight ragged chunks of up to 511 tokens behind contexts of up to 16 k,
        # f32 queries.
        dict(name="prefill 8x511", op="prefill", kind="f16", qd="f32", B=8, Hq=32, Hkv=4, T=511, lo=513, hi=16384,
             W=4096, sink=4),
        # A long prompt in one call, window half its length.
        dict(name="prefill 1x8192", op="prefill", kind="f16", qd="f16", B=1, Hq=32, Hkv=4, T=8192, lo=8192, hi=8192,
             W=4096, sink=64),
        # A single sequence whose keys' weights are accumulated at every step (latency again).
        dict(name="weights 1x513", op="weights", kind="f16", B=1, Hq=16, Hkv=8, lo=513, hi=513, empty=0),
        # The batched decode of mixed contexts up to 32 k: the largest pass over a cache.
        dict(name="weights 64x1k-32k", op="weights", kind="f16", B=64, Hq=32, Hkv=4, lo=1024, hi=32768, empty=0),
        # A q8_0 cache held near a budget of 4096, ragged, with an empty slot.
        dict(name="weights q8 29x1-4k", op="weights", kind="q8", B=29, Hq=16, Hkv=8, lo=1, hi=4160, empty=1),
        # One sequence a page over its budget.
        dict(name="evict 1x544", op="evict", kind="f16", B=1, Hkv=8, lo=544, hi=544, budget=512, sink=4, recent=64),
        # A batch held at 4096 keys, evicting every 64 tokens; the shorter rows are below their budget.
        dict(name="evict 64x4k", op="evict", kind="f16", B=64, Hkv=4, lo=4000, hi=4160, budget=4096, sink=4,
             recent=256),
        # Prompts of up to 32 k cut to 8 k of their keys after prefill, q8_0 cache.
        dict(name="evict q8 16x16k-32k", op="evict", kind="q8", B=16, Hkv=4, lo=16385, hi=32768, budget=8192, sink=33,
             recent=1000),
    ]


def log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["window", "prefill", "weights", "evict"])
    kind = rng.choice(["f16", "f16", "q8"])
    if op in ("window", "weights"):
        Hq, Hkv = rng.choice([(16, 8), (32, 4), (32, 8), (28, 4), (12, 2), (8, 8)])
        B = log_int(rng, 1, 192)
        hi = log_int(rng, 8, min(32768, 1000000 // B))
        lo = rng.choice([1, max(1, hi // 16), hi])
        c = dict(op=op, kind=kind, B=B, Hq=Hq, Hkv=Hkv, lo=lo, hi=hi, empty=rng.choice([0, 1]) if B > 1 else 0)
        if op == "window":
            c.update(W=log_int(rng, 1, 8192), sink=rng.choice([0, 1, 4, 31, 32, 64, 100]))
        return c
    if op == "prefill":
        Hq, Hkv = rng.choice([(16, 8), (32, 4), (32, 8), (8, 8)])
        B = log_int(rng, 1, 12)
        T = log_int(rng, 1, 2048 // B)
        hi = T + log_int(rng, 1, 12000)
        return dict(op=op, kind=kind, qd=rng.choice(["f16", "f32"]), B=B, Hq=Hq, Hkv=Hkv, T=T,
                    lo=rng.choice([T, hi]), hi=hi, W=log_int(rng, 1, 8192), sink=rng.choice([0, 1, 4, 33, 100]))
    B = log_int(rng, 1, 64)
    budget = log_int(rng, 16, min(16384, 300000 // B))
    hi = budget + log_int(rng, 1, min(2 * budget, 500000 // B))
    sink = min(rng.choice([0, 1, 4, 33]), budget)
    return dict(op=op, kind=kind, B=B, Hkv=rng.choice([2, 4, 8]), lo=rng.choice([max(1, budget // 2), budget + 1, hi]),
                hi=hi, budget=budget, sink=sink, recent=rng.randint(0, budget - sink))


def spread(case):
    """The sequences' lengths, in order (the seed only shuffles them)."""
    n = max(1, case["B"] - 1)
    lens = [case["lo"] + (case["hi"] - case["lo"]) * i // n for i in range(case["B"])] if case["B"] > 1 else [case["hi"]]
    if case.get("empty"):
        lens[0] = 0
    return lens


def chunks(case):
    """(query tokens, keys) of each sequence of a prefill: chunks of T, T - 1 / 7 T, ... behind their contexts."""
    return [(max(1, case["T"] - (case["T"] * i) // (7 * case["B"])), n) for i, n in enumerate(spread(case))]


def work(case):
    cell = case["Hkv"] * (256 if case["kind"] == "f16" else 136)  # bytes of one token's K (or V)
    if case["op"] == "window":
        keys = sum(min(n, case["W"] + min(case["sink"], max(0, n - case["W"]))) for n in spread(case))
        rows = case["B"] * case["Hq"]
        return {"bytes": 2 * cell * keys + rows * (256 + 256 + 4), "flops": 4.0 * D * case["Hq"] * keys}
    if case["op"] == "weights":
        keys = sum(spread(case))
        rows = case["B"] * case["Hq"]
        return {"bytes": (2 * cell + 8) * keys + rows * (256 + 256 + 4), "flops": 4.0 * D * case["Hq"] * keys}
    if case["op"] == "prefill":
        pairs = keys = rows = 0
        for t, n in chunks(case):
            p0 = n - t
            for p in range(p0, n):
                pairs += min(p + 1, case["W"] + min(case["sink"], max(0, p + 1 - case["W"])))
            first = max(0, p0 + 1 - case["W"])
            keys += n - first + min(case["sink"], first)
            rows += t * case["Hq"]
        return {"bytes": 2 * cell * keys + rows * ((4 if case["qd"] == "f32" else 2) + 2) * D,
                "flops": 4.0 * D * case["Hq"] * pairs}
    # evict: each weight once; the positions' held part once; each moved row read and written once. Every key
    # outside the sinks and the recent ones is as likely to stay as any other.
    weights = moves = 0
    for n in spread(case):
        if n > case["budget"]:
            weights += n
            mid, free = n - case["sink"] - case["recent"], case["budget"] - case["sink"] - case["recent"]
            over = n - case["budget"]
            tail = min(case["recent"], over)
            moves += tail + max(0, over - tail) * free / max(1, mid)
    return {"bytes": 8 * weights + moves * (4 * cell + 8), "flops": 2.0 * weights}


# ---- inputs ----------------------------------------------------------------------------------------


def page_tables(lens_or_cells, gen, dev):
    """Block tables over a seeded permutation of all pages; unused entries repeat a page of the pool."""
    need = [(n + PAGE - 1) // PAGE for n in lens_or_cells]
    n_pages = sum(need) + 3
    order = torch.randperm(n_pages, generator=gen, device=dev, dtype=torch.int64)
    width = max(1, max(need))
    t = torch.full((len(need), width), int(n_pages - 1), dtype=torch.int64, device=dev)
    at = 0
    for b, k in enumerate(need):
        t[b, :k] = order[at:at + k]
        at += k
    return t.to(torch.int32), n_pages


def unit_rows(shape, gen, dev):
    x = torch.randn(shape, generator=gen, device=dev)
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6)


def caches(n_cells, Hkv, kind, gen, dev):
    """K rows normalised as the QK-norm leaves them, V rows N(0, 1); as f16 tensors or as q8_0 planes."""
    out = {}
    for name in ("k", "v"):
        x = unit_rows((n_cells, Hkv, D), gen, dev) if name == "k" else torch.randn((n_cells, Hkv, D), generator=gen, device=dev)
        if kind == "f16":
            out[name] = x.half()
        else:
            blk = x.view(n_cells, Hkv, D // 32, 32)
            d = blk.abs().amax(-1) / 127.0
            out[name] = torch.round(blk / d[..., None]).to(torch.int8).view(n_cells, Hkv, D)
            out[name + "d"] = d.half()
    return out


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    lens = spread(case)
    perm = torch.randperm(len(lens), generator=gen, device=dev).tolist()
    s = dict(case=case)
    if case["op"] == "evict":
        lens = [lens[i] for i in perm]
        width = max(lens) + PAGE - 1 - (max(lens) - 1) % PAGE  # every row's table covers the longest row
        s["table"], n_pages = page_tables([width] * len(lens), gen, dev)
        s.update(caches(n_pages * PAGE, case["Hkv"], case["kind"], gen, dev))
        B = len(lens)
        s["lens"] = torch.tensor(lens, dtype=torch.int32, device=dev)
        # accumulated weights are heavy-tailed, and a part of the keys has never been attended to within f32
        acc = torch.exp(2.5 * torch.randn((B, width), generator=gen, device=dev) - 4.0)
        acc *= torch.rand((B, width), generator=gen, device=dev) > 0.1
        # the rows have been through an eviction: the first `held` keys carry recorded positions, in no order
        s["held"] = torch.clamp(s["lens"], max=case["budget"])
        s["shift"] = torch.randint(0, 50000, (B,), generator=gen, device=dev, dtype=torch.int32)
        ages = torch.rand((B, width), generator=gen, device=dev).argsort(-1)
        inside = ages.masked_fill(torch.arange(width, device=dev)[None] >= s["held"][:, None], width)
        rank = inside.argsort(-1).argsort(-1)  # a permutation of [0, held) in the first `held` entries
        s["pos"] = torch.where(rank < case["sink"], rank, rank + s["shift"][:, None]).to(torch.int32)
        s["acc"] = acc.masked_fill(torch.arange(width, device=dev)[None] >= s["lens"][:, None], 0.0).contiguous()
        if own:
            import localstack_b200 as L
            s["weights"] = L.KvWeights.from_tensors(s["acc"], s["pos"], s["held"], s["shift"])
    elif case["op"] == "prefill":
        both = [chunks(case)[i] for i in perm]
        s["table"], n_pages = page_tables([n for _, n in both], gen, dev)
        s.update(caches(n_pages * PAGE, case["Hkv"], case["kind"], gen, dev))
        i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
        starts = [0]
        for t, _ in both:
            starts.append(starts[-1] + t)
        s["start"], s["pos0"], s["lens"] = i32(starts), i32([n - t for t, n in both]), i32([n for _, n in both])
        s["max_q"], s["max_len"] = max(t for t, _ in both), max(n for _, n in both)
        # queries after the QK-norm's gain, whose spread sharpens some heads
        q = unit_rows((starts[-1], case["Hq"], D), gen, dev) * (0.5 + 2.0 * torch.rand((case["Hq"], 1), generator=gen, device=dev))
        s["q"] = q.half() if case["qd"] == "f16" else q
    else:
        lens = [lens[i] for i in perm]
        s["table"], n_pages = page_tables(lens, gen, dev)
        s.update(caches(n_pages * PAGE, case["Hkv"], case["kind"], gen, dev))
        s["lens"] = torch.tensor(lens, dtype=torch.int32, device=dev)
        s["max_len"] = max(lens)
        q = unit_rows((len(lens), case["Hq"], D), gen, dev) * (0.5 + 2.0 * torch.rand((case["Hq"], 1), generator=gen, device=dev))
        s["q"] = q.half()
        if case["op"] == "weights":
            width = s["table"].shape[1] * PAGE
            s["acc"] = torch.rand((len(lens), width), generator=gen, device=dev)
        if own:
            import localstack_b200 as L
            ws = L.DecodeWorkspace if case["op"] == "window" else L.WeightsWorkspace
            more = () if case["op"] == "window" else (s["max_len"],)
            s["ws"] = ws(len(lens), case["Hq"], case["Hkv"], *more)
    if own and case["kind"] == "q8":
        import localstack_b200 as L
        s["kq"], s["vq"] = L.Q8Cache.from_planes(s["k"], s["kd"]), L.Q8Cache.from_planes(s["v"], s["vd"])
    return s


# ---- the plain forms -------------------------------------------------------------------------------


def quantised(q):
    """The query row as q8_0 holds it (per 32 values d = amax / 127, q = round(x * (1 / d)), d kept in f16), as values."""
    x = q.float().view(*q.shape[:-1], D // 32, 32)
    d = x.abs().amax(-1, keepdim=True) / 127.0
    inv = torch.where(d != 0, 1.0 / d, torch.zeros_like(d))
    return (torch.round(x * inv) * d.half().float()).view(q.shape)


def rows_of(s, name, cells, dtype):
    """The K (or V) rows of the given cells as `dtype` values [..., Hkv, D]."""
    x = s[name][cells].to(dtype)
    if s["case"]["kind"] == "q8":
        x = x * s[name + "d"][cells].to(dtype).repeat_interleave(32, -1)
    return x


def query_of(s, dtype):
    """The query values the scores use: rounded to the K type (f16, or q8_0 blocks)."""
    return (quantised(s["q"]) if s["case"]["kind"] == "q8" and s["case"]["op"] != "prefill" else s["q"].half()).to(dtype)


def cells_of(s, pos):
    """The cells of positions pos [B, N] through the block tables."""
    page = s["table"].long().gather(1, (pos // PAGE).clamp(0, s["table"].shape[1] - 1))
    return page * PAGE + pos % PAGE


def attend(q, k, v, seen):
    """q [B, T, Hq, D], k / v [B, S, Hkv, D], seen [B, T, S]: outputs, lse and probabilities [B, Hkv, G, T, S]."""
    B, T, Hq, _ = q.shape
    Hkv = k.shape[2]
    qh = q.view(B, T, Hkv, Hq // Hkv, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, Hq // Hkv * T, D)
    x = (qh @ k.permute(0, 2, 3, 1)).view(B, Hkv, Hq // Hkv, T, -1) * SCALE
    x = x.masked_fill(~seen[:, None, None], -math.inf)
    top = x.amax(-1, keepdim=True).clamp_min(-1e30)
    p = (x - top).exp_()
    total = p.sum(-1, keepdim=True)
    lse = (total.log() + top).squeeze(-1)
    p = p / torch.where(total > 0, total, torch.ones_like(total))
    o = (p.view(B, Hkv, Hq // Hkv * T, -1) @ v.permute(0, 2, 1, 3)).view(B, Hkv, Hq // Hkv, T, D)
    lse = torch.where(total.squeeze(-1) > 0, lse, torch.full_like(lse, -math.inf))
    return o.permute(0, 3, 1, 2, 4).reshape(B, T, Hq, D), lse.permute(0, 3, 1, 2).reshape(B, T, Hq), p


def plain_window(s):
    c, lens = s["case"], s["lens"].long()[:, None]
    first = (lens - c["W"]).clamp_min(0)  # the window's first key
    n = min(c["W"], s["max_len"])
    i = torch.arange(c["sink"] + n, device=lens.device)[None]
    pos = torch.where(i < c["sink"], i, first + i - c["sink"])
    seen = torch.where(i < c["sink"], i < first, pos < lens)
    cells = cells_of(s, pos)
    v = rows_of(s, "v", cells, torch.float32)
    o, lse, _ = attend(query_of(s, torch.float32)[:, None], rows_of(s, "k", cells, torch.float32), v, seen[:, None])
    return o[:, 0].bfloat16(), lse[:, 0]


def plain_weights(s):
    lens = s["lens"].long()[:, None]
    pos = torch.arange(s["max_len"], device=lens.device)[None].expand(lens.shape[0], -1)
    seen = pos < lens
    cells = cells_of(s, pos)
    o, lse, p = attend(query_of(s, torch.float32)[:, None], rows_of(s, "k", cells, torch.float32),
                       rows_of(s, "v", cells, torch.float32), seen[:, None])
    s["acc"][:, :s["max_len"]] += p.sum((1, 2, 3))
    return o[:, 0].bfloat16(), lse[:, 0], s["acc"]


def plain_prefill(s):
    c = s["case"]
    B, Tq, S = s["lens"].shape[0], s["max_q"], s["max_len"]
    dev = s["q"].device
    starts = s["start"].long()
    t = torch.arange(Tq, device=dev)[None]
    row = (starts[:-1, None] + t).clamp_max(s["q"].shape[0] - 1)
    key = torch.arange(S, device=dev)[None, None]
    at = (s["pos0"].long()[:, None] + t)[..., None]
    seen = (key <= at) & (key < s["lens"][:, None, None]) & ((key > at - c["W"]) | (key < c["sink"]))
    cells = cells_of(s, torch.arange(S, device=dev)[None].expand(B, -1))
    # the prefill of a q8_0 cache reads its values rounded once to f16
    k = rows_of(s, "k", cells, torch.float32).half().float()
    v = rows_of(s, "v", cells, torch.float32).half().float()
    o, _, _ = attend(query_of(s, torch.float32)[row], k, v, seen)
    seq = torch.bucketize(torch.arange(s["q"].shape[0], device=dev), starts[1:], right=True)
    return o[seq, torch.arange(s["q"].shape[0], device=dev) - starts[seq]].bfloat16()


def plain_evict(s):
    c = s["case"]
    K, lens, acc = c["budget"], s["lens"].long()[:, None], s["acc"]
    B, width = acc.shape
    i = torch.arange(width, device=acc.device)[None].expand(B, -1)
    pos = torch.where(i < s["held"][:, None], s["pos"].long(), i + s["shift"][:, None])
    now = lens + s["shift"][:, None]  # tokens that each row has seen
    safe = (pos < c["sink"]) | (pos >= now - c["recent"])
    # ranked by (there, protected, weight), ties to the lower index: three stable sorts, least first
    order = acc.sort(dim=-1, descending=True, stable=True).indices
    order = order.gather(1, safe.gather(1, order).to(torch.int8).sort(dim=-1, descending=True, stable=True).indices)
    order = order.gather(1, (i < lens).gather(1, order).to(torch.int8).sort(dim=-1, descending=True, stable=True).indices)
    kept = torch.zeros_like(safe).scatter_(1, order[:, :K], True)
    over = lens > K
    hole = over & (i < K) & ~kept
    mover = over & (i >= K) & (i < lens) & kept
    cap = min(K, width - K)
    at = lambda m: torch.where(m, m.cumsum(-1) - 1, torch.full_like(i, cap))  # noqa: E731
    blank = torch.full((B, cap + 1), -1, dtype=torch.int64, device=acc.device)
    src = blank.clone().scatter_(1, at(mover), i)[:, :cap]
    dst = blank.clone().scatter_(1, at(hole), i)[:, :cap]
    live = torch.arange(cap, device=acc.device)[None] < mover.sum(-1, keepdim=True)
    # rows without a j-th move copy their cell K, which is never written, onto itself
    a = cells_of(s, torch.where(live, src, torch.full_like(src, K))).reshape(-1)
    b = cells_of(s, torch.where(live, dst, torch.full_like(dst, K))).reshape(-1)
    for plane in ("k", "v", "kd", "vd"):
        if plane in s:
            s[plane][b] = s[plane][a]
    src, dst = (torch.where(live, x, torch.full_like(x, -1)).int() for x in (src, dst))
    return dict(n=mover.sum(-1).int(), src=src, dst=dst, **planes(s))


def planes(s):
    """The caches as values: q8_0 integers and their scales stay as they are held."""
    return {n: s[n] for n in ("k", "v", "kd", "vd") if n in s}


PLAIN = dict(window=plain_window, weights=plain_weights, prefill=plain_prefill, evict=plain_evict)


# ---- the framework's calls -------------------------------------------------------------------------


def own_run(s):
    import localstack_b200 as L

    c = s["case"]
    q8 = c["kind"] == "q8"
    kv = (s["kq"], s["vq"]) if q8 else (s["k"], s["v"])
    if c["op"] == "window":
        f = L.attn_decode_window_q8 if q8 else L.attn_decode_window
        return f(*kv, s["q"], s["table"], s["lens"], c["W"], c["sink"], max_seq_len=s["max_len"], out_dtype=torch.bfloat16,
                 want_lse=True, workspace=s["ws"])
    if c["op"] == "weights":
        f = L.attn_decode_weights_q8 if q8 else L.attn_decode_weights
        out, lse = f(*kv, s["q"], s["table"], s["lens"], s["acc"], max_seq_len=s["max_len"], out_dtype=torch.bfloat16,
                     want_lse=True, workspace=s["ws"])
        return out, lse, s["acc"]
    if c["op"] == "prefill":
        f = L.attn_prefill_window_q8 if q8 else L.attn_prefill_window
        return f(*kv, s["q"], s["start"], s["pos0"], s["lens"], s["table"], s["max_q"], c["W"], c["sink"],
                 out_dtype=torch.bfloat16)
    moves = s["weights"].select(s["lens"], c["budget"], c["sink"], c["recent"])
    (L.kv_move_q8 if q8 else L.kv_move)(*kv, s["table"], moves)
    return dict(n=moves.n, src=moves.src, dst=moves.dst, **planes(s))


def run(state):
    return own_run(state) if own else PLAIN[state["case"]["op"]](state)


# ---- in 64 bits ------------------------------------------------------------------------------------


def exact_rows(q, k, v, seen):
    """One sequence in f64: q [T, Hq, D], k / v [S, Hkv, D], seen [T, S]."""
    T, Hq, _ = q.shape
    G = Hq // k.shape[1]
    o = torch.zeros((T, Hq, D), dtype=torch.float64, device=q.device)
    lse = torch.full((T, Hq), -math.inf, dtype=torch.float64, device=q.device)
    w = torch.zeros(k.shape[0], dtype=torch.float64, device=q.device)
    some = seen.any(1)
    for h in range(Hq):
        x = (q[:, h] @ k[:, h // G].T) / math.sqrt(D)
        x[~seen] = -math.inf
        l = torch.logsumexp(x, 1)
        p = torch.exp(x - torch.where(some, l, torch.zeros_like(l))[:, None])
        o[:, h] = p @ v[:, h // G]
        lse[:, h] = l
        w += p.sum(0)
    return o, lse, w


def exact(case, seed):
    if case["op"] == "evict":
        return None  # whole numbers and moved rows: equal or not
    s = prepare(case, seed)
    out, lses = [], []
    acc = s["acc"].double() if case["op"] == "weights" else None
    q = query_of(s, torch.float64)
    starts = s["start"].tolist() if case["op"] == "prefill" else None
    for b, n in enumerate(s["lens"].tolist()):
        page = s["table"][b].long()
        pos = torch.arange(n, device=q.device)
        if case["op"] == "prefill":
            rows = slice(starts[b], starts[b + 1])
            at = int(s["pos0"][b]) + torch.arange(starts[b + 1] - starts[b], device=q.device)[:, None]
        else:
            rows, at = slice(b, b + 1), torch.full((1, 1), n - 1, device=q.device)
        seen = (pos[None] <= at) & (pos[None] < n)
        if case["op"] != "weights":
            seen &= (at - pos[None] < case["W"]) | (pos[None] < case["sink"])
        cells = page[pos // PAGE] * PAGE + pos % PAGE
        k, v = rows_of(s, "k", cells, torch.float64), rows_of(s, "v", cells, torch.float64)
        if case["op"] == "prefill" and case["kind"] == "q8":
            k, v = k.half().double(), v.half().double()
        o, lse, w = exact_rows(q[rows], k, v, seen)
        out.append(o)
        lses.append(lse)
        if acc is not None:
            acc[b, :n] += w
    if case["op"] == "prefill":
        return torch.cat(out)
    return (torch.cat(out), torch.cat(lses)) + ((acc,) if acc is not None else ())
