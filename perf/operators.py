"""Cases, plain forms and exact values of the streaming-attention operators.

Operators: attention with a sliding window and visible first tokens over contiguous
K/V ("window") and over a paged cache ("paged"), attention of one new token over a
paged cache ("decode"), and the cache's own page work: appending tokens ("append"),
forking sequences with copy-on-write ("branch") and compacting the pool ("compact").

`run` computes an operator in elementary torch operations (`own` false) or through
the framework's calls (`own` true); `exact` computes it in 64 bits from the definition.
Lengths are drawn from the case (its "shape"), values from the seed.
"""

import math
import os
import sys

import numpy as np
import torch

own = False

D = 128  # head dimension throughout the framework's attention
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "e4m3": torch.float8_e4m3fn}
ALL = 1 << 30  # a window that no sequence leaves


def listed():
    return [
        # One short prompt through a small grouped-head layer: a call whose latency counts.
        dict(name="window_short", op="window", seqs=1, tokens=333, spread=0.0, past=0, heads=8, kv_heads=2,
             window=128, sinks=4, chunk=1, dtype="bf16", shape=1),
        # A batch of prompts of very different lengths, encoded together.
        dict(name="window_prompts", op="window", seqs=11, tokens=500, spread=0.8, past=0, heads=32, kv_heads=8,
             window=1024, sinks=4, chunk=1, dtype="fp16", shape=2),
        # One long document, most of it outside the window of its last tokens.
        dict(name="window_long", op="window", seqs=1, tokens=8192, spread=0.0, past=0, heads=32, kv_heads=8,
             window=4096, sinks=16, chunk=1, dtype="bf16", shape=3),
        # The next 720p latent frame (45 x 80 tokens) of a streamed video: it sees the prompt prefix,
        # itself and the three frames before it, out of a cache that holds five.
        dict(name="paged_frame", op="paged", seqs=1, tokens=3600, spread=0.0, past=509 + 5 * 3600, heads=32,
             kv_heads=32, window=4 * 3600, sinks=509, chunk=3600, page=64, dtype="bf16", shape=4),
        # Follow-up questions: short chunks of new tokens against longer histories.
        dict(name="paged_followup", op="paged", seqs=6, tokens=90, spread=0.5, past=2900, heads=32, kv_heads=8,
             window=ALL, sinks=0, chunk=1, page=16, dtype="bf16", shape=5),
        # One user, one token.
        dict(name="decode_one", op="decode", seqs=1, tokens=701, spread=0.0, heads=32, kv_heads=8, window=ALL,
             sinks=0, page=16, dtype="bf16", cache="bf16", shape=6),
        # A serving batch of ragged conversations under a sliding window with sinks, out of an 8-bit cache.
        dict(name="decode_batch_e4m3", op="decode", seqs=96, tokens=3500, spread=0.7, heads=32, kv_heads=8,
             window=4096, sinks=64, page=32, dtype="bf16", cache="e4m3", shape=8),
        # Two very long contexts: too few rows to fill the card without splitting their length.
        dict(name="decode_long", op="decode", seqs=2, tokens=150001, spread=0.1, heads=32, kv_heads=8, window=ALL,
             sinks=0, page=128, dtype="bf16", cache="bf16", shape=9),
        # One decoded token of each of 200 sequences goes into the cache (and is taken back).
        dict(name="append_step", op="append", seqs=200, tokens=1, spread=0.0, past=700, kv_heads=8, page=16,
             dtype="bf16", cache="bf16", shape=10),
        # Prompts go into an 8-bit cache, with the rounding that this takes.
        dict(name="append_prompts_e4m3", op="append", seqs=5, tokens=6000, spread=0.5, past=40, kv_heads=8, page=64,
             dtype="bf16", cache="e4m3", shape=11),
        # Eight continuations of each of 16 prompts take their first own token: shared last pages are copied.
        dict(name="branch", op="branch", parents=16, children=8, past=1500, spread=0.3, kv_heads=8, layers=8, page=16,
             dtype="bf16", cache="bf16", shape=12),
        # Sequences ended all over the pool: what lives moves to its front, in every layer.
        dict(name="compact", op="compact", seqs=150, tokens=1800, spread=0.5, kv_heads=8, layers=4, page=32,
             dtype="bf16", cache="bf16", shape=13),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["window", "window", "paged", "paged", "decode", "decode", "decode", "append", "branch", "compact"])
    case = dict(op=op, shape=rng.randrange(1 << 20), dtype=rng.choice(["bf16", "bf16", "fp16"]),
                spread=round(rng.choice([0.0, rng.uniform(0.1, 0.9)]), 3))
    kv = rng.choice([1, 2, 4, 8, 8, 16])
    if op == "window":
        case |= dict(kv_heads=kv, heads=kv * rng.choice([1, 2, 3, 4, 6, 8] if kv <= 4 else [1, 2, 4] if kv == 8 else [1, 2]))
        seqs = _log(rng, 1, 20)
        most = int(min(7000, 42000 / math.sqrt(case["heads"])))
        case |= dict(seqs=seqs, tokens=_log(rng, 2, max(3, most // seqs)), past=rng.choice([0, 0, _log(rng, 1, 900)]),
                     window=rng.choice([ALL, _log(rng, 16, 5000)]), sinks=rng.choice([0, rng.randrange(1, 9), _log(rng, 8, 700)]),
                     chunk=rng.choice([1, 1, 1, _log(rng, 2, 1500)]))
    elif op == "paged":
        kv = rng.choice([kv, 32])
        case |= dict(kv_heads=kv, heads=kv * rng.choice([1, 2, 4] if kv <= 8 else [1, 2] if kv <= 16 else [1]))
        seqs = _log(rng, 1, 6)
        case |= dict(seqs=seqs, tokens=_log(rng, 1, 4000 // seqs), past=_log(rng, 8, 16000 // seqs),
                     window=rng.choice([ALL, _log(rng, 16, 9000)]), sinks=rng.choice([0, rng.randrange(1, 9), _log(rng, 8, 700)]),
                     chunk=rng.choice([1, 1, _log(rng, 2, 1500)]), page=rng.choice([16, 32, 64, 128]))
    elif op == "decode":
        kv = min(kv, 8)
        seqs = _log(rng, 1, 150)
        case |= dict(kv_heads=kv, heads=kv * rng.choice([1, 2, 3, 4, 6, 8, 16]), seqs=seqs,
                     tokens=_log(rng, 1, 240000 // seqs), window=rng.choice([ALL, ALL, _log(rng, 16, 9000)]),
                     sinks=rng.choice([0, rng.randrange(1, 9), _log(rng, 8, 700)]), page=rng.choice([16, 32, 64, 128]),
                     cache=rng.choice(["e4m3", case["dtype"]]))
    elif op == "append":
        case |= dict(kv_heads=kv, seqs=_log(rng, 1, 300), page=rng.choice([16, 32, 64, 128]), cache=rng.choice(["e4m3", case["dtype"]]))
        case |= dict(tokens=rng.choice([1, _log(rng, 1, 30000 // case["seqs"])]), past=_log(rng, 1, 60000 // case["seqs"]))
    elif op == "branch":
        parents = _log(rng, 1, 24)
        case |= dict(kv_heads=kv, parents=parents, children=_log(rng, 1, 8), past=_log(rng, 1, 20000 // parents),
                     layers=rng.choice([1, 2, 4]), page=rng.choice([16, 32, 64, 128]), cache=case["dtype"])
    else:
        seqs = _log(rng, 2, 200)
        case |= dict(kv_heads=min(kv, 8), seqs=seqs, tokens=_log(rng, 4, 200000 // seqs), layers=rng.choice([1, 2, 4]),
                     page=rng.choice([16, 32, 64, 128]), cache=case["dtype"])
    return case


# ------------------------------------------------------------------------------------ shapes

def lengths(case, count, mean, salt=0):
    """`count` lengths around `mean`, the same for every seed."""
    r = np.random.RandomState((case["shape"] * 7919 + salt) % (1 << 31))
    f = np.exp(case["spread"] * r.randn(count) - 0.5 * case["spread"] ** 2)
    return np.clip(np.round(mean * f), 1, 4 * mean + 1).astype(np.int64)


def pages_of(tokens, page):
    return -(-tokens // page)


def new_tokens(case):
    if case["tokens"] == 1:
        return np.ones(case["seqs"], np.int64)
    return lengths(case, case["seqs"], case["tokens"], 1)


def visible_ends(case, lq, lk):
    """For each of lq queries right-aligned to lk keys: (first windowed key, one past the last key, sinks seen)."""
    p = lk - lq + np.arange(lq)
    last = p.copy()
    if case.get("chunk", 1) > 1:
        c, s = case["chunk"], case["sinks"]
        last = np.where(p < s, s - 1, s + ((p - s) // c + 1) * c - 1)
    end = np.where(p < 0, 0, np.minimum(last + 1, lk))
    lo = np.minimum(np.maximum(last - case["window"] + 1, 0), end)
    return lo, end, np.minimum(np.minimum(case["sinks"], lo), end)


def work(case):
    op = case["op"]
    if op in ("window", "paged", "decode"):
        if op == "decode":
            lk = lengths(case, case["seqs"], case["tokens"])
            lq = np.ones_like(lk)
            size = 1 if case["cache"] == "e4m3" else 2
        else:
            lq = lengths(case, case["seqs"], case["tokens"])
            lk = lq + case["past"]
            size = 2
        pairs = keys = 0
        for a, b in zip(lq, lk):
            lo, end, s = visible_ends(case, int(a), int(b))
            pairs += int((end - lo + s).sum())
            seen = np.zeros(int(b) + 1, np.int64)  # each key that any query sees is read once
            np.add.at(seen, lo, 1)
            np.add.at(seen, end, -1)
            n = np.cumsum(seen)[:-1] > 0
            n[: int(s.max())] = True
            keys += int(n.sum())
        return {"flops": 4.0 * D * case["heads"] * pairs,
                "bytes": 4.0 * D * case["heads"] * float(lq.sum()) + 2.0 * size * D * case["kv_heads"] * keys}
    row = case["kv_heads"] * D
    if op == "append":
        size = 1 if case["cache"] == "e4m3" else 2
        return {"bytes": 2.0 * row * float(new_tokens(case).sum()) * (2 + size), "flops": 0.0}
    if op == "branch":
        past = lengths(case, case["parents"], case["past"])
        copied = float((past % case["page"]).sum()) * case["children"]
        token = case["parents"] * case["children"]
        return {"bytes": 2.0 * 2 * row * (2 * copied * case["layers"] + 2 * token)
                + 2.0 * 4 * case["children"] * float(pages_of(past, case["page"]).sum()), "flops": 0.0}
    table, live, total, _ = compact_layout(case)
    moved = int((live >= live.size).sum())
    return {"bytes": 2.0 * 2 * 2 * row * case["page"] * moved * case["layers"] + 8.0 * table.size, "flops": 0.0}


def compact_layout(case):
    """A pool after half of its sequences ended: (table, the pages that live, pages in the pool, lengths)."""
    lens = lengths(case, case["seqs"], case["tokens"])
    need = pages_of(lens, case["page"])
    r = np.random.RandomState(case["shape"] + 17)
    total = int(need.sum())
    order = r.permutation(total)
    table = np.full((case["seqs"], int(need.max()) + 1), -1, np.int64)
    keep = r.permutation(case["seqs"])[: max(1, case["seqs"] // 2)]
    at = np.concatenate([[0], np.cumsum(need)])
    for i in keep:
        table[i, : need[i]] = order[at[i]: at[i + 1]]
    kept = np.zeros_like(lens)
    kept[keep] = lens[keep]
    return table, np.sort(table[table >= 0]), total, kept


# ------------------------------------------------------------------------------------ inputs

def _i32(x):
    return torch.from_numpy(np.ascontiguousarray(x).astype(np.int32)).cuda()


def _starts(lens):
    return _i32(np.concatenate([[0], np.cumsum(lens)]))


def _pool(case, pages, layers, g):
    """K and V pools [layers, pages, kv heads, page, 128]: keys with per-channel offsets, as projected keys have
    them; 8-bit pools hold the rows over their head's scale."""
    shape = (layers, pages, case["kv_heads"], case["page"], D)
    off = torch.randn(shape[2], 1, D, device="cuda", generator=g)
    dt = DTYPES[case["cache"]]
    if dt is torch.float8_e4m3fn:
        ks, vs = (torch.full((layers, shape[2]), x, device="cuda") * (1 + torch.rand(layers, shape[2], device="cuda", generator=g))
                  for x in (0.012, 0.009))
    else:
        ks = vs = None
    pools = []
    for scale, shift in ((ks, off), (vs, 0.0)):
        out = torch.empty(shape, device="cuda", dtype=dt)
        for i in range(layers):
            x = torch.randn(shape[1:], device="cuda", dtype=torch.float16, generator=g).float() + shift
            if scale is not None:
                x = (x / scale[i].view(1, -1, 1, 1)).clamp(-448, 448)
            out[i] = x.to(dt)
        pools.append(out)
    return pools[0], pools[1], ks, vs


def _cache(case, lens, layers, g, extra_pages, slots=None, extra_tokens=0):
    """A cache whose sequences' pages lie scattered over the pool."""
    need = pages_of(lens, case["page"])
    total = int(need.sum()) + extra_pages
    order = np.random.RandomState(case["shape"] + 29).permutation(total)
    slots = slots or len(lens)
    table = np.full((slots, int(pages_of(int(lens.max()) + extra_tokens, case["page"])) + 1), -1, np.int64)
    at = np.concatenate([[0], np.cumsum(need)])
    for i in range(len(lens)):
        table[i, : need[i]] = order[at[i]: at[i + 1]]
    refs = np.zeros(total, np.int64)
    refs[order[: at[-1]]] = 1
    all_lens = np.zeros(slots, np.int64)
    all_lens[: len(lens)] = lens
    k, v, ks, vs = _pool(case, total, layers, g)
    return dict(k=k, v=v, table=_i32(table), lens=_i32(all_lens), refs=_i32(refs),
                status=torch.zeros(1, device="cuda", dtype=torch.int32), k_scale=ks, v_scale=vs)


def _rows(case, tokens, heads, g, offset=False):
    x = torch.randn(tokens, heads, D, device="cuda", generator=g)
    if offset:
        x += torch.randn(1, heads, D, device="cuda", generator=g)
    return x.to(DTYPES[case["dtype"]])


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed * 1000003 + case["shape"])
    op = case["op"]
    s = {"case": case}
    if op == "window":
        lq = lengths(case, case["seqs"], case["tokens"])
        lk = lq + case["past"]
        s |= dict(q=_rows(case, int(lq.sum()), case["heads"], g), k=_rows(case, int(lk.sum()), case["kv_heads"], g, True),
                  v=_rows(case, int(lk.sum()), case["kv_heads"], g), q_starts=_starts(lq), k_starts=_starts(lk))
    elif op == "paged":
        lq = lengths(case, case["seqs"], case["tokens"])
        s["cache"] = _cache(case | {"cache": case["dtype"]}, lq + case["past"], 1, g, 7)
        s |= dict(q=_rows(case, int(lq.sum()), case["heads"], g), q_starts=_starts(lq),
                  slots=_i32(np.arange(case["seqs"])))
    elif op == "decode":
        lens = lengths(case, case["seqs"], case["tokens"])
        s["cache"] = _cache(case, lens, 1, g, 5)
        s |= dict(q=_rows(case, case["seqs"], case["heads"], g),
                  slots=_i32(np.random.RandomState(case["shape"]).permutation(case["seqs"])))
    elif op == "append":
        n = new_tokens(case)
        past = lengths(case, case["seqs"], case["past"])
        extra = int((pages_of(past + n, case["page"]) - pages_of(past, case["page"])).sum()) + 3
        s["cache"] = _cache(case, past, 1, g, extra, extra_tokens=int(n.max()))
        s |= dict(k=_rows(case, int(n.sum()), case["kv_heads"], g, True), v=_rows(case, int(n.sum()), case["kv_heads"], g),
                  slots=_i32(np.arange(case["seqs"])[::-1]), starts=None if case["tokens"] == 1 else _starts(n[::-1]),
                  before=_i32(past[::-1]), most=int(n.max()))
    elif op == "branch":
        past = lengths(case, case["parents"], case["past"])
        kids = case["parents"] * case["children"]
        s["cache"] = _cache(case, past, case["layers"], g, kids + 3, case["parents"] + kids, 1)
        s |= dict(k=_rows(case, kids, case["kv_heads"], g, True), v=_rows(case, kids, case["kv_heads"], g),
                  src=_i32(np.repeat(np.arange(case["parents"]), case["children"])),
                  dst=_i32(case["parents"] + np.arange(kids)), most=1)
    else:
        table, live, total, lens = compact_layout(case)
        refs = np.zeros(total, np.int64)
        refs[live] = 1
        k, v, ks, vs = _pool(case, total, case["layers"], g)
        s["cache"] = dict(k=k, v=v, table=_i32(table), lens=_i32(lens), refs=_i32(refs),
                          status=torch.zeros(1, device="cuda", dtype=torch.int32), k_scale=ks, v_scale=vs)
        s |= dict(table=_i32(table), refs=_i32(refs))
    return s


# ------------------------------------------------------------------------------------ one pass

def run(state):
    return (_run_own if own else _run_plain)(state)


def _h3b():
    if "h3b" not in sys.modules:
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "x-minimaxh3_b200"))
    import h3b
    return h3b


def _run_own(s):
    h3b, case = _h3b(), s["case"]
    op = case["op"]
    if op == "window":
        return h3b.window_attention(s["q"], s["k"], s["v"], window=case["window"], sinks=case["sinks"],
                                    chunk=case["chunk"], query_starts=s["q_starts"], key_starts=s["k_starts"])
    cache = h3b.PagedKVCache(**s["cache"])
    if op == "paged":
        return h3b.paged_window_attention(s["q"], cache, s["slots"], window=case["window"], sinks=case["sinks"],
                                          chunk=case["chunk"], query_starts=s["q_starts"])
    if op == "decode":
        return h3b.decode_attention(s["q"], cache, s["slots"], window=case["window"], sinks=case["sinks"])
    if op == "append":  # taken back afterwards, as a rejected draft is, so that every pass appends to the same cache
        cache.append(s["slots"], s["k"], s["v"], starts=s["starts"])
        cache.truncate(s["slots"], s["before"])
    elif op == "branch":
        cache.fork(s["src"], s["dst"])
        cache.append(s["dst"], s["k"], s["v"])
        cache.free(s["dst"])
    else:  # the scattered tables are put back first: the pages that they name still hold their rows
        cache.table.copy_(s["table"])
        cache.refs.copy_(s["refs"])
        cache.compact()
    return cache.k, cache.v, cache.table, cache.lens, cache.refs


# ---- plain forms

def _masked_softmax_product(q, k, v, see, scale):
    """q [..., Lq, D], k, v [..., Lk, D] in fp32, see [..., Lq, Lk]: rows that see nothing give 0."""
    w = torch.matmul(q, k.transpose(-1, -2)).mul_(scale).masked_fill_(~see, -math.inf)
    w = w.sub_(w.amax(-1, keepdim=True).clamp_min(torch.finfo(torch.float32).min)).exp_()
    total = w.sum(-1, keepdim=True)
    return torch.matmul(w, v) / torch.where(total > 0, total, 1.0)


def _see(case, p, j, j_len):
    """Whether the query at position p sees key j of a sequence of j_len keys."""
    last = p
    c, s = case.get("chunk", 1), case["sinks"]
    if c > 1:
        last = torch.where(p < s, s - 1, s + (torch.div(p - s, c, rounding_mode="floor") + 1) * c - 1)
    return (p >= 0) & (j < j_len) & (j <= last) & ((last - j < case["window"]) | (j < s))


def _segments(starts, n):
    at = torch.arange(n, device=starts.device, dtype=torch.int32)
    seg = torch.searchsorted(starts[1:].contiguous(), at, right=True)
    return seg, at - starts[seg]


def _plain_varlen(case, q, k, v, q_seg, q_at, q_len, k_seg, k_at, k_len):
    """q [Tq, Hq, D], k / v [Tk, Hkv, D]; segment, place in it and lengths of every row."""
    group = case["heads"] // case["kv_heads"]
    see = (q_seg[:, None] == k_seg[None]) & _see(case, (k_len[q_seg] - q_len[q_seg] + q_at)[:, None], k_at[None],
                                                 k_len[q_seg][:, None])
    qh = q.float().permute(1, 0, 2).reshape(case["kv_heads"], group, -1, D)
    kh = k.float().permute(1, 0, 2)[:, None]
    vh = v.float().permute(1, 0, 2)[:, None]
    o = _masked_softmax_product(qh, kh, vh, see, 1 / math.sqrt(D))
    return o.reshape(case["heads"], -1, D).permute(1, 0, 2).to(q.dtype)


def _rows_of_pages(pool, scale, pages):
    """[n, kv heads, tokens, D] in fp32 of layer 0's pages [n, w] (-1: any page, to be masked)."""
    x = pool[0].view(torch.uint8 if pool.element_size() == 1 else torch.int16)[pages.clamp_min(0).long()]
    x = x.view(pool.dtype).permute(0, 2, 1, 3, 4).float()
    x = x.reshape(x.shape[0], x.shape[1], -1, D)
    return x if scale is None else x * scale[0].view(1, -1, 1, 1)


def _allocate(c, slots, count, most):
    """Pages for count[i] more tokens of slot i: the lowest free ones, a copy of a shared last page first."""
    page, table, lens, refs = c["k"].shape[3], c["table"], c["lens"], c["refs"]
    old = lens[slots.long()]
    new = old + count
    have, need = (old + page - 1) // page, (new + page - 1) // page
    rows = torch.arange(slots.numel(), device=slots.device)
    row = table[slots.long()]
    tail = row[rows, (have - 1).clamp_min(0).long()].clamp_min(0)
    copies = (old % page != 0) & (count > 0) & (refs[tail.long()] > 1)
    asked = need - have + copies
    first = torch.cumsum(asked, 0) - asked
    free = torch.argsort((refs > 0).to(torch.int8), stable=True).to(torch.int32)
    r = torch.arange(most // page + 2, device=slots.device)
    given = free[(first[:, None] + r).clamp_max(free.numel() - 1)]
    column = (have - copies.int())[:, None] + r
    takes = r < asked[:, None]
    row.scatter_(1, torch.where(takes, column, row.shape[1] - 1).long(),
                 torch.where(takes, given, row[:, -1:]))
    # rows that take no page wrote their own last column back
    refs.scatter_add_(0, tail.long(), -copies.to(torch.int32))
    refs.scatter_add_(0, torch.where(takes, given, 0).reshape(-1).long(), takes.reshape(-1).to(torch.int32))
    table[slots.long()] = row
    lens[slots.long()] = new
    return old, tail, torch.where(copies, given[:, 0], tail)


def _put(pool, scale, where, at, x):
    if scale is not None:
        x = (x.float() / scale[0][:, None]).clamp(-448, 448)
    raw = torch.uint8 if pool.element_size() == 1 else torch.int16
    pool[0].view(raw)[where, :, at] = x.to(pool.dtype).view(raw)


def _move(pool, src, dst, part=True):
    """Pages src over pages dst in every layer, the rows of `part`."""
    pool[:, dst] = torch.where(part, pool[:, src], pool[:, dst]) if part is not True else pool[:, src]


def _write(c, slots, old, starts, k, v):
    page = c["k"].shape[3]
    seg, at = _segments(starts, k.shape[0])
    pos = old[seg] + at
    where = c["table"][slots[seg].long(), (pos // page).long()].long()
    _put(c["k"], c["k_scale"], where, (pos % page).long(), k)
    _put(c["v"], c["v_scale"], where, (pos % page).long(), v)


def _release(c, slots, keep):
    """Slot i keeps its first keep[i] tokens."""
    page, table = c["k"].shape[3], c["table"]
    row = table[slots.long()]
    kept = (keep + page - 1) // page
    goes = (row >= 0) & (torch.arange(row.shape[1], device=row.device) >= kept[:, None])
    c["refs"].scatter_add_(0, row.clamp_min(0).reshape(-1).long(), -goes.reshape(-1).to(torch.int32))
    table[slots.long()] = torch.where(goes, -1, row)
    c["lens"][slots.long()] = keep


def _run_plain(s):
    case = s["case"]
    op = case["op"]
    if op == "window":
        n, m = s["q"].shape[0], s["k"].shape[0]
        return _plain_varlen(case, s["q"], s["k"], s["v"], *_segments(s["q_starts"], n), s["q_starts"].diff(),
                             *_segments(s["k_starts"], m), s["k_starts"].diff())
    c = s["cache"]
    page = c["k"].shape[3]
    if op in ("paged", "decode"):
        pages = c["table"][s["slots"].long()]
        lens = c["lens"][s["slots"].long()]
        k, v = _rows_of_pages(c["k"], c["k_scale"], pages), _rows_of_pages(c["v"], c["v_scale"], pages)
        if op == "paged":
            n, kv, w, _ = k.shape
            seg = torch.arange(n, device=k.device).repeat_interleave(w)
            at = torch.arange(w, device=k.device, dtype=torch.int32).repeat(n)
            return _plain_varlen(case, s["q"], k.transpose(1, 2).reshape(n * w, kv, D), v.transpose(1, 2).reshape(n * w, kv, D),
                                 *_segments(s["q_starts"], s["q"].shape[0]), s["q_starts"].diff(), seg, at, lens)
        j = torch.arange(k.shape[2], device=k.device)
        see = _see(case, (lens - 1)[:, None], j[None], lens[:, None])[:, None, None]
        q = s["q"].float().view(s["q"].shape[0], case["kv_heads"], -1, D)
        return _masked_softmax_product(q, k, v, see, 1 / math.sqrt(D)).reshape(s["q"].shape).to(s["q"].dtype)
    if op == "append":
        starts = s["starts"] if s["starts"] is not None else torch.arange(s["slots"].numel() + 1, device="cuda", dtype=torch.int32)
        old, _, _ = _allocate(c, s["slots"], starts.diff(), s["most"])
        _write(c, s["slots"], old, starts, s["k"], s["v"])
        _release(c, s["slots"], s["before"])
    elif op == "branch":
        src, dst = s["src"].long(), s["dst"].long()
        row = c["table"][src]
        c["table"][dst] = row
        c["lens"][dst] = c["lens"][src]
        c["refs"].scatter_add_(0, row.clamp_min(0).reshape(-1).long(), (row >= 0).reshape(-1).to(torch.int32))
        starts = torch.arange(s["dst"].numel() + 1, device="cuda", dtype=torch.int32)
        old, tail, to = _allocate(c, s["dst"], starts.diff(), s["most"])
        # the rows that the shared page holds; a sequence without a copy writes its own page back to itself
        part = (torch.arange(page, device="cuda") < (old % page)[:, None])[:, None, :, None]
        _move(c["k"], tail.long(), to.long(), part)
        _move(c["v"], tail.long(), to.long(), part)
        _write(c, s["dst"], old, starts, s["k"], s["v"])
        _release(c, s["dst"], torch.zeros_like(old))
    else:
        c["table"].copy_(s["table"])
        c["refs"].copy_(s["refs"])
        used = c["refs"] > 0
        n = used.sum()
        at = torch.arange(used.numel(), device="cuda")
        # the i-th used page at or after n goes to the i-th free page before it
        moves, holes = used & (at >= n), ~used & (at < n)
        count = int(moves.sum())
        src = torch.argsort((~moves).to(torch.int8), stable=True)
        dst = torch.argsort((~holes).to(torch.int8), stable=True)
        src, dst = src[:count], dst[:count]
        _move(c["k"], src, dst)
        _move(c["v"], src, dst)
        to = at.clone()
        to[src] = dst
        c["table"].copy_(torch.where(c["table"] >= 0, to[c["table"].clamp_min(0).long()].to(torch.int32), c["table"]))
        c["refs"][dst] = c["refs"][src]
        c["refs"][src] = 0
    return c["k"], c["v"], c["table"], c["lens"], c["refs"]


# ------------------------------------------------------------------------------------ from the definition, in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op in ("window", "paged", "decode"):
        return _exact_attention(case, s)
    return _exact_pages(case, s)


def _exact_attention(case, s):
    q, op = s["q"], case["op"]
    group = case["heads"] // case["kv_heads"]
    out = torch.zeros(q.shape, device="cuda", dtype=torch.float64)
    if op == "decode":
        at_q = np.arange(case["seqs"] + 1)
    else:
        at_q = s["q_starts"].cpu().numpy()
    for i in range(case["seqs"]):
        a, b = int(at_q[i]), int(at_q[i + 1])
        if op == "window":
            lo, hi = (int(x) for x in s["k_starts"][i: i + 2].cpu())
            k, v = s["k"][lo:hi].double().transpose(0, 1), s["v"][lo:hi].double().transpose(0, 1)
        else:
            c = s["cache"]
            slot = int(s["slots"][i])
            n = int(c["lens"][slot])
            pages = c["table"][slot, : pages_of(n, case["page"])].cpu().tolist()
            k, v = (torch.cat([x[0, p].float() for p in pages], 1)[:, :n].double() for x in (c["k"], c["v"]))
            if c["k_scale"] is not None:
                k, v = k * c["k_scale"][0].double().view(-1, 1, 1), v * c["v_scale"][0].double().view(-1, 1, 1)
        lq, lk = b - a, k.shape[1]
        lo, end, sinks = (torch.from_numpy(x).cuda() for x in visible_ends(case, lq, lk))
        for r in range(0, lq, 1024):
            j = torch.arange(lk, device="cuda")
            rows = slice(r, min(lq, r + 1024))
            see = (j < end[rows, None]) & ((j >= lo[rows, None]) | (j < sinks[rows, None]))
            for h in range(case["heads"]):
                w = q[a:b, h][rows].double() @ k[h // group].T / math.sqrt(D)
                w = torch.where(see, w, -math.inf)
                top = w.max(-1, keepdim=True).values
                w = torch.where(see, torch.exp(w - torch.where(torch.isfinite(top), top, 0.0)), 0.0)
                total = w.sum(-1, keepdim=True)
                o = (w @ v[h // group]) / torch.where(total > 0, total, 1.0)
                out[a + r: a + r + o.shape[0], h] = o
    return out


def _exact_pages(case, s):
    """The page work step by step on the host, and the rows that it moves."""
    c, op, page = s["cache"], case["op"], case["page"]
    table, lens, refs = (c[x].cpu().numpy().astype(np.int64) for x in ("table", "lens", "refs"))
    k, v = c["k"], c["v"]
    if c["k_scale"] is not None:
        k, v = k.float(), v.float()  # the codes' values; appended rows are put in below as they are before rounding

    def take():
        return int(np.flatnonzero(refs == 0)[0])

    def append(slots, counts, rows_k, rows_v):
        at = 0
        shared = refs.copy()
        dropped = []
        for slot, n in zip(slots, counts):
            if lens[slot] % page and n and shared[table[slot, lens[slot] // page]] > 1:
                old = int(table[slot, lens[slot] // page])
                new = take()
                refs[new] = 1
                dropped.append(old)
                table[slot, lens[slot] // page] = new
                part = int(lens[slot] % page)
                for pool in (k, v):
                    pool[:, new, :, :part] = pool[:, old, :, :part]
            for col in range(int(pages_of(lens[slot], page)), int(pages_of(lens[slot] + n, page))):
                table[slot, col] = take()
                refs[table[slot, col]] = 1
        for old in dropped:
            refs[old] -= 1
        for slot, n in zip(slots, counts):
            pos = lens[slot] + np.arange(n)
            p = torch.from_numpy(table[slot, pos // page]).cuda()
            o = torch.from_numpy(pos % page).cuda()
            for pool, rows, scale in ((k, rows_k, c["k_scale"]), (v, rows_v, c["v_scale"])):
                x = rows[at: at + n]
                if scale is not None:
                    x = (x.double() / scale[0].double()[:, None]).clamp(-448, 448).float()
                pool[0][p, :, o] = x.to(pool.dtype)
            at += n
            lens[slot] += n

    def release(slots, keep):
        for slot, n in zip(slots, keep):
            for col in range(int(pages_of(n, page)), int(pages_of(lens[slot], page))):
                refs[table[slot, col]] -= 1
                table[slot, col] = -1
            lens[slot] = n

    if op == "append":
        slots = s["slots"].cpu().numpy()
        counts = np.ones(len(slots), np.int64) if s["starts"] is None else np.diff(s["starts"].cpu().numpy())
        append(slots, counts, s["k"], s["v"])
        release(slots, s["before"].cpu().numpy())
    elif op == "branch":
        dst = s["dst"].cpu().numpy()
        for a, b in zip(s["src"].cpu().numpy(), dst):
            table[b], lens[b] = table[a], lens[a]
            refs[table[b][table[b] >= 0]] += 1
        append(dst, np.ones(len(dst), np.int64), s["k"], s["v"])
        release(dst, np.zeros(len(dst), np.int64))
    else:
        used = np.flatnonzero(refs)
        holes = np.flatnonzero(refs[: used.size] == 0)
        for new, old in zip(holes, used[used >= used.size]):
            for pool in (k, v):
                pool[:, int(new)] = pool[:, int(old)]
            refs[new], refs[old] = refs[old], 0
            table[table == old] = new
    return k, v, *(_i32(x) for x in (table, lens, refs))
