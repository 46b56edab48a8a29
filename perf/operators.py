"""Cases of the generation operators: shared-prefix attention, sampling, and the page operations of the cache.

``own`` false computes each operator in plain torch operations in 32 bits;
``own`` true makes the calls of :mod:`mini_nccl_b200.ops.generation` that a
program generating many continuations of one prompt makes.
"""

from __future__ import annotations

import math
import random

import torch

own = False
DEV = "cuda"


# ---- cases -----------------------------------------------------------------------------


def listed():
    A, S, P = dict(op="attention"), dict(op="sample"), dict(op="pages")
    return [
        # one decode step of four continuations of a short prompt, GPT-124M heads: latency counts
        A | dict(name="decode_few", batch=4, heads=12, kv_heads=12, dim=64, page=16, prefix=300, own=17, chunk=1, idle=0),
        # one decode step of 192 rollouts of one long prompt, the 24-layer GPT's heads
        A | dict(name="decode_many", batch=192, heads=16, kv_heads=16, dim=128, page=16, prefix=8191, own=401, chunk=1, idle=3),
        # a few agents behind one very long shared document, grouped heads, ragged and empty continuations
        A | dict(name="decode_long", batch=16, heads=32, kv_heads=8, dim=128, page=64, prefix=65537, own=1000, chunk=1, idle=2),
        # questions of 1 to 300 tokens appended to one shared prompt in one pass, the 32-layer GPT's heads
        A | dict(name="chunk_ragged", batch=24, heads=32, kv_heads=32, dim=128, page=32, prefix=4001, own=411, chunk=300, idle=0),
        # the next token of one sequence, GPT vocabulary
        S | dict(name="sample_one", rows=1, vocab=50304, dtype="bfloat16", mix="topk", banned=0.0),
        # a served batch in which each row has its own settings, greedy rows among them
        S | dict(name="sample_mixed", rows=64, vocab=50304, dtype="float32", mix="mixed", banned=0.02),
        # nucleus sampling of many rollouts
        S | dict(name="sample_nucleus", rows=512, vocab=50304, dtype="bfloat16", mix="topp", banned=0.0),
        # a large odd vocabulary with min-p
        S | dict(name="sample_wide", rows=129, vocab=130003, dtype="float32", mix="minp", banned=0.01),
        # four branches of one sequence of GPT-124M: the last, part-filled page is copied in all layers
        P | dict(name="fork_few", kind="fork", layers=12, kv_heads=12, dim=64, page=16, pool=512, parents=1, count=4, tokens=1000),
        # a tree step: 128 children of 32 parents at once
        P | dict(name="fork_many", kind="fork", layers=24, kv_heads=16, dim=128, page=16, pool=640, parents=32, count=128, tokens=235),
        # the live half of a fragmented pool moved to its front
        P | dict(name="compact_half", kind="compact", layers=12, kv_heads=12, dim=64, page=16, pool=2048, parents=0, count=64, tokens=511),
        # the keys and values of a packed prompt batch written to one layer's pages
        P | dict(name="append_prompts", kind="append", layers=1, kv_heads=16, dim=128, page=32, pool=512, parents=0, count=13, tokens=1013),
    ]


def _log(rng, lo, hi):
    """A whole number, uniform over the logarithm."""
    return min(hi, max(lo, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    """One more case; none costs more than the largest listed one."""
    most = {k: max(work(c)[k] for c in listed()) for k in ("bytes", "flops")}
    while True:
        case = _draw(rng)
        if all(v <= most[k] for k, v in work(case).items()):
            return case


def _draw(rng):
    op = rng.choice(("attention", "attention", "sample", "pages"))
    if op == "sample":
        rows = _log(rng, 1, 512)
        vocab = _log(rng, 1000, min(130003, 26_000_000 // rows))
        return dict(op=op, rows=rows, vocab=vocab, dtype=rng.choice(("bfloat16", "float32")),
                    mix=rng.choice(("topk", "topp", "minp", "mixed", "none")), banned=rng.choice((0.0, 0.02, 0.5)))
    if op == "pages":
        kind = rng.choice(("fork", "compact", "append"))
        dim, kv = rng.choice((64, 128)), rng.choice((2, 3, 8, 12, 16))
        page = rng.choice((16, 32, 64))
        if kind == "append":
            count, tokens = _log(rng, 1, 24), _log(rng, 1, 600)
            return dict(op=op, kind=kind, layers=1, kv_heads=kv, dim=dim, page=page, parents=0, count=count, tokens=tokens,
                        pool=count * -(-tokens // page) + rng.randrange(1, 40))
        layers = rng.choice((1, 4, 7, 12))
        parents, count, tokens = _log(rng, 1, 24), _log(rng, 1, 64), _log(rng, 17, 400)
        if kind == "compact":
            parents = 0
        held = (parents or count) * -(-tokens // page)
        return dict(op=op, kind=kind, layers=layers, kv_heads=kv, dim=dim, page=page, parents=parents, count=count, tokens=tokens,
                    pool=held + count + rng.randrange(1, 100))
    chunk = rng.choice((1, 1, 1, _log(rng, 2, 300)))
    batch = _log(rng, 1, 192 if chunk == 1 else max(1, min(64, 3000 // chunk)))
    kv = rng.choice((2, 4, 8, 12, 16))
    group = rng.choice((1, 1, 2, 4, 8))
    if kv * group > 32:
        group = 1
    prefix = _log(rng, 33, 65537)
    rows = batch * (1 if chunk == 1 else 0.6 * chunk) * kv * group
    prefix = max(33, min(prefix, int(5e8 / rows)))  # keeps the plain form's score table to the largest listed one's
    return dict(op=op, batch=batch, heads=kv * group, kv_heads=kv, dim=rng.choice((64, 128)), page=rng.choice((8, 16, 32, 64, 128)),
                prefix=prefix, own=max(chunk, _log(rng, 1, 700)), chunk=chunk, idle=rng.choice((0, 0, 1)) if batch > 1 and chunk == 1 else 0)


def _spread(n, lo, hi, turn):
    """n whole numbers over lo..hi, alike for every seed up to their order."""
    return [lo + int((hi - lo + 1) * ((i + 1) * turn % 1.0)) for i in range(n)]


def _lengths(case):
    """(own length, new tokens) of each sequence; the idle ones hold nothing."""
    n = case["batch"] - case["idle"]
    length = _spread(n, 1, case["own"], 0.6180339887)
    new = [1] * n if case["chunk"] == 1 else [min(a, b) for a, b in zip(length, _spread(n, 1, case["chunk"], 0.7548776662))]
    return length + [0] * case["idle"], new + [1 if case["chunk"] == 1 else 0] * case["idle"]


def work(case):
    if case["op"] == "attention":
        length, new = _lengths(case)
        # every key and value once, the prefix's once for all; queries in, outputs and log-sum-exps out
        tokens = case["prefix"] + sum(length)
        n, H, D = sum(new), case["heads"], case["dim"]
        pairs = sum(t * case["prefix"] + t * max(0, m - t) + t * (t + 1) // 2 for m, t in zip(length, new) if m) \
            + sum(t * case["prefix"] for m, t in zip(length, new) if not m)
        return {"bytes": 2 * tokens * case["kv_heads"] * D * 2 + 2 * n * H * D * 2 + 4 * n * H, "flops": 4 * pairs * H * D}
    if case["op"] == "sample":
        n = case["rows"] * case["vocab"]
        # logits once; the noise of tokens that a filter drops is not needed, so it counts only where nothing is dropped
        return {"bytes": n * (2 if case["dtype"] == "bfloat16" else 4) + (4 * n if case["mix"] == "none" else 0), "flops": 4 * n}
    token = 2 * case["kv_heads"] * case["dim"] * 2 * case["layers"]
    if case["kind"] == "fork":
        part = case["tokens"] % case["page"]
        return {"bytes": token * part * (case["count"] + min(case["parents"], case["count"])) + 8 * case["count"], "flops": 0}
    if case["kind"] == "append":
        return {"bytes": 2 * token * case["count"] * case["tokens"], "flops": 0}
    live, pages = _compact_pages(case)
    moved = live * (1 - live / case["pool"])  # expected, for pages placed at random
    return {"bytes": 2 * token * case["page"] * max(1, int(moved)) + 8 * case["pool"], "flops": 0}


def _compact_pages(case):
    """(live pages, pages of each sequence): every second sequence has ended."""
    pages = [-(-t // case["page"]) for t in _spread(case["count"], 1, case["tokens"], 0.6180339887)]
    return sum(pages[::2]), pages


# ---- inputs ----------------------------------------------------------------------------


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def prepare(case, seed):
    rng = random.Random(seed)
    gen = torch.Generator(device=DEV).manual_seed(seed)

    def normal(*shape, dtype=torch.bfloat16):
        return torch.randn(*shape, generator=gen, device=DEV, dtype=dtype)

    s = dict(case)
    if case["op"] == "attention":
        length, new = _lengths(case)
        order = list(range(case["batch"]))
        rng.shuffle(order)
        length, new = [length[i] for i in order], [new[i] for i in order]
        page, D, Hk = case["page"], case["dim"], case["kv_heads"]
        n_prefix = -(-case["prefix"] // page)
        per = max(1, -(-case["own"] // page))
        need = n_prefix + sum(-(-m // page) for m in length)
        ids = list(range(need + 5))
        rng.shuffle(ids)
        s["kv"] = normal(2, len(ids), page, Hk, D)
        s["prefix_pages"] = _int32(ids[:n_prefix])
        at, table = n_prefix, []
        for m in length:
            k = -(-m // page)
            table.append(ids[at:at + k] + [-1] * (per - k))
            at += k
        s["page_table"], s["seq_lens"] = _int32(table), _int32(length)
        # queries as they leave a fused projection: one part of its rows
        C = case["heads"] * D
        s["q"] = (normal(sum(new), C + 2 * Hk * D) * 1.5)[:, :C].view(-1, case["heads"], D)
        s["q_offsets"] = None
        if case["chunk"] > 1:
            s["q_offsets"] = _int32([sum(new[:i]) for i in range(len(new) + 1)])
        s["max_q_len"] = max(new)
    elif case["op"] == "sample":
        R, V = case["rows"], case["vocab"]
        x = normal(R, V, dtype=torch.float32) * (1.5 + 2.5 * torch.rand(R, 1, generator=gen, device=DEV))
        if case["banned"]:
            x.masked_fill_(torch.rand(R, V, generator=gen, device=DEV) < case["banned"], float("-inf"))
        s["logits"] = x.to(getattr(torch, case["dtype"]))
        s["noise"] = torch.empty(R, V, device=DEV).exponential_(generator=gen).log_().neg_()

        def some(values, dtype=torch.float32):
            return torch.tensor([rng.choice(values) for _ in range(R)], dtype=dtype, device=DEV)

        mix = case["mix"]
        s["temperature"] = some((0.0, 0.7, 1.0, 1.3) if mix == "mixed" else (0.8, 1.0))
        s["top_k"] = some({"topk": (50,), "mixed": (0, 1, 40, 300)}.get(mix, (0,)), torch.int32)
        s["top_p"] = some({"topp": (0.9, 0.95), "mixed": (1.0, 0.9, 0.99)}.get(mix, (1.0,)))
        s["min_p"] = some({"minp": (0.05, 0.1), "mixed": (0.0, 0.02)}.get(mix, (0.0,)))
    else:
        page = case["page"]
        s["kv"] = normal(case["layers"], 2, case["pool"], page, case["kv_heads"], case["dim"])
        ids = list(range(case["pool"]))
        rng.shuffle(ids)
        refs = [0] * case["pool"]
        if case["kind"] == "compact":
            _, pages = _compact_pages(case)
            pages = [k if i % 2 == 0 else 0 for i, k in enumerate(pages)]
            rng.shuffle(pages)
        else:
            pages = [-(-case["tokens"] // page)] * (case["parents"] or case["count"])
        rows, at, width = [], 0, max(1, -(-case["tokens"] // page) + 1)
        for k in pages:
            rows.append(ids[at:at + k] + [-1] * (width - k))
            for p in ids[at:at + k]:
                refs[p] = 1
            at += k
        if case["kind"] == "fork":
            rows += [[-1] * width] * case["count"]
            s["parents"] = _int32([rng.randrange(case["parents"]) for _ in range(case["count"])])
            s["children"] = _int32([case["parents"] + i for i in range(case["count"])])
            s["lens"] = _int32([case["tokens"]] * case["parents"] + [0] * case["count"])
        if case["kind"] == "append":
            n = case["count"] * case["tokens"]
            kv = normal(n, 2, case["kv_heads"], case["dim"])
            s["k"], s["v"] = kv[:, 0], kv[:, 1]
            slot = torch.arange(n, device=DEV, dtype=torch.int32) // case["tokens"]
            s["slots"], s["positions"] = slot, torch.arange(n, device=DEV, dtype=torch.int32) - slot * case["tokens"]
        s["page_table"], s["refs"] = _int32(rows), _int32(refs)
    return s


# ---- one pass --------------------------------------------------------------------------


def run(s):
    if s["op"] == "attention":
        return (_own_attention if own else _plain_attention)(s)
    if s["op"] == "sample":
        return (_own_sample if own else _plain_sample)(s)
    return (_own_pages if own else _plain_pages)(s)


def _own_attention(s):
    from mini_nccl_b200.ops import generation as G

    o, lse = G.shared_prefix_attention(
        s["q"], s["kv"][0], s["kv"][1], s["prefix_pages"], s["prefix"], s["page_table"], s["seq_lens"],
        q_offsets=s["q_offsets"], max_q_len=s["max_q_len"], max_seq_len=s["own"], return_lse=True)
    return {"o": o, "lse": lse}


def _own_sample(s):
    from mini_nccl_b200.ops import generation as G

    token, logprob = G.sample(s["logits"], s["noise"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"],
                              min_p=s["min_p"], return_logprob=True)
    return {"token": token, "logprob": logprob}


def _own_pages(s):
    from mini_nccl_b200.ops import generation as G

    kv, table, refs = s["kv"], s["page_table"], s["refs"]
    if s["kind"] == "fork":
        G.fork_sequences(kv, table, s["lens"], refs, s["parents"], s["children"])
        held = {"table": table.clone(), "lens": s["lens"].clone(), "held": refs.clone()}
        G.free_sequences(table, s["lens"], refs, s["children"])
        return held | {"kv": kv, "refs": refs}
    if s["kind"] == "append":
        G.append_kv(kv[0, 0], kv[0, 1], s["k"], s["v"], table, s["positions"], s["slots"])
        return {"kv": kv}
    table, refs = G.compact_pages(kv, table, refs)
    return {"kv": kv, "table": table, "refs": refs}


# ---- the plain forms -------------------------------------------------------------------


def _part(scores, allowed, v):
    """Maximum, sum and weighted values of one part of a softmax, over the last axis."""
    if allowed is not None:
        scores = torch.where(allowed, scores, float("-inf"))
    m = scores.amax(-1) if scores.shape[-1] else scores.new_full(scores.shape[:-1], float("-inf"))
    p = torch.exp(scores - torch.where(m == float("-inf"), 0.0, m)[..., None])
    return m, p.sum(-1), p @ v


def _plain_attention(s):
    q, (k_pages, v_pages) = s["q"], s["kv"]
    N, H, D = q.shape
    Hk, page = k_pages.shape[2], k_pages.shape[1]
    G, B, L = H // Hk, s["batch"], s["own"]
    lens = s["seq_lens"].long()
    qf = q.float().view(N, Hk, G, D) / math.sqrt(D)
    # the prefix: one product for all rows of a head
    k1, v1 = (t[s["prefix_pages"].long()].reshape(-1, Hk, D)[: s["prefix"]].float().transpose(0, 1) for t in (k_pages, v_pages))
    rows = qf.transpose(0, 1).reshape(Hk, N * G, D)
    m1, l1, o1 = _part(rows @ k1.transpose(1, 2), None, v1)
    m1, l1, o1 = (t.reshape(Hk, N, G, -1).transpose(0, 1) for t in (m1, l1, o1))
    # each sequence's own tokens, padded to the longest
    if s["q_offsets"] is None:
        first, new = torch.arange(B, device=q.device), torch.ones(B, dtype=torch.long, device=q.device)
    else:
        first, new = s["q_offsets"][:-1].long(), s["q_offsets"].long().diff()
    t = torch.arange(s["max_q_len"], device=q.device)
    pages = s["page_table"].long().clamp(min=0)
    k2, v2 = (x[pages].reshape(B, -1, Hk, D)[:, :L].float().transpose(1, 2) for x in (k_pages, v_pages))
    at = (first[:, None] + t).clamp(max=N - 1)
    mine = qf[at].permute(0, 2, 1, 3, 4).reshape(B, Hk, -1, D)
    last = (lens - new)[:, None] + t  # the newest key that each row may see
    j = torch.arange(L, device=q.device)
    allowed = (j <= last[..., None]) & (j < lens[:, None, None])
    allowed = allowed[:, None, :, None].expand(B, 1, len(t), G, L).reshape(B, 1, -1, L)
    m2, l2, o2 = _part(mine @ k2.transpose(2, 3), allowed, v2)
    n = torch.arange(N, device=q.device)
    b = torch.searchsorted(first + new, n, right=True)
    m2, l2, o2 = (x.reshape(B, Hk, len(t), G, -1)[b, :, n - first[b]] for x in (m2, l2, o2))
    # joined
    m = torch.maximum(m1, m2)
    base = torch.where(m == float("-inf"), 0.0, m)
    a1, a2 = torch.exp(m1 - base), torch.exp(m2 - base)
    total = l1 * a1 + l2 * a2
    o = torch.where(total > 0, (o1 * a1 + o2 * a2) / total, 0.0)
    lse = torch.where(total > 0, base + torch.log(total), float("-inf"))
    return {"o": o.reshape(N, H, D).to(q.dtype), "lse": lse.reshape(N, H)}


def _plain_sample(s):
    x = s["logits"].float()
    R, V = x.shape
    T = s["temperature"][:, None]
    xs, order = torch.sort(x, dim=-1, descending=True, stable=True)
    top = xs[:, :1]
    heat = torch.where(T > 0, T, 1.0)
    rank = torch.arange(V, device=x.device)
    k = torch.where(s["top_k"] > 0, s["top_k"], V)[:, None]
    k = torch.where(T > 0, k, 1)
    w = torch.where((rank < k) & (xs > float("-inf")), torch.exp((xs - top) / heat), 0.0)
    before = torch.cumsum(w, -1) - w
    keep = (w > 0) & ((s["top_p"][:, None] >= 1) | (before < s["top_p"][:, None] * w.sum(-1, keepdim=True)))
    keep = keep & (w >= s["min_p"][:, None])
    total = torch.where(keep, w, 0.0).sum(-1)
    kept = torch.zeros_like(keep).scatter_(1, order, keep)
    score = torch.where(kept, x / heat + s["noise"], float("-inf"))
    best = score.amax(-1, keepdim=True)
    token = torch.where(kept & (score == best), rank, V).amin(-1)
    chosen = x.gather(1, token.clamp(max=V - 1)[:, None])
    logprob = ((chosen - top) / heat)[:, 0] - torch.log(total)
    return {"token": token, "logprob": logprob}


def _plain_pages(s):
    kv, page = s["kv"], s["page"]
    table, refs = s["page_table"], s["refs"]
    width = table.shape[1]
    if s["kind"] == "append":
        positions, slots = s["positions"].long(), s["slots"].long()
        at = table[slots, positions // page].long()
        kv[0, 0, at, positions % page] = s["k"]
        kv[0, 1, at, positions % page] = s["v"]
        return {"kv": kv}
    if s["kind"] == "compact":
        live = refs > 0
        n = live.sum()
        at = torch.arange(s["pool"], device=kv.device)
        src, dst = at[live & (at >= n)], at[~live & (at < n)]
        kv[:, :, dst] = kv[:, :, src]
        to = at.clone()
        to[src] = dst
        moved = torch.zeros_like(refs)
        moved[to[live]] = refs[live]
        return {"kv": kv, "table": torch.where(table >= 0, to[table.long().clamp(min=0)].int(), -1), "refs": moved}
    parents, children, lens = s["parents"].long(), s["children"].long(), s["lens"]
    length = lens[parents].long()
    full, part = length // page, length % page
    rank = (part > 0).long().cumsum(0) - (part > 0).long()
    fresh = torch.nonzero(refs == 0)[:, 0][: len(children)][rank]
    column = torch.arange(width, device=kv.device)
    rows = torch.where(column < full[:, None], table[parents], -1)
    refs.index_add_(0, rows.clamp(min=0).reshape(-1), (rows >= 0).int().reshape(-1))
    source = table[parents, full.clamp(max=width - 1)].long().clamp(min=0)
    rows = torch.where((column == full[:, None]) & (part > 0)[:, None], fresh[:, None].int(), rows)
    token = (torch.arange(page, device=kv.device) < part[:, None])[:, :, None, None]
    kv[:, :, fresh] = torch.where(token, kv[:, :, source], kv[:, :, fresh])
    refs.index_add_(0, fresh, (part > 0).int())
    table[children], lens[children] = rows, length.int()
    held = {"table": table.clone(), "lens": lens.clone(), "held": refs.clone()}
    refs.index_add_(0, rows.clamp(min=0).reshape(-1), -(rows >= 0).int().reshape(-1))
    table[children], lens[children] = -1, 0
    return held | {"kv": kv, "refs": refs}


# ---- in 64 bits ------------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "attention":
        H, D, Hk = case["heads"], case["dim"], case["kv_heads"]
        offsets = list(range(case["batch"] + 1)) if s["q_offsets"] is None else s["q_offsets"].tolist()

        def tokens(pool, ids, n):  # [Hk, n, D]
            return pool[ids.long()].reshape(-1, Hk, D)[:n].double().transpose(0, 1)

        head = [tokens(pool, s["prefix_pages"], case["prefix"]) for pool in s["kv"]]
        outs, sums = [], []
        for b, m in enumerate(s["seq_lens"].tolist()):
            q = s["q"][offsets[b]:offsets[b + 1]].double()
            n = q.shape[0]
            ids = s["page_table"][b, : -(-m // case["page"])]
            keys, values = (torch.cat([h, tokens(pool, ids, m)], 1) for h, pool in zip(head, s["kv"]))
            scores = torch.einsum("nhgd,hkd->nhgk", q.view(n, Hk, H // Hk, D), keys) * D ** -0.5
            where = torch.arange(case["prefix"] + m, device=DEV) - case["prefix"]  # < 0: the prefix
            hidden = where[None] > (m - n + torch.arange(n, device=DEV))[:, None].clamp(min=-1)
            scores.masked_fill_(hidden[:, None, None], float("-inf"))
            outs.append(torch.einsum("nhgk,hkd->nhgd", torch.softmax(scores, -1), values).reshape(n, H, D))
            sums.append(torch.logsumexp(scores, -1).reshape(n, H))
        return {"o": torch.cat(outs), "lse": torch.cat(sums)}
    if case["op"] == "sample":
        logprobs = []
        for r in range(case["rows"]):
            T, k, p, least = (s[name][r].item() for name in ("temperature", "top_k", "top_p", "min_p"))
            x = s["logits"][r].double()
            if T == 0:
                logprobs.append(0.0)
                continue
            order = torch.argsort(x, descending=True, stable=True)
            order = order[torch.isfinite(x[order])][: k or None]
            prob = torch.softmax(x[order] / T, 0)
            n = len(order)
            if p < 1:
                n = min(n, int((torch.cumsum(prob, 0) < p).sum()) + 1)
            n = max(1, min(n, int((prob >= least * prob[0]).sum())))
            score = x[order[:n]] / T + s["noise"][r, order[:n]].double()
            logprobs.append(torch.log_softmax(x[order[:n]] / T, 0)[score.argmax()].item())
        return {"token": None, "logprob": torch.tensor(logprobs, dtype=torch.float64)}
    return None
