"""Cases of the 8-bit key / value cache (attention over it, appending to it) and of the logits' adjustment before sampling.

``own`` false computes each operator in plain torch operations in 32 bits;
``own`` true makes the calls of :mod:`mini_nccl_b200.ops.generation` that a
program generating text makes.

A cache in 8 bits holds codes (int8, or float8_e4m3fn) and one fp32 scale, a
power of two, for each page and kv head; a code stands for ``code * scale``.
"""

from __future__ import annotations

import math
import random

import torch

own = False
DEV = "cuda"

TOP = {"int8": 127.0, "float8_e4m3fn": 448.0}  # the largest code
LEAST = -60  # the scales' least exponent


# ---- cases -----------------------------------------------------------------------------


def listed():
    A, P, L = dict(op="attention"), dict(op="append"), dict(op="logits")
    return [
        # one decode step of four continuations of a short prompt, GPT-124M heads: latency counts
        A | dict(name="q8_few", dtype="int8", batch=4, heads=12, kv_heads=12, dim=64, page=16, prefix=411, own=23, chunk=1, idle=0),
        # one decode step of many rollouts of one long prompt, the 24-layer GPT's heads
        A | dict(name="q8_many", dtype="float8_e4m3fn", batch=160, heads=16, kv_heads=16, dim=128, page=16, prefix=8003, own=509, chunk=1,
                 idle=2),
        # a few agents behind one very long shared document, grouped heads, ragged and empty continuations
        A | dict(name="q8_long", dtype="int8", batch=12, heads=32, kv_heads=8, dim=128, page=64, prefix=100003, own=1500, chunk=1, idle=1),
        # a served batch without a shared prompt: every sequence reads its own history
        A | dict(name="q8_own", dtype="int8", batch=48, heads=32, kv_heads=8, dim=128, page=32, prefix=0, own=6001, chunk=1, idle=0),
        # questions of 1 to 250 tokens appended to one shared prompt in one pass, the 32-layer GPT's heads
        A | dict(name="q8_chunk", dtype="float8_e4m3fn", batch=20, heads=32, kv_heads=32, dim=128, page=32, prefix=3001, own=333, chunk=250,
                 idle=0),
        # the next token of each of 160 sequences into part-filled pages of one layer
        P | dict(name="append_step", dtype="int8", kv_heads=16, dim=128, page=16, count=160, held=300, tokens=1),
        # the next token of a few sequences, GPT-124M heads: latency counts
        P | dict(name="append_few", dtype="float8_e4m3fn", kv_heads=12, dim=64, page=16, count=4, held=40, tokens=1),
        # the keys and values of a packed prompt batch written to one layer's pages
        P | dict(name="append_prompts", dtype="float8_e4m3fn", kv_heads=16, dim=128, page=32, count=13, held=0, tokens=1001),
        # the next token of one sequence with penalties for the tokens it and its prompt hold, GPT vocabulary
        L | dict(name="logits_one", dtype="bfloat16", rows=1, vocab=50304, prompt=411, history=200, bias=0, masks=0, share=1.0, penalties=True),
        # a served batch: penalties, biases, and a few grammars that allow a small part of the vocabulary
        L | dict(name="logits_grammar", dtype="float32", rows=64, vocab=50304, prompt=0, history=700, bias=40, masks=5, share=0.04,
                 penalties=True),
        # penalties for many rollouts of one prompt
        L | dict(name="logits_many", dtype="bfloat16", rows=512, vocab=50304, prompt=900, history=800, bias=0, masks=0, share=1.0,
                 penalties=True),
        # a large odd vocabulary with biases and masks that forbid little
        L | dict(name="logits_wide", dtype="float32", rows=129, vocab=130003, prompt=0, history=0, bias=100, masks=129, share=0.98,
                 penalties=False),
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
    op = rng.choice(("attention", "attention", "append", "logits"))
    dtype = rng.choice(("int8", "float8_e4m3fn"))
    if op == "logits":
        rows = _log(rng, 1, 512)
        vocab = _log(rng, 1000, min(130003, 26_000_000 // rows))
        penalties = rng.random() < 0.75
        masks = rng.choice((0, 0, 1, min(rows, 7), rows))
        return dict(op=op, dtype=rng.choice(("bfloat16", "float32")), rows=rows, vocab=vocab, prompt=rng.choice((0, _log(rng, 1, 4000))),
                    history=_log(rng, 1, 2000) if penalties else 0, bias=rng.choice((0, _log(rng, 1, 300))), masks=masks,
                    share=rng.choice((0.01, 0.3, 0.99)) if masks else 1.0, penalties=penalties)
    if op == "append":
        tokens = rng.choice((1, 1, _log(rng, 2, 900)))
        count = _log(rng, 1, 256 if tokens == 1 else max(1, min(24, 12000 // tokens)))
        return dict(op=op, dtype=dtype, kv_heads=rng.choice((1, 2, 3, 8, 12, 16)), dim=rng.choice((32, 64, 128)),
                    page=rng.choice((8, 16, 32, 64, 128)), count=count, held=rng.choice((0, _log(rng, 1, 300))), tokens=tokens)
    chunk = rng.choice((1, 1, 1, _log(rng, 2, 250)))
    batch = _log(rng, 1, 192 if chunk == 1 else max(1, min(64, 2500 // chunk)))
    kv = rng.choice((2, 4, 8, 12, 16))
    group = rng.choice((1, 1, 2, 4, 8))
    if kv * group > 32:
        group = 1
    longest = _log(rng, 1, max(700, min(6000, 300_000 // batch)) if chunk == 1 else 700)
    prefix = rng.choice((0, _log(rng, 33, 100003), _log(rng, 33, 100003)))
    rows = batch * (1 if chunk == 1 else 0.6 * chunk) * kv * group
    prefix = min(prefix, max(33, int(4e8 / rows)))  # keeps the plain form's score table to the largest listed one's
    return dict(op=op, dtype=dtype, batch=batch, heads=kv * group, kv_heads=kv, dim=rng.choice((32, 64, 128, 128)),
                page=rng.choice((8, 16, 32, 64, 128)), prefix=prefix, own=max(chunk, longest), chunk=chunk,
                idle=rng.choice((0, 0, 1)) if batch > 1 and chunk == 1 else 0)


def _spread(n, lo, hi, turn):
    """n whole numbers over lo..hi, alike for every seed up to their order."""
    return [lo + int((hi - lo + 1) * ((i + 1) * turn % 1.0)) for i in range(n)]


def _lengths(case):
    """(own length, new tokens) of each sequence; the idle ones hold nothing."""
    n = case["batch"] - case["idle"]
    length = _spread(n, 1, case["own"], 0.6180339887)
    new = [1] * n if case["chunk"] == 1 else [min(a, b) for a, b in zip(length, _spread(n, 1, case["chunk"], 0.7548776662))]
    return length + [0] * case["idle"], new + [1 if case["chunk"] == 1 else 0] * case["idle"]


def _runs(case):
    """(tokens held before, new tokens) of each sequence of an append."""
    held = _spread(case["count"], 0, case["held"], 0.6180339887)
    return held, [1] * case["count"] if case["tokens"] == 1 else _spread(case["count"], 1, case["tokens"], 0.7548776662)


def _histories(case):
    return _spread(case["rows"], 0, case["history"], 0.6180339887)


def work(case):
    if case["op"] == "attention":
        length, new = _lengths(case)
        # every code once, the prefix's once for all, and the scales; queries in, outputs and log-sum-exps out
        tokens, pages = case["prefix"] + sum(length), -(-case["prefix"] // case["page"]) + sum(-(-m // case["page"]) for m in length)
        n, H, D = sum(new), case["heads"], case["dim"]
        pairs = sum(t * case["prefix"] + t * max(0, m - t) + t * (t + 1) // 2 for m, t in zip(length, new) if m) \
            + sum(t * case["prefix"] for m, t in zip(length, new) if not m)
        return {"bytes": 2 * case["kv_heads"] * (tokens * D + 4 * pages) + 2 * n * H * D * 2 + 4 * n * H, "flops": 4 * pairs * H * D}
    if case["op"] == "append":
        held, new = _runs(case)
        # keys and values in, their codes out, and the touched pages' scales; codes that are held already need not be touched
        pages = sum((a + n - 1) // case["page"] - a // case["page"] + 1 for a, n in zip(held, new))
        return {"bytes": 2 * case["kv_heads"] * (3 * sum(new) * case["dim"] + 8 * pages) + 8 * sum(new), "flops": 0}
    n, size = case["rows"] * case["vocab"], 2 if case["dtype"] == "bfloat16" else 4
    # logits of the tokens that are allowed in, all out; the tokens that penalties and biases name, and the masks
    named = 8 * (sum(_histories(case)) + case["prompt"]) + 12 * case["rows"] * case["bias"]
    return {"bytes": int(n * size * (1 + case["share"])) + named + case["masks"] * -(-case["vocab"] // 32) * 4, "flops": 4 * n}


# ---- inputs ----------------------------------------------------------------------------


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _exponent(most, dtype):
    """The least e with most <= TOP 2^e, from LEAST on (32-bit whole numbers)."""
    m, x = torch.frexp(most)
    top, shift = math.frexp(TOP[dtype])
    return torch.where(most > 0, x - shift + (m > top).int(), LEAST).clamp(min=LEAST)


def _round(x, dtype):
    return torch.round(x).to(torch.int8) if dtype == "int8" else x.to(torch.float8_e4m3fn)


def _held(gen, pages, page, heads, dim, dtype):
    """Codes and scales of full pages, keys and values of normal data whose size differs from block to block."""
    kv = torch.empty(2, pages, page, heads, dim, dtype=getattr(torch, dtype), device=DEV)
    scales = torch.empty(2, pages, heads, device=DEV)
    for i in (0, 1):
        x = torch.randn(pages, page, heads, dim, generator=gen, device=DEV)
        x *= 0.5 + 1.5 * torch.rand(pages, 1, heads, 1, generator=gen, device=DEV)
        e = _exponent(x.abs().amax((1, 3)), dtype)
        scales[i] = torch.ldexp(torch.ones_like(scales[i]), e)
        kv[i] = _round(x / scales[i][:, None, :, None], dtype)
    return kv, scales


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
        ids = list(range(n_prefix + sum(-(-m // page) for m in length) + 5))
        rng.shuffle(ids)
        s["kv"], s["scales"] = _held(gen, len(ids), page, Hk, D, case["dtype"])
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
    elif case["op"] == "append":
        held, new = _runs(case)
        page, H, D = case["page"], case["kv_heads"], case["dim"]
        columns = max(-(-(a + n) // page) for a, n in zip(held, new))
        ids = list(range(sum(-(-(a + n) // page) for a, n in zip(held, new)) + 3))
        rng.shuffle(ids)
        s["kv"], s["scales"] = _held(gen, len(ids), page, H, D, case["dtype"])
        at, table = 0, []
        for a, n in zip(held, new):
            k = -(-(a + n) // page)
            table.append(ids[at:at + k] + [-1] * (columns - k))
            at += k
        s["page_table"] = _int32(table)
        # keys and values as they leave a fused projection, and some tokens larger than what their pages hold
        qkv = normal(sum(new), 3, H, D)
        qkv *= torch.where(torch.rand(sum(new), 1, 1, 1, generator=gen, device=DEV) < 0.1, 4.0, 1.0)
        s["k"], s["v"] = qkv[:, 1], qkv[:, 2]
        s["positions"] = torch.cat([torch.arange(a, a + n, device=DEV, dtype=torch.int32) for a, n in zip(held, new)])
        s["slots"] = torch.repeat_interleave(torch.arange(len(new), device=DEV, dtype=torch.int32), torch.tensor(new, device=DEV))
    else:
        R, V = case["rows"], case["vocab"]
        x = normal(R, V, dtype=torch.float32) * (1.5 + 2.5 * torch.rand(R, 1, generator=gen, device=DEV))
        s["logits"] = x.to(getattr(torch, case["dtype"]))

        def tokens(*shape):  # a text repeats its frequent tokens
            return (V * torch.rand(*shape, generator=gen, device=DEV, dtype=torch.float64).pow(3)).long().clamp(max=V - 1)

        def some(values):
            return torch.tensor([rng.choice(values) for _ in range(R)], device=DEV)

        s["prompt"] = tokens(case["prompt"]) if case["prompt"] else None
        s["history"] = tokens(R, case["history"]) if case["history"] else None
        lens = _histories(case)
        rng.shuffle(lens)
        s["history_lens"] = _int32(lens) if case["history"] else None
        s["repetition"] = some((1.0, 1.1, 1.3)) if case["penalties"] else 1.0
        s["presence"] = some((0.0, 0.4)) if case["penalties"] else 0.0
        s["frequency"] = some((0.0, 0.1, 0.3)) if case["penalties"] else 0.0
        s["bias_tokens"] = s["bias"] = s["allowed"] = s["mask_of"] = None
        if n := case["bias"]:  # tokens of a row are distinct
            first, step = torch.randint(0, V, (R, 1), generator=gen, device=DEV), V // (n + 1)
            s["bias_tokens"] = ((first + step * torch.arange(n, device=DEV)) % V).int()
            s["bias_tokens"][:, n - n // 4:] = -1  # lists shorter than the longest
            s["bias"] = normal(R, n, dtype=torch.float32) * 5
        if M := case["masks"]:
            bits = torch.rand(M, -(-V // 32) * 32, generator=gen, device=DEV) < case["share"]
            weight = torch.tensor([1 << i if i < 31 else -(1 << 31) for i in range(32)], device=DEV)
            s["allowed"] = (bits.view(M, -1, 32) * weight).sum(-1).int()
            s["mask_of"] = _int32([rng.randrange(-1 if M < R else 0, M) for _ in range(R)]) if M != R else None
    return s


# ---- one pass --------------------------------------------------------------------------


def run(s):
    if s["op"] == "attention":
        return (_own_attention if own else _plain_attention)(s)
    if s["op"] == "append":
        return (_own_append if own else _plain_append)(s)
    return (_own_logits if own else _plain_logits)(s)


def _own_attention(s):
    from mini_nccl_b200.ops import generation as G

    o, lse = G.shared_prefix_attention(
        s["q"], s["kv"][0], s["kv"][1], s["prefix_pages"], s["prefix"], s["page_table"], s["seq_lens"], k_scales=s["scales"][0],
        v_scales=s["scales"][1], q_offsets=s["q_offsets"], max_q_len=s["max_q_len"], max_seq_len=s["own"], return_lse=True)
    return {"o": o, "lse": lse}


def _own_append(s):
    from mini_nccl_b200.ops import generation as G

    G.append_kv(s["kv"][0], s["kv"][1], s["k"], s["v"], s["page_table"], s["positions"], s["slots"], k_scales=s["scales"][0],
                v_scales=s["scales"][1])
    # the cache itself: its definition fixes every code and scale, so they are compared as they are held
    return {"kv": s["kv"], "scales": s["scales"]}


def _own_logits(s):
    from mini_nccl_b200.ops import generation as G

    return G.adjust_logits(
        s["logits"], prompt=s["prompt"], history=s["history"], history_lens=s["history_lens"], repetition=s["repetition"],
        presence=s["presence"], frequency=s["frequency"], bias_tokens=s["bias_tokens"], bias=s["bias"], allowed=s["allowed"],
        mask_of=s["mask_of"])


# ---- the plain forms -------------------------------------------------------------------


def _part(scores, allowed, v):
    """Maximum, sum and weighted values of one part of a softmax, over the last axis."""
    if allowed is not None:
        scores = torch.where(allowed, scores, float("-inf"))
    m = scores.amax(-1) if scores.shape[-1] else scores.new_full(scores.shape[:-1], float("-inf"))
    p = torch.exp(scores - torch.where(m == float("-inf"), 0.0, m)[..., None])
    return m, p.sum(-1), p @ v


def _plain_attention(s):
    q = s["q"]
    N, H, D = q.shape
    Hk, page = s["kv_heads"], s["page"]
    G, B, L = H // Hk, s["batch"], s["own"]
    lens = s["seq_lens"].long()
    qf = q.float().view(N, Hk, G, D) / math.sqrt(D)

    def values(i, ids):  # of the pages ids, in fp32
        return s["kv"][i][ids].float() * s["scales"][i][ids][..., None, :, None]

    # the prefix: one product for all rows of a head
    ids = s["prefix_pages"].long()
    k1, v1 = (values(i, ids).reshape(-1, Hk, D)[: s["prefix"]].transpose(0, 1) for i in (0, 1))
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
    k2, v2 = (values(i, pages).reshape(B, -1, Hk, D)[:, :L].transpose(1, 2) for i in (0, 1))
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


def _plain_append(s):
    positions, slots, page = s["positions"].long(), s["slots"].long(), s["page"]
    at, place = s["page_table"][slots, positions // page].long(), positions % page
    kv, scales = s["kv"], s["scales"]
    new = torch.stack((s["k"], s["v"])).float()
    most = new.abs().amax(-1)  # [2, tokens, heads]
    block = torch.zeros_like(scales).scatter_reduce_(1, at[None, :, None].expand_as(most), most, "amax")
    touched = torch.zeros(scales.shape[1], dtype=torch.bool, device=kv.device).index_fill_(0, at, True)[:, None]
    # a page whose first place is written begins anew
    begun = torch.zeros(scales.shape[1], device=kv.device).index_add_(0, at, (place == 0).float())[:, None] > 0
    held = torch.where(begun, 0.0, scales)
    need = torch.ldexp(torch.ones_like(scales), _exponent(block, s["dtype"]))
    now = torch.where(touched, torch.maximum(held, need), scales)
    # what a page holds already under a larger scale
    grows = (touched & ~begun & (now > scales))[:, :, None, :, None]
    again = _round(kv.float() * (scales / now)[:, :, None, :, None], s["dtype"])
    kv.copy_(torch.where(grows, again.float(), kv.float()))
    scales.copy_(now)
    kv.view(torch.int8)[:, at, place] = _round(new / now[:, at][..., None], s["dtype"]).view(torch.int8)
    return {"kv": kv, "scales": scales}


def _plain_logits(s):
    x = s["logits"].float()
    R, V = x.shape

    def column(v):
        return v[:, None] if isinstance(v, torch.Tensor) else v

    count = torch.zeros(R, V, device=x.device)
    seen = torch.zeros(R, V, device=x.device)
    if s["history"] is not None:
        held = torch.arange(s["history"].shape[1], device=x.device) < s["history_lens"][:, None]
        count.scatter_add_(1, s["history"], held.float())
    if s["prompt"] is not None:
        seen[:, s["prompt"]] = 1.0
    there = count > 0
    repetition = column(s["repetition"])
    x = torch.where(there | (seen > 0), torch.where(x > 0, x / repetition, x * repetition), x)
    x = torch.where(there, x - (column(s["frequency"]) * count + column(s["presence"])), x)
    if s["bias"] is not None:
        named = s["bias_tokens"] >= 0
        x = x.scatter_add(1, s["bias_tokens"].long().clamp(min=0), torch.where(named, s["bias"], 0.0))
    if s["allowed"] is not None:
        v = torch.arange(V, device=x.device)
        bits = (s["allowed"][:, v // 32] >> (v % 32).int()) & 1
        if s["mask_of"] is not None:
            of = s["mask_of"].long()[:, None]
            bits = torch.where(of >= 0, bits[of[:, 0].clamp(min=0)], 1)
        x = torch.where(bits != 0, x, float("-inf"))
    return x.to(s["logits"].dtype)


# ---- in 64 bits ------------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "attention":
        return _exact_attention(case, s)
    if case["op"] == "append":
        return _exact_append(case, s)
    out = s["logits"].double()
    for r in range(case["rows"]):
        def of(name):
            return float(s[name][r]) if isinstance(s[name], torch.Tensor) else s[name]

        tokens = s["history"][r, : int(s["history_lens"][r])] if s["history"] is not None else torch.empty(0, dtype=torch.long, device=DEV)
        mine, times = torch.unique(tokens, return_counts=True)
        both = mine if s["prompt"] is None else torch.unique(torch.cat([mine, s["prompt"]]))
        x = out[r]
        old, rho = x[both], of("repetition")
        x[both] = torch.where(old > 0, old / rho, old * rho)
        x[mine] -= of("frequency") * times.double() + of("presence")
        if case["bias"]:
            named = s["bias_tokens"][r] >= 0
            x[s["bias_tokens"][r][named].long()] += s["bias"][r][named].double()
        which = -1 if not case["masks"] else r if s["mask_of"] is None else int(s["mask_of"][r])
        if which >= 0:
            words = s["allowed"][which].long()
            bits = torch.stack([(words >> i) & 1 for i in range(32)], 1).reshape(-1)[: case["vocab"]]
            x[bits == 0] = float("-inf")
    return out


def _exact_attention(case, s):
    H, D, Hk = case["heads"], case["dim"], case["kv_heads"]
    offsets = list(range(case["batch"] + 1)) if s["q_offsets"] is None else s["q_offsets"].tolist()

    def tokens(i, ids, n):  # [Hk, n, D]
        ids = ids.long()
        return (s["kv"][i][ids].double() * s["scales"][i][ids].double()[:, None, :, None]).reshape(-1, Hk, D)[:n].transpose(0, 1)

    head = [tokens(i, s["prefix_pages"], case["prefix"]) for i in (0, 1)]
    outs, sums = [], []
    for b, m in enumerate(s["seq_lens"].tolist()):
        q = s["q"][offsets[b]:offsets[b + 1]].double()
        n = q.shape[0]
        ids = s["page_table"][b, : -(-m // case["page"])]
        keys, values = (torch.cat([h, tokens(i, ids, m)], 1) for i, h in enumerate(head))
        scores = torch.einsum("nhgd,hkd->nhgk", q.view(n, Hk, H // Hk, D), keys) * D ** -0.5
        where = torch.arange(case["prefix"] + m, device=DEV) - case["prefix"]  # < 0: the prefix
        hidden = where[None] > (m - n + torch.arange(n, device=DEV))[:, None].clamp(min=-1)
        scores.masked_fill_(hidden[:, None, None], float("-inf"))
        if keys.shape[1]:
            outs.append(torch.einsum("nhgk,hkd->nhgd", torch.softmax(scores, -1), values).reshape(n, H, D))
            sums.append(torch.logsumexp(scores, -1).reshape(n, H))
        else:
            outs.append(torch.zeros(n, H, D, dtype=torch.float64, device=DEV))
            sums.append(torch.full((n, H), float("-inf"), dtype=torch.float64, device=DEV))
    return {"o": torch.cat(outs), "lse": torch.cat(sums)}


def _exact_append(case, s):
    """Page by page: every value that the page is to hold, then the least power of two that takes them all."""
    page, top = case["page"], TOP[case["dtype"]]
    kv, scales = s["kv"].double(), s["scales"].double()
    positions, slots = s["positions"].tolist(), s["slots"].tolist()
    rows = s["page_table"].tolist()
    of_page = {}
    for i, (pos, slot) in enumerate(zip(positions, slots)):
        of_page.setdefault(rows[slot][pos // page], []).append((i, pos % page))
    for p, named in of_page.items():
        tokens, places = (torch.tensor(x, device=DEV) for x in zip(*named))
        for i, x in enumerate((s["k"], s["v"])):
            new = x[tokens].double()
            for h in range(case["kv_heads"]):
                most = float(new[:, h].abs().max())
                scale = 2.0 ** max(LEAST, math.ceil(math.log2(most / top)) if most > 0 else LEAST)
                if int(places.min()) > 0:
                    was = float(scales[i, p, h])
                    scale = max(scale, was)
                    kv[i, p, :, h] = _nearest(kv[i, p, :, h] * (was / scale), case["dtype"])
                scales[i, p, h] = scale
                kv[i, p, places, h] = _nearest(new[:, h] / scale, case["dtype"])
    return {"kv": kv.to(torch.int8) if case["dtype"] == "int8" else kv, "scales": scales}


def _nearest(x, dtype):
    """The nearest code, of two the even one, in 64 bits."""
    if dtype == "int8":
        return torch.round(x)
    step = torch.ldexp(torch.ones_like(x), (torch.frexp(x)[1] - 1).clamp(min=-6) - 3)  # 3 bits behind the first, down to 2^-6
    return torch.round(x / step) * step
