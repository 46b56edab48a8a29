"""Edges of the 8-bit cache and of the logits' adjustment, and both as generation uses them.

References are in 64 bits, with the tolerances of ``test_generation_8bit.py``.
"""

from __future__ import annotations

import math
import random
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

import pytest
import torch

from mini_nccl_b200.models.generation import BranchedGeneration, sample_continuations
from mini_nccl_b200.ops import generation as G
from test_generation import DEVICES, ints, settle
from test_generation_8bit import TYPES, U, Problem, adjusted, tokens_of, values_of, words_of
from test_generation_edges import out_of_range
from test_generation_path import model_on

# few rows, many rows, several tokens of a sequence, and enough of a prefix for the tensor cores
FEW = dict(lens=[60, 3, 0], new=[1, 1, 1], kv_heads=2, group=2, page=16, prefix=129)
MANY = dict(lens=[40] * 50, new=[1] * 50, kv_heads=2, group=1, page=32, prefix=100)
RAGGED = dict(lens=[70, 90], new=[60, 90], kv_heads=2, group=2, page=8, prefix=333)
WIDE = dict(lens=[9] * 30, new=[1] * 30, kv_heads=16, group=1, page=16, prefix=4101)
FORMS = [(FEW, 32), (FEW, 128), (MANY, 32), (MANY, 64), (RAGGED, 64), (RAGGED, 128), (WIDE, 64), (WIDE, 128)]
# (the plain path has no forms)
CALLS = [("cpu", FEW, 128), ("cpu", RAGGED, 64)] + [pytest.param("cuda", *f, marks=pytest.mark.gpu) for f in FORMS]


# ---- attention ---------------------------------------------------------------------------


@pytest.mark.parametrize("device,form,dim", CALLS)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("scale,scale_q", [(0.0, 1.0), (-0.2, 1.0), (None, 0.0), (None, 40.0)])
def test_attention_scales_of_scores(device, dtype, form, dim, scale, scale_q):
    p = Problem(**form, dim=dim, device=device, dtype=dtype, scale_q=scale_q)
    p.check(*p.run(scale=scale), scale=scale)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("form,dim", [(FEW, 64), (RAGGED, 32), (WIDE, 128)])
def test_attention_layouts_and_bounds(device, dtype, form, dim):
    p = Problem(**form, dim=dim, device=device, dtype=dtype, heads_first=True)
    o, lse = p.run(max_seq_len=max(form["lens"]), scale=0.3)
    p.check(o, lse, scale=0.3)
    args, named = p.arguments(max_seq_len=max(form["lens"]), scale=0.3)
    named["return_lse"] = False
    assert torch.equal(G.shared_prefix_attention(*args, **named), o)
    # a tight bound and none, and a layer's pages and scales as slices of a larger pool
    plain = Problem(**form, dim=dim, device=device, dtype=dtype)
    want = plain.run()
    plain.check(*want)
    pool = plain.pool.view(torch.uint8)
    plain.pool = torch.stack([pool, 255 - pool], 1).view(dtype)[:, 0]
    plain.scales = torch.stack([plain.scales * 2, plain.scales], 1)[:, 1]
    again = plain.run(max_seq_len=max(form["lens"]))
    plain.check(*again)


@pytest.mark.parametrize("device,form,dim", CALLS)
@pytest.mark.parametrize("dtype", TYPES)
def test_attention_scales_far_apart(device, dtype, form, dim):
    """Pages whose scales differ by up to 2^14: errors are those of the row's largest value, in whichever column it is."""
    p = Problem(**form, dim=dim, device=device, dtype=dtype, exponents=(-14, 0))
    o, lse = (t.cpu().double() for t in p.run())
    at = 0
    for m, n, own in zip(p.lens, p.new, p.own):
        k, v = torch.cat([p.head, own], 1).repeat_interleave(p.group, 2).transpose(1, 2)
        for t in range(n):
            seen = p.prefix + max(0, m - n + 1 + t)
            q = p.q[at].cpu().double()
            s = torch.einsum("hd,hkd->hk", q, k[:, :seen]) * dim ** -0.5
            off = dim * U * (torch.einsum("hd,hkd->hk", q.abs(), k[:, :seen].abs()) * dim ** -0.5).amax(-1) + 8 * U * (s.abs().amax(-1) + 60)
            w = torch.softmax(s, -1)[..., None]
            want, spread = (w * v[:, :seen]).sum(1), (w * v[:, :seen].abs()).sum(1).amax(-1, keepdim=True)
            assert torch.all((lse[at] - torch.logsumexp(s, -1)).abs() <= off)
            assert torch.all((o[at] - want).abs() <= 2.0 ** -8 * want.abs() + (2.0 ** -11 + 2 * off[:, None]) * spread)
            at += 1


@pytest.mark.parametrize("device,form,dim", CALLS)
@pytest.mark.parametrize("dtype", TYPES)
def test_attention_pages_that_nothing_was_written_to(device, dtype, form, dim):
    """Scales of 0, and codes of 0 beside scales that are none."""
    p = Problem(**form, dim=dim, device=device, dtype=dtype)
    p.scales[:] = 0
    o, lse = p.run()
    seen = torch.tensor([p.prefix + max(0, m - n + 1 + t) for m, n in zip(p.lens, p.new) for t in range(n)]).double()
    assert torch.all(o.abs() <= 448 * 2.0 ** -60)
    assert torch.all((lse.cpu().double() - seen.log()[:, None]).abs() <= 8 * U * 64)
    # half of the pages are empty: their tokens have a score of 0 and no values
    p = Problem(**form, dim=dim, device=device, dtype=dtype)
    empty = torch.arange(p.pool.shape[1]) % 2 == 0
    p.pool.view(torch.uint8)[:, empty] = 0
    p.scales[:, empty] = 0
    for t, page_of in [(p.head, p.prefix_pages)] + list(zip(p.own, p.rows)):
        for i in range(t.shape[1]):
            if empty[page_of[i // form["page"]]]:
                t[:, i] = 0
    p.check(*p.run())


@pytest.mark.parametrize("device,form,dim", CALLS)
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_attention_shows_queries_that_are_no_numbers(device, form, dim, bad):
    p = Problem(**form, dim=dim, device=device, dtype=torch.int8)
    want, want_lse = (t.cpu() for t in p.run())
    sound = p.q.clone()
    p.q[1, 1, 5] = bad
    o, lse = (t.cpu() for t in p.run())
    assert torch.all(o[1, 1].isnan()) and (lse[1, 1].isnan() or bad == math.inf)
    # the other rows hold to the definition (not to the bit: where one of a warp's rows has scores past 2^24, all of them are
    # rounded before their base is taken off)
    p.q = sound
    o[1, 1], lse[1, 1] = want[1, 1], want_lse[1, 1]
    p.check(o, lse)


@pytest.mark.parametrize("device,form,dim", CALLS)
def test_attention_shows_nan_in_visible_tokens(device, form, dim):
    group, page = form["group"], form["page"]
    for part in (0, 1):
        for at in range(0, p_len(form), 37):  # one token of the prefix: every row of its head sees it
            p = Problem(**form, dim=dim, device=device, dtype=torch.float8_e4m3fn)
            p.pool.view(torch.uint8)[part, p.prefix_pages[at // page], at % page, 1, 3] = 0xff
            o, lse = (t.cpu() for t in p.run())
            hit = o[:, group:2 * group]
            assert torch.all(hit.isnan() if part == 0 else hit[..., 3].isnan()), (part, at)
            assert part == 1 or torch.all(lse[:, group:2 * group].isnan())
            rest = torch.cat([o[:, :group], o[:, 2 * group:]], 1)
            assert not rest.isnan().any() and not lse[:, :group].isnan().any()
    # the first token of a sequence's own
    p = Problem(**form, dim=dim, device=device, dtype=torch.float8_e4m3fn)
    want, _ = p.run()
    p.pool.view(torch.uint8)[0, p.rows[1][0], 0, 0, 0] = 0x7f
    o, _ = p.run()
    first = form["new"][0]
    seen = torch.zeros(o.shape[:2], dtype=torch.bool)
    seen[first + max(0, form["new"][1] - form["lens"][1]): first + form["new"][1], :group] = True
    assert torch.equal(o.isnan().all(-1).cpu(), seen)


def p_len(form):
    return min(form["prefix"], 300)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("lens,new,kv_heads,group,dim,page,prefix", [
    ([7, 5], [7, 5], 1, 1, 32, 8, 0),
    ([70, 33, 0, 5], [33, 1, 0, 5], 2, 2, 64, 16, 100),
    ([130, 7, 129], [130, 7, 2], 1, 3, 128, 8, 0),
    ([90, 31], [77, 31], 1, 1, 128, 64, 191),
    ([9 + i % 5 for i in range(230)], [4] * 230, 4, 1, 128, 8, 0),
])
def test_attention_leaves_out_hidden_values(device, lens, new, kv_heads, group, dim, page, prefix):
    """A query's result does not depend on tokens behind it, whatever they hold; those that see the token show it."""
    p = Problem(lens, new, kv_heads=kv_heads, group=group, dim=dim, page=page, prefix=prefix, device=device, dtype=torch.float8_e4m3fn)
    want, want_lse = (t.cpu() for t in p.run())
    first = torch.tensor([0] + new).cumsum(0).tolist()
    sees = torch.zeros(sum(new), dtype=torch.bool)
    codes = p.pool.view(torch.uint8)
    for b, (m, n) in enumerate(zip(lens, new)):
        if n < 2:
            continue
        at = m - n + n // 2  # the place of query n // 2
        codes[1, p.rows[b][at // page], at % page, 0, 1::2] = 0x7f
        codes[0, p.rows[b][at // page], at % page, kv_heads - 1, 0] = 0xff  # and its key in another head
        sees[first[b] + n // 2: first[b + 1]] = True
    o, lse = (t.cpu() for t in p.run())
    p.check(torch.where(sees[:, None, None], want, o), torch.where(sees[:, None], want_lse, lse))
    values = o[sees][:, :group] if kv_heads > 1 else o[sees][:0]
    assert values[..., 1::2].isnan().all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
def test_attention_no_rows_and_no_tokens(device, dtype):
    pool, scales = torch.zeros(2, 4, 8, 4, 64, device=device).to(dtype), torch.ones(2, 4, 4, device=device)
    sc = dict(k_scales=scales[0], v_scales=scales[1], return_lse=True)
    none = torch.empty(0, 2, dtype=torch.int32, device=device)
    q = torch.randn(3, 4, 64, device=device).to(torch.bfloat16)
    o, lse = G.shared_prefix_attention(q[:0], pool[0], pool[1], ints([1], device), 3, none, ints([], device), **sc)
    assert o.shape == (0, 4, 64) and lse.shape == (0, 4)
    o, lse = G.shared_prefix_attention(q, pool[0], pool[1], ints([], device), 0, torch.empty(3, 0, dtype=torch.int32, device=device),
                                       ints([0, 0, 0], device), **sc)
    settle(device)
    assert torch.all(o == 0) and torch.all(lse == -math.inf)
    p = Problem([0] * 30, [1] * 30, kv_heads=2, group=2, dim=64, page=16, prefix=140, device=device, dtype=dtype)
    p.check(*p.run(max_seq_len=0))
    if device == "cuda":
        p = Problem([0] * 30, [1] * 30, kv_heads=16, group=1, dim=64, page=16, prefix=4200, device=device, dtype=dtype)
        p.check(*p.run(max_seq_len=0))
    # some sequences without a new token, at most one each
    for prefix in (0, 70):
        p = Problem([5, 9, 0, 70, 3], [1, 0, 1, 1, 0], kv_heads=2, group=3, dim=128, page=8, prefix=prefix, device=device, dtype=dtype)
        p.check(*p.run())


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("lens,new,kv_heads,group,dim,page,prefix", [
    ([5, 70, 0], [1, 1, 1], 1, 71, 64, 16, 50),
    ([5, 70, 3], [2, 9, 1], 1, 40, 128, 16, 50),
    ([5, 70, 3], [1, 1, 1], 2, 64, 32, 8, 0),
    pytest.param([5, 70, 3], [2, 9, 1], 1, 64, 128, 16, 5000, marks=pytest.mark.gpu),
    ([300], [300], 1, 1, 64, 256, 0),
])
def test_attention_many_heads_to_one(device, lens, new, kv_heads, group, dim, page, prefix):
    p = Problem(lens, new, kv_heads=kv_heads, group=group, dim=dim, page=page, prefix=prefix, device=device, dtype=torch.int8)
    p.check(*p.run())


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
def test_attention_on_a_pool_without_pages(device, dtype):
    pool, scales = torch.zeros(0, 8, 2, 64, device=device).to(dtype), torch.zeros(0, 2, device=device)
    q = torch.randn(3, 4, 64, device=device).to(torch.bfloat16)

    def call(prefix, lens):
        return G.shared_prefix_attention(q, pool, pool, ints([0], device), prefix, ints([[-1], [-1], [0]], device), ints(lens, device),
                                         k_scales=scales, v_scales=scales)

    assert torch.all(call(0, [0, 0, 0]) == 0)
    settle(device)
    for prefix, lens in ((5, [0, 0, 0]), (0, [0, 0, 3])):
        o = out_of_range(device, lambda: call(prefix, lens))
        assert o is None or torch.all(o == 0)


@pytest.mark.parametrize("device", DEVICES)
def test_attention_refusals(device):
    def call(dtype=torch.int8, v_dtype=None, scales=(4, 2), of=torch.float32, only_k=False, q=(3, 4, 64), rows=3, **more):
        pool = [torch.zeros(4, 8, 2, 64, device=device).to(t) for t in (dtype, v_dtype or dtype)]
        s = None if scales is None else torch.ones(*scales, device=device, dtype=of)
        G.shared_prefix_attention(torch.zeros(*q, device=device, dtype=torch.bfloat16), *pool, ints([3], device), 5,
                                  ints([[0], [1], [2]][:rows], device), ints([1, 2, 3], device), k_scales=s, v_scales=None if only_k else s,
                                  **more)

    call()
    call(torch.float8_e4m3fn)
    call(torch.bfloat16, scales=None)
    for bad in (dict(scales=None), dict(only_k=True), dict(dtype=torch.bfloat16), dict(v_dtype=torch.float8_e4m3fn), dict(scales=(4, 3)),
                dict(scales=(3, 2)), dict(scales=(4, 2, 1)), dict(of=torch.float64), dict(of=torch.bfloat16), dict(q=(3, 5, 64)),
                dict(q=(2, 4, 64)), dict(q=(3, 4, 32)), dict(rows=2)):
        with pytest.raises(ValueError):
            call(**bad)
    settle(device)


@pytest.mark.gpu
def test_attention_refuses_other_layouts_on_the_gpu():
    pool, scales = torch.zeros(2, 8, 8, 2, 64, dtype=torch.int8, device="cuda"), torch.ones(2, 8, 2, device="cuda")
    q = torch.zeros(1, 2, 64, dtype=torch.bfloat16, device="cuda")

    def call(k, v, a, b):
        G.shared_prefix_attention(q, k, v, ints([3], "cuda"), 5, ints([[1]], "cuda"), ints([1], "cuda"), k_scales=a, v_scales=b)

    call(pool[0], pool[1], scales[0], scales[1])
    flat = torch.zeros(pool[0].numel() + 1, dtype=torch.int8, device="cuda")
    for bad in ((flat[1:].view(8, 8, 2, 64), pool[1], scales[0], scales[1]),  # not on 16 bytes
                (pool[0].transpose(0, 1), pool[1].transpose(0, 1).contiguous().transpose(0, 1).transpose(0, 1), scales[0], scales[1]),
                (pool[0], pool[1], scales[0], scales[1].t().contiguous().t()),  # scales of two layouts
                (pool[0], pool[1], scales[0].cpu(), scales[1]),
                (pool[0].cpu(), pool[1], scales[0], scales[1])):
        with pytest.raises((ValueError, RuntimeError)):
            call(*bad)
    settle("cuda")


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dim,prefix", [(32, 0), (64, 40), (128, 600), (64, 6000)])
@pytest.mark.parametrize("offsets,most,limit", [
    ([3, 40, 60, 70], 60, 90), ([0, 40, 60, 65], 60, 90), ([0, 50, 40, 70], 60, 90), ([0, 40, 60, 90], 60, 90), ([-4, 40, 60, 70], 60, 90),
    ([0, 40, 60, 70], 25, 90), ([0, 40, 60, 70], 60, 50), ([0, 40, 69, 70], 60, 0),
])
def test_attention_reports_offsets_and_bounds_that_do_not_hold(device, dim, prefix, offsets, most, limit):
    p = Problem([60, 90, 33], [40, 20, 10], kv_heads=8, group=1, dim=dim, page=16, prefix=prefix, device=device, dtype=torch.int8)
    if device == "cuda":  # what the allocator hands out next holds NaN
        stale = torch.full((32 << 20,), math.nan, device=device)
        del stale
    args, named = p.arguments(max_seq_len=limit)
    named.update(q_offsets=ints(offsets, device), max_q_len=most)
    out = out_of_range(device, lambda: G.shared_prefix_attention(*args, **named))
    if out is None:
        return
    if limit == 90:  # rows without a sequence of their own: the own tokens of the whole call are left out
        p.lens, p.own, p.new = [0] * 3, [t[:, :0] for t in p.own], [40, 20, 10]
        p.check(*out)
    else:
        assert not any(t.isnan().any() for t in out)


@pytest.mark.gpu
@pytest.mark.parametrize("form,dim", [(FEW, 64), (MANY, 32), (RAGGED, 128), (WIDE, 128)])
def test_attention_reports_bad_pages_and_lengths(form, dim):
    def bad_call(i, change):
        p = Problem(**form, dim=dim, device="cuda", dtype=torch.float8_e4m3fn)
        args, named = p.arguments()
        args = list(args)
        args[i] = args[i].clone()
        change(args[i], p)
        out = out_of_range("cuda", lambda: G.shared_prefix_attention(*args, **named))
        assert not any(t.isnan().any() for t in out)
        p.check(*out)

    def prefix_page(t, p):  # pages outside the pool read as zeros
        t[1], t[2] = 10 ** 6, -7
        page = form["page"]
        p.head[:, page:3 * page] = 0

    def own_page(t, p):
        t[1, 0] = -1
        p.own[1][:, :form["page"]] = 0

    def length(value):
        def change(t, p):
            t[1] = value
            p.lens[1], p.own[1] = 0, p.own[1][:, :0]
        return change

    bad_call(3, prefix_page)
    bad_call(5, own_page)
    bad_call(6, length(-3))
    bad_call(6, length(10 ** 6))


@pytest.mark.gpu
@pytest.mark.parametrize("form", [FEW, WIDE])
def test_attention_over_the_prefix_alone_reports_lengths(form):
    p = Problem(**{**form, "lens": [0] * len(form["lens"])}, dim=64, device="cuda", dtype=torch.int8)
    args, named = p.arguments(max_seq_len=0)
    args = (*args[:6], ints([0, 7] + [0] * (len(form["lens"]) - 2), "cuda"))
    out = out_of_range("cuda", lambda: G.shared_prefix_attention(*args, **named))
    p.check(*out)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_pages_beyond_32_bit_offsets(dtype):
    page, heads, dim = 256, 16, 128
    pages = (1 << 32) // (page * heads * dim) + 40  # ids whose first byte lies past 2^32
    pool = torch.empty(2, pages, page, heads, dim, dtype=torch.uint8, device="cuda").view(dtype)
    scales = torch.zeros(2, pages, heads, device="cuda")
    for rows in (2, 40):
        small = Problem([300, 2] + [0] * (rows - 2), [1] * rows, kv_heads=heads, group=1, dim=dim, page=page, prefix=4100 if rows > 2 else 700,
                        device="cuda", dtype=dtype)
        base = pages - small.pool.shape[1]
        pool.view(torch.uint8)[:, base:] = small.pool.view(torch.uint8)
        scales[:, base:] = small.scales
        args, named = small.arguments()
        q, _, _, head, prefix, table, lens = args
        named.update(k_scales=scales[0], v_scales=scales[1])
        out = G.shared_prefix_attention(q, pool[0], pool[1], head + base, prefix, torch.where(table < 0, table, table + base), lens, **named)
        settle("cuda")
        small.check(*out)
    k, v = tokens_of(5, heads, dim, "cuda", 3)
    near = torch.zeros(2, 1, page, heads, dim, dtype=torch.uint8, device="cuda").view(dtype)
    near_scales = torch.zeros(2, 1, heads, device="cuda")
    for kv, sc, last in ((pool, scales, pages - 1), (near, near_scales, 0)):
        G.append_kv(kv[0], kv[1], k, v, ints([[last]], "cuda"), ints([0, 1, 2, 3, 4], "cuda"), ints([0] * 5, "cuda"), k_scales=sc[0],
                    v_scales=sc[1])
    settle("cuda")
    assert torch.equal(pool.view(torch.uint8)[:, -1, :5], near.view(torch.uint8)[:, 0, :5])
    assert torch.equal(scales[:, -1], near_scales[:, 0])


@pytest.mark.gpu
def test_gradients_are_refused_not_lost():
    p = Problem(**FEW, dim=64, device="cuda", dtype=torch.int8)
    want, _ = p.run()
    p.q = p.q.detach().requires_grad_()
    o, lse = p.run()
    assert torch.equal(o, want)
    for out in (o, lse):
        with pytest.raises(RuntimeError, match="no gradient"):
            out.float().sum().backward()
    p.q = p.q.detach()
    p.scales.requires_grad_()
    with pytest.raises(RuntimeError, match="no gradient"):
        p.run()[0].float().sum().backward()
    x, b = torch.randn(2, 50, device="cuda", requires_grad=True), torch.randn(1, device="cuda", requires_grad=True)
    for y in (G.adjust_logits(x, repetition=2.0, prompt=ints([3], "cuda")),
              G.adjust_logits(x.detach(), bias_tokens=ints([3], "cuda"), bias=b)):
        with pytest.raises(RuntimeError, match="no gradient"):
            y.sum().backward()
    with pytest.raises(ValueError, match="in place"):
        G.adjust_logits(x, prompt=ints([3], "cuda"), out=x)
    with torch.no_grad():
        assert not G.adjust_logits(x, prompt=ints([3], "cuda")).requires_grad


# ---- pages with scales -------------------------------------------------------------------


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
def test_page_operations_take_the_scales_along(device, dtype):
    layers, page, heads, dim = 2, 8, 3, 32
    c = G.PagedKVCache(layers, 24, page, heads, dim, max_seqs=8, max_seq_len=40, device=device, dtype=dtype)
    lens = {0: 19, 3: 8, 4: 5, 6: 33}
    c.extend(list(lens), list(lens.values()))
    places, slots = [t for n in lens.values() for t in range(n)], [s for s, n in lens.items() for _ in range(n)]
    given = [tokens_of(len(places), heads, dim, device, layer) for layer in range(layers)]
    for layer, (k, v) in enumerate(given):
        c.append(layer, k, v, ints(places, device), ints(slots, device))

    def tokens(slot):
        ids = c.page_table[slot, : -(-c.lengths[slot] // page)].long().cpu()
        return torch.stack([values_of(c.kv[i, j], c.scales[i, j])[ids].flatten(0, 1)[: c.lengths[slot]]
                            for i in range(layers) for j in range(2)])

    want = {s: tokens(s) for s in lens}
    # within half a step of what was given: 2^-4 of a value, or half a scale of the page's largest value / 127 (or twice it)
    for layer, (k, v) in enumerate(given):
        for part, x in enumerate((k, v)):
            x, got = x.cpu().double(), torch.cat([want[s][2 * layer + part] for s in lens])
            if dtype == torch.float8_e4m3fn:
                largest = torch.stack([x[[j for j in range(len(places)) if (slots[j], places[j] // page) == (slots[i], places[i] // page)]]
                                       .abs().amax((0, 2)) for i in range(len(places))])
                assert torch.all((got - x).abs() <= 2.0 ** -4 * x.abs() + largest[..., None] * 2.0 ** -17)
    c.fork([0, 6, 0], [1, 2, 5])
    c.free([0])
    c.compact()
    settle(device)
    for child, parent in ((1, 0), (2, 6), (5, 0), (3, 3), (4, 4), (6, 6)):
        assert torch.equal(tokens(child), want[parent]), (child, parent)
    # a fork goes on by itself: larger values change the scale of its own page only
    c.extend([1], [1])
    k, v = tokens_of(1, heads, dim, device, 9, size=100.0)
    c.append(0, k, v, ints([19], device), ints([1], device))
    settle(device)
    assert torch.equal(tokens(5), want[0])
    src, dst = ints([int(c.page_table[3, 0])], device), ints([23], device)
    G.copy_pages(c.kv, src, dst, c.scales)
    settle(device)
    assert torch.equal(c.scales[:, :, 23], c.scales[:, :, int(src[0])])
    for bad in (c.scales[:, :, :5], c.scales.double(), c.scales[0], c.scales.transpose(2, 3)):
        with pytest.raises(ValueError):
            G.copy_pages(c.kv, src, dst, bad)
        with pytest.raises(ValueError):
            G.compact_pages(c.kv, c.page_table, c.refs, bad)


@pytest.mark.parametrize("device", DEVICES)
def test_append_refuses_scales_that_share_memory(device):
    pool, scales = torch.zeros(2, 4, 8, 2, 16, dtype=torch.int8, device=device), torch.zeros(2, 4, 2, device=device)
    k, v = tokens_of(1, 2, 16, device, 0)
    for a, b in ((scales[0], scales[0]), (scales[0, :, :1].expand(4, 2), scales[1, :, :1].expand(4, 2)),
                 (scales[0, :1].expand(4, 2), scales[1, :1].expand(4, 2))):
        with pytest.raises(ValueError, match="of their own"):
            G.append_kv(pool[0], pool[1], k, v, ints([[1]], device), ints([0], device), k_scales=a, v_scales=b)
    settle(device)


# ---- logits ------------------------------------------------------------------------------


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("R,V,H", [(2, 900, 5000), (200, 50304, 1500), (3, 1 << 20, 3001)])
def test_adjust_logits_long_lists(device, dtype, R, V, H):
    """More named tokens in a block's part of a row than it keeps."""
    gen = torch.Generator().manual_seed(H)
    x = (torch.randn(R, V, generator=gen) * 4).to(dtype)
    low = min(V, 7000)
    history, prompt = torch.randint(0, low, (R, H), generator=gen), torch.randint(0, low, (R, 1100), generator=gen)
    tokens, bias = torch.randint(0, low, (R, 4095), generator=gen).int(), torch.randn(R, 4095, generator=gen)
    bits = torch.rand(1, V, generator=gen) < 0.7
    y = G.adjust_logits(x.to(device), prompt=prompt.to(device), history=history.to(device), repetition=1.2, presence=0.5, frequency=0.125,
                        bias_tokens=tokens.to(device), bias=bias.to(device), allowed=words_of(bits).to(device)).cpu()
    settle(device)
    for r in range(0, R, 67):
        named = {int(t): float(b) for t, b in zip(tokens[r], bias[r])}
        rho = float(torch.tensor(1.2))
        want, room = adjusted(x[r], prompt[r].tolist(), history[r].tolist(), rho, 0.5, 0.125, named, bits[0])
        off, fine = (y[r].double() - want).abs(), bits[0]
        assert torch.all(y[r][~fine] == -math.inf)
        assert torch.all(off[fine] <= (room + torch.finfo(dtype).eps / 2 * (want.abs() + room))[fine])


@pytest.mark.parametrize("device", DEVICES)
def test_adjust_logits_reports_what_there_is_not(device):
    x = torch.randn(3, 77).to(device)
    good = dict(history=torch.tensor([[5, 6], [7, -1], [8, 8]], device=device), presence=1.0)
    want = G.adjust_logits(x, **good)

    def bad(**change):
        return out_of_range(device, lambda: G.adjust_logits(x, **{**good, **change}))

    y = bad(history=torch.tensor([[5, 6], [7, 77], [8, 8]], device=device))
    assert y is None or torch.equal(y, want)
    y = bad(prompt=torch.tensor([1 << 40], device=device))
    assert y is None or torch.equal(y, want)
    for lens in ([2, 3, 2], [2, -1, 2]):
        y = bad(history_lens=ints(lens, device))
        assert y is None or (torch.equal(y[[0, 2]], want[[0, 2]]) and torch.equal(y[1], x[1]))
    y = bad(bias_tokens=torch.tensor([80], device=device), bias=torch.ones(1, device=device))
    assert y is None or torch.equal(y, want)
    y = bad(allowed=torch.full((2, 3), -1, dtype=torch.int32, device=device), mask_of=ints([0, 2, -1], device))
    assert y is None or torch.equal(y[[0, 2]], want[[0, 2]])
    none = torch.empty(0, 3, dtype=torch.int32, device=device)
    y = bad(allowed=none, mask_of=ints([-1, 0, -1], device))
    assert y is None or torch.equal(y, want)
    assert torch.equal(G.adjust_logits(x, **good, allowed=none, mask_of=ints([-1, -1, -1], device)), want)
    settle(device)


@pytest.mark.gpu
def test_adjust_logits_refuses_memory_that_overlaps():
    flat = torch.zeros(3 * 100 + 64, device="cuda")
    x = flat[:300].view(3, 100)
    for out in (flat[4:304].view(3, 100), flat[300:].expand(3, 64),
                torch.as_strided(flat, (3, 100), (104, 1))):
        with pytest.raises(ValueError):
            G.adjust_logits(x, prompt=ints([1], "cuda"), out=out)
    with pytest.raises(ValueError):
        G.adjust_logits(x, prompt=torch.tensor([1]))
    with pytest.raises(ValueError):
        G.adjust_logits(x.t()[:3], prompt=ints([1], "cuda"))
    settle("cuda")


# ---- streams, graphs, threads ------------------------------------------------------------


@pytest.mark.gpu
def test_operators_follow_the_current_stream():
    p = Problem(**RAGGED, dim=64, device="cuda", dtype=torch.int8)
    want, _ = p.run()
    args, named = p.arguments()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)  # what the side stream computes is late for every other stream
        pool, scales = [t * 1 for t in p.pool], p.scales * 1
        named.update(k_scales=scales[0], v_scales=scales[1])
        got, _ = G.shared_prefix_attention(args[0] * 1, *pool, *args[3:], **named)
        x = torch.zeros(3, 1000, device="cuda") + 4
        y = G.adjust_logits(x, prompt=ints([7], "cuda"), repetition=2.0)
        kv, sc = torch.zeros(2, 2, 8, 1, 16, dtype=torch.int8, device="cuda"), torch.zeros(2, 2, 1, device="cuda")
        G.append_kv(kv[0], kv[1], *[(torch.ones(1, 1, 16, device="cuda") * 127).to(torch.bfloat16)] * 2, ints([[1]], "cuda"),
                    ints([0], "cuda"), k_scales=sc[0], v_scales=sc[1])
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want) and torch.all(y[:, 7] == 2) and float(y.sum()) == 3 * (999 * 4 + 2)
    assert torch.all(kv[:, 1, 0] == 127) and sc[:, 1].flatten().tolist() == [1, 1]
    settle("cuda")


@pytest.mark.gpu
def test_operators_from_several_threads():
    """Calls of very different sizes at once, each thread on a stream of its own."""
    forms = [(FEW, 128), (WIDE, 128), (RAGGED, 64), (MANY, 32), (WIDE, 64), (FEW, 32)]

    def work(i):
        form, dim = forms[i]
        p = Problem(**form, dim=dim, device="cuda", dtype=TYPES[i % 2], seed=i)
        args, named = p.arguments()
        want, _ = G.shared_prefix_attention(*args, **named)
        x, tokens = torch.randn(3 + 50 * i, 5000, device="cuda"), torch.randint(0, 5000, (40 * i + 1,), device="cuda")
        want_y = G.adjust_logits(x, prompt=tokens, repetition=1.5)
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            got = [G.shared_prefix_attention(*args, **named)[0] for _ in range(30)]
            ys = [G.adjust_logits(x, prompt=tokens, repetition=1.5) for _ in range(30)]
        stream.synchronize()
        return all(torch.equal(t, want) for t in got) and all(torch.equal(t, want_y) for t in ys)

    with ThreadPoolExecutor(3) as pool:
        assert all(pool.map(work, range(len(forms))))
    settle("cuda")


@pytest.mark.gpu
def test_two_graphs_of_attention_replayed_in_turn():
    runs = []
    for i, (form, dim) in enumerate([(WIDE, 128), (RAGGED, 64), (FEW, 128)]):
        p = Problem(**form, dim=dim, device="cuda", dtype=TYPES[i % 2], seed=i)
        args, named = p.arguments()
        want = G.shared_prefix_attention(*args, **named)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = G.shared_prefix_attention(*args, **named)
        runs.append((graph, out, want, p, args, named))  # (a graph reads its inputs where they were: they stay)
    for turn in range(3):
        for graph, out, *_ in runs:
            for t in out:
                t.fill_(math.nan)
            graph.replay()
        for _, out, want, *_ in runs:
            assert all(torch.equal(a, b) for a, b in zip(out, want))
    settle("cuda")


@pytest.mark.gpu
def test_launch_counts_of_the_forms_of_a_call():
    from mini_nccl_b200.utils import launches

    def kernels(call):
        before = launches.count()
        call()
        return launches.count() - before

    def attention(form, **more):
        p = Problem(**form, dim=64, device="cuda", dtype=torch.int8)
        return kernels(lambda: p.run(**more))

    assert attention(FEW) == attention(MANY) == attention(RAGGED) == 2  # pieces, join
    assert attention(WIDE) == 3  # own pieces, the prefix on tensor cores, join
    x = torch.zeros(2, 9, device="cuda")
    assert kernels(lambda: G.adjust_logits(x)) == 1 and kernels(lambda: G.adjust_logits(x[:0])) == 0
    kv, sc = torch.zeros(2, 2, 8, 1, 16, dtype=torch.int8, device="cuda"), torch.zeros(2, 2, 1, device="cuda")
    k = torch.zeros(3, 1, 16, dtype=torch.bfloat16, device="cuda")
    for n, want in ((3, 1), (0, 0)):
        assert kernels(lambda: G.append_kv(kv[0], kv[1], k[:n], k[:n], ints([[0]], "cuda"), ints([0, 1, 2][:n], "cuda"),
                                           ints([0, 0, 0][:n], "cuda"), k_scales=sc[0], v_scales=sc[1])) == want


# ---- as generation uses them -------------------------------------------------------------


def decode_step(c, w, tokens, step, history, masks, noise, prefix, prefix_len, slots, ones):
    """One token of every sequence through a layer that is a table of queries, keys and values."""
    G.reserve_pages(c.page_table, c.lens, c.refs, slots, ones, c.page_size)
    q, k, v = w[tokens].unbind(1)
    table, lens = c.page_table[slots.long()], c.lens[slots.long()]
    c.append(0, k, v, lens - 1, slots)
    y = G.shared_prefix_attention(q, c.kv[0, 0], c.kv[0, 1], prefix, prefix_len, table, lens, **c.scales_of(0))
    logits = G.adjust_logits(y.flatten(1) @ w[:, 0].flatten(1).t(), history=history, history_lens=step, repetition=1.3, presence=0.5,
                             frequency=0.25, allowed=masks)
    token = G.sample(logits, noise, temperature=0.7, top_k=20)
    history.scatter_(1, step.long()[:, None], token[:, None])
    step += 1
    tokens.copy_(token)
    return logits


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
def test_a_run_of_the_operators(device, dtype):
    """Reserve, append, attend, adjust and draw, step by step; on the GPU a captured step gives what the calls give, and each
    step agrees with the plain implementations on the same cache."""
    n, heads, dim, V, P, steps = 5, 2, 64, 100, 37, 20
    gen = torch.Generator().manual_seed(3)
    w = torch.randn(V, 3, heads, dim, generator=gen).to(torch.bfloat16).to(device)
    noise = -(-torch.rand(n, V, generator=gen).clamp(1e-6, 1 - 1e-6).log()).log().to(device)
    bits = torch.rand(1, V, generator=gen) < 0.8
    masks = words_of(bits).to(device)

    def fresh():
        c = G.PagedKVCache(1, 24, 8, heads, dim, max_seqs=n + 1, max_seq_len=40, device=device, dtype=dtype)
        c.extend([0], [P])
        k, v = tokens_of(P, heads, dim, device, 8)
        c.append(0, k, v, ints(list(range(P)), device), ints([0] * P, device))
        state = dict(tokens=torch.arange(n, device=device), step=ints([0] * n, device), history=torch.full((n, steps + 1), -1, device=device))
        return c, state, dict(masks=masks, noise=noise, prefix=c.page_table[0, :5].clone(), prefix_len=P,
                              slots=ints(list(range(1, n + 1)), device), ones=ints([1] * n, device))

    c, state, fixed = fresh()
    for t in range(steps):
        before = {k: x.clone() for k, x in state.items()}
        got = decode_step(c, w, **state, **fixed)
        settle(device)
        assert c.lens.tolist() == [P] + [t + 1] * n
        for b in range(n):  # the step in 64 bits, from what the cache holds
            ids = torch.cat([fixed["prefix"], c.page_table[b + 1, : -(-(t + 1) // 8)]]).long().cpu()
            held = [values_of(c.kv[0, i], c.scales[0, i])[ids] for i in (0, 1)]
            k, v = (torch.cat([x[:5].flatten(0, 1)[:P], x[5:].flatten(0, 1)[: t + 1]]).transpose(0, 1) for x in held)
            q = w[before["tokens"][b], 0].cpu().double()
            s = torch.einsum("hd,hkd->hk", q, k) * dim ** -0.5
            p = torch.softmax(s, -1)[..., None]
            o = (p * v).sum(1)
            off = (2.0 ** -8 * o.abs() + (2.0 ** -11 + 2 * dim * U * 40) * (p * v.abs()).sum(1)).flatten()
            table = w[:, 0].flatten(1).cpu().double()
            x = table @ o.flatten()
            # the products' own rounding to bf16, and fp32 sums
            room = table.abs() @ off + 2.0 ** -8 * x.abs() + 130 * U * (table.abs() @ o.abs().flatten())
            want, more = adjusted(x, [], [int(i) for i in before["history"][b] if i >= 0], float(torch.tensor(1.3)), 0.5, 0.25, {}, bits[0])
            off = (got[b].cpu().double() - want).abs()[bits[0]]
            assert torch.all(off <= (1.3 * 1.01 * room + more + 2.0 ** -8 * want.abs())[bits[0]])
            assert torch.all(got[b].cpu()[~bits[0]] == -math.inf)
    assert bool(bits[0][state["history"][:, :steps].cpu()].all())
    if device == "cpu":
        return
    want = state["history"].clone()
    c, state, fixed = fresh()
    decode_step(c, w, **state, **fixed)  # (warm)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        decode_step(c, w, **state, **fixed)
    for _ in range(steps - 1):
        graph.replay()
    settle(device)
    assert torch.equal(state["history"], want)


def rounded_cache(dtype, plain=G.PagedKVCache):
    """A cache in the model's type that holds what one of ``dtype`` would."""

    class Cache(plain):
        codes = None

        def append(self, layer, k, v, positions, slots=None):
            if self.codes is None:
                L, _, pages, page, heads, dim = self.kv.shape
                self.codes = plain(L, pages, page, heads, dim, max_seqs=1, max_seq_len=1, device="cpu", dtype=dtype)
            c = self.codes
            G.append_kv(c.kv[layer, 0], c.kv[layer, 1], k.cpu(), v.cpu(), self.page_table.cpu(), positions.cpu(), slots.cpu(),
                        **c.scales_of(layer))
            for i in (0, 1):
                self.kv[layer, i] = values_of(c.kv[layer, i], c.scales[layer, i]).to(self.kv.dtype).to(self.kv.device)

    return Cache


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
def test_generation_with_the_cache_in_8_bits(device, dtype, monkeypatch):
    """The logits are those over a cache of the rounded keys and values: on the CPU to the bit; on the GPU both are bf16
    networks, whose roundings differ, and a key or value of the second layer may fall on the next code (off by 2^-3 of itself
    at most, few of them): 1e-1 of the largest logit."""
    m = model_on(device)
    prompt = torch.arange(20, device=device)
    state = BranchedGeneration(m, prompt, max_branches=3, max_new_tokens=30, cache_dtype=dtype)
    assert state.cache.kv.dtype == dtype
    monkeypatch.setattr(G, "PagedKVCache", rounded_cache(dtype))
    other = BranchedGeneration(m, prompt, max_branches=3, max_new_tokens=30)
    for s in (state, other):
        s.select([0] * 3)
    gen = torch.Generator().manual_seed(2)
    for _ in range(25):
        tokens = torch.randint(0, 96, (3,), generator=gen).to(device)
        a, b = state.step(tokens), other.step(tokens)
        if device == "cpu":
            assert torch.equal(a, b)
        else:
            assert torch.all((a.float() - b.float()).abs() <= 0.1 * b.float().abs().max())
    settle(device)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [None, *TYPES])
def test_sampled_continuations_follow_penalties_and_masks(device, dtype):
    m = model_on(device)
    prompt = torch.arange(20, device=device)

    def draw(**more):
        gen = torch.Generator(device=device).manual_seed(5)
        out = sample_continuations(m, prompt, 6, 30, generator=gen, cache_dtype=dtype, **more)
        settle(device)
        return out

    plain, _ = draw()
    assert torch.equal(plain, draw(repetition=1.0)[0])
    once, _ = draw(frequency=1e9)  # nothing twice
    assert all(len(set(row)) == 30 for row in once.tolist())
    new, _ = draw(repetition=1e9, temperature=0.0)  # what was seen has no positive logit left
    assert not set(new[0, :1].tolist()) & set(range(20))
    bits = torch.zeros(1, 96, dtype=torch.bool)
    bits[0, 40:60] = True
    masked, logprobs = draw(allowed=words_of(bits).to(device), resample_every=7)
    assert torch.all((masked >= 40) & (masked < 60)) and torch.all(logprobs > -math.inf)

    def even_then_odd(tokens):  # a mask for each branch from what it has
        rows = torch.zeros(6, 96, dtype=torch.bool)
        last = tokens[:, -1].cpu() if tokens.shape[1] else torch.zeros(6)
        for r in range(6):
            rows[r, int(1 - last[r] % 2)::2] = True
        return words_of(rows).to(device)

    turns, _ = draw(allowed=even_then_odd)
    assert torch.all(turns[:, 0] % 2 == 1) and torch.all(turns[:, 1:] % 2 != turns[:, :-1] % 2)
    biased, _ = draw(bias_tokens=torch.tensor([7], device=device), bias=torch.tensor([1e6], device=device))
    assert torch.all(biased == 7)


def test_generation_refusals():
    m = model_on("cpu")
    for bad in (torch.float16, torch.uint8, torch.float8_e5m2):
        with pytest.raises(ValueError, match="cache_dtype"):
            BranchedGeneration(m, torch.arange(9), max_branches=1, max_new_tokens=2, cache_dtype=bad)
    for bad in (0.0, -1.0, math.nan):
        with pytest.raises(ValueError, match="repetition"):
            sample_continuations(m, torch.arange(9), 2, 2, repetition=bad)
    assert BranchedGeneration(m, torch.arange(9), max_branches=1, max_new_tokens=2, cache_dtype=torch.float32).cache.scales is None


@pytest.mark.examples
@pytest.mark.parametrize("device", DEVICES)
def test_example(device):
    command = [sys.executable, "examples/sample_gpt.py", "--device", device, "--steps", "2", "--n-layer", "2", "--branches", "5",
               "--new-tokens", "24", "--resample-every", "8", "--cache-dtype", "e4m3", "--repetition", "1.2", "--frequency", "0.1",
               "--only", "abcdefgh "]
    run = subprocess.run(command, cwd=Path(__file__).resolve().parent.parent, capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stdout[-2000:] + run.stderr[-2000:]
    assert "sampled 5 continuations of 24 tokens" in run.stdout
