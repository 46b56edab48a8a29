"""Edges of the generation operators: special values, damaged requests, bounds, and forms that few calls reach.

The references are in 64 bits; tolerances as in ``test_generation.py``.
"""

from __future__ import annotations

import math

import pytest
import torch

from mini_nccl_b200.ops import generation as G
from test_generation import DEVICES, Books, Problem, ints, logits_of, settle


def out_of_range(device, call, match="outside its tensor"):
    """The call raises (CPU), or is reported afterwards (GPU); returns what it returned on the GPU."""
    if device == "cpu":
        with pytest.raises((RuntimeError, IndexError)):
            call()
        return None
    from mini_nccl_b200.ops import kernels as K

    out = call()
    with pytest.raises(RuntimeError, match=match):
        K.check_status()
    return out


# ---- tokens that are none ----------------------------------------------------------------


@pytest.mark.gpu
def test_embedding_reports_ids_outside_the_table():
    from mini_nccl_b200.ops import kernels as K

    wte = torch.randn(40, 24, device="cuda").to(torch.bfloat16).requires_grad_()
    wpe = torch.randn(4, 24, device="cuda").to(torch.bfloat16).requires_grad_()
    idx = torch.tensor([[3, -1, 39, 40], [1 << 40, 0, -(1 << 50), 7]], device="cuda")
    y = out_of_range("cuda", lambda: K.Embedding.apply(idx, wte, wpe))
    known = (idx >= 0) & (idx < 40)
    want = torch.where(known[..., None], wte[idx.clamp(0, 39)].float(), 0.0) + wpe.float()
    assert torch.equal(y, want.to(torch.bfloat16))
    y.backward(torch.ones_like(y))
    count = torch.bincount(idx[known], minlength=40)
    assert torch.equal(wte.grad.float(), count[:, None].float().expand(40, 24))
    assert torch.all(wpe.grad == 2)
    settle("cuda")


@pytest.mark.parametrize("device", DEVICES)
def test_a_model_of_nan_is_reported(device):
    """Its logits are NaN, nothing can be drawn from them (-1), and -1 is no token that could be fed back."""
    from mini_nccl_b200.models.generation import sample_continuations
    from mini_nccl_b200.models.gpt import GPT

    torch.manual_seed(0)
    m = GPT(96, 64, 2, 2, 64)
    m.blocks[1].proj.bias.data[5] = math.nan
    m = m.to(device, torch.bfloat16) if device == "cuda" else m
    prompt = torch.arange(20, device=device)
    tokens, logprobs = sample_continuations(m, prompt, 3, 1)
    settle(device)
    assert torch.all(tokens == -1) and torch.all(logprobs == -math.inf)
    out = out_of_range(device, lambda: sample_continuations(m, prompt, 3, 5))
    assert out is None or torch.all(out[0] == -1)


# ---- pages -------------------------------------------------------------------------------


@pytest.mark.gpu
def test_page_plans_are_read_when_they_are_there():
    """Calls back to back, each with other requests in the same workspace: a copy named by the last plan would show."""
    page, S, pages = 8, 64, 600
    kv = torch.randn(2, 2, pages, page, 2, 64).to(torch.bfloat16).cuda()
    table, lens, refs = ints([[-1] * 5] * S, "cuda"), ints([0] * S, "cuda"), ints([0] * pages, "cuda")
    G.reserve_pages(table, lens, refs, ints(range(S // 2), "cuda"), ints([9 + i % 20 for i in range(S // 2)], "cuda"), page)
    gen = torch.Generator().manual_seed(0)
    plans = []
    for _ in range(40):
        n = int(torch.randint(1, S // 2, (1,), generator=gen))
        plans.append((torch.randint(0, S // 2, (n,), generator=gen).int().cuda(), (S // 2 + torch.randperm(S // 2, generator=gen)[:n]).int().cuda()))
    parents_of, copies = [], []
    for parents, children in plans:
        G.fork_sequences(kv, table, lens, refs, parents, children)
        rows = table[children.long()].long().clamp(min=0)
        copies.append((kv[:, :, rows].clone(), lens[children.long()].clone()))
        rows = table[parents.long()].long().clamp(min=0)
        parents_of.append(kv[:, :, rows].clone())
        G.free_sequences(table, lens, refs, children)
        table, refs = G.compact_pages(kv, table, refs)
    settle("cuda")
    for (got, n), want in zip(copies, parents_of):
        inside = (torch.arange(5 * page, device="cuda") < n[:, None]).view(1, 1, -1, 5, page, 1, 1)
        assert torch.equal(torch.where(inside, got, 0), torch.where(inside, want, 0))


# ---- attention: memory -------------------------------------------------------------------


@pytest.mark.parametrize("device", DEVICES)
def test_attention_on_a_pool_without_pages(device):
    """No page can be read, not even of the tensor that the pool is a part of."""
    for rows in (3, 60):
        q = torch.randn(rows, 2, 64).to(torch.bfloat16).to(device)
        whole = torch.full((2, 6, 8, 2, 64), math.nan, dtype=torch.bfloat16, device=device)
        for pool in (whole[:, 3:3], torch.empty(2, 0, 8, 2, 64, dtype=torch.bfloat16, device=device)):
            table = ints([[0, -1]] * rows, device)

            def call(prefix, lens):
                return G.shared_prefix_attention(q, pool[0], pool[1], ints([0] * 17, device), prefix, table, ints(lens, device),
                                                 return_lse=True)

            o, lse = call(0, [0] * rows)
            settle(device)
            assert torch.all(o == 0) and torch.all(lse == -math.inf)
            for prefix, lens in ((130, [0] * rows), (0, [1] * rows), (130, [5] * rows)):
                out = out_of_range(device, lambda: call(prefix, lens))
                assert out is None or torch.all(out[0] == 0), "the keys that are not there read as zeros"


@pytest.mark.parametrize("device", DEVICES)
def test_reserve_past_the_range_of_lengths(device):
    """A row whose pages hold more than 2^31 tokens: lengths are int32, so it ends before."""
    page, columns, last = 1 << 20, 2100, (1 << 31) - 1
    table, lens, refs = ints([[-1] * columns], device), ints([last - 50], device), ints([0] * 4, device)
    before = table.clone()
    out_of_range(device, lambda: G.reserve_pages(table, lens, refs, ints([0], device), ints([60], device), page), match=".")
    assert torch.equal(table, before) and lens.tolist() == [last - 50] and refs.tolist() == [0] * 4
    G.reserve_pages(table, lens, refs, ints([0], device), ints([50], device), page)  # up to the last length
    settle(device)
    assert lens.tolist() == [last] and torch.equal(table, before)
    lens.fill_(last - page - 7)
    G.reserve_pages(table, lens, refs, ints([0], device), ints([page], device), page)
    settle(device)
    assert lens.tolist() == [last - 7] and table[0, 2047].item() == 0 and int(refs.sum()) == 1


# ---- models ------------------------------------------------------------------------------


def _sharded_gpt_is_refused(pg):
    from mini_nccl_b200.fsdp import FullyShardedDataParallel
    from mini_nccl_b200.models.generation import BranchedGeneration, sample_continuations
    from mini_nccl_b200.models.gpt import GPT, Block

    torch.manual_seed(0)
    model, prompt = GPT(96, 64, 2, 2, 64), torch.arange(20)
    with torch.no_grad():
        want = model(prompt[None])[0][:, -1]
    plain = GPT(96, 64, 2, 2, 64)
    fsdp = FullyShardedDataParallel(model, pg, unit_cls=Block)
    for m in (model, fsdp):
        with pytest.raises(ValueError, match="Block|blocks"):
            sample_continuations(m, prompt, 2, 1)
        with pytest.raises(ValueError, match="Block|blocks"):
            BranchedGeneration(m, prompt, max_branches=1, max_new_tokens=3)
    plain.load_state_dict(fsdp.full_state_dict(), strict=False)
    assert torch.allclose(BranchedGeneration(plain, prompt, max_branches=1, max_new_tokens=3).logits, want, atol=1e-4)


@pytest.mark.parametrize("ranks", [1, 2])
def test_generation_refuses_a_sharded_model(ranks):
    from mini_nccl_b200.launcher import run

    run(_sharded_gpt_is_refused, ranks)


def test_generation_refuses_blocks_that_do_something_else():
    from mini_nccl_b200.models.generation import BranchedGeneration
    from mini_nccl_b200.models.gpt import GPT, Block

    class Scaled(Block):
        def forward(self, x):
            return super().forward(x) * 0.5

    class Named(Block):
        pass

    class Around(torch.nn.Module):
        def __init__(self, block):
            super().__init__()
            self.block = block

        def forward(self, x):
            return self.block(x)

    for change, ok in ((lambda b: Scaled(64, 2), False), (Around, False), (lambda b: Named(64, 2), True), (lambda b: b, True)):
        m = GPT(96, 64, 2, 2, 64)
        m.blocks[1] = change(m.blocks[1])
        call = lambda: BranchedGeneration(m, torch.arange(9), max_branches=1, max_new_tokens=3)  # noqa: E731
        if not ok:
            with pytest.raises(ValueError, match="Block"):
                call()
            continue
        with torch.no_grad():
            assert torch.allclose(call().logits, m(torch.arange(9)[None])[0][:, -1], atol=1e-4)


# ---- attention: values -------------------------------------------------------------------


# few and many rows of a kv head, prefixes that end inside a tile and behind one
ROWS = [([60, 3, 0], [1, 1, 1], 1, 129), ([40] * 50, [1] * 50, 1, 129), ([70, 90], [60, 90], 2, 333), ([5] * 70, [1] * 70, 4, 256)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dim", [32, 64, 128])
@pytest.mark.parametrize("lens,new,group,prefix", ROWS)
@pytest.mark.parametrize("scale", [0.0, -0.2])
def test_attention_scale_of_zero_and_below(device, dim, lens, new, group, prefix, scale):
    p = Problem(lens, new, kv_heads=2, group=group, dim=dim, page=16, prefix=prefix, device=device)
    p.check(*p.run(scale=scale), scale=scale)


def aligned_problem(device, dim, size, rows, prefix, group=1, lens=None, new=None):
    """Every query and key lies along one direction, so scores are products of two bf16 numbers: +-`size` and near it."""
    lens = [3] * rows if lens is None else lens
    p = Problem(lens, [1] * len(lens) if new is None else new, kv_heads=1, group=group, dim=dim, page=16, prefix=prefix, device=device)
    p.q = torch.zeros_like(p.q)
    p.q[..., 0] = 128.0
    keys = p.pool[0]
    g = torch.Generator().manual_seed(1)
    along = (size / 128 + torch.randn(keys.shape[:3], generator=g).mul_(abs(size) * 2.0 ** -15)).to(torch.bfloat16)
    keys[:] = 0
    keys[..., 0] = along.to(device)
    p.head[0].zero_()
    ids = torch.tensor(p.prefix_pages)
    p.head[0][..., 0] = along[ids].reshape(-1, 1)[:prefix].double()
    for own, row, m in zip(p.own, p.rows, lens):
        own[0].zero_()
        own[0][..., 0] = along[torch.tensor(row[: -(-m // 16)], dtype=torch.long)].reshape(-1, 1)[:m].double()
    return p


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("size", [1.2e4, -1.2e4, 2.9e4, 1.5e5, -3e6, 2e9, 1e12, -1e15, 1e30])
@pytest.mark.parametrize("rows,prefix", [(2, 300), (40, 300), (40, 500), (200, 2100)])
def test_attention_scores_far_from_zero(device, dim, size, rows, prefix):
    # log2 units: size / ln 2.  Beyond 2^14 a step of bf16 is 128 and more, beyond 2^31 one of fp32 is
    p = aligned_problem(device, dim, size, rows, prefix)
    p.check(*p.run(scale=1.0), scale=1.0)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dim", [32, 64, 128])
@pytest.mark.parametrize("rows,prefix", [(3, 140), (3, 0), (50, 140), (50, 0), (50, 1300), (300, 700)])
def test_attention_shows_nan_in_queries_and_visible_keys(device, dim, rows, prefix):
    def fresh():
        return Problem([4] * rows, [1] * rows, kv_heads=2, group=1, dim=dim, page=16, prefix=prefix, device=device)

    p = fresh()
    p.q[1, 1] = math.nan
    o, lse = (t.cpu() for t in p.run())
    assert torch.all(o[1, 1].isnan()) and lse[1, 1].isnan(), "a query of NaN"
    p.q[1, 1] = 0
    rest, rest_lse = (t.cpu() for t in p.run())
    others = torch.ones(rows, 2, dtype=torch.bool)
    others[1, 1] = False
    assert torch.equal(o[others], rest[others]) and torch.equal(lse[others], rest_lse[others])
    # one key of the prefix: every row of its head sees it, wherever it lies in its tile
    for at in range(0, min(prefix, 140), 1 if rows == 50 and dim == 64 else 23):
        p = fresh()
        p.pool[0, p.prefix_pages[at // 16], at % 16, 1, 3] = math.nan
        o, lse = p.run()
        assert torch.all(o[:, 1].isnan()) and torch.all(lse[:, 1].isnan()), at
        assert not o[:, 0].isnan().any() and not lse[:, 0].isnan().any()
    # one key of a sequence's own
    p = fresh()
    p.pool[0, p.rows[2][0], 3, 0, 0] = math.nan
    o, lse = p.run()
    hit = torch.zeros(rows, 2, dtype=torch.bool)
    hit[2, 0] = True
    assert torch.equal(o.isnan().all(-1).cpu(), hit) and torch.equal(lse.isnan().cpu(), hit)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("lens,new,kv_heads,group,dim,page,prefix", [
    ([7, 5], [7, 5], 1, 1, 32, 8, 0),
    ([70, 33, 0, 5], [33, 1, 0, 5], 2, 2, 64, 16, 100),
    ([130, 7, 129], [130, 7, 2], 1, 3, 128, 8, 0),
    ([90, 31], [77, 31], 1, 1, 128, 64, 191),
    ([9 + i % 5 for i in range(230)], [4] * 230, 5, 2, 64, 8, 40),
    ([9 + i % 5 for i in range(230)], [4] * 230, 4, 1, 128, 8, 0),
])
def test_attention_leaves_out_hidden_values(device, bad, lens, new, kv_heads, group, dim, page, prefix):
    """A query's result does not depend on tokens behind it, whatever they hold; those that see the token show it."""
    p = Problem(lens, new, kv_heads=kv_heads, group=group, dim=dim, page=page, prefix=prefix, device=device)
    want, want_lse = (t.cpu() for t in p.run())
    first = torch.tensor([0] + new).cumsum(0).tolist()
    sees = torch.zeros(sum(new), dtype=torch.bool)
    for b, (m, n) in enumerate(zip(lens, new)):
        if n < 2:
            continue
        at = m - n + n // 2  # the place of query n // 2
        page_id = p.rows[b][at // page]
        p.pool[1, page_id, at % page, 0, 1::2] = bad
        p.pool[0, page_id, at % page, kv_heads - 1, 0] = bad  # and its key in another head
        sees[first[b] + n // 2: first[b + 1]] = True
    o, lse = (t.cpu() for t in p.run())
    # (the rows that see it are checked below: here they get what they were without it)
    p.check(torch.where(sees[:, None, None], want, o), torch.where(sees[:, None], want_lse, lse))
    values = o[sees][:, :group] if kv_heads > 1 else o[sees][:0]
    assert not values[..., 1::2].isfinite().any()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dim,prefix", [(32, 0), (32, 40), (64, 0), (64, 40), (64, 3000), (128, 200)])
@pytest.mark.parametrize("offsets,most,limit", [
    ([3, 40, 60, 70], 60, 90),    # the first rows belong to nobody
    ([0, 40, 60, 65], 60, 90),    # nor do the last
    ([0, 50, 40, 70], 60, 90),    # a descent
    ([0, 40, 60, 90], 60, 90),    # past the rows
    ([-4, 40, 60, 70], 60, 90),
    ([0, 40, 60, 70], 25, 90),    # longer than max_q_len
    ([0, 40, 60, 70], 60, 50),    # lengths beyond max_seq_len
    ([0, 40, 60, 70], 60, 0),
    ([0, 40, 69, 70], 60, 0),
])
def test_attention_reports_offsets_and_bounds_that_do_not_hold(device, dim, prefix, offsets, most, limit):
    p = Problem([60, 90, 33], [40, 20, 10], kv_heads=2, group=1, dim=dim, page=16, prefix=prefix, device=device)
    if device == "cuda":  # what the allocator hands out next holds NaN
        stale = torch.full((32 << 20,), math.nan, device=device)
        del stale

    def call():
        return G.shared_prefix_attention(p.q, p.pool[0], p.pool[1], ints(p.prefix_pages, device), prefix, ints(p.rows, device),
                                         ints(p.lens, device), q_offsets=ints(offsets, device), max_q_len=most, max_seq_len=limit,
                                         return_lse=True)

    out = out_of_range(device, call)
    if out is None:
        return
    o, lse = out
    if limit == 90:  # rows without a sequence of their own: the own tokens of the whole call are left out
        p.lens, p.own, p.new = [0] * 3, [t[:, :0] for t in p.own], [40, 20, 10]
        p.check(o, lse)
    else:
        assert not o.isnan().any() and not lse.isnan().any()


@pytest.mark.parametrize("device", DEVICES)
def test_attention_bounds_that_no_call_can_keep(device):
    p = Problem([20, 5], [3, 2], kv_heads=1, group=1, dim=64, page=16, prefix=10, device=device)
    args = (p.q, p.pool[0], p.pool[1], ints(p.prefix_pages, device), 10)
    with pytest.raises(ValueError, match="max_q_len"):
        G.shared_prefix_attention(*args, ints(p.rows, device), ints(p.lens, device), q_offsets=ints([0, 3, 5], device), max_q_len=0)
    with pytest.raises(ValueError, match="q_offsets"):
        G.shared_prefix_attention(*args, torch.empty(0, 2, dtype=torch.int32, device=device), ints([], device),
                                  q_offsets=ints([0], device), max_q_len=5)


@pytest.mark.parametrize("device", DEVICES)
def test_attention_over_the_prefix_alone(device):
    # a bound of 0 with lengths of 0 is a sound request
    for rows in (3, 60):
        p = Problem([0] * rows, [1] * rows, kv_heads=2, group=1, dim=64, page=16, prefix=140, device=device)
        p.check(*p.run(max_seq_len=0))


@pytest.mark.gpu
def test_attention_leaves_out_a_sequence_with_a_bad_length():
    for lens, bound in (([20, -3, 30], 48), ([20, 49, 30], 48)):
        p = Problem([20, 48, 30], [1, 1, 1], kv_heads=2, group=1, dim=64, page=16, prefix=40, device="cuda")
        o, lse = out_of_range("cuda", lambda: G.shared_prefix_attention(
            p.q, p.pool[0], p.pool[1], ints(p.prefix_pages, "cuda"), 40, ints(p.rows, "cuda"), ints(lens, "cuda"), max_seq_len=bound,
            return_lse=True))
        p.lens[1], p.own[1] = 0, p.own[1][:, :0]
        p.check(o, lse)


# ---- status ------------------------------------------------------------------------------


def test_check_status_reports_a_pipeline_and_a_request_at_once(monkeypatch):
    from mini_nccl_b200.ops import kernels as K

    word = torch.zeros(4, dtype=torch.int32)
    monkeypatch.setattr(K, "_STATUS", {0: word})
    K.check_status()
    for value, match in (([2, 0, 4, 0], "pipeline status 2.*too few free pages"), ([2, 0, 0, 0], "pipeline status 2$"),
                         ([0, 0, 5, 0], "^request left out on cuda:0.*outside its tensor")):
        word.copy_(torch.tensor(value))
        with pytest.raises(RuntimeError, match=match):
            K.check_status()
        K.check_status()  # the words were cleared


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("many", [False, True])
@pytest.mark.parametrize("bad", [-1, 10 ** 6, -(1 << 31)])
@pytest.mark.parametrize("column", [0, 1, 2])
def test_fork_of_a_damaged_sequence_is_left_out(device, bad, column, many):
    """A parent whose row names no page of the pool: in the middle, or where the part-filled last page is."""
    lens = [20, 13, 17] + [9] * (300 if many else 2)
    b = Books(device, lens, slots=2 * len(lens), columns=4, pages=1300)
    want = [b.tokens(s) for s in range(len(lens))]
    b.table[2, column] = bad
    table, n, refs = b.table.clone(), b.lens.clone(), b.refs.clone()
    at = len(lens)
    parents = [0, 2, 1] + list(range(3, len(lens)))
    children = list(range(at, 2 * at))
    out_of_range(device, lambda: G.fork_sequences(b.kv, b.table, b.lens, b.refs, ints(parents, device), ints(children, device)))
    assert torch.equal(b.table[:at], table[:at]) and torch.equal(b.lens[:at], n[:at])
    if device == "cpu":
        assert torch.equal(b.table, table) and torch.equal(b.lens, n) and torch.equal(b.refs, refs)
        return
    assert int(b.lens[at + 1]) == 0 and torch.all(b.table[at + 1] == -1)
    for p, c in zip(parents, children):
        if p != 2:
            assert torch.equal(b.tokens(c), want[p])
    held = b.table[(b.table >= 0) & (b.table < 1300)].long()
    missing = torch.bincount(held, minlength=1300).int()
    gap = b.refs - missing
    assert int(gap.sum()) == 1 and int(gap.min()) == 0, "only the page that the damaged row no longer names"


def test_reserve_without_room_changes_nothing_on_the_cpu():
    c = G.PagedKVCache(1, 4, 8, 1, 32, max_seqs=3, max_seq_len=32, device="cpu")
    c.extend([0], [9])
    with pytest.raises(RuntimeError, match="too few free pages"):
        c.extend([1, 2], [16, 8])
    assert c.lengths == [9, 0, 0] and c.lens.tolist() == c.lengths and c.pages_in_use() == 2
    assert torch.all(c.page_table[1:] == -1)
    c.extend([2], [16])
    assert c.lens.tolist() == c.lengths == [9, 0, 16]


@pytest.mark.gpu
def test_gradients_are_refused_not_lost():
    p = Problem([20, 5], [1, 1], kv_heads=2, group=1, dim=64, page=16, prefix=40, device="cuda")
    want, want_lse = p.run()
    p.q = p.q.detach().requires_grad_()
    o, lse = p.run()
    assert torch.equal(o, want) and torch.equal(lse, want_lse) and o.requires_grad and lse.requires_grad
    for out in (o, lse):
        with pytest.raises(RuntimeError, match="no gradient"):
            out.float().sum().backward()
    with torch.no_grad():
        assert not p.run()[0].requires_grad
    x = torch.randn(3, 100, device="cuda", requires_grad=True)
    token, logprob = G.sample(x, torch.zeros(3, 100, device="cuda"), return_logprob=True)
    assert not token.requires_grad and logprob.requires_grad
    with pytest.raises(RuntimeError, match="no gradient"):
        logprob.sum().backward()


# ---- sampling ----------------------------------------------------------------------------


@pytest.mark.gpu
def test_sample_from_several_threads():
    """Rows of very different lengths at once, each thread on a stream of its own: a launch may not lower another's limits."""
    from concurrent.futures import ThreadPoolExecutor

    def work(vocab):
        x, noise = (t.cuda() for t in logits_of(3, vocab, torch.float32, seed=vocab))
        want = G.sample(x, noise, top_p=0.9)
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            got = [G.sample(x, noise, top_p=0.9) for _ in range(60)]
        stream.synchronize()
        return all(torch.equal(t, want) for t in got)

    with ThreadPoolExecutor(4) as pool:
        assert all(pool.map(work, [300, 50304, 9001, 130003, 20000, 40000]))
    settle("cuda")


# ---- counted launches --------------------------------------------------------------------


def test_launch_counts_follow_what_the_extension_says():
    from types import SimpleNamespace

    from mini_nccl_b200.utils import launches

    last = []
    target = SimpleNamespace(sample=lambda n: last.append(n) or n, gelu_fwd=lambda: None, generation_launches=lambda: last[-1])
    proxy = launches.CountingProxy(target)
    before = launches.count()
    assert proxy.sample(3) == 3 and proxy.sample(0) == 0 and proxy.gelu_fwd() is None
    assert launches.count() - before == 4


@pytest.mark.gpu
def test_launch_counts_of_the_forms_of_a_call():
    from mini_nccl_b200.utils import launches

    def kernels(call):
        before = launches.count()
        call()
        return launches.count() - before

    def attention(rows, prefix, lens=5, dim=64, **more):
        p = Problem([lens] * rows, [1] * rows, kv_heads=2, group=1, dim=dim, page=16, prefix=prefix, device="cuda")
        return kernels(lambda: p.run(**more))

    assert attention(3, 40) == 2  # pieces, join
    assert attention(60, 40) == 2  # own pieces, and the prefix on tensor cores, which joins them
    assert attention(60, 9000) == 3  # the prefix in several pieces
    assert attention(60, 40, lens=0, max_seq_len=0) == 2  # the check of the lengths, and the prefix
    assert attention(3, 0, lens=0, max_seq_len=0) == 2  # the check, and the join that writes zeros
    b = Books("cuda", [9, 20], slots=4, columns=4, pages=40)
    assert kernels(lambda: b.fork([0], [2])) == 2 and kernels(lambda: b.fork([], [])) == 0
    assert kernels(lambda: G.compact_pages(b.kv, b.table, b.refs)) == 2
    assert kernels(lambda: G.compact_pages(b.kv, b.table.repeat(1100, 1), b.refs)) == 3
    assert kernels(lambda: G.copy_pages(b.kv, ints([], "cuda"), ints([], "cuda"))) == 0
    x = torch.zeros(2, 9, device="cuda")
    assert kernels(lambda: G.sample(x, x)) == 1 and kernels(lambda: G.sample(x[:0], x[:0])) == 0


# ---- forms that few calls reach ----------------------------------------------------------

@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("lens,new,kv_heads,group,dim,page,prefix", [
    # more sequences than a block keeps the lengths of
    ([i % 23 for i in range(1100)], [1] * 1100, 1, 1, 64, 8, 40),
    ([i % 9 for i in range(1030)], [i % 3 for i in range(1030)], 2, 1, 32, 8, 0),
    # four kv heads to a piece at head dim 32, the last of them fewer
    ([(3 * i) % 31 for i in range(300)], [1] * 300, 7, 1, 32, 8, 0),
    ([(3 * i) % 31 for i in range(300)], [1] * 300, 4, 4, 32, 64, 0),
])
def test_attention_many_sequences(device, lens, new, kv_heads, group, dim, page, prefix):
    p = Problem(lens, new, kv_heads=kv_heads, group=group, dim=dim, page=page, prefix=prefix, device=device)
    p.check(*p.run())


@pytest.mark.gpu
@pytest.mark.parametrize("lens,new,kv_heads,group,dim,prefix", [
    ([17, 300, 5, 90], [1] * 4, 12, 1, 64, 300),
    ([(11 * i) % 400 for i in range(96)], [1] * 96, 8, 1, 128, 3000),
    ([(11 * i) % 700 for i in range(16)], [1] * 16, 8, 4, 128, 9000),
    ([200, 77, 300, 150], [200, 60, 150, 1], 4, 2, 128, 1500),
    ([4] * 200, [1] * 200, 8, 1, 64, 64),
])
def test_attention_repeats_itself_to_the_bit(lens, new, kv_heads, group, dim, prefix):
    p = Problem(lens, new, kv_heads=kv_heads, group=group, dim=dim, page=16, prefix=prefix, device="cuda")
    o, lse = p.run()
    for _ in range(10):
        again, lse_again = p.run()
        assert torch.equal(again, o) and torch.equal(lse_again, lse)


@pytest.mark.gpu
def test_attention_exponential_on_the_fma_pipe():
    """The polynomial is off by 1.1e-7 at most; its last rounding adds 2^-24 and the earlier ones together less than 2^-25."""
    from mini_nccl_b200.ops import kernels as K

    x = torch.cat([torch.linspace(-126, 20, 1 << 20), torch.arange(-126.0, 20), torch.tensor([-126.5, -1e30, -math.inf, -0.0])]).cuda()
    y = torch.empty_like(x)
    K.ext().prefix_exp2_eval(x, y)
    want = torch.exp2(x.double().clamp(min=-126))
    assert float(((y.double() - want).abs() / want).max()) <= 1.1e-7 + 2.0 ** -24 + 2.0 ** -25
    whole = y[1 << 20: -4]
    assert torch.equal(whole, torch.exp2(torch.arange(-126.0, 20).double()).float().cuda()), "exact at whole numbers"


# ---- the embedding's other arguments -----------------------------------------------------


@pytest.mark.gpu
def test_embedding_of_strided_ids_and_of_too_many_positions():
    from mini_nccl_b200.ops import kernels as K

    wte = torch.randn(40, 24, device="cuda").to(torch.bfloat16).requires_grad_()
    wpe = torch.randn(6, 24, device="cuda").to(torch.bfloat16).requires_grad_()
    flat = torch.arange(12, device="cuda")
    for idx in (flat.view(4, 3).t(), flat[:4].expand(3, 4), flat.view(3, 4)[:, ::2]):
        wte.grad = None
        K.Embedding.apply(idx, wte, wpe).sum().backward()
        count = torch.bincount(idx.reshape(-1), minlength=40)
        assert torch.equal(wte.grad.float(), count[:, None].float().expand(40, 24))
    with pytest.raises(RuntimeError, match="positions"):
        K.Embedding.apply(flat.view(1, 12), wte, wpe)
    settle("cuda")


# ---- after an error ----------------------------------------------------------------------


@pytest.mark.parametrize("device", DEVICES)
def test_a_step_that_was_refused_changes_nothing(device):
    from mini_nccl_b200.models.generation import BranchedGeneration
    from mini_nccl_b200.models.gpt import GPT

    torch.manual_seed(0)
    m = GPT(96, 64, 2, 2, 64)
    m = m.to(device, torch.bfloat16) if device == "cuda" else m
    prompt, good = torch.arange(20, device=device), torch.tensor([5], device=device)
    # a dtype that the embedding does not take, and (seen on the CPU only) a token that is none
    for bad in [good.float()] + ([good + 1000] if device == "cpu" else []):
        states = [BranchedGeneration(m, prompt, max_branches=1, max_new_tokens=4) for _ in range(2)]
        with pytest.raises((RuntimeError, IndexError)):
            states[0].step(bad)
        assert states[0].length == 0 and states[0].cache.lengths == [20, 0] and states[0].cache.lens.tolist() == [20, 0]
        assert torch.equal(states[0].step(good), states[1].step(good))
    settle(device)


# ---- sizes at the ends of their types ----------------------------------------------------


@pytest.mark.parametrize("device", DEVICES)
def test_sample_top_k_beyond_32_bits_keeps_all(device):
    x, noise = (t.to(device) for t in logits_of(2, 300, torch.float32, seed=1))
    want = G.sample(x, noise)
    for k in (1 << 40, (1 << 31) - 1, 300, 0, -1, -(1 << 40)):
        assert torch.equal(G.sample(x, noise, top_k=k), want)


@pytest.mark.parametrize("device", DEVICES)
def test_single_entries_of_strided_tensors(device):
    """An axis of one entry has any stride: a column of a wider table, an entry of a wider list."""
    p = Problem([7], [1], kv_heads=2, group=1, dim=64, page=8, prefix=5, device=device)
    want, _ = p.run()
    table = ints([[p.rows[0][0], 9, 9]] * 2, device)
    lens, prefix = ints([7, 0, 3, 0], device), ints([p.prefix_pages[0], 4, 4], device)
    got = G.shared_prefix_attention(p.q, p.pool[0], p.pool[1], prefix[::3], 5, table[:1, ::3], lens[::4])
    assert torch.equal(got, want)
    settle(device)
