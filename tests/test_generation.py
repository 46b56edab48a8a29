"""The generation operators against plain 64-bit implementations, on CPU and (marked gpu) on the kernels.

Tolerances follow from the arithmetic: outputs are rounded to bf16 once
(2^-9 of the value) and the probabilities once (2^-9 of each, so 2^-9 of the
softmax average of |v|); a score is an fp32 sum of D products of bf16 values,
off by at most D 2^-24 sum |q_i k_i|.
"""

from __future__ import annotations

import math
import random

import pytest
import torch

from mini_nccl_b200.ops import generation as G

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
U = 2.0 ** -24


def ints(values, device):
    return torch.tensor(values, dtype=torch.int32, device=device)


def settle(device):
    if device == "cuda":
        from mini_nccl_b200.ops import kernels as K

        torch.cuda.synchronize()
        K.check_status()


# ---- attention -------------------------------------------------------------------------


class Problem:
    """A shared prefix, ragged own lengths and their pages in a pool whose other places hold NaN."""

    def __init__(self, lens, new, *, kv_heads, group, dim, page, prefix, device, seed=0, scale_q=1.0, heads_first=False):
        rng, gen = random.Random(seed), torch.Generator().manual_seed(seed)
        B, H = len(lens), kv_heads * group
        n_prefix = -(-prefix // page)
        need = n_prefix + sum(-(-m // page) for m in lens)
        ids = list(range(need + 3))
        rng.shuffle(ids)
        pool = torch.full((2, len(ids), page, kv_heads, dim), math.nan, dtype=torch.bfloat16)
        self.prefix_pages, at = ids[:n_prefix], n_prefix
        columns = max(1, -(-max(lens) // page))
        self.rows = []
        for m in lens:
            k = -(-m // page)
            self.rows.append(ids[at:at + k] + [-1] * (columns - k))
            at += k

        def fill(pages, n):
            data = torch.randn(2, n, kv_heads, dim, generator=gen).to(torch.bfloat16)
            for t in range(n):
                pool[:, pages[t // page], t % page] = data[:, t]
            return data.double()

        self.head = fill(self.prefix_pages, prefix)
        self.own = [fill(r, m) for r, m in zip(self.rows, lens)]
        self.lens, self.new, self.prefix, self.dim, self.group = lens, new, prefix, dim, group
        wide = (torch.randn(sum(new), (H + 1) * dim, generator=gen) * scale_q).to(torch.bfloat16).to(device)
        self.q = wide[:, dim:].view(-1, H, dim)  # a slice of a wider projection
        pool = pool.to(device)
        if heads_first:
            pool = pool.transpose(2, 3).contiguous().transpose(2, 3)
        self.pool = pool
        self.device = device

    def run(self, **more):
        offsets = None
        if any(n != 1 for n in self.new):
            offsets = ints([sum(self.new[:i]) for i in range(len(self.new) + 1)], self.device)
            more.setdefault("max_q_len", max(self.new))
        out = G.shared_prefix_attention(
            self.q, self.pool[0], self.pool[1], ints(self.prefix_pages, self.device), self.prefix,
            ints(self.rows, self.device), ints(self.lens, self.device), q_offsets=offsets, return_lse=True, **more)
        settle(self.device)
        return out

    def check(self, o, lse, scale=None):
        scale = self.dim ** -0.5 if scale is None else scale
        q, at = self.q.cpu().double(), 0
        o, lse = o.cpu().double(), lse.cpu().double()
        for m, n, own in zip(self.lens, self.new, self.own):
            k, v = torch.cat([self.head, own], 1).repeat_interleave(self.group, 2).transpose(1, 2)
            for t in range(n):
                seen = self.prefix + max(0, m - n + 1 + t)
                qt = q[at]
                if not seen:
                    assert torch.all(o[at] == 0) and torch.all(lse[at] == -math.inf)
                else:
                    s = torch.einsum("hd,hkd->hk", qt, k[:, :seen]) * scale
                    p = torch.softmax(s, -1)[..., None]
                    want, spread = (p * v[:, :seen]).sum(1), (p * v[:, :seen].abs()).sum(1)
                    off = self.dim * U * (torch.einsum("hd,hkd->hk", qt.abs(), k[:, :seen].abs()) * abs(scale)).amax(-1) \
                        + 8 * U * s.abs().amax(-1) + 2.0 ** -20
                    assert torch.all((lse[at] - torch.logsumexp(s, -1)).abs() <= off)
                    bound = 2.0 ** -8 * want.abs() + (2.0 ** -8 + 2 * off[:, None]) * spread
                    assert torch.all((o[at] - want).abs() <= bound), ((o[at] - want).abs() - bound).max()
                at += 1


SHAPES = [
    # lens, new, kv_heads, group, dim, page, prefix
    ([1], [1], 1, 1, 32, 8, 1),
    ([3, 17, 1], [1] * 3, 2, 1, 64, 16, 0),
    ([65, 0, 64, 63, 1], [1] * 5, 3, 4, 64, 8, 63),
    ([64, 128], [1, 1], 2, 8, 128, 64, 64),
    ([200 - 11 * i for i in range(17)], [1] * 17, 2, 5, 128, 32, 129),
    ([i % 41 for i in range(70)], [1] * 70, 1, 1, 64, 16, 515),
    ([0, 0], [1, 1], 1, 2, 64, 16, 33),
    ([70, 33, 0, 5], [33, 1, 0, 5], 2, 2, 64, 16, 100),
    ([130, 7, 129], [130, 7, 2], 1, 3, 128, 8, 0),
    ([300, 64, 65], [64, 64, 17], 2, 1, 32, 256, 257),
    ([9, 9], [9, 4], 4, 1, 128, 16, 1000),
    ([2, 0], [5, 3], 1, 1, 64, 8, 0),  # more queries than tokens: the first ones see nothing
    ([700], [1], 1, 1, 128, 16, 5),
    ([40] * 9, [30] * 9, 1, 1, 128, 16, 400),  # 270 rows
    ([3] * 150, [1] * 150, 2, 1, 64, 32, 2000),
    ([31, 90, 500], [31, 77, 200], 1, 4, 64, 64, 191),
    # many short sequences: four kv heads at a time, the last of them fewer
    ([i % 37 for i in range(230)], [1] * 230, 13, 1, 64, 8, 70),
    ([(7 * i) % 50 for i in range(225)], [1] * 225, 16, 2, 128, 32, 0),
    ([(5 * i) % 21 for i in range(450)], [i % 3 for i in range(450)], 6, 3, 32, 16, 40),
]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("lens,new,kv_heads,group,dim,page,prefix", SHAPES)
def test_attention(device, lens, new, kv_heads, group, dim, page, prefix):
    p = Problem(lens, new, kv_heads=kv_heads, group=group, dim=dim, page=page, prefix=prefix, device=device)
    p.check(*p.run())


@pytest.mark.parametrize("device", DEVICES)
def test_attention_layouts_and_bounds(device):
    shape = dict(kv_heads=3, group=2, dim=64, page=16, prefix=77, device=device)
    p = Problem([20, 5, 64], [4, 5, 1], heads_first=True, **shape)
    o, lse = p.run(max_seq_len=64, scale=0.3)
    p.check(o, lse, scale=0.3)
    again, _ = p.run(max_seq_len=64, scale=0.3)
    assert torch.equal(o, again)
    alone = G.shared_prefix_attention(
        p.q, p.pool[0], p.pool[1], ints(p.prefix_pages, device), p.prefix, ints(p.rows, device), ints(p.lens, device),
        q_offsets=ints([0, 4, 9, 10], device), max_q_len=5, max_seq_len=64, scale=0.3)
    assert torch.equal(o, alone)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("scale_q", [0.0, 40.0])
def test_attention_flat_and_steep_scores(device, scale_q):
    for new in ([1, 1, 1], [50, 3, 90]):
        p = Problem([60, 3, 90], new, kv_heads=2, group=1, dim=128, page=16, prefix=333, device=device, scale_q=scale_q)
        p.check(*p.run())


@pytest.mark.parametrize("device", DEVICES)
def test_attention_no_rows(device):
    empty = torch.empty(0, 4, 64, dtype=torch.bfloat16, device=device)
    pool = torch.zeros(2, 4, 8, 4, 64, dtype=torch.bfloat16, device=device)
    o = G.shared_prefix_attention(empty, pool[0], pool[1], ints([1], device), 3, torch.empty(0, 2, dtype=torch.int32, device=device),
                                  ints([], device))
    assert o.shape == (0, 4, 64)


@pytest.mark.parametrize("device", DEVICES)
def test_attention_refusals(device):
    def call(q=(2, 4, 64), pages=(4, 8, 2, 64), ids=2, prefix=9, table=(2, 2), lens=2, **more):
        z = lambda *s: torch.zeros(*s, dtype=torch.bfloat16, device=device)  # noqa: E731
        i = lambda *s: torch.zeros(*s, dtype=torch.int32, device=device)  # noqa: E731
        kv = z(2, *pages)
        return G.shared_prefix_attention(z(*q), kv[0], kv[1], i(ids), prefix, i(*table), i(lens), **more)

    call()
    for bad in (dict(q=(2, 4, 48), pages=(4, 8, 2, 48)), dict(pages=(4, 8, 3, 64)), dict(pages=(4, 12, 2, 64)),
                dict(pages=(4, 8, 2, 128)), dict(prefix=17), dict(prefix=-1), dict(lens=3), dict(q=(3, 4, 64)),
                dict(max_seq_len=17), dict(q_offsets=ints([0, 2], device), max_q_len=2),
                dict(q_offsets=ints([0, 1, 2], device)), dict(q_offsets=torch.zeros(3, device=device), max_q_len=1)):
        with pytest.raises(ValueError):
            call(**bad)


@pytest.mark.gpu
def test_attention_reports_bad_pages_and_lengths_without_reading_them():
    from mini_nccl_b200.ops import kernels as K

    p = Problem([20, 30], [1, 1], kv_heads=1, group=1, dim=64, page=16, prefix=40, device="cuda")
    args = [p.q, p.pool[0], p.pool[1], ints(p.prefix_pages, "cuda"), p.prefix, ints(p.rows, "cuda"), ints(p.lens, "cuda")]
    for i, bad in ((3, [10 ** 6, -5, 0]), (5, [[-1, 2], [10 ** 6, 1]]), (6, [-3, 10 ** 6])):
        G.shared_prefix_attention(*args[:i], ints(bad, "cuda"), *args[i + 1:])
        with pytest.raises(RuntimeError, match="outside its tensor"):
            K.check_status()


@pytest.mark.gpu
def test_attention_beyond_32_bit_offsets():
    page, heads, dim = 256, 16, 128
    pages = (1 << 31) // (page * heads * dim) + 40  # ids whose first element lies past 2^31
    pool = torch.empty(2, pages, page, heads, dim, dtype=torch.bfloat16, device="cuda")
    small = Problem([300, 2], [1, 1], kv_heads=heads, group=1, dim=dim, page=page, prefix=700, device="cuda")
    base = pages - small.pool.shape[1]
    pool[:, base:] = small.pool
    o, lse = G.shared_prefix_attention(
        small.q, pool[0], pool[1], ints(small.prefix_pages, "cuda") + base, small.prefix, ints(small.rows, "cuda") + base,
        ints(small.lens, "cuda"), return_lse=True)
    settle("cuda")
    small.check(o, lse)


@pytest.mark.gpu
def test_operators_follow_the_current_stream():
    p = Problem([60, 3], [1, 1], kv_heads=2, group=1, dim=64, page=16, prefix=333, device="cuda")
    want, _ = p.run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)  # what the side stream computes is late for every other stream
        pool = p.pool * 1
        q = p.q * 1
        got = G.shared_prefix_attention(q, pool[0], pool[1], ints(p.prefix_pages, "cuda"), p.prefix, ints(p.rows, "cuda"),
                                        ints(p.lens, "cuda"))
        x = torch.zeros(3, 1000, device="cuda").index_fill_(1, torch.tensor([7], device="cuda"), 9.0)
        token = G.sample(x, torch.zeros_like(x))
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want) and token.tolist() == [7, 7, 7]


# ---- sampling --------------------------------------------------------------------------


def reference_sample(x, noise, T, k, p, least, slack=0.0):
    """(token, log-probability) of one row, from the definition in 64 bits; the scores are the fp32 ones.

    ``slack`` moves the mass that top-p keeps by that share of itself."""
    order = torch.argsort(torch.where(x.isnan(), -math.inf, x), descending=True, stable=True)
    order = order[x[order] > -math.inf]
    if not len(order):
        return -1, -math.inf
    if not T > 0:
        return int(order[0]), 0.0
    if 0 < k < len(x):
        order = order[:k]
    top = x[order[0]]

    def power(v):
        return torch.where(v == top, 0.0, (v - top) / T)

    w = torch.exp(power(x[order]))
    before = torch.cumsum(w, 0) - w
    keep = (w >= least) & ((before < p * (1 + slack) * w.sum()) if p < 1 else True)
    keep[0] = True
    kept = order[keep].sort().values
    score = x[kept].float() / torch.tensor(T, dtype=torch.float32) + noise[kept]
    score = torch.where(score.isnan(), -math.inf, score)
    best = kept[score == score.max()][0]
    return int(best), float(power(x[best]) - torch.log(w[keep].sum()))


def check_sample(device, x, noise, T, k, p, least, tensors=True):
    R = x.shape[0]
    lists = [[v] * R if not isinstance(v, list) else v for v in (T, k, p, least)]
    f = lambda v: torch.tensor(v, dtype=torch.float32, device=device)  # noqa: E731
    if tensors:
        settings = dict(temperature=f(lists[0]), top_k=ints(lists[1], device), top_p=f(lists[2]), min_p=f(lists[3]))
    else:
        settings = dict(temperature=T, top_k=k, top_p=p, min_p=least)
    token, logprob = G.sample(x.to(device), noise.to(device), return_logprob=True, **settings)
    assert torch.equal(token, G.sample(x.to(device), noise.to(device), **settings))
    rows = x.double()
    r32 = lambda v: float(torch.tensor(v, dtype=torch.float32))  # noqa: E731
    for r in range(R):
        a, b, c, d = (v[r] for v in lists)
        want, lp = reference_sample(rows[r], noise[r], r32(a), b, r32(c), r32(d))
        got = float(logprob[r])
        # weights: two roundings of the exponent (at most 64 here) and one of the power; sums of at most V terms in blocks
        if int(token[r]) == want and (got == lp or abs(got - lp) <= 2e-5 + 4 * U * abs(lp)):
            continue
        # top-p compares two fp32 sums: where a token lies within their rounding (16 of them) of the cut, either side is right
        near = [reference_sample(rows[r], noise[r], r32(a), b, r32(c), r32(d), slack) for slack in (-16 * U, 16 * U)]
        assert int(token[r]) in [i for i, _ in near], (r, int(token[r]), want)
        assert min(v for _, v in near) - 2e-5 <= got <= max(v for _, v in near) + 2e-5, (r, got, lp, near)


def logits_of(rows, vocab, dtype, seed, spread=3.0):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, vocab, generator=g) * spread).to(dtype)
    noise = -torch.empty(rows, vocab).exponential_(generator=g).log()
    return x, noise


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [1, 2, 31, 1000, 4097, 50304])
def test_sample_filters(device, dtype, vocab):
    T, k = [1.0, 0.7, 0.0, 1.3, 1.0, 0.5, 2.0, 1.0], [0, 1, 5, 40, 0, 700, 0, 3]
    p, least = [1.0, 1.0, 0.5, 0.9, 0.95, 0.99, 0.3, 0.0], [0.0, 0.0, 0.0, 0.0, 0.0, 0.01, 0.2, 0.0]
    x, noise = logits_of(8, vocab, dtype, seed=vocab)
    check_sample(device, x, noise, T, k, p, least)
    check_sample(device, x[:2], noise[:2], 0.8, 50, 0.9, 0.001, tensors=False)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("spread", [0.0, 0.02, 1.0, 30.0])
def test_sample_ties_flat_and_steep_rows(device, dtype, spread):
    x, noise = logits_of(6, 9001, dtype, seed=5, spread=spread)
    x = (x * 4).round() / 4 if spread else x  # equal logits everywhere
    check_sample(device, x, noise, [1.0, 1.0, 0.9, 1.0, 1.1, 3.0], [0, 4444, 0, 17, 8000, 0], [0.37, 1.0, 0.999, 0.5, 0.83, 1.0],
                 [0.0, 0.0, 0.0, 0.0, 0.0, 0.5])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("rows,vocab", [(3, 300001), (1, 1 << 20), (2, 130003), (320, 2500), (150, 26000)])
def test_sample_row_splits(device, rows, vocab):
    # rows that one block takes, that several share, and that are too long to be kept on the chip
    for dtype in (torch.float32, torch.bfloat16):
        x, noise = logits_of(rows, vocab, dtype, seed=rows)
        each = [(1.0, 0, 0.9, 0.0), (0.8, 50, 1.0, 0.0), (1.0, 0, 1.0, 0.05), (0.0, 0, 1.0, 0.0), (1.2, 2000, 0.7, 0.01),
                (1.0, 500, 0.99, 0.0)]
        for j in range(0 if rows > 6 else len(each) - rows + 1):
            check_sample(device, x, noise, *map(list, zip(*each[j:j + rows])))
        if rows > 6:
            check_sample(device, x, noise, *map(list, zip(*[each[r % 6] for r in range(rows)])))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("rows,vocab,dtype", [(1, 12288, torch.float32), (1, 25013, torch.bfloat16), (9, 17001, torch.float32),
                                              (17, 26000, torch.bfloat16), (35, 13001, torch.float32)])
def test_sample_few_rows_without_top_k(device, rows, vocab, dtype):
    # settings as numbers, so that a row may be spread over more blocks than hold it
    x, noise = logits_of(rows, vocab, dtype, seed=vocab)
    x[0, 5:] = x[0, 5]  # ties across the blocks' slices
    if rows > 1:
        x[1] = -math.inf
    for T, p, least in ((0.8, 1.0, 0.0), (1.0, 0.9, 0.0), (1.3, 0.99, 0.02), (0.0, 1.0, 0.0)):
        check_sample(device, x, noise, T, 0, p, least, tensors=False)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("spread", [1e-3, 0.1])
def test_sample_nearly_flat_rows(device, spread):
    # thousands of tokens within one bin of the log-weight, a far maximum, and the type's lowest value as a mask
    x, noise = logits_of(3, 40001, torch.float32, seed=8, spread=spread)
    x[1, 77] = 5.0
    x[2, ::2] = torch.finfo(torch.float32).min
    for p in (0.5, 0.99):
        check_sample(device, x, noise, 1.0, 0, p, 0.0)
        check_sample(device, x, noise, 1.0, [9000, 7, 1500], p, 0.0)


@pytest.mark.parametrize("device", DEVICES)
def test_sample_scores_that_nearly_tie(device):
    # the winner is decided by the last bit of logit / temperature + noise, or by the index
    g = torch.Generator().manual_seed(1)
    x = torch.randn(4, 6000, generator=g)
    T = 0.7
    noise = 3.0 - x / T
    noise[1] = 3.0 - (x[1] / T).nextafter(torch.tensor(9.0))
    check_sample(device, x, noise, T, 0, 0.97, 0.0)
    check_sample(device, x, noise, T, 0, 1.0, 0.0)
    check_sample(device, x, noise, T, 100, 1.0, 0.0)


@pytest.mark.parametrize("device", DEVICES)
def test_sample_masked_rows_and_special_values(device):
    inf, nan = math.inf, math.nan
    x = torch.full((9, 777), -inf)
    noise = logits_of(9, 777, torch.float32, seed=2)[1]
    x[1, 700] = -3e38
    x[2, 5], x[2, 6] = nan, 1.0
    x[3, 10], x[3, 20], x[3, 30] = inf, inf, 2.0
    x[4] = torch.finfo(torch.float32).min  # a mask of the type's lowest value
    x[4, 300] = 0.0
    x[5] = -0.0
    x[5, ::2] = 0.0  # equal to -0.0
    x[6, :4] = torch.tensor([1.0, 2.0, 3.0, 4.0])
    noise[6, :4] = torch.tensor([nan, -inf, -inf, -inf])
    x[7] = nan
    x[8, 100:200] = torch.arange(100.0)
    noise[8] = inf
    check_sample(device, x, noise, 1.0, 0, 1.0, 0.0)
    check_sample(device, x, noise, 0.0, 0, 1.0, 0.0)
    check_sample(device, x, noise, 0.7, 3, 0.8, 0.05)
    check_sample(device, x, noise, 1.0, 0, 0.5, 0.0)


@pytest.mark.parametrize("device", DEVICES)
def test_sample_strided_rows(device):
    x, noise = logits_of(6, 3000, torch.float32, seed=9)
    wide_x, wide_n = torch.zeros(6, 3101), torch.zeros(6, 3007)
    wide_x[:, 5:3005], wide_n[:, 3:3003] = x, noise
    a = G.sample(wide_x.to(device)[:, 5:3005], wide_n.to(device)[:, 3:3003], top_p=0.9)
    assert torch.equal(a, G.sample(x.to(device), noise.to(device), top_p=0.9))
    assert torch.equal(a[::2], G.sample(x.to(device)[::2], noise.to(device)[::2], top_p=0.9))
    assert G.sample(x[:0].to(device), noise[:0].to(device)).shape == (0,)


@pytest.mark.parametrize("device", DEVICES)
def test_sample_draws_the_filtered_softmax(device):
    g = torch.Generator().manual_seed(3)
    n, x = 20000, torch.tensor([2.0, 1.0, 0.0, -1.0, 1.5, -9.0])
    noise = -torch.empty(n, 6).exponential_(generator=g).log()
    token = G.sample(x.expand(n, 6).contiguous().to(device), noise.to(device), temperature=1.5, top_k=4).cpu()
    want = torch.softmax(torch.where(torch.tensor([1, 1, 1, 0, 1, 0]).bool(), x, -math.inf) / 1.5, 0)
    share = torch.bincount(token, minlength=6) / n
    # five standard deviations of a share
    assert torch.all((share - want).abs() <= 5 * (want * (1 - want) / n).sqrt() + 1e-9), (share, want)


@pytest.mark.parametrize("device", DEVICES)
def test_sample_refusals(device):
    x = torch.zeros(2, 8, device=device)
    G.sample(x, x)
    for bad in (dict(logits=x.half()), dict(logits=x[0], noise=x[0]), dict(noise=x.double()), dict(noise=x[:, :7]),
                dict(logits=x[:, :0], noise=x[:, :0]), dict(top_k=torch.zeros(2, device=device)),
                dict(top_p=torch.zeros(3, device=device)), dict(temperature=torch.zeros(2, dtype=torch.int32, device=device))):
        with pytest.raises(ValueError):
            G.sample(**{"logits": x, "noise": x} | bad)


# ---- pages -----------------------------------------------------------------------------


class Books:
    """A pool with some sequences in it, and what each sequence's tokens should be."""

    def __init__(self, device, lens, *, slots, columns, pages, page=8, planes=(2, 2), tail=(3, 16), dtype=torch.bfloat16, seed=0):
        g = torch.Generator().manual_seed(seed)
        kv = torch.randn(*planes, pages, page, *tail, generator=g) * 10
        self.kv = kv.to(dtype).to(device)
        self.table = ints([[-1] * columns] * slots, device)
        self.lens, self.refs = ints([0] * slots, device), ints([0] * pages, device)
        self.page, self.device = page, device
        G.reserve_pages(self.table, self.lens, self.refs, ints(range(len(lens)), device), ints(lens, device), page)
        settle(device)

    def tokens(self, slot):
        n, pool = int(self.lens[slot]), self.kv.flatten(0, -5)
        ids = self.table[slot, : -(-n // self.page)].long()
        assert torch.all(ids >= 0) and torch.all(self.table[slot, len(ids):] == -1)
        return pool[:, ids].flatten(1, 2)[:, :n].cpu()

    def consistent(self):
        """refs counts the rows that name each page."""
        held = self.table[self.table >= 0].long()
        assert torch.equal(torch.bincount(held, minlength=len(self.refs)).int(), self.refs), "refs"

    def fork(self, parents, children):
        G.fork_sequences(self.kv, self.table, self.lens, self.refs, ints(parents, self.device), ints(children, self.device))
        settle(self.device)

    def free(self, slots):
        G.free_sequences(self.table, self.lens, self.refs, ints(slots, self.device))
        settle(self.device)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype,tail,page", [(torch.bfloat16, (3, 16), 8), (torch.float32, (1, 4), 7), (torch.int8, (5, 48), 16),
                                             (torch.bfloat16, (16, 128), 16)])
def test_fork_free_and_compact_keep_every_sequence(device, dtype, tail, page):
    b = Books(device, [3 * page, 0, 2 * page + 3, 1, 5 * page - 1], slots=12, columns=6, pages=40, page=page, tail=tail, dtype=dtype)
    b.consistent()
    assert int(b.table[0, 0]) == 0 and int((b.refs > 0).sum()) == 3 + 3 + 1 + 5
    want = {s: b.tokens(s) for s in range(5)}
    b.fork([2, 0, 2, 4, 1], [7, 5, 6, 9, 11])
    b.consistent()
    for p, c in ((2, 7), (0, 5), (2, 6), (4, 9), (1, 11)):
        assert torch.equal(b.tokens(c), want[p]) and torch.equal(b.tokens(p), want[p])
    assert int(b.table[7, 2]) == 12 and int(b.table[6, 2]) == 13, "the lowest free pages, in order"
    assert b.table[5].tolist() == b.table[0].tolist(), "full pages are shared"
    # writing to a child leaves its parent alone
    b.kv.flatten(0, -5)[:, int(b.table[7, 2]), 0] += 1
    assert torch.equal(b.tokens(2), want[2])
    want[7] = b.tokens(7)
    b.free([2, 0, 4, 4])
    b.consistent()
    assert b.lens.tolist()[:5] == [0, 0, 0, 1, 0]
    for s, p in ((5, 0), (6, 2), (9, 4)):
        assert torch.equal(b.tokens(s), want[p])
    old_table, old_refs = b.table.clone(), b.refs.clone()
    b.table, b.refs = G.compact_pages(b.kv, b.table, b.refs)
    settle(device)
    b.consistent()
    live = int((b.refs > 0).sum())
    assert torch.all(b.refs[:live] > 0) and live == int((old_refs > 0).sum()) and not torch.equal(old_table, b.table)
    for s, p in ((5, 0), (6, 2), (9, 4), (3, 3)):
        assert torch.equal(b.tokens(s), want[p])
    assert torch.equal(b.tokens(7), want[7])


@pytest.mark.parametrize("device", DEVICES)
def test_page_operations_on_larger_books(device):
    rng = random.Random(4)
    lens = [rng.randrange(0, 90) for _ in range(150)]
    b = Books(device, lens, slots=1500, columns=12, pages=4500, planes=(1,), tail=(1, 8))
    b.consistent()
    want = {s: b.tokens(s) for s in range(150)}
    children = list(range(150, 1350))
    rng.shuffle(children)
    parents = [rng.randrange(150) for _ in children]
    b.fork(parents, children)
    b.consistent()
    gone = rng.sample(range(1350), 700)
    b.free(gone)
    b.consistent()
    b.table, b.refs = G.compact_pages(b.kv, b.table, b.refs)
    settle(device)
    b.consistent()
    origin = {s: s for s in range(150)} | dict(zip(children, parents))
    for s in sorted(set(range(1350)) - set(gone))[::7]:
        assert torch.equal(b.tokens(s), want[origin[s]])


@pytest.mark.parametrize("device", DEVICES)
def test_reserve_and_append(device):
    b = Books(device, [0, 13, 8], slots=4, columns=4, pages=12, planes=(1, 2), tail=(2, 16))
    want = {s: b.tokens(s) for s in (1, 2)}
    grow = {2: 9, 0: 1, 1: 3}
    G.reserve_pages(b.table, b.lens, b.refs, ints(list(grow), device), ints(list(grow.values()), device), b.page)
    b.consistent()
    assert b.lens.tolist() == [1, 16, 17, 0]
    slots = [s for s, n in grow.items() for _ in range(n)] + [3]
    places = [int(b.lens[s]) - n + t for s, n in grow.items() for t in range(n)] + [-1]
    new = torch.randn(len(slots), 2, 3, 16).to(torch.bfloat16).to(device)  # two of three heads: a strided slice
    G.append_kv(b.kv[0, 0], b.kv[0, 1], new[:, 0, 1:], new[:, 1, 1:], b.table, ints(places, device), ints(slots, device))
    settle(device)
    at = 0
    for s, n in grow.items():
        got = b.tokens(s)
        if s in want:
            assert torch.equal(got[:, :-n], want[s])
        assert torch.equal(got[:, -n:], new[at:at + n, :, 1:].transpose(0, 1).cpu())
        at += n
    # token i to row i
    G.append_kv(b.kv[0, 0], b.kv[0, 1], new[:3, 0, 1:], new[:3, 1, 1:], b.table, ints([0, 2, -1], device))
    settle(device)
    assert torch.equal(b.tokens(1)[:, 2], new[1, :, 1:].cpu()) and torch.equal(b.tokens(0)[:, 0], new[0, :, 1:].cpu())


@pytest.mark.parametrize("device", DEVICES)
def test_copy_pages(device):
    kv = torch.randn(3, 2, 9, 8, 1, 24).to(torch.bfloat16).to(device)
    want = kv.clone()
    want[:, :, [1, 8]] = want[:, :, [0, 5]]
    G.copy_pages(kv, ints([0, -1, 5, 3], device), ints([1, 2, 8, -1], device))
    settle(device)
    assert torch.equal(kv, want)
    G.copy_pages(kv, ints([], device), ints([], device))
    assert torch.equal(kv, want)


@pytest.mark.parametrize("device", DEVICES)
def test_page_requests_that_cannot_be_met(device):
    def refused(match, call, *args):
        with pytest.raises(RuntimeError, match=match):
            call(*args)
            settle(device)

    b = Books(device, [13, 8], slots=5, columns=2, pages=4)
    table, lens, refs = b.table.clone(), b.lens.clone(), b.refs.clone()
    one = ints([1], device)
    refused(".", b.fork, [0], [1])  # not empty
    refused(".", b.fork, [0], [7])
    refused(".", b.fork, [-1], [2])
    refused(".", b.fork, [3, 0], [2, 3])  # a parent that is a child
    b.free([3, 2])  # on the GPU the sound half of the last request was done
    refused(".", b.free, [9])
    refused("too few free pages", G.reserve_pages, b.table, b.lens, b.refs, ints([2], device), ints([16], device), 8)
    refused(".", G.reserve_pages, b.table, b.lens, b.refs, ints([0], device), ints([4], device), 8)  # past the row
    refused(".", G.reserve_pages, b.table, b.lens, b.refs, ints([0], device), ints([-1], device), 8)
    refused(".", G.append_kv, b.kv[0, 0], b.kv[0, 1], b.kv[0, 0, 0, :1], b.kv[0, 1, 0, :1], b.table, ints([9], device), one)
    refused(".", G.append_kv, b.kv[0, 0], b.kv[0, 1], b.kv[0, 0, 0, :1], b.kv[0, 1, 0, :1], b.table, ints([0], device), ints([4], device))
    refused(".", G.copy_pages, b.kv, ints([0], device), ints([4], device))
    assert torch.equal(b.table, table) and torch.equal(b.lens, lens) and torch.equal(b.refs, refs)
    b.fork([0], [2])
    refused("too few free pages", b.fork, [0], [3])
    b.consistent()
    assert int(b.lens[3]) == 0


@pytest.mark.parametrize("device", DEVICES)
def test_page_refusals(device):
    b = Books(device, [13], slots=2, columns=2, pages=4)
    one = ints([1], device)
    for call in (
        lambda: G.copy_pages(b.kv[..., :5], one, one), lambda: G.copy_pages(b.kv, one.long(), one.long()),
        lambda: G.copy_pages(b.kv, one, ints([1, 2], device)),
        lambda: G.copy_pages(torch.zeros(4, 8, 1, 3, device=device), one, one),
        lambda: G.fork_sequences(b.kv, b.table, b.lens, b.refs[:3], one, one),
        lambda: G.fork_sequences(b.kv, b.table, b.lens[:1], b.refs, one, one),
        lambda: G.fork_sequences(b.kv, b.table.long(), b.lens, b.refs, one, one),
        lambda: G.reserve_pages(b.table, b.lens, b.refs, one, ints([1, 2], device), 8),
        lambda: G.reserve_pages(b.table, b.lens, b.refs, one, one, 0),
        lambda: G.free_sequences(b.table, b.lens, b.refs, one[None]),
        lambda: G.compact_pages(b.kv, b.table, b.refs[:3]),
        lambda: G.append_kv(b.kv[0, 0], b.kv[0, 1], b.kv[0, 0, 0], b.kv[0, 1, 0], b.table, one),
        lambda: G.append_kv(b.kv[0, 0], b.kv[0, 1], b.kv[0, 0, 0, :, :2], b.kv[0, 1, 0, :, :2], b.table, ints([0] * 8, device),
                            ints([0] * 8, device)),
    ):
        with pytest.raises(ValueError):
            call()


@pytest.mark.gpu
def test_page_copies_beyond_32_bit_offsets():
    pages = (1 << 31) // (256 * 16 * 128) + 8
    kv = torch.empty(2, pages, 256, 16, 128, dtype=torch.bfloat16, device="cuda")
    kv[:, -1], kv[:, -2] = 3, 5
    G.copy_pages(kv, ints([pages - 1], "cuda"), ints([pages - 2], "cuda"))
    settle("cuda")
    assert torch.all(kv[:, -2] == 3)


@pytest.mark.parametrize("device", DEVICES)
def test_cache_class(device):
    c = G.PagedKVCache(2, 32, 8, 2, 32, max_seqs=6, max_seq_len=40, device=device)
    c.extend([0, 3], [11, 8])
    k = torch.randn(19, 2, 32).to(torch.bfloat16).to(device)
    places, slots = ints([*range(11), *range(8)], device), ints([0] * 11 + [3] * 8, device)
    for layer in range(2):
        c.append(layer, k + layer, -k, places, slots)
    c.fork([0, 3], [1, 2])
    assert c.lengths == [11, 11, 8, 8, 0, 0] and c.lens.tolist() == c.lengths and c.pages_in_use() == 4
    c.free([0])
    c.compact()
    assert c.pages_in_use() == 3
    got = c.kv[1, 0][c.page_table[1, :2].long()].flatten(0, 1)[:11]
    assert torch.equal(got, k[:11] + 1)
    settle(device)
    for call in (lambda: c.extend([0], [41]), lambda: c.extend([6], [1]), lambda: c.extend([1, 1], [1, 1]),
                 lambda: c.fork([1], [2]), lambda: c.fork([1, 4], [4, 5]), lambda: c.free([-1]),
                 lambda: G.PagedKVCache(1, 4, 12, 1, 32, max_seqs=1, max_seq_len=8, device=device)):
        with pytest.raises(ValueError):
            call()


@pytest.mark.gpu
@pytest.mark.parametrize("seed", range(4))
def test_page_operations_agree_bit_for_bit_with_the_plain_ones(seed):
    """A run of random operations on both: every value of the pool and the books stays the same, unused pages included."""
    rng = random.Random(seed)
    page, heads, dim = rng.choice([(8, 3, 16), (16, 2, 64), (5, 1, 8)])
    kv = torch.randn(3, 2, 400, page, heads, dim).to(torch.bfloat16)
    S, W = 300, 9
    sides = []
    for device in ("cpu", "cuda"):
        sides.append([kv.clone().to(device), ints([[-1] * W] * S, device), ints([0] * S, device), ints([0] * 400, device)])
    lens = [0] * S
    for _ in range(25):
        live = [s for s in range(S) if lens[s]]
        op = rng.choice(["grow", "grow", "fork", "free", "compact", "append"])
        if op == "grow":
            slots = rng.sample(range(S), rng.randrange(1, 12))
            counts = [rng.randrange(0, min(2 * page, W * page - lens[s]) + 1) for s in slots]
            if sum(-(-c // page) + 1 for c in counts) > int((sides[0][3] == 0).sum()):
                continue
            for k, t, n, r in sides:
                G.reserve_pages(t, n, r, ints(slots, t.device), ints(counts, t.device), page)
            for s, c in zip(slots, counts):
                lens[s] += c
        elif op == "fork" and live:
            empty = [s for s in range(S) if not lens[s]]
            children = rng.sample(empty, min(len(empty), rng.choice([1, 5, 270])))
            children = children[: int((sides[0][3] == 0).sum())]
            parents = [rng.choice(live) for _ in children]
            for k, t, n, r in sides:
                G.fork_sequences(k, t, n, r, ints(parents, t.device), ints(children, t.device))
            for p, c in zip(parents, children):
                lens[c] = lens[p]
        elif op == "free" and live:
            gone = rng.sample(live, max(1, len(live) // 2))
            for k, t, n, r in sides:
                G.free_sequences(t, n, r, ints(gone, t.device))
            for s in gone:
                lens[s] = 0
        elif op == "compact":
            for side in sides:
                side[1], side[3] = G.compact_pages(side[0], side[1], side[3])
        elif op == "append" and live:
            # only pages with one holder may be written
            alone = [s for s in live if int(sides[0][3][int(sides[0][1][s, (lens[s] - 1) // page])]) == 1]
            if not alone:
                continue
            new = torch.randn(len(alone), 2, heads, dim).to(torch.bfloat16)
            for k, t, n, r in sides:
                x = new.to(t.device)
                G.append_kv(k[1, 0], k[1, 1], x[:, 0], x[:, 1], t, ints([lens[s] - 1 for s in alone], t.device), ints(alone, t.device))
        settle("cuda")
        for a, b in zip(*sides):
            assert torch.equal(a, b.cpu()), op
