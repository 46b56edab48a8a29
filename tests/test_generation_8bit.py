"""The cache in 8 bits and the logits' adjustment against plain 64-bit implementations, on CPU and (marked gpu) on the kernels.

Tolerances follow from the arithmetic.  Appending is exact but for the one
rounding that its definition has, so codes and scales have to be equal.  In
the attention the weights are rounded to f16 (2^-11 of each) and the outputs to
bf16 (2^-8 of the value); a score is an fp32 sum of D products, off by at most
D 2^-24 sum |q_i k_i|, and is held in fp32 beside the logarithm of a scale
(2^-24 of their sum, in log2 units), as is the row's base.  Codes may be 0, so a
column of the output may come from tokens of next to no weight alone: f16 holds
a weight to 2^-25 absolutely where the largest of its row, times its scale (or
the largest scale near it), is held as 2^7 or more, so a weight may also be off
by 2^-32 of that, times each token's code.  The adjustment of
logits is a chain of at most five fp32 operations, each off by 2^-24 of its
result, and a rounding to the logits' type.
"""

from __future__ import annotations

import math
import random

import pytest
import torch

from mini_nccl_b200.ops import generation as G
from test_generation import DEVICES, ints, settle

TYPES = [torch.int8, torch.float8_e4m3fn]
TOP = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}
U = 2.0 ** -24


def nearest(x, dtype):
    """The nearest code in 64 bits, of two the even one."""
    if dtype == torch.int8:
        return torch.round(x)
    step = torch.ldexp(torch.ones_like(x), (torch.frexp(x)[1] - 1).clamp(min=-6) - 3)
    return torch.round(x / step) * step


def least_scale(most, dtype):
    return 2.0 ** max(-60, math.ceil(math.log2(most / TOP[dtype]))) if most > 0 else 2.0 ** -60


def values_of(pages, scales):
    return pages.view(torch.uint8).cpu().view(pages.dtype).double() * scales.cpu().double()[:, None, :, None]


# ---- appending ---------------------------------------------------------------------------


class Cache:
    """Pages and what they should hold: 64-bit codes and scales, kept by the definition."""

    def __init__(self, pages, page, heads, dim, dtype, device, seed=0, layout="plain"):
        gen = torch.Generator().manual_seed(seed)
        self.page, self.dtype, self.device = page, dtype, device
        code = torch.randint(-127, 128, (2, pages, page, heads, dim), generator=gen).double()
        code = code if dtype == torch.int8 else nearest(code * 3, dtype)
        scale = torch.ldexp(torch.ones(2, pages, heads), torch.randint(-9, 0, (2, pages, heads), generator=gen)).double()
        self.code, self.scale = code, scale
        kv = code.to(torch.int8) if dtype == torch.int8 else code.float().to(dtype)
        kv = kv.view(torch.uint8).to(device)
        if layout == "heads first":
            kv = kv.transpose(2, 3).contiguous().transpose(2, 3)
        self.kv = kv.view(dtype)
        self.scales = scale.float().to(device)
        if layout == "heads first":
            self.scales = self.scales.transpose(1, 2).contiguous().transpose(1, 2)

    def append(self, table, positions, slots, k, v):
        G.append_kv(self.kv[0], self.kv[1], k, v, ints(table, self.device), ints(positions, self.device),
                    None if slots is None else ints(slots, self.device), k_scales=self.scales[0], v_scales=self.scales[1])
        named = {}
        for i, pos in enumerate(positions):
            if pos >= 0:
                named.setdefault(table[i if slots is None else slots[i]][pos // self.page], []).append((i, pos % self.page))
        for p, tokens in named.items():
            which, places = [i for i, _ in tokens], dict((at, i) for i, at in tokens)
            for part, x in enumerate((k.cpu().double(), v.cpu().double())):
                for h in range(x.shape[1]):
                    mine = x[which, h]
                    scale = least_scale(float(mine[mine.isfinite()].abs().max()) if mine.isfinite().any() else 0.0, self.dtype)
                    if 0 not in places:
                        held = float(self.scale[part, p, h])
                        scale = max(scale, held)
                        self.code[part, p, :, h] = nearest(self.code[part, p, :, h] * (held / scale), self.dtype)
                    self.scale[part, p, h] = scale
                    for at, i in places.items():
                        code = nearest(x[i, h].clamp(-TOP[self.dtype] * scale, TOP[self.dtype] * scale) / scale, self.dtype)
                        self.code[part, p, at, h] = code

    def check(self):
        settle(self.device)
        assert torch.equal(self.scales.cpu().double(), self.scale)
        got = self.kv.view(torch.uint8).cpu().view(self.dtype).double()
        assert torch.equal(got.nan_to_num(nan=7777.0), self.code.nan_to_num(nan=7777.0))


def tokens_of(n, heads, dim, device, seed, size=1.0):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(n, 3, heads, dim, generator=gen) * size
    x *= torch.where(torch.rand(n, 1, heads, 1, generator=gen) < 0.2, 20.0, 1.0)  # some do not fit what is there
    x = x.to(torch.bfloat16).to(device)
    return x[:, 1], x[:, 2]  # slices of a fused projection


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,dim,page", [(1, 16, 8), (3, 64, 16), (2, 128, 32), (5, 32, 8), (1, 256, 64), (2, 96, 16)])
def test_append(device, dtype, heads, dim, page):
    rng = random.Random(dim)
    S, columns = 9, 5
    ids = list(range(S * columns + 2))
    rng.shuffle(ids)
    table = [ids[i * columns:(i + 1) * columns] for i in range(S)]
    c = Cache(len(ids), page, heads, dim, dtype, device)
    # prompts of ragged lengths, packed
    lens = [1, page, page + 1, 3 * page - 1, 2, 4 * page, 0, 7, page - 1]
    positions = [t for n in lens for t in range(n)]
    slots = [s for s, n in enumerate(lens) for _ in range(n)]
    c.append(table, positions, slots, *tokens_of(len(positions), heads, dim, device, 1))
    c.check()
    # then token by token, some larger than what their pages hold, and twice a few at once
    for step in range(4):
        c.append(table, lens, None, *tokens_of(S, heads, dim, device, 10 + step, size=2.0 ** step))
        lens = [n + 1 for n in lens]
    c.check()
    few = [s for s, n in enumerate(lens) if n + 3 <= columns * page]
    c.append(table, [lens[s] + i for s in few for i in range(3)], [s for s in few for _ in range(3)],
             *tokens_of(3 * len(few), heads, dim, device, 30))
    c.check()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
def test_append_padding_orders_and_layouts(device, dtype):
    heads, dim, page = 3, 64, 16
    table = [[4, 2, -1], [0, 3, 7], [6, 1, 5]]
    c = Cache(9, page, heads, dim, dtype, device, layout="heads first")
    c.append(table, [], [], *tokens_of(0, heads, dim, device, 1))
    # padding inside a page's tokens, and more of it than a warp looks at; descending places; a place named twice
    positions = [5, -1, 6, -1, -1, 3] + [-3] * 70 + [4, 17, 16, -1, 18, 18, 30, 18] + [-1] * 40
    slots = [0] * 76 + [0] + [2, 2, 99, 2, 2, 2, 2] + [-5] * 40
    c.append(table, positions, slots, *tokens_of(len(positions), heads, dim, device, 2, size=9.0))
    c.append(table, [30, -1, 0], None, *tokens_of(3, heads, dim, device, 3))
    c.check()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
def test_append_ranges(device, dtype):
    """Zeros, the least and the largest bf16 values, borders of the scale, ties, and pages that nothing was written to."""
    top = TOP[dtype]
    c = Cache(8, 8, 1, 16, dtype, device)
    c.scales.zero_(), c.scale.zero_()
    c.kv.view(torch.uint8).zero_(), c.code.zero_()
    rows = [[0.0] * 16, [1e-38, -1e-40] + [0.0] * 14, [3.38e38, -3e38] + [1.0] * 14, [top, -top] + [0.5, 1.5, 2.5, -0.5] * 3 + [17.0, 19.0],
            [top * 1.01, 1.0] + [3.0, 5.0] * 7, [2.0 ** -60 * top, 2.0 ** -61] + [0.0] * 14, [0.0625, 0.0635] * 8]
    x = torch.tensor(rows).to(torch.bfloat16).view(-1, 1, 16).to(device)
    c.append([[i] for i in range(7)], [0] * 7, None, x, -x)
    c.check()
    c.append([[i] for i in range(7)], [3] * 7, None, x.flip(0), x.flip(0))  # small beside large, and large after small
    c.check()
    c.append([[7]], [5], None, x[3:4], x[4:5])  # a page that is not begun by its first place
    c.check()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
def test_append_not_finite(device, dtype):
    c = Cache(3, 8, 2, 32, dtype, device)
    k, v = tokens_of(6, 2, 32, device, 4)
    k, v = k.contiguous(), v.contiguous()
    k[1, 0, 3], k[2, 1, 0], v[4, 0, 31], v[5] = math.inf, -math.inf, math.inf, -math.inf
    c.append([[1, 2]], [0, 1, 2, 3, 8, 9], [0] * 6, k, v)
    c.check()
    k[3, 1, 5] = math.nan
    if dtype == torch.float8_e4m3fn:
        c.append([[1, 2]], [0, 1, 2, 3, 8, 9], [0] * 6, k, v)
        assert int(c.code.isnan().sum()) == 1
        c.check()
    elif device == "cpu":
        with pytest.raises(RuntimeError):
            c.append([[1, 2]], [0, 1, 2, 3, 8, 9], [0] * 6, k, v)
    else:
        from mini_nccl_b200.ops import kernels as K

        c.append([[1, 2]], [0, 1, 2, 3, 8, 9], [0] * 6, k, v)
        with pytest.raises(RuntimeError, match="NaN among"):
            K.check_status()
        c.code[0, 1, 3, 1, 5] = 0.0
        c.check()


@pytest.mark.parametrize("device", DEVICES)
def test_append_in_pieces_is_the_same_cache(device):
    """However a page's tokens are split over calls, e4m3 holds the same, int8 within one step of the last scale (a page
    that begins with its first place)."""
    k, v = tokens_of(40, 2, 64, device, 5)
    for dtype in TYPES:
        held = []
        for step in (40, 7, 1):
            c = Cache(3, 16, 2, 64, dtype, device)
            for i in range(0, 40, step):
                n = min(40, i + step) - i
                c.append([[2, 0, 1]], list(range(i, i + n)), [0] * n, k[i:i + n], v[i:i + n])
            c.check()
            held.append(values_of(c.kv[0], c.scales[0])[[2, 0, 1]].reshape(-1, 2, 64)[:40])
            scale = c.scale[0][[2, 0, 1]].repeat_interleave(16, 0)[:40, :, None]
        for other in held[1:]:
            off = (other - held[0]).abs()
            # (e4m3 rounds twice only below its normal range, 2^-6 times the scale, by half a step of 2^-9)
            assert torch.all(off <= (scale if dtype == torch.int8 else scale * 2.0 ** -9))


@pytest.mark.parametrize("device", DEVICES)
def test_append_refusals(device):
    def call(dtype=torch.int8, pages=(4, 8, 2, 32), scales=(4, 2), k=(3, 2, 32), v_dtype=None, of=torch.float32):
        kv = [torch.zeros(*pages, device=device).to(t) for t in (dtype, v_dtype or dtype)]
        sc = {} if scales is None else dict(k_scales=torch.zeros(*scales, device=device, dtype=of), v_scales=torch.zeros(*scales, device=device, dtype=of))
        x = torch.zeros(*k, dtype=torch.bfloat16, device=device)
        G.append_kv(kv[0], kv[1], x, x, ints([[0], [1], [2]], device), ints([0, 1, 2], device), **sc)

    call()
    call(torch.float8_e4m3fn)
    call(torch.bfloat16, scales=None)
    for bad in (dict(scales=None), dict(scales=(4, 3)), dict(scales=(3, 2)), dict(of=torch.float64), dict(dtype=torch.bfloat16),
                dict(v_dtype=torch.float8_e4m3fn), dict(pages=(4, 8, 2, 24), k=(3, 2, 24)), dict(pages=(4, 8, 2, 272), k=(3, 2, 272))):
        with pytest.raises(ValueError):
            call(**bad)
    settle(device)


def test_append_refuses_scattered_pages_on_the_cpu():
    c = Cache(4, 8, 1, 16, torch.int8, "cpu")
    with pytest.raises(ValueError, match="follow one another"):
        G.append_kv(c.kv[0], c.kv[1], *tokens_of(3, 1, 16, "cpu", 0), ints([[0, 1]], "cpu"), ints([0, 8, 1], "cpu"), ints([0, 0, 0], "cpu"),
                    k_scales=c.scales[0], v_scales=c.scales[1])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_append_leaves_out_tokens_that_come_back_to_a_page(dtype):
    from mini_nccl_b200.ops import kernels as K

    k, v = tokens_of(5, 2, 64, "cuda", 0)
    held = []
    for positions, slots in (([0, 8, 1, 9, 2], [0, 1, 0, 1, 0]), ([0, 8], [0, 1])):
        c = Cache(6, 8, 2, 64, dtype, "cuda")
        n = len(positions)
        G.append_kv(c.kv[0], c.kv[1], k[:n], v[:n], ints([[4, 0], [2, 5]], "cuda"), ints(positions, "cuda"), ints(slots, "cuda"),
                    k_scales=c.scales[0], v_scales=c.scales[1])
        held.append(c)
        if n == 5:
            with pytest.raises(RuntimeError, match="do not follow one another"):
                K.check_status()
    settle("cuda")
    assert torch.equal(held[0].kv.view(torch.uint8), held[1].kv.view(torch.uint8)) and torch.equal(held[0].scales, held[1].scales)


@pytest.mark.gpu
def test_append_leaves_bad_requests_out():
    from mini_nccl_b200.ops import kernels as K

    for table, positions, slots in (([[9, 1]], [0, 8], [0, 0]), ([[-1, 1]], [3, 9], [0, 0]), ([[0, 1]], [16, 9], [0, 0]),
                                    ([[0, 1]], [2, 9], [5, 0]), ([[0, 1]], [2, 9], [-1, 0])):
        c = Cache(4, 8, 2, 64, torch.int8, "cuda")
        k, v = tokens_of(2, 2, 64, "cuda", 0)
        G.append_kv(c.kv[0], c.kv[1], k, v, ints(table, "cuda"), ints(positions, "cuda"), ints(slots, "cuda"), k_scales=c.scales[0],
                    v_scales=c.scales[1])
        with pytest.raises(RuntimeError, match="outside its tensor"):
            K.check_status()
        before = Cache(4, 8, 2, 64, torch.int8, "cuda")
        before.append([[0, 1]], positions[1:], [0], k[1:], v[1:])
        assert torch.equal(c.kv, before.kv) and torch.equal(c.scales, before.scales)


# ---- attention ---------------------------------------------------------------------------


class Problem:
    """A shared prefix, ragged own lengths and their pages in a pool whose other places hold anything (NaN in e4m3)."""

    def __init__(self, lens, new, *, kv_heads, group, dim, page, prefix, device, dtype, seed=0, scale_q=1.0, heads_first=False,
                 exponents=(-7, -4)):
        rng, gen = random.Random(seed), torch.Generator().manual_seed(seed)
        H = kv_heads * group
        n_prefix = -(-prefix // page)
        ids = list(range(n_prefix + sum(-(-m // page) for m in lens) + 3))
        rng.shuffle(ids)
        pool = torch.full((2, len(ids), page, kv_heads, dim), 0x7f, dtype=torch.uint8)
        scales = torch.ldexp(torch.ones(2, len(ids), kv_heads), torch.randint(exponents[0], exponents[1] + 1, (2, len(ids), kv_heads), generator=gen))
        self.prefix_pages, at = ids[:n_prefix], n_prefix
        columns = max(1, -(-max(lens, default=0) // page))
        self.rows = []
        for m in lens:
            k = -(-m // page)
            self.rows.append(ids[at:at + k] + [-1] * (columns - k))
            at += k

        def fill(pages, n):
            code = torch.randn(2, n, kv_heads, dim, generator=gen) * 32
            code = (code.clamp(-127, 127).round().to(torch.int8) if dtype == torch.int8 else code.to(dtype)).view(torch.uint8)
            for t in range(n):
                pool[:, pages[t // page], t % page] = code[:, t]
            of = scales[:, [pages[t // page] for t in range(n)]].double()
            self.largest = max(self.largest, float(of[1].max()) if n else 0.0)
            return code.view(dtype).double() * of[..., None]

        self.largest = 0.0  # of the values' scales
        self.head = fill(self.prefix_pages, prefix)
        self.own = [fill(r, m) for r, m in zip(self.rows, lens)]
        self.top = TOP[dtype]
        self.lens, self.new, self.prefix, self.dim, self.group, self.least = lens, new, prefix, dim, group, exponents[0]
        wide = (torch.randn(sum(new), (H + 1) * dim, generator=gen) * scale_q).to(torch.bfloat16).to(device)
        self.q = wide[:, dim:].view(-1, H, dim)  # a slice of a wider projection
        pool, self.scales = pool.to(device), scales.to(device)
        if heads_first:
            pool = pool.transpose(2, 3).contiguous().transpose(2, 3)
            self.scales = self.scales.transpose(1, 2).contiguous().transpose(1, 2)
        self.pool = pool.view(dtype)
        self.device = device

    def arguments(self, **more):
        offsets = None
        if any(n != 1 for n in self.new):
            offsets = ints([sum(self.new[:i]) for i in range(len(self.new) + 1)], self.device)
            more.setdefault("max_q_len", max(self.new))
        return (self.q, self.pool[0], self.pool[1], ints(self.prefix_pages, self.device), self.prefix, ints(self.rows, self.device),
                ints(self.lens, self.device)), dict(q_offsets=offsets, return_lse=True, k_scales=self.scales[0], v_scales=self.scales[1], **more)

    def run(self, **more):
        args, named = self.arguments(**more)
        out = G.shared_prefix_attention(*args, **named)
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
                        + 8 * U * (s.abs().amax(-1) + abs(self.least) + 40)
                    assert torch.all((lse[at] - torch.logsumexp(s, -1)).abs() <= off), ((lse[at] - torch.logsumexp(s, -1)).abs() / off).max()
                    lost = 2.0 ** -32 * self.largest * self.top * (v[:, :seen] != 0).sum(1) * p.amax(1)
                    bound = 2.0 ** -8 * (want.abs() + lost) + (2.0 ** -11 + 2 * off[:, None]) * spread + lost
                    assert torch.all((o[at] - want).abs() <= bound), ((o[at] - want).abs() / bound).max()
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
    ([i % 37 for i in range(230)], [1] * 230, 13, 1, 64, 8, 70),
    ([(5 * i) % 21 for i in range(450)], [i % 3 for i in range(450)], 6, 3, 32, 16, 40),
    ([1200, 3], [1, 1], 1, 1, 128, 128, 4500),
    ([33] * 1100, [1] * 1100, 1, 1, 32, 8, 0),  # more sequences than a block keeps the lengths of
    # enough of a prefix for the tensor cores: rows in both streams, and in one; ends inside a tile and a page
    ([2] * 180, [1] * 180, 12, 1, 128, 16, 1491),
    ([i % 3 for i in range(40)], [1] * 40, 8, 4, 64, 64, 2500),
    ([5, 0, 9] * 4, [1] * 12, 8, 4, 128, 8, 6001),
    ([7] * 30, [1] * 30, 16, 1, 64, 128, 4100),
    ([70, 90, 64], [60, 90, 34], 4, 3, 128, 32, 1000),
]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lens,new,kv_heads,group,dim,page,prefix", SHAPES)
def test_attention(device, dtype, lens, new, kv_heads, group, dim, page, prefix):
    p = Problem(lens, new, kv_heads=kv_heads, group=group, dim=dim, page=page, prefix=prefix, device=device, dtype=dtype)
    o, lse = p.run()
    p.check(o, lse)
    if device == "cuda":
        again, _ = p.run()
        assert torch.equal(o, again)


# ---- logits ------------------------------------------------------------------------------


def words_of(bits):
    """Truth values [masks, vocabulary] as int32 words."""
    M, V = bits.shape
    padded = torch.zeros(M, -(-V // 32) * 32, dtype=torch.int64)
    padded[:, :V] = bits
    words = (padded.view(M, -1, 32) << torch.arange(32)).sum(-1)
    return torch.where(words >= 1 << 31, words - (1 << 32), words).int()


def adjusted(x, prompt, history, rho, alpha, phi, named, bits):
    """One row in 64 bits, and how far fp32 arithmetic may be off."""
    x, room = x.double().clone(), torch.zeros(x.shape[0], dtype=torch.float64)
    for v in set(prompt) | set(history):
        if 0 <= v:
            x[v] = x[v] / rho if x[v] > 0 else x[v] * rho
            room[v] += U * abs(x[v])
    for v in set(history):
        if 0 <= v:
            off = phi * history.count(v) + alpha
            x[v] -= off
            room[v] += U * (2 * abs(off) + abs(x[v]))
    for v, b in named.items():
        x[v] += b
        room[v] += U * abs(x[v])
    x[~bits] = -math.inf
    return x, 1.01 * room


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("R,V", [(1, 1), (1, 50), (3, 777), (2, 4099), (5, 8192), (2, 40007), (160, 333)])
def test_adjust_logits(device, dtype, R, V):
    gen, rng = torch.Generator().manual_seed(R * V), random.Random(V)
    x = (torch.randn(R, V + 3, generator=gen) * 4).to(dtype)[:, 3:]  # rows that begin anywhere
    x[0, V // 2] = -math.inf
    H, P, B = 37, 19, min(V, 11)
    history = torch.randint(-1, V, (R, H), generator=gen)
    history[:, 5:9] = history[:, :1]
    lens = [rng.randrange(H + 1) for _ in range(R)]
    prompt = torch.randint(-1, V, (P,), generator=gen)
    bias_tokens = torch.randint(-1, V, (R, B), generator=gen).int()
    bias = torch.randn(R, B, generator=gen) * 3
    M = min(4, R)
    bits = torch.rand(M, V, generator=gen) < torch.tensor([0.02, 0.5, 0.999, 0.0])[:M, None]
    mask_of = [rng.randrange(-1, M) for _ in range(R)]
    rho, alpha, phi = (torch.tensor([rng.choice(c) for _ in range(R)]) for c in ((1.0, 1.3, 0.8), (0.0, 0.7), (0.0, 0.25)))
    on = lambda t: t.to(device)  # noqa: E731

    def check(y, use_prompt, use_history, use_bias, use_mask, rho=rho, alpha=alpha, phi=phi):
        settle(device)
        assert y.dtype == dtype and y.shape == (R, V)
        for r in range(R):
            named = {}
            if use_bias:
                named = {int(t): float(b) for t, b in zip(bias_tokens[r], bias[r]) if t >= 0}
            seen = torch.ones(V, dtype=torch.bool) if not use_mask or mask_of[r] < 0 else bits[mask_of[r]]
            want, room = adjusted(x[r], prompt.tolist() if use_prompt else [], history[r, :lens[r]].tolist() if use_history else [],
                                  float(rho[r]), float(alpha[r]), float(phi[r]), named, seen)
            got = y[r].cpu().double()
            assert torch.equal(got == -math.inf, want == -math.inf)
            fine = want > -math.inf
            off = (got - want).abs()[fine]
            assert torch.all(off <= (room + torch.finfo(dtype).eps / 2 * (want.abs() + room))[fine])

    where = on(x)
    full = dict(prompt=on(prompt), history=on(history), history_lens=ints(lens, device), repetition=on(rho), presence=on(alpha),
                frequency=on(phi), bias_tokens=on(bias_tokens), bias=on(bias), allowed=on(words_of(bits)), mask_of=ints(mask_of, device))
    y = G.adjust_logits(where, **full)
    check(y, True, True, True, True)
    assert torch.equal(where.cpu(), x)
    check(G.adjust_logits(where, allowed=full["allowed"], mask_of=full["mask_of"]), False, False, False, True)
    check(G.adjust_logits(where, bias_tokens=full["bias_tokens"], bias=full["bias"]), False, False, True, False)
    numbers = dict(repetition=1.5, presence=0.25, frequency=-0.5)
    z = G.adjust_logits(where, prompt=full["prompt"].int(), history=full["history"].int(), history_lens=full["history_lens"], **numbers)
    of = {k: torch.full((R,), v) for k, v in numbers.items()}
    check(z, True, True, False, False, of["repetition"], of["presence"], of["frequency"])
    assert torch.equal(G.adjust_logits(where).cpu(), x)
    # in place, in a part of a wider tensor whose other columns stay as they are
    wide = torch.full((R, V + 7), 5.0, dtype=dtype, device=device)
    wide[:, 2:2 + V] = where
    assert G.adjust_logits(wide[:, 2:2 + V], **full, out=wide[:, 2:2 + V]).data_ptr() == wide[:, 2:].data_ptr()
    assert torch.equal(wide[:, 2:2 + V], y) and torch.all(wide[:, :2] == 5) and torch.all(wide[:, 2 + V:] == 5)
    wide[:, 2:2 + V] = 5.0
    G.adjust_logits(where, **full, out=wide[:, 5:5 + V])
    assert torch.equal(wide[:, 5:5 + V], y) and torch.all(wide[:, :5] == 5) and torch.all(wide[:, 5 + V:] == 5)


@pytest.mark.parametrize("device", DEVICES)
def test_adjust_logits_special_values(device):
    V = 100
    x = torch.randn(2, V).to(device)
    x[:, 3], x[:, 4], x[:, 5] = math.nan, math.inf, -math.inf
    tokens = torch.tensor([[3, 4, 5, 6]] * 2, device=device)
    bits = torch.ones(1, V, dtype=torch.bool)
    bits[0, [3, 7]] = False
    y = G.adjust_logits(x, history=tokens, repetition=2.0, presence=1.0, allowed=words_of(bits).to(device))
    settle(device)
    assert torch.all(y[:, [3, 5, 7]] == -math.inf) and torch.all(y[:, 4] == math.inf)
    y = G.adjust_logits(x, history=tokens, repetition=2.0)
    assert torch.all(y[:, 3].isnan())
    nothing = G.adjust_logits(x, allowed=torch.zeros(1, 4, dtype=torch.int32, device=device))
    assert torch.all(nothing == -math.inf)
    token = G.sample(nothing, torch.zeros_like(nothing))
    assert torch.all(token == -1)
    assert G.adjust_logits(x[:0], history=tokens[:0]).shape == (0, V)
    assert torch.equal(G.adjust_logits(x, history=tokens[:, :0], prompt=tokens[0, :0])[:, 6:], x[:, 6:])
    # a token that has two biases gets the later one, whichever row the list is for
    two = G.adjust_logits(torch.zeros(2, V, device=device), bias_tokens=torch.tensor([9, -1, 8, 9], device=device),
                          bias=torch.tensor([1.0, 2.0, 3.0, 4.0], device=device))
    settle(device)
    assert torch.all(two[:, 9] == 4) and torch.all(two[:, 8] == 3) and float(two.sum()) == 14


@pytest.mark.parametrize("device", DEVICES)
def test_adjust_logits_refusals(device):
    x = torch.zeros(2, 40, device=device)
    t = lambda *s, dtype=torch.int64: torch.zeros(*s, dtype=dtype, device=device)  # noqa: E731
    for bad in (dict(history=t(3, 4)), dict(history=t(4)), dict(history=t(2, 4, dtype=torch.int16)), dict(prompt=t(3, 4)),
                dict(history_lens=t(2, dtype=torch.int32)), dict(history=t(2, 4), history_lens=t(3, dtype=torch.int32)),
                dict(history=t(2, 4), history_lens=t(2)), dict(bias_tokens=t(2, 3)), dict(bias=t(2, 3, dtype=torch.float32)),
                dict(bias_tokens=t(2, 3), bias=t(2, 4, dtype=torch.float32)), dict(bias_tokens=t(2, 3), bias=t(2, 3, dtype=torch.float64)),
                dict(bias_tokens=t(2, 4096), bias=t(2, 4096, dtype=torch.float32)), dict(allowed=t(1, 1, dtype=torch.int32)),
                dict(allowed=t(3, 2, dtype=torch.int32)), dict(allowed=t(1, 2)), dict(mask_of=t(2, dtype=torch.int32)),
                dict(allowed=t(1, 2, dtype=torch.int32), mask_of=t(3, dtype=torch.int32)),
                dict(repetition=t(3, dtype=torch.float32)), dict(presence=t(2)), dict(out=t(2, 40)), dict(out=x[:, :39]),
                dict(history=t(2, 1 << 19))):
        with pytest.raises(ValueError):
            G.adjust_logits(x, **bad)
    with pytest.raises(ValueError):
        G.adjust_logits(x.half())
    with pytest.raises(ValueError):
        G.adjust_logits(x[0])
    settle(device)
