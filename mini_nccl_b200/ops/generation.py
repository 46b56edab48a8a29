"""Operators for generating many continuations of one prompt.

* :func:`shared_prefix_attention` -- attention of new tokens over a prefix that
  the whole batch shares (computed once for all rows) and over each
  sequence's own tokens, both in a paged cache;
* :func:`sample` -- temperature, top-k, top-p and min-p sampling from given
  random numbers;
* :func:`append_kv`, :func:`copy_pages`, :func:`fork_sequences`,
  :func:`reserve_pages`, :func:`free_sequences`, :func:`compact_pages` -- the
  page operations, and :class:`PagedKVCache`, which holds the tensors they
  work on.

As in :mod:`mini_nccl_b200.ops.functional`, a CUDA tensor runs the sm_100a
kernel (and raises where the extension is missing), a CPU tensor the plain
PyTorch expression of the same definition.  Arguments that do not fit raise
``ValueError``.  What only the device knows -- page ids, lengths, a pool that
runs out of pages -- cannot raise without waiting for the GPU: the kernels
leave such a request out, never touch memory outside the tensors, and set the
device's status word, which :func:`mini_nccl_b200.ops.kernels.check_status`
turns into an error (the CPU path raises at once).  Nothing here has a
gradient on CUDA: these operators serve, they do not train, and a backward pass
through an output or a log-probability raises.
"""

from __future__ import annotations

import math
from collections.abc import Sequence

import torch


_KERNELS = None


def _kernels():
    global _KERNELS
    if _KERNELS is None:
        from . import kernels

        _KERNELS = kernels
    return _KERNELS


def _need(ok: bool, message: str) -> None:
    if not ok:
        raise ValueError(message)


def _ints(t: torch.Tensor, dim: int, what: str) -> None:
    _need(t.dtype == torch.int32 and t.dim() == dim, f"{what}: a {dim}-d int32 tensor")


class _NoGradient(torch.autograd.Function):
    """A kernel's result as a function of its inputs, for inputs that want a gradient: asking for it raises."""

    @staticmethod
    def forward(ctx, name, out, *inputs):
        ctx.name = name
        return out.view_as(out)

    @staticmethod
    def backward(ctx, *grads):
        raise RuntimeError(f"{ctx.name} has no gradient on CUDA: it serves, it does not train")


# ---- attention -----------------------------------------------------------------------


def shared_prefix_attention(
    q: torch.Tensor,
    k_pages: torch.Tensor,
    v_pages: torch.Tensor,
    prefix_pages: torch.Tensor,
    prefix_len: int,
    page_table: torch.Tensor,
    seq_lens: torch.Tensor,
    *,
    q_offsets: torch.Tensor | None = None,
    max_q_len: int | None = None,
    max_seq_len: int | None = None,
    scale: float | None = None,
    return_lse: bool = False,
) -> torch.Tensor | tuple[torch.Tensor, torch.Tensor]:
    """``softmax(scale q k^T) v`` over a shared prefix and each sequence's own tokens.

    ``q`` is ``[tokens, heads, head_dim]`` bf16 (any token and head stride; a
    slice of a fused projection is used in place); ``k_pages`` and ``v_pages``
    are ``[num_pages, page_size, kv_heads, head_dim]``, ``heads`` a multiple of
    ``kv_heads`` (query head h reads kv head ``h // (heads // kv_heads)``).
    Every token sees the ``prefix_len`` tokens in the pages ``prefix_pages``.
    Sequence b has ``seq_lens[b]`` tokens of its own, in the pages of row b of
    ``page_table``, the newest of which are its queries: tokens
    ``q_offsets[b]`` to ``q_offsets[b + 1]`` of ``q`` (``q_offsets`` ascends
    from 0 to ``tokens``; ``max_q_len`` bounds the differences), or token b
    alone without ``q_offsets``.  A query sees its sequence's own tokens up to
    and including itself.  A token that sees nothing gets zeros and a
    log-sum-exp of ``-inf``.  ``max_seq_len`` bounds ``seq_lens`` (default:
    what ``page_table`` can hold); a tight bound means fewer idle blocks.

    Returns ``o`` like ``q`` (contiguous) and, with ``return_lse``, the natural
    log-sum-exp of the scaled scores, fp32 ``[tokens, heads]``.  Head dims 32,
    64 and 128; page sizes 8 to 256, powers of two.

    On the device, a page id outside the pool reads as zeros, a sequence whose
    length is negative or above its bound has no tokens of its own, and with
    ``q_offsets`` that do not give every token to one sequence no token has;
    all are reported.
    """
    if scale is None:
        scale = 1.0 / math.sqrt(max(1, q.shape[-1]))
    if q.is_cuda:
        K = _kernels()
        o, lse = K.ext().shared_prefix_attention(
            q, k_pages, v_pages, prefix_pages, prefix_len, page_table, seq_lens, q_offsets,
            -1 if max_q_len is None else max_q_len, -1 if max_seq_len is None else max_seq_len, scale, return_lse,
            K.status_word(q.device))
        if torch.is_grad_enabled() and (q.requires_grad or k_pages.requires_grad or v_pages.requires_grad):
            o, lse = (None if t is None else _NoGradient.apply("shared_prefix_attention", t, q, k_pages, v_pages) for t in (o, lse))
        return (o, lse) if return_lse else o
    _need(q.dim() == 3 and k_pages.dim() == 4 and k_pages.shape == v_pages.shape,
          "q: [tokens, heads, head_dim]; k_pages and v_pages: [num_pages, page_size, kv_heads, head_dim]")
    _ints(prefix_pages, 1, "prefix_pages")
    _ints(page_table, 2, "page_table")
    _ints(seq_lens, 1, "seq_lens")
    N, H, D = q.shape
    pages, page, Hk, B = k_pages.shape[0], k_pages.shape[1], k_pages.shape[2], page_table.shape[0]
    _need(D in (32, 64, 128) and k_pages.shape[3] == D, "head_dim: 32, 64 or 128, the same in q and the pages")
    _need(Hk > 0 and H > 0 and H % Hk == 0, "heads: a multiple of the pages' kv heads")
    _need(8 <= page <= 256 and page & (page - 1) == 0, "page_size: a power of two from 8 to 256")
    _need(seq_lens.shape[0] == B, "seq_lens: one length for each row of page_table")
    _need(0 <= prefix_len <= prefix_pages.shape[0] * page, "prefix_len: 0 to the tokens of prefix_pages")
    room = page_table.shape[1] * page
    _need(max_seq_len is None or max_seq_len <= room, "max_seq_len: at most the tokens of a row of page_table")
    if q_offsets is None:
        _need(N == B, "without q_offsets there is one token for each sequence")
        offsets = list(range(B + 1))
    else:
        _ints(q_offsets, 1, "q_offsets")
        _need(q_offsets.shape[0] == B + 1, "q_offsets: one more entry than page_table has rows")
        _need(max_q_len is not None and max_q_len >= 0, "max_q_len: needed with q_offsets")
        _need(N == 0 or B > 0, "q_offsets: no sequence for the tokens")
        _need(N == 0 or max_q_len > 0, "max_q_len: at least 1 where there are tokens")
        offsets = q_offsets.tolist()
        if offsets[0] != 0 or offsets[-1] != N or any(not 0 <= b - a <= max_q_len for a, b in zip(offsets, offsets[1:])):
            raise RuntimeError("q_offsets: ascending from 0 to the number of tokens, in steps of at most max_q_len")
    limit = room if max_seq_len is None or max_seq_len < 0 else max_seq_len

    def tokens(ids: torch.Tensor, n: int) -> tuple[torch.Tensor, torch.Tensor]:
        if n and (int(ids.min()) < 0 or int(ids.max()) >= pages):
            raise RuntimeError("a page id outside the pool")
        k, v = (p[ids.long()].reshape(-1, Hk, D)[:n].float().transpose(0, 1) for p in (k_pages, v_pages))
        return k, v

    o = torch.zeros(N, H, D, dtype=q.dtype)
    lse = torch.full((N, H), -math.inf)
    k0, v0 = tokens(prefix_pages[: -(-prefix_len // page)], prefix_len)
    for b, length in enumerate(seq_lens.tolist()):
        if not 0 <= length <= limit:
            raise RuntimeError(f"seq_lens[{b}] = {length}, outside 0 to {limit}")
        n = offsets[b + 1] - offsets[b]
        if not n:
            continue
        k1, v1 = tokens(page_table[b, : -(-length // page)], length)
        k, v = torch.cat([k0, k1], 1), torch.cat([v0, v1], 1)
        if not k.shape[1]:
            continue
        qb = q[offsets[b]: offsets[b + 1]].float().view(n, Hk, H // Hk, D)
        s = torch.einsum("nhgd,hkd->nhgk", qb, k) * scale
        seen = prefix_len + (length - n + 1 + torch.arange(n)).clamp(min=0)
        s.masked_fill_((torch.arange(k.shape[1]) >= seen[:, None])[:, None, None], -math.inf)
        m = torch.logsumexp(s, -1, keepdim=True)
        p = torch.exp(s - torch.where(m == -math.inf, 0.0, m))
        if n > 1 and not torch.isfinite(v).all():  # a weight of 0 times a hidden value that is no number would be NaN
            y = torch.stack([torch.einsum("hgk,hkd->hgd", p[t, ..., :e], v[:, :e]) for t, e in enumerate(seen.tolist())])
        else:
            y = torch.einsum("nhgk,hkd->nhgd", p, v)
        o[offsets[b]: offsets[b + 1]] = y.reshape(n, H, D).to(q.dtype)
        lse[offsets[b]: offsets[b + 1]] = m.reshape(n, H)
    return (o, lse) if return_lse else o


# ---- sampling ------------------------------------------------------------------------

Setting = float | torch.Tensor


def sample(
    logits: torch.Tensor,
    noise: torch.Tensor,
    *,
    temperature: Setting = 1.0,
    top_k: int | torch.Tensor = 0,
    top_p: Setting = 1.0,
    min_p: Setting = 0.0,
    return_logprob: bool = False,
) -> torch.Tensor | tuple[torch.Tensor, torch.Tensor]:
    """Draw one token for each row of ``logits`` ``[rows, vocabulary]`` (bf16 or fp32).

    Order a row by logit, equal logits by index.  ``top_k`` keeps the first k
    tokens (0, or a k of at least the vocabulary: all); ``top_p`` those before
    which less than p of the remaining probability lies (1 or more: all; the
    first token always stays); ``min_p`` (at most 1) those with at least
    ``min_p`` times the first one's probability.  The token with the largest
    ``logit / temperature + noise`` among what is left is returned, of equals
    the one with the lowest index: with ``noise`` from the standard Gumbel
    distribution, fp32 ``[rows, vocabulary]``, that is a draw from the
    filtered softmax, and the same noise gives the same token whatever the
    batch (except that ``top_p`` compares fp32 sums, whose order depends on the
    number of rows: a token within their rounding of the cut may fall on either
    side).  A temperature of 0 (or less) takes the first token.  Each setting
    is a number or a tensor with one entry for each row (fp32; ``top_k``
    int32).  Logits of ``-inf`` and NaN are never drawn, and a row without any
    other returns token -1.

    Returns int64 tokens and, with ``return_logprob``, the log-probability of
    each under its row's filtered distribution (fp32).
    """
    if logits.is_cuda:

        def split(x, whole):
            return (x, whole(0)) if isinstance(x, torch.Tensor) else (None, whole(x))

        K = _kernels()
        heat, nucleus, least = split(temperature, float), split(top_p, float), split(min_p, float)
        token, logprob = K.ext().sample(logits, noise, *heat, *split(top_k, int), *nucleus, *least, return_logprob,
                                        K.status_word(logits.device))
        if return_logprob and torch.is_grad_enabled() and (
                logits.requires_grad or noise.requires_grad or (heat[0] is not None and heat[0].requires_grad)
                or (nucleus[0] is not None and nucleus[0].requires_grad) or (least[0] is not None and least[0].requires_grad)):
            logprob = _NoGradient.apply("sample", logprob, logits, noise, heat[0], nucleus[0], least[0])
        return (token, logprob) if return_logprob else token
    _need(logits.dim() == 2 and logits.dtype in (torch.bfloat16, torch.float32),
          "logits: a bf16 or fp32 tensor [rows, vocabulary]")
    R, V = logits.shape
    _need(1 <= V <= 1 << 20, f"vocabulary: 1 to 1048576 tokens, got {V}")
    _need(noise.shape == logits.shape and noise.dtype == torch.float32, "noise: an fp32 tensor of the logits' shape")

    def column(x, dtype, what):
        if isinstance(x, torch.Tensor):
            _need(x.dtype == dtype and x.shape == (R,), f"{what}: a number, or a {dtype} tensor with one entry for each row")
            return x[:, None]
        return torch.full((R, 1), x, dtype=dtype)

    if not isinstance(top_k, torch.Tensor):
        top_k = min(max(int(top_k), 0), V)
    T, k = column(temperature, torch.float32, "temperature"), column(top_k, torch.int32, "top_k")
    p, least = column(top_p, torch.float32, "top_p"), column(min_p, torch.float32, "min_p").clamp(max=1)
    x = logits.float()
    x = torch.where(x.isnan(), -math.inf, x)
    xs, order = torch.sort(x, dim=-1, descending=True, stable=True)
    top = xs[:, :1]
    heat = torch.where(T > 0, T, 1.0)
    rank = torch.arange(V)
    k = torch.where(T > 0, torch.where(k > 0, k, V), 1)
    delta = torch.where(xs == top, 0.0, (xs - top) / heat)
    left = (rank < k) & (xs > -math.inf)
    w = torch.where(left, torch.exp(delta), 0.0)
    before = torch.cumsum(w, -1) - w
    keep = left & ((p >= 1) | (before < p * w.sum(-1, keepdim=True))) & (w >= least)
    keep |= left & (rank == 0)
    total = torch.where(keep, w, 0.0).sum(-1)
    kept = torch.zeros_like(keep).scatter_(1, order, keep)
    score = torch.where(kept, x / heat + noise, -math.inf)
    score = torch.where(score.isnan(), -math.inf, score)
    token = torch.where(kept & (score == score.amax(-1, keepdim=True)), rank, V).amin(-1)
    token = torch.where(token == V, -1, token)
    if not return_logprob:
        return token
    chosen = x.gather(1, token.clamp(min=0)[:, None])
    logprob = torch.where(chosen == top, 0.0, (chosen - top) / heat)[:, 0] - torch.log(total)
    return token, torch.where(token < 0, -math.inf, logprob)


# ---- pages ---------------------------------------------------------------------------


def _pool(kv: torch.Tensor) -> torch.Tensor:
    """The pool as ``[planes, num_pages, page_size, kv_heads, head_dim]``."""
    _need(kv.dim() >= 4 and kv.is_contiguous() and kv.numel() > 0,
          "kv: a contiguous tensor [..., num_pages, page_size, kv_heads, head_dim]")
    _need(kv.shape[-1] * kv.shape[-2] * kv.element_size() % 16 == 0, "kv: a token's keys must be a multiple of 16 bytes")
    return kv.view(-1, *kv.shape[-4:])


def _state(page_table: torch.Tensor, lens: torch.Tensor, refs: torch.Tensor) -> None:
    _ints(page_table, 2, "page_table")
    _ints(lens, 1, "lens")
    _ints(refs, 1, "refs")
    _need(lens.shape[0] == page_table.shape[0], "lens: one entry for each row of page_table")


def _ids(*named: tuple[torch.Tensor, str]) -> list[list[int]]:
    for t, what in named:
        _ints(t, 1, what)
    _need(len({t.shape[0] for t, _ in named}) == 1, " and ".join(w for _, w in named) + ": one entry for each other")
    return [t.tolist() for t, _ in named]


def _free_ids(refs: torch.Tensor) -> list[int]:
    return torch.nonzero(refs == 0)[:, 0].tolist()


def append_kv(
    k_pages: torch.Tensor,
    v_pages: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    page_table: torch.Tensor,
    positions: torch.Tensor,
    slots: torch.Tensor | None = None,
) -> None:
    """Write the keys and values of tokens into their sequences' pages.

    Token i of ``k`` and ``v`` ``[tokens, kv_heads, head_dim]`` goes to place
    ``positions[i]`` of the sequence in row ``slots[i]`` of ``page_table`` (row
    i without ``slots``); a negative position is padding and is left out.  The
    pages have to be there (:func:`reserve_pages`) and must not be shared.
    """
    if k_pages.is_cuda:
        K = _kernels()
        K.ext().append_kv(k_pages, v_pages, k, v, page_table, positions, slots, K.status_word(k_pages.device))
        return
    _need(k_pages.dim() == 4 and v_pages.shape == k_pages.shape and k.shape == v.shape and k.dim() == 3
          and k.shape[1:] == k_pages.shape[2:], "k, v: [tokens, kv_heads, head_dim] as in the pages")
    _ints(page_table, 2, "page_table")
    named = [(positions, "positions")] + ([(slots, "slots")] if slots is not None else [])
    where = _ids(*named)
    _need(len(where[0]) == k.shape[0], "positions: one for each token")
    _need(slots is not None or k.shape[0] <= page_table.shape[0],
          "without slots, token i belongs to row i of page_table: too many tokens")
    page, rows = k_pages.shape[1], page_table.tolist()
    for i, pos in enumerate(where[0]):
        if pos < 0:
            continue
        s = where[1][i] if slots is not None else i
        if not (0 <= s < len(rows) and pos // page < len(rows[s]) and 0 <= rows[s][pos // page] < k_pages.shape[0]):
            raise RuntimeError(f"token {i}: no page for place {pos} of sequence {s}")
        k_pages[rows[s][pos // page], pos % page] = k[i]
        v_pages[rows[s][pos // page], pos % page] = v[i]


def copy_pages(kv: torch.Tensor, src: torch.Tensor, dst: torch.Tensor) -> None:
    """Copy page ``src[i]`` to page ``dst[i]`` in every plane of ``kv``.

    ``kv`` is ``[..., num_pages, page_size, kv_heads, head_dim]``, of any
    dtype; the leading axes are the planes.  Pairs with a negative id are left
    out; no destination may be named twice or be a source as well.
    """
    if kv.is_cuda:
        K = _kernels()
        K.ext().copy_pages(kv, src, dst, K.status_word(kv.device))
        return
    pool = _pool(kv)
    for a, b in zip(*_ids((src, "src"), (dst, "dst"))):
        if a < 0 or b < 0:
            continue
        if max(a, b) >= pool.shape[1]:
            raise RuntimeError("a page id outside the pool")
        pool[:, b] = pool[:, a]


def fork_sequences(
    kv: torch.Tensor,
    page_table: torch.Tensor,
    lens: torch.Tensor,
    refs: torch.Tensor,
    parents: torch.Tensor,
    children: torch.Tensor,
) -> None:
    """Make the empty sequence ``children[i]`` a copy of sequence ``parents[i]``.

    Full pages are shared (their ``refs`` grow); the tokens of a part-filled
    last page are copied, in every plane of ``kv``, to a page of the child's
    own, so appending to either never touches the other.  New pages are the
    lowest free ids, in the order of the requests.  Children are distinct,
    empty (length 0) and nobody's parent in the same call; a request that
    breaks this, finds no free page, or whose parent's row names a page outside
    the pool, is left out and reported.
    """
    if kv.is_cuda:
        K = _kernels()
        K.ext().fork_sequences(kv, page_table, lens, refs, parents, children, K.status_word(kv.device))
        return
    pool = _pool(kv)
    _state(page_table, lens, refs)
    _need(refs.shape[0] == pool.shape[1], "refs: one count for each page of kv")
    ps, cs = _ids((parents, "parents"), (children, "children"))
    page, (S, W) = pool.shape[2], page_table.shape
    for i, (p, c) in enumerate(zip(ps, cs)):
        if not (0 <= p < S and 0 <= c < S and cs.index(c) == i and p not in cs and int(lens[c]) == 0
                and 0 <= int(lens[p]) <= W * page):
            raise RuntimeError(f"fork {i}: sequence {p} to {c} (children are distinct, empty and nobody's parent)")
        held = page_table[p, : -(-int(lens[p]) // page)]
        if held.numel() and (int(held.min()) < 0 or int(held.max()) >= pool.shape[1]):
            raise RuntimeError(f"fork {i}: the row of sequence {p} names a page outside the pool")
    free = _free_ids(refs)
    if sum(int(lens[p]) % page > 0 for p in ps) > len(free):
        raise RuntimeError("the pool has too few free pages")
    for p, c in zip(ps, cs):
        full, part = divmod(int(lens[p]), page)
        row = page_table[p].clone()
        row[full:] = -1
        refs.index_add_(0, row[:full].long(), torch.ones(full, dtype=torch.int32))
        if part:
            row[full] = free.pop(0)
            pool[:, row[full], :part] = pool[:, page_table[p, full], :part]
            refs[row[full]] = 1
        page_table[c], lens[c] = row, lens[p]


def reserve_pages(
    page_table: torch.Tensor,
    lens: torch.Tensor,
    refs: torch.Tensor,
    slots: torch.Tensor,
    counts: torch.Tensor,
    page_size: int,
) -> None:
    """Make sequence ``slots[i]`` longer by ``counts[i]`` tokens, with pages for them.

    ``lens`` grows at once; :func:`append_kv` fills the new places.  New pages
    are the lowest free ids, in the order of the requests; a request whose
    pages (with those of the requests before it) the pool does not have is
    left out and reported.
    """
    if page_table.is_cuda:
        K = _kernels()
        K.ext().reserve_pages(page_table, lens, refs, slots, counts, page_size, K.status_word(page_table.device))
        return
    _need(page_size >= 1, "page_size: at least 1")
    _state(page_table, lens, refs)
    ss, ns = _ids((slots, "slots"), (counts, "counts"))
    S, W = page_table.shape
    for i, (s, n) in enumerate(zip(ss, ns)):
        if not (0 <= s < S and n >= 0 and ss.index(s) == i and int(lens[s]) + n <= min(W * page_size, 2 ** 31 - 1)):
            raise RuntimeError(f"reserve {i}: {n} tokens for sequence {s}")
    free = _free_ids(refs)
    new = [range(-(-int(lens[s]) // page_size), -(-(int(lens[s]) + n) // page_size)) for s, n in zip(ss, ns)]
    if sum(map(len, new)) > len(free):
        raise RuntimeError("the pool has too few free pages")
    for s, n, columns in zip(ss, ns, new):
        for column in columns:
            page_table[s, column] = free.pop(0)
            refs[page_table[s, column]] = 1
        lens[s] += n


def free_sequences(page_table: torch.Tensor, lens: torch.Tensor, refs: torch.Tensor, slots: torch.Tensor) -> None:
    """Empty the sequences ``slots``: each of their pages loses one holder.

    A page without holders is free (``refs`` 0).  Naming a slot twice frees it
    once.  On the device a row is emptied also where it names a page that is
    none, or that nobody holds: that entry is dropped and reported.
    """
    if page_table.is_cuda:
        K = _kernels()
        K.ext().free_sequences(page_table, lens, refs, slots, K.status_word(page_table.device))
        return
    _state(page_table, lens, refs)
    (ss,) = _ids((slots, "slots"))
    for s in ss:
        if not 0 <= s < page_table.shape[0]:
            raise RuntimeError(f"no sequence {s}")
        held = page_table[s][page_table[s] >= 0].long()
        if held.numel() and (int(held.max()) >= refs.shape[0] or int(refs[held].min()) <= 0):
            raise RuntimeError(f"sequence {s} names a page that nobody holds")
        refs.index_add_(0, held, torch.full((held.numel(),), -1, dtype=torch.int32))
        page_table[s], lens[s] = -1, 0


def compact_pages(
    kv: torch.Tensor, page_table: torch.Tensor, refs: torch.Tensor
) -> tuple[torch.Tensor, torch.Tensor]:
    """Move the pages in use to the front of the pool; returns the new ``(page_table, refs)``.

    With n pages in use, those with ids from n on move, in ascending order, to
    the free ids below n, in every plane of ``kv``.  The given tables are left
    as they are.  Entries of ``page_table`` for free pages become -1.
    """
    if kv.is_cuda:
        K = _kernels()
        return K.ext().compact_pages(kv, page_table, refs, K.status_word(kv.device))
    pool = _pool(kv)
    _ints(page_table, 2, "page_table")
    _ints(refs, 1, "refs")
    _need(refs.shape[0] == pool.shape[1], "refs: one count for each page of kv")
    live = refs > 0
    n, at = int(live.sum()), torch.arange(refs.shape[0])
    src, dst = at[live & (at >= n)], at[~live & (at < n)]
    pool[:, dst] = pool[:, src]
    to = torch.where(live, at, -1)
    to[src] = dst
    moved = torch.zeros_like(refs)
    moved[to[live]] = refs[live]
    inside = (page_table >= 0) & (page_table < refs.shape[0])
    return torch.where(inside, to[torch.where(inside, page_table, 0).long()].int(), -1), moved


class PagedKVCache:
    """Keys and values of up to ``max_seqs`` sequences, in pages of ``page_size`` tokens.

    ``kv`` is ``[n_layer, 2, num_pages, page_size, n_kv_head, head_dim]`` (keys
    are ``kv[layer, 0]``, values ``kv[layer, 1]``); a page id names the same
    page of every layer.  ``page_table``, ``lens`` and ``refs`` are the device
    tensors that the operators of this module work on; ``lengths`` is the
    host's copy of ``lens``, so planning a step needs no synchronisation.
    Sequences are named by slots, whole numbers below ``max_seqs``.
    """

    def __init__(self, n_layer: int, num_pages: int, page_size: int, n_kv_head: int, head_dim: int, *, max_seqs: int,
                 max_seq_len: int, device: torch.device | str = "cuda", dtype: torch.dtype = torch.bfloat16) -> None:
        _need(min(n_layer, num_pages, n_kv_head, head_dim, max_seqs, max_seq_len) > 0, "every size: at least 1")
        _need(8 <= page_size <= 256 and page_size & (page_size - 1) == 0, "page_size: a power of two from 8 to 256")
        self.page_size = page_size
        self.kv = torch.zeros(n_layer, 2, num_pages, page_size, n_kv_head, head_dim, dtype=dtype, device=device)
        ints = dict(dtype=torch.int32, device=device)
        self.page_table = torch.full((max_seqs, -(-max_seq_len // page_size)), -1, **ints)
        self.lens = torch.zeros(max_seqs, **ints)
        self.refs = torch.zeros(num_pages, **ints)
        self.lengths = [0] * max_seqs

    def _tensor(self, values: Sequence[int]) -> torch.Tensor:
        return torch.tensor(list(values), dtype=torch.int32, device=self.kv.device)

    def _slots(self, slots: Sequence[int]) -> None:
        _need(all(0 <= s < len(self.lengths) for s in slots), f"slots: 0 to {len(self.lengths) - 1}")

    def extend(self, slots: Sequence[int], counts: Sequence[int], slot_ids: torch.Tensor | None = None,
               count_ids: torch.Tensor | None = None) -> None:
        """Room for ``counts[i]`` more tokens in each slot (``slot_ids`` / ``count_ids``: the same
        numbers on the device, where a loop has them already)."""
        self._slots(slots)
        _need(len(slots) == len(counts) and len(set(slots)) == len(slots), "slots: distinct, one count for each")
        room = self.page_table.shape[1] * self.page_size
        _need(all(n >= 0 and self.lengths[s] + n <= room for s, n in zip(slots, counts)),
              f"a sequence holds at most {room} tokens")
        reserve_pages(self.page_table, self.lens, self.refs, self._tensor(slots) if slot_ids is None else slot_ids,
                      self._tensor(counts) if count_ids is None else count_ids, self.page_size)
        for s, n in zip(slots, counts):
            self.lengths[s] += n

    def append(self, layer: int, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor,
               slots: torch.Tensor | None = None) -> None:
        """Keys and values of one layer, for places that :meth:`extend` made (see :func:`append_kv`)."""
        append_kv(self.kv[layer, 0], self.kv[layer, 1], k, v, self.page_table, positions, slots)

    def fork(self, parents: Sequence[int], children: Sequence[int]) -> None:
        """Each child, an empty slot, becomes a copy of its parent (see :func:`fork_sequences`)."""
        self._slots(parents)
        self._slots(children)
        _need(len(parents) == len(children) and len(set(children)) == len(children)
              and not set(parents) & set(children) and all(self.lengths[c] == 0 for c in children),
              "children: one for each parent, distinct, empty and nobody's parent")
        if not children:
            return
        fork_sequences(self.kv, self.page_table, self.lens, self.refs, self._tensor(parents), self._tensor(children))
        for p, c in zip(parents, children):
            self.lengths[c] = self.lengths[p]

    def free(self, slots: Sequence[int]) -> None:
        """Empty the slots; pages that nobody else holds become free."""
        self._slots(slots)
        if not slots:
            return
        free_sequences(self.page_table, self.lens, self.refs, self._tensor(slots))
        for s in slots:
            self.lengths[s] = 0

    def compact(self) -> None:
        """Move the pages in use to the front of the pool (see :func:`compact_pages`)."""
        self.page_table, self.refs = compact_pages(self.kv, self.page_table, self.refs)

    def pages_in_use(self) -> int:
        """Number of pages that some sequence holds (waits for the device)."""
        return int((self.refs > 0).sum())
