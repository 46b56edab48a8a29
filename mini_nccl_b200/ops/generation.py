"""Operators for generating many continuations of one prompt.

* :func:`shared_prefix_attention` -- attention of new tokens over a prefix that
  the whole batch shares (computed once for all rows) and over each
  sequence's own tokens, both in a paged cache;
* :func:`adjust_logits` -- penalties for repeated tokens, biases and masks (of a
  grammar) on logits, before :func:`sample`;
* :func:`sample` -- temperature, top-k, top-p and min-p sampling from given
  random numbers;
* :func:`append_kv`, :func:`copy_pages`, :func:`fork_sequences`,
  :func:`reserve_pages`, :func:`free_sequences`, :func:`compact_pages` -- the
  page operations, and :class:`PagedKVCache`, which holds the tensors they
  work on.

A cache is held in bf16, or in 8 bits: codes (int8 or float8_e4m3fn) and one
fp32 scale for each page and kv head, a power of two.  A code stands for
``code * scale``; :func:`append_kv` chooses the scales, and the functions that
take pages take the scales with them.

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


#: The largest code of each type that an 8-bit cache may have.
TOP_CODE = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}
_LEAST_EXPONENT = -60  # of a scale


def _held_in_8_bits(k_pages: torch.Tensor, v_pages: torch.Tensor, k_scales: torch.Tensor | None, v_scales: torch.Tensor | None) -> bool:
    _need(k_pages.dim() == 4 and k_pages.shape == v_pages.shape and k_pages.dtype == v_pages.dtype,
          "k_pages and v_pages: [num_pages, page_size, kv_heads, head_dim] of one type")
    coded = k_pages.dtype in TOP_CODE
    _need((k_scales is not None and v_scales is not None) if coded else (k_scales is None and v_scales is None),
          "k_scales and v_scales: needed with pages of int8 or float8_e4m3fn, and only with them")
    for s in (k_scales, v_scales):
        _need(s is None or (s.dtype == torch.float32 and s.shape == (k_pages.shape[0], k_pages.shape[2])),
              "k_scales and v_scales: fp32 tensors [num_pages, kv_heads]")
    return coded


def _values(pages: torch.Tensor, scales: torch.Tensor | None, ids: torch.Tensor) -> torch.Tensor:
    """What the pages ``ids`` hold, in fp32 (CPU)."""
    if scales is None:
        return pages[ids].float()
    return pages.view(torch.uint8)[ids].view(pages.dtype).float() * scales[ids][:, None, :, None]


def _code(x: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """The nearest code to each of ``x``, of two the even one (CPU)."""
    top = TOP_CODE[dtype]
    if dtype == torch.int8:
        return torch.round(x.clamp(-top, top)).to(torch.int8)
    return x.clamp(-top, top).to(dtype)


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
    k_scales: torch.Tensor | None = None,
    v_scales: torch.Tensor | None = None,
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

    Pages of int8 or float8_e4m3fn come with ``k_scales`` and ``v_scales``, fp32
    ``[num_pages, kv_heads]`` of one layout: page p's keys of head h are
    ``k_pages[p, :, h] * k_scales[p, h]``.  Scales are powers of two from
    ``2 ** -60`` to ``2 ** 60`` (a smaller or no positive scale of values
    counts as ``2 ** -60``), as :func:`append_kv` leaves them for values up to
    1e20, or 0 where nothing was written; others only cost accuracy, as do
    scales more than ``2 ** 15`` apart within 128 tokens of the prefix, of which
    the smaller ones' values lose their lowest bits.

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
            -1 if max_q_len is None else max_q_len, -1 if max_seq_len is None else max_seq_len, scale, return_lse, k_scales, v_scales,
            K.status_word(q.device))
        if torch.is_grad_enabled() and (q.requires_grad or k_pages.requires_grad or v_pages.requires_grad
                                        or (k_scales is not None and (k_scales.requires_grad or v_scales.requires_grad))):
            o, lse = (None if t is None else _NoGradient.apply("shared_prefix_attention", t, q, k_pages, v_pages, k_scales, v_scales)
                      for t in (o, lse))
        return (o, lse) if return_lse else o
    _need(q.dim() == 3 and k_pages.dim() == 4 and k_pages.shape == v_pages.shape,
          "q: [tokens, heads, head_dim]; k_pages and v_pages: [num_pages, page_size, kv_heads, head_dim]")
    _held_in_8_bits(k_pages, v_pages, k_scales, v_scales)
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
        k, v = (_values(p, s, ids.long()).reshape(-1, Hk, D)[:n].transpose(0, 1) for p, s in ((k_pages, k_scales), (v_pages, v_scales)))
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


def adjust_logits(
    logits: torch.Tensor,
    *,
    prompt: torch.Tensor | None = None,
    history: torch.Tensor | None = None,
    history_lens: torch.Tensor | None = None,
    repetition: Setting = 1.0,
    presence: Setting = 0.0,
    frequency: Setting = 0.0,
    bias_tokens: torch.Tensor | None = None,
    bias: torch.Tensor | None = None,
    allowed: torch.Tensor | None = None,
    mask_of: torch.Tensor | None = None,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """Penalties, biases and masks on ``logits`` ``[rows, vocabulary]`` (bf16 or fp32), for :func:`sample`.

    With x the logit of token v in row r, and c the number of times that v is
    among the row's ``history``, in this order and in fp32, rounded once:

    * ``x = x / repetition`` if x is above 0, else ``x * repetition``, where v is
      in the history or in the ``prompt``;
    * ``x = x - (frequency * c + presence)`` where v is in the history;
    * ``x = x + bias[r, i]`` where ``bias_tokens[r, i]`` is v (of a token that is
      named twice the later one);
    * ``x = -inf`` where the row's mask does not allow v.

    ``history`` is ``[rows, n]``, its first ``history_lens`` (int32, one for each
    row; default all) tokens counting; ``prompt`` ``[rows, n]``, or ``[n]`` for
    all rows, as are ``bias_tokens`` and ``bias`` (fp32).  Tokens are int64 or
    int32; negative ones are padding.  ``repetition`` (above 0), ``presence`` and
    ``frequency`` are numbers or fp32 tensors with one entry for each row.
    ``allowed`` holds masks, int32 ``[masks, (vocabulary + 31) // 32]``: bit
    ``v % 32`` of word ``v // 32`` allows token v.  Row r has mask
    ``mask_of[r]`` (int32, a negative one is no mask); without ``mask_of`` mask r,
    or the only one.

    Returns a new tensor, or ``out``, which may be ``logits`` itself (then tokens
    that nothing names are neither read nor written) but no other memory that
    overlaps it.  A token or a mask that there is none of, and a length outside
    the history (the history then counts for nothing), are reported.
    """
    if logits.is_cuda:
        K, tensor = _kernels(), torch.Tensor
        rho, by_rho = (repetition, 0.0) if isinstance(repetition, tensor) else (None, repetition)
        alpha, by_alpha = (presence, 0.0) if isinstance(presence, tensor) else (None, presence)
        phi, by_phi = (frequency, 0.0) if isinstance(frequency, tensor) else (None, frequency)
        wanted = torch.is_grad_enabled() and (
            logits.requires_grad or (rho is not None and rho.requires_grad) or (alpha is not None and alpha.requires_grad)
            or (phi is not None and phi.requires_grad) or (bias is not None and bias.requires_grad))
        _need(not wanted or out is not logits, "out: not in place where a gradient is wanted")
        y = K.ext().adjust_logits(logits, out, prompt, history, history_lens, rho, by_rho, alpha, by_alpha, phi, by_phi, bias_tokens, bias,
                                  allowed, mask_of, K.status_word(logits.device))
        return _NoGradient.apply("adjust_logits", y, logits, rho, alpha, phi, bias) if wanted else y if out is None else out
    _need(logits.dim() == 2 and logits.dtype in (torch.bfloat16, torch.float32),
          "logits: a bf16 or fp32 tensor [rows, vocabulary]")
    R, V = logits.shape
    _need(1 <= V <= 1 << 20, f"vocabulary: 1 to 1048576 tokens, got {V}")
    if out is None:
        out = torch.empty(logits.shape, dtype=logits.dtype)
    _need(out.shape == logits.shape and out.dtype == logits.dtype, "out: a tensor like logits")

    def column(x, what):
        if isinstance(x, torch.Tensor):
            _need(x.dtype == torch.float32 and x.shape == (R,), f"{what}: a number, or an fp32 tensor with one entry for each row")
            return x[:, None]
        return torch.full((R, 1), float(x))

    def listed(t, shared, what):
        _need(t.dtype in (torch.int64, torch.int32) and ((t.dim() == 2 and t.shape[0] == R) or (shared and t.dim() == 1)),
              f"{what}: int64 or int32 tokens [rows, n]" + (" or [n]" if shared else ""))
        if t.numel() and int(t.max()) >= V:
            raise RuntimeError(f"{what}: a token outside the vocabulary")
        return t.long().expand(R, t.shape[-1])

    rho, alpha, phi = column(repetition, "repetition"), column(presence, "presence"), column(frequency, "frequency")
    count, seen = torch.zeros(R, V + 1), torch.zeros(R, V + 1, dtype=torch.bool)  # (the last one is padding's)
    _need(history_lens is None or history is not None, "history_lens: needs history")
    if history is not None:
        ids = listed(history, False, "history")
        _need(ids.shape[1] < 1 << 19, "history: at most 524287 tokens a row")
        if history_lens is not None:
            _ints(history_lens, 1, "history_lens")
            _need(history_lens.shape[0] == R, "history_lens: one length for each row of history")
            if R and (int(history_lens.min()) < 0 or int(history_lens.max()) > ids.shape[1]):
                raise RuntimeError("history_lens: a length outside the history")
            ids = torch.where(torch.arange(ids.shape[1]) < history_lens[:, None], ids, -1)
        count.scatter_add_(1, torch.where(ids < 0, V, ids), torch.ones(ids.shape))
    if prompt is not None:
        ids = listed(prompt, True, "prompt")
        seen.scatter_(1, torch.where(ids < 0, V, ids), True)
    count, seen = count[:, :V], seen[:, :V]
    x = logits.float()
    x = torch.where((count > 0) | seen, torch.where(x > 0, x / rho, x * rho), x)
    x = torch.where(count > 0, x - (phi * count + alpha), x)
    _need((bias is None) == (bias_tokens is None), "bias_tokens and bias: one needs the other")
    if bias is not None:
        _need(bias.dtype == torch.float32 and bias.shape == bias_tokens.shape, "bias: fp32, of the tokens' shape")
        ids = listed(bias_tokens, True, "bias_tokens")
        _need(ids.shape[1] <= 4095, "bias_tokens: at most 4095 a row")
        last = torch.full((R, V + 1), -1).scatter_reduce_(
            1, torch.where(ids < 0, V, ids), torch.arange(ids.shape[1]).expand(R, -1), "amax")[:, :V]
        if ids.shape[1]:
            x = torch.where(last >= 0, x + bias.expand(R, -1).gather(1, last.clamp(min=0)), x)
    _need(mask_of is None or allowed is not None, "mask_of: needs allowed")
    if allowed is not None:
        _ints(allowed, 2, "allowed")
        _need(allowed.shape[1] == -(-V // 32), f"allowed: {-(-V // 32)} words of 32 tokens a mask")
        if mask_of is None:
            _need(allowed.shape[0] in (1, R), "allowed: without mask_of one mask, or one for each row")
            of = torch.arange(R) if allowed.shape[0] == R else torch.zeros(R, dtype=torch.long)
        else:
            _ints(mask_of, 1, "mask_of")
            _need(mask_of.shape[0] == R, "mask_of: one mask for each row")
            of = mask_of.long()
            if R and int(of.max()) >= allowed.shape[0]:
                raise RuntimeError("mask_of: a mask that there is none of")
        if allowed.shape[0]:
            v = torch.arange(V)
            bits = (allowed[of.clamp(min=0)][:, v // 32] >> (v % 32).int()) & 1
            x = torch.where((bits != 0) | (of < 0)[:, None], x, -math.inf)
    return out.copy_(x)


# ---- pages ---------------------------------------------------------------------------


def _pool(kv: torch.Tensor, scales: torch.Tensor | None = None) -> tuple[torch.Tensor, ...]:
    """The pool as ``[planes, num_pages, page_size, kv_heads, head_dim]``, and its scales, if any, as ``[planes, num_pages, kv_heads]``."""
    _need(kv.dim() >= 4 and kv.is_contiguous() and kv.numel() > 0,
          "kv: a contiguous tensor [..., num_pages, page_size, kv_heads, head_dim]")
    _need(kv.shape[-1] * kv.shape[-2] * kv.element_size() % 16 == 0, "kv: a token's keys must be a multiple of 16 bytes")
    if kv.dtype == torch.float8_e4m3fn:
        kv = kv.view(torch.uint8)
    if scales is None:
        return (kv.view(-1, *kv.shape[-4:]),)
    _need(scales.dtype == torch.float32 and scales.is_contiguous() and scales.shape == (*kv.shape[:-3], kv.shape[-2]),
          "scales: a contiguous fp32 tensor [..., num_pages, kv_heads] with the leading axes of kv")
    return kv.view(-1, *kv.shape[-4:]), scales.view(-1, *scales.shape[-2:])


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
    *,
    k_scales: torch.Tensor | None = None,
    v_scales: torch.Tensor | None = None,
) -> None:
    """Write the keys and values of tokens into their sequences' pages.

    Token i of ``k`` and ``v`` ``[tokens, kv_heads, head_dim]`` goes to place
    ``positions[i]`` of the sequence in row ``slots[i]`` of ``page_table`` (row
    i without ``slots``); a negative position is padding and is left out.  The
    pages have to be there (:func:`reserve_pages`) and must not be shared.

    Pages of int8 or float8_e4m3fn come with ``k_scales`` and ``v_scales``, fp32
    ``[num_pages, kv_heads]``, which are written too (so they do not share
    memory).  A page's values of one head share a scale, the least power of two
    (from ``2 ** -60`` on) whose multiple by the largest code (127 or 448) is at
    least the largest of them; each value becomes the nearest code, of two the
    even one.  Writing a page's first place begins the page: its scale then comes from this call's tokens
    alone.  Otherwise the scale only grows, and the codes that are there are
    rounded to the new one.  Values that are not finite do not count for the
    scale; an infinite one is stored as the largest code, NaN as float8_e4m3fn's
    NaN, or as int8 zero (and reported).  In a call the tokens of one page follow
    one another (padding aside), in any order; a place that is named twice gets
    the later one.  Tokens that come back to a page are left out and reported
    where a kernel sees it (among 32 tokens one after another, in calls of few);
    further apart what the page then holds is undefined.  Head dims that are multiples of 16, up to 256.
    """
    if k_pages.is_cuda:
        K = _kernels()
        K.ext().append_kv(k_pages, v_pages, k, v, page_table, positions, slots, k_scales, v_scales, K.status_word(k_pages.device))
        return
    _need(k_pages.dim() == 4 and v_pages.shape == k_pages.shape and k.shape == v.shape and k.dim() == 3
          and k.shape[1:] == k_pages.shape[2:], "k, v: [tokens, kv_heads, head_dim] as in the pages")
    coded = _held_in_8_bits(k_pages, v_pages, k_scales, v_scales)
    _need(not coded or (k.shape[2] % 16 == 0 and k.shape[2] <= 256), "head_dim: in 8 bits a multiple of 16, at most 256")
    _need(not coded or k_pages.numel() == 0 or (
        k_scales.data_ptr() != v_scales.data_ptr()
        and all(s.shape[i] <= 1 or s.stride(i) != 0 for s in (k_scales, v_scales) for i in (0, 1))),
        "k_scales and v_scales: memory of their own for each page and head")
    _ints(page_table, 2, "page_table")
    named = [(positions, "positions")] + ([(slots, "slots")] if slots is not None else [])
    where = _ids(*named)
    _need(len(where[0]) == k.shape[0], "positions: one for each token")
    _need(slots is not None or k.shape[0] <= page_table.shape[0],
          "without slots, token i belongs to row i of page_table: too many tokens")
    page, rows = k_pages.shape[1], page_table.tolist()
    runs: list[tuple[int, dict[int, int], list[int]]] = []  # a page, which token its places get, and all that the call has for it
    for i, pos in enumerate(where[0]):
        if pos < 0:
            continue
        s = where[1][i] if slots is not None else i
        if not (0 <= s < len(rows) and pos // page < len(rows[s]) and 0 <= rows[s][pos // page] < k_pages.shape[0]):
            raise RuntimeError(f"token {i}: no page for place {pos} of sequence {s}")
        if not coded:
            k_pages[rows[s][pos // page], pos % page] = k[i]
            v_pages[rows[s][pos // page], pos % page] = v[i]
            continue
        if not runs or runs[-1][0] != rows[s][pos // page]:
            _need(all(r[0] != rows[s][pos // page] for r in runs), "positions: in 8 bits, a page's tokens follow one another")
            runs.append((rows[s][pos // page], {}, []))
        runs[-1][1][pos % page] = i
        runs[-1][2].append(i)
    if coded and k_pages.dtype == torch.int8 and any(bool(x[r[2]].isnan().any()) for r in runs for x in (k, v)):
        raise RuntimeError("NaN cannot be held as int8")
    for p, places, tokens in runs:
        for pages, scales, x in ((k_pages, k_scales, k.float()), (v_pages, v_scales, v.float())):
            most = torch.where(x[tokens].isfinite(), x[tokens].abs(), 0.0).amax((0, 2))
            m, e = torch.frexp(most)
            top, shift = math.frexp(TOP_CODE[pages.dtype])
            e = torch.where(most > 0, e - shift + (m > top).int(), _LEAST_EXPONENT).clamp(min=_LEAST_EXPONENT)
            held = torch.zeros_like(scales[p]) if 0 in places else scales[p].clone()
            need = torch.ldexp(torch.ones_like(held), e)
            now = torch.where(held > need, held, need)
            if 0 not in places:
                ratio = torch.where(held > 0, held / now, 0.0)[:, None]
                again = _code(pages[p].float() * ratio, pages.dtype)
                pages.view(torch.uint8)[p] = torch.where((now != held)[:, None], again.view(torch.uint8), pages[p].view(torch.uint8))
            scales[p] = now
            code = _code(x[list(places.values())] / now[:, None], pages.dtype)
            pages.view(torch.uint8)[p, list(places)] = code.view(torch.uint8)


def copy_pages(kv: torch.Tensor, src: torch.Tensor, dst: torch.Tensor, scales: torch.Tensor | None = None) -> None:
    """Copy page ``src[i]`` to page ``dst[i]`` in every plane of ``kv``.

    ``kv`` is ``[..., num_pages, page_size, kv_heads, head_dim]``, of any
    dtype; the leading axes are the planes.  Pairs with a negative id are left
    out; no destination may be named twice or be a source as well.  ``scales``,
    fp32 ``[..., num_pages, kv_heads]``, are those of a cache in 8 bits and go
    with their pages (here and in the functions below).
    """
    if kv.is_cuda:
        K = _kernels()
        K.ext().copy_pages(kv, src, dst, scales, K.status_word(kv.device))
        return
    pools = _pool(kv, scales)
    for a, b in zip(*_ids((src, "src"), (dst, "dst"))):
        if a < 0 or b < 0:
            continue
        if max(a, b) >= pools[0].shape[1]:
            raise RuntimeError("a page id outside the pool")
        for pool in pools:
            pool[:, b] = pool[:, a]


def fork_sequences(
    kv: torch.Tensor,
    page_table: torch.Tensor,
    lens: torch.Tensor,
    refs: torch.Tensor,
    parents: torch.Tensor,
    children: torch.Tensor,
    scales: torch.Tensor | None = None,
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
        K.ext().fork_sequences(kv, page_table, lens, refs, parents, children, scales, K.status_word(kv.device))
        return
    pool, *of_scales = _pool(kv, scales)
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
            for t in of_scales:
                t[:, row[full]] = t[:, page_table[p, full]]
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
    kv: torch.Tensor, page_table: torch.Tensor, refs: torch.Tensor, scales: torch.Tensor | None = None
) -> tuple[torch.Tensor, torch.Tensor]:
    """Move the pages in use to the front of the pool; returns the new ``(page_table, refs)``.

    With n pages in use, those with ids from n on move, in ascending order, to
    the free ids below n, in every plane of ``kv``.  The given tables are left
    as they are.  Entries of ``page_table`` for free pages become -1.
    """
    if kv.is_cuda:
        K = _kernels()
        return K.ext().compact_pages(kv, page_table, refs, scales, K.status_word(kv.device))
    pool, *of_scales = _pool(kv, scales)
    _ints(page_table, 2, "page_table")
    _ints(refs, 1, "refs")
    _need(refs.shape[0] == pool.shape[1], "refs: one count for each page of kv")
    live = refs > 0
    n, at = int(live.sum()), torch.arange(refs.shape[0])
    src, dst = at[live & (at >= n)], at[~live & (at < n)]
    for t in (pool, *of_scales):
        t[:, dst] = t[:, src]
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
        self.scales = torch.zeros(n_layer, 2, num_pages, n_kv_head, device=device) if dtype in TOP_CODE else None
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
        append_kv(self.kv[layer, 0], self.kv[layer, 1], k, v, self.page_table, positions, slots, **self.scales_of(layer))

    def scales_of(self, layer: int) -> dict[str, torch.Tensor]:
        """One layer's scales as the operators' arguments (none for a cache that has none)."""
        return {} if self.scales is None else {"k_scales": self.scales[layer, 0], "v_scales": self.scales[layer, 1]}

    def fork(self, parents: Sequence[int], children: Sequence[int]) -> None:
        """Each child, an empty slot, becomes a copy of its parent (see :func:`fork_sequences`)."""
        self._slots(parents)
        self._slots(children)
        _need(len(parents) == len(children) and len(set(children)) == len(children)
              and not set(parents) & set(children) and all(self.lengths[c] == 0 for c in children),
              "children: one for each parent, distinct, empty and nobody's parent")
        if not children:
            return
        fork_sequences(self.kv, self.page_table, self.lens, self.refs, self._tensor(parents), self._tensor(children),
                       self.scales)
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
        self.page_table, self.refs = compact_pages(self.kv, self.page_table, self.refs, self.scales)

    def pages_in_use(self) -> int:
        """Number of pages that some sequence holds (waits for the device)."""
        return int((self.refs > 0).sum())
