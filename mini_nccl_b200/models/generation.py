"""Many continuations of one prompt from a :class:`~mini_nccl_b200.models.gpt.GPT`.

The prompt runs through the model once and its keys and values stay in a paged
cache; every continuation ("branch") adds pages of its own.  A step feeds one
token per branch: the attention reads the prompt's pages once for all branches
(:func:`~mini_nccl_b200.ops.generation.shared_prefix_attention`), the next
tokens are drawn by :func:`~mini_nccl_b200.ops.generation.sample`, and branches
are copied, dropped and moved together by the page operations.  A CUDA model
(bf16) runs the sm_100a kernels, a CPU model the plain PyTorch path.
"""

from __future__ import annotations

from collections.abc import Callable, Sequence

import torch

from ..ops import functional as F
from ..ops import generation as G
from .gpt import GPT, Block


def _add_linear(x: torch.Tensor, layer: torch.nn.Linear, resid: torch.Tensor) -> torch.Tensor:
    """``resid + layer(x)``; the addition rides in the GEMM's epilogue on CUDA."""
    if x.is_cuda:
        from ..ops import kernels as K

        return K.Linear.apply(x, layer.weight, layer.bias, resid)
    return resid + F.linear(x, layer.weight, layer.bias)


def _plain_blocks(model: GPT) -> list[Block]:
    """The model's blocks, which are run layer by layer here; a wrapped or changed one would not be what the model runs."""
    blocks = list(getattr(model, "blocks", ()))
    for b in blocks:
        if getattr(type(b), "forward", None) is not Block.forward or getattr(type(b), "_forward_cuda", None) is not Block._forward_cuda:
            raise ValueError(f"generation with a cache runs the layers of GPT's own Block, not of {type(b).__name__} "
                             "(of a sharded model, load the full weights into a plain GPT)")
    if not blocks:
        raise ValueError(f"a GPT with blocks, not {type(model).__name__}")
    return blocks


class BranchedGeneration:
    """The state of up to ``max_branches`` continuations of one prompt, which grow in step.

    ``logits`` holds the scores of the next token, one row for each of
    ``branches``; at first there is one branch, which holds nothing yet.
    The model is a plain :class:`GPT`: one whose blocks are wrapped (sharded
    by ``FullyShardedDataParallel``) is refused with ``ValueError``.
    """

    @torch.no_grad()
    def __init__(self, model: GPT, prompt: torch.Tensor, *, max_branches: int, max_new_tokens: int, page_size: int = 16) -> None:
        prompt = prompt.reshape(-1)
        P, self._blocks = prompt.numel(), _plain_blocks(model)
        if P < 1 or max_branches < 1 or max_new_tokens < 1:
            raise ValueError("a prompt of at least one token, one branch and one new token")
        if P + max_new_tokens > model.block_size:
            raise ValueError(f"{P} + {max_new_tokens} tokens are more than the model's {model.block_size} positions")
        self.model, self.prompt_len, self.max_new_tokens = model, P, max_new_tokens
        cfg, w = model.config, model.tok_emb.weight
        self.heads, self.head_dim = cfg.n_head, cfg.n_embd // cfg.n_head
        pages = -(-P // page_size) + max_branches * -(-max_new_tokens // page_size)
        # slot 0 is the prompt's
        self.cache = G.PagedKVCache(cfg.n_layer, pages, page_size, self.heads, self.head_dim, max_seqs=max_branches + 1,
                                    max_seq_len=max(P, max_new_tokens), device=w.device, dtype=w.dtype)
        self.branches = [1]
        self.length = 0  # tokens of each branch
        self._device_ids: dict[tuple[int, ...], torch.Tensor] = {}
        self.cache.extend([0], [P])
        places = torch.arange(P, dtype=torch.int32, device=w.device)
        x = _embed(model, prompt[None], 0)
        for layer, block in enumerate(self._blocks):
            h = F.layer_norm(x, block.ln1.weight, block.ln1.bias, block.ln1.eps)
            qkv = F.linear(h, block.qkv.weight, block.qkv.bias)
            _, k, v = qkv[0].view(P, 3, self.heads, self.head_dim).unbind(1)
            self.cache.append(layer, k, v, places, torch.zeros_like(places))
            x = self._rest(block, F.causal_attention(qkv, self.heads).reshape(1, P, -1), x)
        self.logits = self._head(x[:, -1])

    def _rest(self, block: Block, y: torch.Tensor, x: torch.Tensor) -> torch.Tensor:
        """The block after its attention."""
        x = _add_linear(y, block.proj, x)
        h = F.layer_norm(x, block.ln2.weight, block.ln2.bias, block.ln2.eps)
        return _add_linear(F.linear_gelu(h, block.mlp[0].weight, block.mlp[0].bias), block.mlp[2], x)

    def _head(self, x: torch.Tensor) -> torch.Tensor:
        m = self.model
        return F.linear(F.layer_norm(x, m.ln_f.weight, m.ln_f.bias, m.ln_f.eps), m.tok_emb.weight)

    def _ids(self, slots: Sequence[int]) -> torch.Tensor:
        key = tuple(slots)
        if key not in self._device_ids:
            if len(self._device_ids) >= 64:
                self._device_ids.clear()
            self._device_ids[key] = torch.tensor(key, dtype=torch.int32, device=self.cache.kv.device)
        return self._device_ids[key]

    @torch.no_grad()
    def step(self, tokens: torch.Tensor) -> torch.Tensor:
        """Add ``tokens[i]`` to branch i; returns (and keeps) the scores of the tokens after them."""
        n = len(self.branches)
        if tokens.shape != (n,):
            raise ValueError(f"one token for each of the {n} branches")
        if self.length >= self.max_new_tokens:
            raise ValueError(f"the branches hold {self.max_new_tokens} tokens already")
        c, P = self.cache, self.prompt_len
        ids = self._ids(self.branches)
        x = _embed(self.model, tokens[:, None], P + self.length)[:, 0]  # (first: it refuses tokens that are none)
        c.extend(self.branches, [1] * n, ids, torch.ones_like(ids))
        place = torch.full_like(ids, self.length)
        table, lens = c.page_table[ids.long()], c.lens[ids.long()]
        prefix = c.page_table[0, : -(-P // c.page_size)]
        self.length += 1
        for layer, block in enumerate(self._blocks):
            h = F.layer_norm(x, block.ln1.weight, block.ln1.bias, block.ln1.eps)
            q, k, v = F.linear(h, block.qkv.weight, block.qkv.bias).view(n, 3, self.heads, self.head_dim).unbind(1)
            c.append(layer, k, v, place, ids)
            y = G.shared_prefix_attention(q, c.kv[layer, 0], c.kv[layer, 1], prefix, P, table, lens, max_seq_len=self.length)
            x = self._rest(block, y.reshape(n, -1), x)
        self.logits = self._head(x)
        return self.logits

    @torch.no_grad()
    def select(self, picks: Sequence[int]) -> None:
        """Make the branches copies of the present branches ``picks``, in that order.

        A branch that is picked once goes on as it is, further picks of it are
        forked (full pages stay shared), and one that is not picked gives its
        pages back.  ``logits`` are rearranged with them.
        """
        c = self.cache
        if not picks or not all(0 <= i < len(self.branches) for i in picks):
            raise ValueError("picks: indices of the present branches")
        if len(picks) > len(c.lengths) - 1:
            raise ValueError(f"at most {len(c.lengths) - 1} branches")
        c.free([s for i, s in enumerate(self.branches) if i not in set(picks)])
        kept = {self.branches[i] for i in picks}
        spare = [s for s in range(1, len(c.lengths)) if s not in kept]
        slots, parents, children = [], [], []
        for i in picks:
            slot = self.branches[i]
            if slot in slots:
                parents.append(slot)
                children.append(spare.pop(0))
                slot = children[-1]
            slots.append(slot)
        c.fork(parents, children)
        self.branches = slots
        self.logits = self.logits[torch.tensor(list(picks), device=self.logits.device)]

    def compact(self) -> None:
        """Move the pages in use to the front of the cache's pool."""
        self.cache.compact()


def _embed(model: GPT, idx: torch.Tensor, position: int) -> torch.Tensor:
    """Token embeddings plus the learned positions from ``position`` on, for ``idx`` ``[B, T]``."""
    pos = model.pos_emb[0, position: position + idx.shape[1]]
    if idx.is_cuda:
        from ..ops import kernels as K

        return K.Embedding.apply(idx, model.tok_emb.weight, pos)
    return model.tok_emb(idx) + pos


@torch.no_grad()
def sample_continuations(
    model: GPT,
    prompt: torch.Tensor,
    n: int,
    max_new_tokens: int,
    *,
    temperature: float = 0.8,
    top_k: int = 0,
    top_p: float = 1.0,
    min_p: float = 0.0,
    generator: torch.Generator | None = None,
    resample_every: int = 0,
    score: Callable[[torch.Tensor, torch.Tensor], torch.Tensor] | None = None,
    page_size: int = 16,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Draw ``n`` continuations of ``prompt``; returns ``(tokens, logprobs)``, ``[n, max_new_tokens]`` each.

    The log-probabilities are those of the drawn tokens under the filtered
    distributions (:func:`~mini_nccl_b200.ops.generation.sample`).  With
    ``resample_every``, after every so many tokens the better half of the
    branches, by ``score(tokens, logprobs)`` (default: the mean
    log-probability; larger is better), is copied over the other half.
    """
    state = BranchedGeneration(model, prompt, max_branches=n, max_new_tokens=max_new_tokens, page_size=page_size)
    state.select([0] * n)
    device = state.logits.device
    tokens = torch.empty(n, max_new_tokens, dtype=torch.long, device=device)
    logprobs = torch.empty(n, max_new_tokens, dtype=torch.float32, device=device)
    for t in range(max_new_tokens):
        noise = torch.empty(state.logits.shape, dtype=torch.float32, device=device)
        noise.exponential_(generator=generator).log_().neg_()
        tokens[:, t], logprobs[:, t] = G.sample(state.logits, noise, temperature=temperature, top_k=top_k, top_p=top_p,
                                                min_p=min_p, return_logprob=True)
        if t + 1 == max_new_tokens:
            break
        state.step(tokens[:, t])
        if resample_every and (t + 1) % resample_every == 0 and n > 1:
            done = tokens[:, : t + 1], logprobs[:, : t + 1]
            value = score(*done) if score is not None else done[1].mean(1)
            best = torch.argsort(value, descending=True, stable=True)[: -(-n // 2)].tolist()
            picks = (best + best)[:n]
            state.select(picks)
            state.compact()
            at = torch.tensor(picks, device=device)
            tokens[:, : t + 1], logprobs[:, : t + 1] = done[0][at], done[1][at]
    return tokens, logprobs
