"""Train a small character-level GPT, then draw many continuations of one prompt.

    python examples/sample_gpt.py --steps 200 --branches 8
    python examples/sample_gpt.py --device cuda --branches 64 --top-p 0.95 --resample-every 16

The prompt runs through the model once; the continuations share its keys and
values in a paged cache.  With ``--resample-every`` the likelier half of the
branches replaces the other half every so many tokens (fork, free, compact).
"""

from __future__ import annotations

import argparse
import time

import torch

from _common import batch, encode, load_corpus, to_device

from mini_nccl_b200.models.generation import sample_continuations
from mini_nccl_b200.models.gpt import GPT


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--data", help="a text file (default: a synthetic corpus)")
    ap.add_argument("--device", choices=["cpu", "cuda"], default="cpu")
    ap.add_argument("--steps", type=int, default=200)
    ap.add_argument("--batch-size", type=int, default=16)
    ap.add_argument("--block-size", type=int, default=128)
    ap.add_argument("--n-layer", type=int, default=4)
    ap.add_argument("--n-head", type=int, default=4)
    ap.add_argument("--n-embd", type=int, default=128, help="32, 64 or 128 times --n-head")
    ap.add_argument("--lr", type=float, default=1e-3)
    ap.add_argument("--prompt", default="To be, or not to ")
    ap.add_argument("--branches", type=int, default=8)
    ap.add_argument("--new-tokens", type=int, default=64)
    ap.add_argument("--temperature", type=float, default=0.8)
    ap.add_argument("--top-k", type=int, default=0)
    ap.add_argument("--top-p", type=float, default=0.95)
    ap.add_argument("--min-p", type=float, default=0.0)
    ap.add_argument("--resample-every", type=int, default=0)
    args = ap.parse_args()

    data, vocab = encode(load_corpus(args.data))
    torch.manual_seed(0)
    size = -(-len(vocab) // 8) * 8  # the GEMM kernels take multiples of 8
    model, dev = to_device(GPT(size, args.block_size, args.n_layer, args.n_head, args.n_embd), args.device)
    if dev.type == "cuda":
        from mini_nccl_b200.ops.kernels import FusedAdamW

        opt = FusedAdamW(model.parameters(), lr=args.lr)
    else:
        opt = torch.optim.AdamW(model.parameters(), lr=args.lr)
    loss = None
    for step in range(args.steps):
        x, y = batch(data, args.block_size, args.batch_size, seed=step)
        _, loss = model(x.to(dev), y.to(dev))
        opt.zero_grad()
        loss.backward()
        opt.step()
    if loss is not None:
        print(f"trained {args.steps} steps, loss {float(loss.detach()):.3f}", flush=True)

    prompt = torch.tensor([vocab.index(ch) for ch in args.prompt if ch in vocab], device=dev)
    gen = torch.Generator(device=dev).manual_seed(1)
    start = time.perf_counter()
    tokens, logprobs = sample_continuations(
        model, prompt, args.branches, args.new_tokens, temperature=args.temperature, top_k=args.top_k, top_p=args.top_p,
        min_p=args.min_p, generator=gen, resample_every=args.resample_every)
    tokens, mean = tokens.tolist(), logprobs.mean(1).tolist()
    seconds = time.perf_counter() - start
    if dev.type == "cuda":
        from mini_nccl_b200.ops.kernels import check_status

        check_status(dev)
    for row, value in sorted(zip(tokens, mean), key=lambda r: -r[1]):
        text = "".join(vocab[i] if i < len(vocab) else "?" for i in row)
        print(f"[{value:6.2f}] {args.prompt + text!r}")
    print(f"sampled {args.branches} continuations of {args.new_tokens} tokens in {seconds:.2f} s")


if __name__ == "__main__":
    main()
