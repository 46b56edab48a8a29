"""Generation with the cache against the model run over whole sequences, on CPU and (marked gpu) on the kernels."""

from __future__ import annotations

import subprocess
import sys
from pathlib import Path

import pytest
import torch

from mini_nccl_b200.models.generation import BranchedGeneration, sample_continuations
from mini_nccl_b200.models.gpt import GPT

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def model_on(device, n_head=2, n_embd=64, vocab=96, block=96, seed=0):
    torch.manual_seed(seed)
    m = GPT(vocab, block, 2, n_head, n_embd)
    with torch.no_grad():
        for p in m.parameters():
            p.mul_(4.0)  # scores that differ
    return m.to(device, torch.bfloat16) if device == "cuda" else m


def settle(device):
    if device == "cuda":
        from mini_nccl_b200.ops import kernels as K

        K.check_status()


def close(got, want, device):
    # fp32 on CPU; on the GPU both sides are bf16 networks whose roundings fall differently, layer by layer
    tol = 1e-4 if device == "cpu" else 6e-2
    scale = want.float().abs().max()
    assert torch.all((got.float() - want.float()).abs() <= tol * scale), float((got.float() - want.float()).abs().max() / scale)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("n_head,n_embd,page", [(2, 64, 16), (1, 64, 8), (2, 256, 16)])
def test_steps_match_the_whole_sequence(device, n_head, n_embd, page):
    m = model_on(device, n_head, n_embd)
    g = torch.Generator().manual_seed(1)
    prompt = torch.randint(0, 96, (37,), generator=g).to(device)
    state = BranchedGeneration(m, prompt, max_branches=5, max_new_tokens=40, page_size=page)
    with torch.no_grad():
        close(state.logits, m(prompt[None])[0][:, -1], device)
    state.select([0] * 3)
    rows = [[] for _ in range(3)]

    def advance():
        tokens = torch.randint(0, 96, (len(rows),), generator=g)
        for row, t in zip(rows, tokens.tolist()):
            row.append(t)
        state.step(tokens.to(device))
        whole = torch.cat([prompt.expand(len(rows), -1), torch.tensor(rows, device=device)], 1)
        with torch.no_grad():
            close(state.logits, m(whole)[0][:, -1], device)

    for t in range(38):
        advance()
        if t == 9:  # one goes, two are copied
            picks = [2, 0, 2, 0, 2]
            rows = [list(rows[i]) for i in picks]
            state.select(picks)
        if t == 20:
            state.select([4, 1])
            rows = [list(rows[i]) for i in (4, 1)]
            state.compact()
        if t == 30:
            state.select([1, 1, 0])
            rows = [list(rows[i]) for i in (1, 1, 0)]
    settle(device)
    held = state.cache.page_table[state.cache.page_table >= 0].long()
    assert torch.equal(torch.bincount(held, minlength=len(state.cache.refs)).int(), state.cache.refs)


@pytest.mark.parametrize("device", DEVICES)
def test_sample_continuations(device):
    m = model_on(device)
    prompt = torch.arange(20, device=device)

    def draw(**more):
        gen = torch.Generator(device=device).manual_seed(5)
        return sample_continuations(m, prompt, 6, 30, generator=gen, **more)

    tokens, logprobs = draw(top_k=20, top_p=0.9)
    assert tokens.shape == logprobs.shape == (6, 30) and torch.all((tokens >= 0) & (tokens < 96)) and torch.all(logprobs <= 0)
    again, _ = draw(top_k=20, top_p=0.9)
    assert torch.equal(tokens, again)
    greedy, lp = draw(temperature=0.0)
    assert torch.all(greedy == greedy[:1]) and torch.all(lp == 0)
    with torch.no_grad():
        logits = m(torch.cat([prompt, greedy[0, :-1]])[None])[0][0, 19:].float()
    # the greedy token is the whole model's best, or within the roundings of it
    gap = logits.amax(-1) - logits.gather(1, greedy[0][:, None])[:, 0]
    assert torch.all(gap <= (1e-3 if device == "cpu" else 6e-2) * logits.abs().amax())
    best, lp = draw(resample_every=7)
    assert best.shape == (6, 30) and torch.unique(best[:, :7], dim=0).shape[0] <= 3
    settle(device)


def test_refusals():
    m = model_on("cpu")
    with pytest.raises(ValueError):
        BranchedGeneration(m, torch.arange(90), max_branches=1, max_new_tokens=7)
    with pytest.raises(ValueError):
        BranchedGeneration(m, torch.arange(0), max_branches=1, max_new_tokens=7)
    state = BranchedGeneration(m, torch.arange(9), max_branches=2, max_new_tokens=1)
    for bad in ([], [1], [0, 0, 0]):
        with pytest.raises(ValueError):
            state.select(bad)
    with pytest.raises(ValueError):
        state.step(torch.zeros(2, dtype=torch.long))
    state.step(torch.zeros(1, dtype=torch.long))
    with pytest.raises(ValueError):
        state.step(torch.zeros(1, dtype=torch.long))


@pytest.mark.examples
@pytest.mark.parametrize("device", DEVICES)
def test_example(device):
    command = [sys.executable, "examples/sample_gpt.py", "--device", device, "--steps", "2", "--n-layer", "2", "--branches", "5",
               "--new-tokens", "24", "--resample-every", "8"]
    run = subprocess.run(command, cwd=Path(__file__).resolve().parent.parent, capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stdout[-2000:] + run.stderr[-2000:]
    assert "sampled 5 continuations of 24 tokens" in run.stdout
