"""Rollouts over the 8-bit cache and the update behind them, in one run: groups share a
prompt's pages, every step attends over the cache, projects to logits on the
tensor-core GEMM, samples, takes the behaviour log-probabilities and appends the new
token's K and V; then rewards become advantages and the policy loss its gradient.
Each stage is checked against 64 bits on what the stage before has left."""
import ctypes

import numpy as np
import pytest
import torch

from test_kv8_gpu import check as check_attention
from test_policy_gpu import E, check_policy

pytestmark = pytest.mark.gpu


def gemm_chunk_max(pkg, A, B):
    M, K = A.shape
    N = B.shape[0]
    C = torch.empty(M, N, device=A.device)
    cmax = torch.empty(M, pkg.chunk_max_stride(N), device=A.device)
    p = pkg.rt_gemm_params_t(M, N, K, A.stride(0), B.stride(0), N, 0, 0)
    err = torch.zeros(1, dtype=torch.int32, device=A.device)
    pkg.check(pkg.lib().rt_gemm_bf16_chunk_max(ctypes.byref(p), pkg._ptr(A), pkg._ptr(B),
                                               pkg._ptr(C), None, 0, pkg._ptr(err),
                                               pkg._ptr(cmax), cmax.stride(0),
                                               pkg._stream_ptr(None)), "gemm")
    assert err.item() == 0
    return C, cmax


@pytest.mark.parametrize("fmt", ["e4m3", "s8"])
def test_rollouts_and_update(pkg, cuda, fmt):
    groups, size, prompt, steps = 3, 4, 48, 20
    heads, G, vocab, temperature = 2, 4, 1000, 0.8
    B, d = groups * size, heads * G * 128
    g = torch.Generator(device=cuda).manual_seed(5)
    rand = lambda *s, std=1.0: (torch.randn(*s, generator=g, device=cuda) * std).bfloat16()  # noqa: E731
    embed, w_qkv = rand(vocab, d), rand((heads * G + 2 * heads) * 128, d, std=d ** -0.5)
    w_lm = rand(vocab, d, std=2 * d ** -0.5)

    # a group's prompt pages lie in every member's table; the pages behind are its own
    shared = prompt // 16
    own = (prompt + steps) // 16 + 1 - shared
    n_pages = groups * shared + B * own
    perm = np.random.default_rng(6).permutation(n_pages).astype(np.int32)
    table = np.concatenate([np.repeat(perm[:groups * shared].reshape(groups, shared), size, 0),
                            perm[groups * shared:].reshape(B, own)], 1)
    td = torch.from_numpy(table).to(cuda)
    pages, scales, tail = pkg.kv8_cache(n_pages, B, heads, fmt, cuda)
    error = torch.zeros(1, dtype=torch.int32, device=cuda)

    # the prompts, by each group's first member: one call, the other members bring nothing
    tokens = torch.randint(0, vocab, (groups * prompt,), generator=g, device=cuda)
    kv = (embed[tokens].float() @ w_qkv[heads * G * 128:].float().T).view(-1, 2 * heads, 128)
    new = [prompt if b % size == 0 else 0 for b in range(B)]
    cu = torch.tensor([0] + list(np.cumsum(new)), dtype=torch.int32, device=cuda)
    lens = torch.zeros(B, dtype=torch.int32, device=cuda)
    pkg.kv8_append(kv[:, :heads], kv[:, heads:], cu, lens, td, pages, scales, tail, error=error)
    before = pages.view(torch.int8)[torch.from_numpy(perm[:groups * shared]).long().to(cuda)].clone()

    lens.fill_(prompt)
    ones = torch.arange(B + 1, dtype=torch.int32, device=cuda)
    last = torch.randint(0, vocab, (B,), generator=g, device=cuda).to(torch.int32)
    kept, logits_all = [], []
    for step in range(steps):
        qkv = (embed[last.long()].float() @ w_qkv.float().T).view(B, -1, 128)
        k, v = qkv[:, heads * G:heads * G + heads], qkv[:, heads * G + heads:]
        pkg.kv8_append(k, v, ones, lens, td, pages, scales, tail, error=error)   # fp32 columns
        lens += 1
        q = qkv[:, :heads * G].bfloat16()
        out = pkg.kv8_decode_attention(q, pages, scales, tail, td, lens, prompt + steps, error=error)
        if step in (0, 7, 15, steps - 1):
            check_attention(out, q, pages, scales, tail, table, lens.tolist())
        logits, cmax = gemm_chunk_max(pkg, out.view(B, d).bfloat16().contiguous(), w_lm)
        rows = pkg.sample_row_table(temperature, 50, 0.9, np.arange(B), step, 1234)
        last = pkg.sample_rows_cmax(logits, cmax, torch.from_numpy(rows.view(np.uint8)).to(cuda), vocab)
        lp, h = pkg.token_logprobs(logits, last, temperature=temperature, error=error)
        kept.append((last.clone(), lp, h))
        logits_all.append(logits)
    assert error.item() == 0
    # the shared pages have not been written again
    assert torch.equal(pages.view(torch.int8)[torch.from_numpy(perm[:groups * shared]).long().to(cuda)],
                       before)

    # the update: rows in the order (rollout, step), a policy that has moved a little
    logits = torch.stack(logits_all, 1).reshape(B * steps, vocab)
    acted = torch.stack([t for t, _, _ in kept], 1).reshape(-1).contiguous()
    old = torch.stack([p for _, p, _ in kept], 1).reshape(-1).contiguous()
    ent = torch.stack([h for _, _, h in kept], 1).reshape(-1)
    rewards = torch.rand(B, generator=g, device=cuda)
    adv = pkg.grpo_advantages(rewards, size)
    seq = torch.arange(B, device=cuda).repeat_interleave(steps).to(torch.int32)
    weights = torch.full((B * steps,), 1.0 / (B * steps), device=cuda)
    first = pkg.policy_loss(logits, acted, weights, adv, old, old, seq, temperature=temperature,
                            kl_coef=0.04, entropy_coef=0.01, error=error)
    # the same policy: the same bits as the behaviour's, ratios of 1 and no divergence
    assert torch.equal(first.logprobs, old) and torch.equal(first.entropy, ent)
    assert bool(((first.ratio - 1).abs() <= 2.0 ** -23 * (1 + old.abs())).all())
    assert not bool(first.clipped.any()) and float(first.kl.abs().max()) < 1e-9

    moved = logits + 0.3 * torch.randn(logits.shape, generator=g, device=cuda)
    case = dict(logits=moved, tokens=acted, weights=weights, advantages=adv, old_logprobs=old,
                ref_logprobs=old, row_seq=seq)
    r = check_policy(pkg, case, t=temperature)
    assert bool(r.clipped.any())
    # an update along the gradient, written over the logits, lowers the loss
    start = float(r.stats[0])
    point = moved.clone()
    grad = pkg.policy_loss(**dict(case, logits=point), temperature=temperature, kl_coef=0.04,
                           entropy_coef=0.01, dlogits=point).dlogits
    assert torch.equal(grad, r.dlogits)
    small = 1e-2 / float(grad.norm())
    after = pkg.policy_loss(**dict(case, logits=moved - small * grad), temperature=temperature,
                            kl_coef=0.04, entropy_coef=0.01, backward=False)
    drop, want = start - float(after.stats[0]), small * float(grad.double().square().sum())
    # first order: 1e-2 |grad|; the loss's fp32 rounding and the curvature are far below half
    assert abs(drop - want) <= 0.5 * want + 2.0 ** -22 * abs(start) + E * 1e-2, (drop, want)
    assert error.item() == 0
