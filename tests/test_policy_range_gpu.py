"""The row operators over wide ranges: rows shorter than a vector, large ratios, the longest
rows that a warp takes alone.  References and tolerances are those of test_policy_gpu.py,
except where a test states its own."""
import math

import pytest
import torch

import test_policy_gpu
from test_policy_gpu import (E, case, check_backward, check_forward, check_policy, grad64,
                             logits_of, policy64, rows64)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", range(1, 10))
@pytest.mark.parametrize("extra", [0, 3])
def test_rows_without_gradient_stay_inside(pkg, cuda, dtype, V, extra):
    """Every second row is skipped, has a bad token or has no weight; its gradient is zeros, and
    what lies beside the rows and in them stays: in a buffer of its own, and over the logits."""
    R, stride = 90, V + extra
    for offset in range(8):
        logits, tokens = logits_of(cuda, R, V, dtype, 61 + offset, offset=offset, stride=stride)
        c = case(cuda, R, V, dtype, 62)
        c.update(logits=logits, tokens=tokens)
        off = torch.arange(R, device=cuda) % 2 == 1
        enable = (~off).to(torch.int32)
        wrong = torch.where(off, V + 5, tokens).to(torch.int32)
        c["weights"] = torch.where(off, 0.0, c["weights"])
        one = torch.linspace(-1, 1, R, device=cuda)
        p, logp, d, _, h, _ = rows64(logits, tokens, 1.0)
        ref, tol = grad64(p, logp, d, h, tokens, one.double(), one.double(), 1.0, dtype)
        pol = policy64(logits, tokens, c["weights"], c["advantages"], c["old_logprobs"], None, None,
                       1.0, 0.2, 0.2, 0.0, 0.01)
        pref, ptol = grad64(p, logp, d, h, tokens, pol["g"], pol["gh"], 1.0, dtype)
        hit = torch.zeros_like(pref).scatter_(1, tokens.long()[:, None], 1.0)
        ptol = ptol + pol["e_g"][:, None] * (p + hit)

        def calls(x, dl):
            yield ref, tol, lambda: pkg.token_logprobs_backward(x, tokens, one, one, dlogits=dl,
                                                                row_enable=enable)
            yield ref, tol, lambda: pkg.token_logprobs_backward(x, wrong, one, one, dlogits=dl)
            yield pref, ptol, lambda: pkg.policy_loss(
                **dict(c, logits=x, ref_logprobs=None), entropy_coef=0.01, dlogits=dl)

        for in_place in (False, True):
            for i in range(3):
                flat = torch.full((R * stride + offset + 8,), 5.0, dtype=dtype, device=cuda)
                view = flat[offset:offset + R * stride].view(R, stride)[:, :V]
                inside = torch.zeros_like(flat, dtype=torch.bool)
                inside[offset:offset + R * stride].view(R, stride)[:, :V] = True
                if in_place:
                    view.copy_(logits)
                want, bound, call = list(calls(view if in_place else logits, view))[i]
                call()
                assert bool((flat[~inside] == 5).all())
                assert bool((view[off] == 0).all())
                assert bool(((view[~off].double() - want[~off]).abs() <= bound[~off]).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [50, 5000])
def test_policy_of_large_ratios(pkg, cuda, dtype, V):
    """Log-probabilities far above the old ones: e^gap leaves fp32 at 88.7, its product with an
    advantage of 0 is 0, and with a small one a number.  The product is off by the share that
    its exponent is (lp's error, and half a step of a gap below 256: 2^-17), and by that of two
    exponentials and two products, at most 2^-21 each."""
    gaps = [0.0, 50.0, 88.0, 89.0, 95.0, 120.0, 170.0, 200.0]
    values = [0.0, 1e-30, -1e-30, -1e-3, 1.0, -1.0]
    R = len(gaps) * len(values)
    logits, tokens = logits_of(cuda, R, V, dtype, 71)
    gap = torch.tensor(gaps, dtype=torch.float64, device=cuda).repeat_interleave(len(values))
    adv = torch.tensor(values, device=cuda).repeat(len(gaps))
    p, logp, d, lp, h, _ = rows64(logits, tokens, 1.0)
    old = (lp - gap).float()
    w = torch.full((R,), 0.5, device=cuda)
    r = pkg.policy_loss(logits, tokens, w, adv, old)
    ratio = (lp - old.double()).exp()
    a = adv.double()
    cut = ratio * a > ratio.clip(0.8, 1.2) * a
    want = -torch.where(cut, ratio.clip(0.8, 1.2) * a, ratio * a)
    share = E + 2.0 ** -24 * lp.abs() + 2.0 ** -17 + 4 * 2.0 ** -21
    big = torch.finfo(torch.float32).max
    fits = want.abs() < big
    near = (r.row_loss.double() - want).abs() <= share * want.abs()
    assert bool((near | ~fits).all()) and bool((r.row_loss[~fits] == math.inf).all())
    assert bool((r.policy == r.row_loss).all())
    assert torch.equal(r.clipped.bool(), cut)
    # a slope beyond fp32 has no gradient in numbers
    slope = torch.where(cut, 0.0, -ratio * a) * 0.5
    ok = slope.abs() < big
    zero = torch.zeros_like(slope)
    ref, tol = grad64(p, logp, d, h, tokens, torch.where(ok, slope, 0.0), zero, 1.0, dtype)
    hit = torch.zeros_like(ref).scatter_(1, tokens.long()[:, None], 1.0)
    tol = tol + (share * slope.abs())[:, None] * (p + hit)
    assert bool(((r.dlogits[ok].double() - ref[ok]).abs() <= tol[ok]).all())
    assert bool((r.dlogits[adv == 0] == 0).all())
    none = pkg.policy_loss(logits, tokens, w, torch.zeros_like(adv), old)
    assert bool((none.stats[:2] == 0).all()) and bool((none.dlogits == 0).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [50, 5000])
def test_policy_of_large_divergences(pkg, cuda, dtype, V):
    """Reference log-probabilities far above: e^gap leaves fp32 at 88.7, its products with the
    coefficient and the weight later.  Off by the shares that the test above counts."""
    gaps = [79.0, 81.0, 88.0, 89.5, 91.0, 100.0, 120.0]
    weights = [1e-3, 1e-7, 1e-12, 1e-20]
    coef = 1e-2
    R = len(gaps) * len(weights)
    logits, tokens = logits_of(cuda, R, V, dtype, 72)
    logits[::3, 1] = -math.inf
    tokens[::3] = torch.where(tokens[::3] == 1, 2, tokens[::3])
    gap = torch.tensor(gaps, dtype=torch.float64, device=cuda).repeat_interleave(len(weights))
    w = torch.tensor(weights, device=cuda).repeat(len(gaps))
    p, logp, d, lp, h, _ = rows64(logits, tokens, 1.0)
    ref_lp = (lp + gap).float()
    adv = torch.linspace(-1, 1, R, device=cuda)
    r = pkg.policy_loss(logits, tokens, w, adv, None, ref_lp, kl_coef=coef)
    apart = ref_lp.double() - lp
    share = E + 2.0 ** -24 * lp.abs() + 2.0 ** -17 + 4 * 2.0 ** -21
    big = torch.finfo(torch.float32).max

    def same(got, want):
        fits = want < big * 0.99
        near = (got.double() - want).abs() <= share * want.abs()
        assert bool((near | ~fits).all()) and bool((got[want > big * 1.01] == math.inf).all())

    same(r.kl, apart.exp() - apart - 1)
    same(r.row_loss, coef * (apart.exp() - apart - 1) - adv.double())
    slope = (coef * (1 - apart.exp()) - adv.double()) * w.double()
    ok = slope.abs() < big * 0.99
    assert int(ok.sum()) > R // 2
    zero = torch.zeros_like(slope)
    ref, tol = grad64(p, logp, d, h, tokens, torch.where(ok, slope, 0.0), zero, 1.0, dtype)
    hit = torch.zeros_like(ref).scatter_(1, tokens.long()[:, None], 1.0)
    tol = tol + (share * slope.abs())[:, None] * (p + hit)
    assert bool(((r.dlogits[ok].double() - ref[ok]).abs() <= tol[ok]).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("R,V", [(600, 6000), (600, 6001), (593, 5999), (592, 6000), (2500, 1000),
                                 (2500, 1001)])
@pytest.mark.parametrize("offset,extra", [(0, 0), (3, 5)])
def test_rows_at_the_edges_of_a_warp(pkg, cuda, monkeypatch, dtype, R, V, offset, extra):
    """Up to 6,000 logits a row may be a warp's own: each of a lane's two sums has 94 terms, and
    1 + 6 additions behind them, so with two exponentials' shares the relative error of the sum
    is at most 1.37 x 2^-22 + 101 x 2^-24 < 6.4e-6."""
    monkeypatch.setattr(test_policy_gpu, "E", 6.4e-6)
    logits, tokens = logits_of(cuda, R, V, dtype, V, offset=offset, stride=V + extra)
    check_forward(pkg, logits, tokens, 0.8)
    check_backward(pkg, logits, tokens, 0.8)
    g = torch.linspace(-1, 1, R, device=cuda)
    want = pkg.token_logprobs_backward(logits, tokens, g, g)
    flat = torch.empty(R * (V + extra) + offset, dtype=dtype, device=cuda)
    same = flat[offset:].view(R, V + extra)[:, :V]
    same.copy_(logits)
    got = pkg.token_logprobs_backward(same, tokens, g, g, dlogits=same)
    assert torch.equal(got, want)
    if not offset:
        check_policy(pkg, case(cuda, R, V, dtype, R, 20), t=0.8)
