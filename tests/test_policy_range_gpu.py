"""The row operators over wide ranges: rows shorter than a vector, large ratios, the longest
rows that a warp takes alone.  References and tolerances are those of test_policy_gpu.py,
except where a test states its own."""
import pytest
import torch

from test_policy_gpu import case, grad64, logits_of, policy64, rows64

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
