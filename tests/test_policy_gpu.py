"""Token log-probabilities and the policy loss (rt_token_logprobs,
rt_token_logprobs_backward, rt_policy_loss) against plain 64-bit
implementations.

Tolerances count the kernels' roundings.  A thread adds at most 72
exponentials and merges them with the others' in at most 20 steps, each off by
2^-24; an exponential is off by 2^-22 (exp2) and by the share 2^-22 d of its
exponent's roundings, with d e^-d <= 0.37.  So the relative error of the sum is
at most E = 2^-22 + 0.37 x 2^-22 + 92 x 2^-24 < 6e-6: the log-probability is
off by E + 2^-24 |lp|, the entropy by E (1 + sum p |d|) + 2^-24 H, and an
element of the gradient, with the coefficient's own error from lp, by
p |coefficient| (2 E + 2^-22 |d|) + 2^-23 of what is added, + half a step of its
type, and by 2^-126 |coefficient| where an exponential below the normal range is
flushed to 0.  Where log p and H cancel (a vocabulary of one: both are 0) their own
errors stay: p |dentropy| (E + E (1 + sum p |d|)) more.  An exponent of the policy loss magnifies lp's error by its own value."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

E = 6e-6
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


def rows64(logits, tokens, t):
    z = logits.double() / (t if t else 1.0)
    d = z - z.amax(1, keepdim=True)
    logp = torch.log_softmax(z, 1)
    p = logp.exp()
    safe = torch.where(p == 0, 0.0, logp)
    h = -(p * safe).sum(1)
    spread = (p * torch.where(p == 0, 0.0, d).abs()).sum(1)
    return p, safe, d, logp.gather(1, tokens.long()[:, None])[:, 0], h, spread


def grad64(p, logp, d, h, tokens, g, gh, t, dtype):
    """The gradient, and how far the kernel's may be off."""
    t = t if t else 1.0
    inner = g[:, None] + gh[:, None] * (logp + h[:, None])
    ref = -p * inner
    size = p * (g.abs()[:, None] + gh.abs()[:, None] * (logp.abs() + h.abs()[:, None]))
    spread = (p * torch.where(p == 0, 0.0, d).abs()).sum(1)
    off = size * (2 * E + 2.0 ** -22 * torch.where(p == 0, 0.0, d).abs())
    off += p * (gh.abs() * E * (2 + spread))[:, None]
    off += 2.0 ** -126 * (g.abs()[:, None] + gh.abs()[:, None] * (logp.abs() + h.abs()[:, None]))
    hit = tokens.long()[:, None]
    ref.scatter_add_(1, hit, g[:, None])
    off.scatter_add_(1, hit, g.abs()[:, None] * 2.0 ** -23)
    ref, off = ref / t, off / t
    return ref, off + 2.0 ** -23 * ref.abs() + HALF[dtype] * ref.abs() * (1 + 1e-3) + 1e-37


def logits_of(dev, R, V, dtype, seed, std=2.0, offset=0, stride=None):
    """Rows that start `offset` elements into a buffer with the given row stride."""
    g = torch.Generator(device=dev).manual_seed(seed)
    stride = stride or V
    flat = torch.full((R * stride + offset + 8,), float("nan"), dtype=dtype, device=dev)
    view = flat[offset:offset + R * stride].view(R, stride)[:, :V]
    view.copy_(torch.randn(R, V, generator=g, device=dev) * std)
    tokens = torch.randint(0, V, (R,), generator=g, device=dev).to(torch.int32)
    return view, tokens


def check_forward(pkg, logits, tokens, t, **kw):
    lp, h = pkg.token_logprobs(logits, tokens, temperature=t, **kw)
    _, _, _, want, ent, spread = rows64(logits, tokens, t)
    assert bool(((lp.double() - want).abs() <= E + 2.0 ** -24 * want.abs()).all())
    assert bool(((h.double() - ent).abs() <= E * (1 + spread) + 2.0 ** -24 * ent).all())


def check_backward(pkg, logits, tokens, t, seed=0, **kw):
    g = torch.Generator(device=logits.device).manual_seed(seed)
    R = logits.shape[0]
    dlp = torch.randn(R, generator=g, device=logits.device)
    dh = torch.randn(R, generator=g, device=logits.device)
    p, logp, d, _, h, _ = rows64(logits, tokens, t)
    ref, off = grad64(p, logp, d, h, tokens, dlp.double(), dh.double(), t, logits.dtype)
    got = pkg.token_logprobs_backward(logits, tokens, dlp, dh, temperature=t, **kw)
    assert got.dtype == logits.dtype
    assert bool(((got.double() - ref).abs() <= off).all())


SIZES = [(1, 1), (3, 2), (5, 3), (2, 7), (4, 8), (3, 9), (1, 15), (33, 100), (7, 1001), (300, 4097),
         (2, 32000), (700, 32000), (5, 50001), (3, 131077), (2, 262144),
         (700, 1), (1500, 37), (9000, 100), (2000, 1001), (640, 2290), (600, 4500), (1000, 8191)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("R,V", SIZES)
def test_logprobs_sizes(pkg, cuda, R, V, dtype):
    logits, tokens = logits_of(cuda, R, V, dtype, seed=V)
    check_forward(pkg, logits, tokens, 0.8)
    check_backward(pkg, logits, tokens, 0.8)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [1, 5, 6, 7, 8, 37, 32003])
@pytest.mark.parametrize("offset,extra", [(1, 0), (0, 1), (3, 5), (7, 2)])
def test_logprobs_alignments(pkg, cuda, dtype, V, offset, extra):
    """Rows that start anywhere; what lies between and behind them is NaN."""
    logits, tokens = logits_of(cuda, 6, V, dtype, 3, offset=offset, stride=V + extra)
    check_forward(pkg, logits, tokens, 1.0)
    check_backward(pkg, logits, tokens, 1.0)
    # a gradient with another alignment and stride than its logits, and nothing outside it
    wide = torch.full((6, V + 9), 5.0, dtype=dtype, device=cuda)
    check_backward(pkg, logits, tokens, 1.0, dlogits=wide[:, 2:V + 2])
    assert bool((wide[:, :2] == 5).all()) and bool((wide[:, V + 2:] == 5).all())
    same = torch.full((6 * (V + extra) + offset + 8,), 5.0, dtype=dtype, device=cuda)
    view = same[offset:offset + 6 * (V + extra)].view(6, V + extra)[:, :V]
    check_backward(pkg, logits, tokens, 1.0, dlogits=view)
    keep = torch.ones_like(same, dtype=torch.bool)
    keep[offset:offset + 6 * (V + extra)].view(6, V + extra)[:, :V] = False
    assert bool((same[keep] == 5).all())


@pytest.mark.parametrize("t", [0.0, 1e-3, 0.7, 100.0])
def test_logprobs_temperatures(pkg, cuda, t):
    logits, tokens = logits_of(cuda, 9, 5000, torch.float32, 5)
    if t == 1e-3:
        logits.mul_(1e-3)
    check_forward(pkg, logits, tokens, t)
    check_backward(pkg, logits, tokens, t)


def test_logprobs_masked_columns(pkg, cuda):
    """-infinity and the type's lowest value as masks, at a row's ends, in runs, everywhere but
    at one place, and before and behind the maximum."""
    low = torch.finfo(torch.float32).min
    logits, tokens = logits_of(cuda, 8, 3001, torch.float32, 6)
    tokens.fill_(1500)
    for r, mask in enumerate([-math.inf, low] * 4):
        where = [slice(0, 1400), slice(1600, None), slice(0, None, 2), slice(0, None)][r // 2]
        keep = logits[r, 1500].item()
        logits[r, where] = mask
        logits[r, 1500] = keep
    check_forward(pkg, logits, tokens, 0.9)
    check_backward(pkg, logits, tokens, 0.9)
    dlp = torch.ones(8, device=cuda)
    grad = pkg.token_logprobs_backward(logits, tokens, dlp, dlp, temperature=0.9)
    assert bool((grad[logits < -1e30] == 0).all())
    # a masked token: its log-probability is -infinity, the entropy is the others'
    lp, h = pkg.token_logprobs(logits[:1], torch.tensor([3], dtype=torch.int32, device=cuda))
    assert lp.item() == -math.inf and math.isfinite(h.item())
    # nothing but the lowest value: uniform
    lp, h = pkg.token_logprobs(torch.full((1, 1000), low, device=cuda), tokens[:1] * 0)
    assert abs(lp.item() + math.log(1000)) < 1e-6 + E and abs(h.item() - math.log(1000)) < 1e-6 + E


def test_logprobs_without_a_number(pkg, cuda):
    """NaN, +infinity, or nothing but -infinity give NaN in their rows alone."""
    logits, tokens = logits_of(cuda, 5, 2000, torch.float32, 7)
    logits[1, 77] = math.nan
    logits[2, 78] = math.inf
    logits[3] = -math.inf
    lp, h = pkg.token_logprobs(logits, tokens)
    g = torch.ones(5, device=cuda)
    grad = pkg.token_logprobs_backward(logits, tokens, g, g)
    for r in range(5):
        assert math.isnan(lp[r].item()) == (r in (1, 2, 3))
        assert math.isnan(h[r].item()) == (r in (1, 2, 3))
        assert bool(torch.isnan(grad[r]).all()) == (r in (1, 2, 3))
    check_forward(pkg, logits[[0, 4]].contiguous(), tokens[[0, 4]].contiguous(), 1.0)


def test_logprobs_rows_skipped_and_bad_tokens(pkg, cuda):
    logits, tokens = logits_of(cuda, 4, 500, torch.float32, 8)
    tokens[2] = 500
    logits[1] = math.nan
    enable = torch.tensor([1, 0, 1, 1], dtype=torch.int32, device=cuda)
    lp, h = torch.full((4,), 9.0, device=cuda), torch.full((4,), 8.0, device=cuda)
    error = torch.zeros(1, dtype=torch.int32, device=cuda)
    pkg.token_logprobs(logits, tokens, row_enable=enable, logprobs=lp, entropy=h, error=error)
    assert error.item() == 1
    assert lp[1].item() == 9.0 and h[1].item() == 8.0 and lp[2].item() == 0.0 and h[2].item() == 0.0
    error.zero_()
    g = torch.ones(4, device=cuda)
    grad = pkg.token_logprobs_backward(logits, tokens, g, row_enable=enable, error=error)
    assert error.item() == 1
    assert bool((grad[1:3] == 0).all()) and bool((grad[[0, 3]] != 0).any())
    check_forward(pkg, logits[[0, 3]].contiguous(), tokens[[0, 3]].contiguous(), 1.0)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("R,V", [(700, 900), (6, 9000)])
@pytest.mark.parametrize("step", [30.0, 60.0, 68.0, 72.0, 200.0])
def test_logprobs_of_rows_in_steps(pkg, cuda, R, V, dtype, step):
    """Rows that rise by `step` and fall again, so that what a warp sees first is far below or
    far above the row's maximum (in base 2: up to 288 either way); with gradients of 1e-7."""
    logits, tokens = logits_of(cuda, R, V, dtype, 41)
    at = torch.arange(V, device=cuda)
    logits += (step * ((at // 97) % 2)).to(dtype)
    logits[1::2] -= (step * (at < V // 3)).to(dtype)
    tokens[::3] = torch.where(at % 194 > 97, logits[::3], -1e30).argmax(1).to(torch.int32)
    check_forward(pkg, logits, tokens, 1.0)
    check_backward(pkg, logits, tokens, 1.0)
    p, logp, d, _, h, _ = rows64(logits, tokens, 1.0)
    g = torch.full((R,), 1e-7, device=cuda)
    ref, off = grad64(p, logp, d, h, tokens, g.double(), g.double(), 1.0, dtype)
    got = pkg.token_logprobs_backward(logits, tokens, g, g)
    assert bool(((got.double() - ref).abs() <= off).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("R,V", [(700, 2000), (40, 32000)])
@pytest.mark.parametrize("gap", [3.0, 6.0, 11.0, 16.0, 30.0, 60.0])
def test_logprobs_of_peaked_rows(pkg, cuda, R, V, dtype, gap):
    """One element far above the others, wherever it lies, which is the row's token or not.
    With gaps above 16 the others are less than 2^-7 of the sum (32000 e^(1/2) e^-16), and what
    the log-probability is off by is the one large summand's: 2^-22 of its exp2, 2^-22 of its
    exponent's rounding (below 12 in base 2), and at most 92 additions of 2^-24."""
    logits, tokens = logits_of(cuda, R, V, dtype, 47, std=1.0)
    logits.clamp_(-5, 5)
    tokens[:] = torch.linspace(0, V - 1, R, device=cuda).to(torch.int32)
    logits[torch.arange(R, device=cuda), tokens.long()] = 5.0 + gap
    tokens[::2] = (tokens[::2] * 7 + 1) % V
    check_forward(pkg, logits, tokens, 1.0)
    check_backward(pkg, logits, tokens, 1.0)
    if gap > 16:
        lp, _ = pkg.token_logprobs(logits, tokens)
        want = rows64(logits, tokens, 1.0)[3]
        bound = 2.0 ** -21 + 92 * 2.0 ** -24 + 2.0 ** -24 * want.abs()
        assert bool(((lp.double() - want).abs() <= bound).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("R,V", [(900, 555), (60, 20011)])
def test_logprobs_awkward_rows_among_others(pkg, cuda, R, V, dtype):
    """Rows without a number, masked rows, rows of logits in the millions (of which one at the
    top of the fp32 range), skipped rows and bad tokens, each beside ordinary ones; short rows
    and long ones, at odd strides."""
    logits, tokens = logits_of(cuda, R, V, dtype, 31, offset=1, stride=V + 2)
    low = torch.finfo(dtype).min
    for r in range(R):
        kind = r % 10
        if kind == 0:
            logits[r, r % V] = math.nan
        elif kind == 1:
            logits[r, r % V] = math.inf
        elif kind == 2:
            logits[r] = -math.inf
        elif kind == 3:
            logits[r] = low
        elif kind == 4:
            logits[r] *= 3e6
        elif kind == 5:
            logits[r, : V // 2] = low
        elif kind == 6:
            logits[r] = logits[r] * 1e3 - 1e30
        elif kind == 7:
            logits[r, 0] = 3e38
    tokens[8::10] = V
    enable = torch.ones(R, dtype=torch.int32, device=cuda)
    enable[9::20] = 0
    error = torch.zeros(1, dtype=torch.int32, device=cuda)
    lp, h = torch.full((R,), 9.0, device=cuda), torch.full((R,), 9.0, device=cuda)
    pkg.token_logprobs(logits, tokens, row_enable=enable, logprobs=lp, entropy=h, error=error)
    assert error.item() == 1
    one = torch.ones(R, device=cuda)
    grad = pkg.token_logprobs_backward(logits, tokens, one, one, row_enable=enable)
    at = torch.arange(R, device=cuda)
    bad, off = at % 10 == 8, at % 20 == 9
    assert bool((lp[bad] == 0).all()) and bool((h[bad] == 0).all())
    assert bool((lp[off] == 9).all()) and bool((h[off] == 9).all())
    assert bool((grad[bad | off] == 0).all())
    p, logp, d, want, ent, spread = rows64(logits, tokens.clamp(max=V - 1), 1.0)
    nan = (at % 10 < 3) & ~bad & ~off
    assert bool(torch.isnan(lp[nan]).all()) and bool(torch.isnan(h[nan]).all())
    assert bool(torch.isnan(grad[nan]).all())
    ok = ~nan & ~bad & ~off
    assert bool(((lp[ok].double() - want[ok]).abs() <= E + 2.0 ** -24 * want[ok].abs()).all())
    assert bool(((h[ok].double() - ent[ok]).abs() <= E * (1 + spread[ok]) + 2.0 ** -24 * ent[ok]).all())
    ref, tol = grad64(p, logp, d, ent, tokens.clamp(max=V - 1), one.double(), one.double(), 1.0, dtype)
    assert bool(((grad[ok].double() - ref[ok]).abs() <= tol[ok]).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("R,V", [(700, 300), (5, 1003), (400, 32000), (2, 200000)])
def test_gradient_in_place(pkg, cuda, R, V, dtype):
    logits, tokens = logits_of(cuda, R, V, dtype, 9)
    g = torch.linspace(-1, 1, R, device=cuda)
    want = pkg.token_logprobs_backward(logits, tokens, g, g)
    got = pkg.token_logprobs_backward(logits, tokens, g, g, dlogits=logits)
    assert got.data_ptr() == logits.data_ptr() and torch.equal(got, want)


# ---------------------------------------------------------------- policy loss
def policy64(logits, tokens, w, adv, old, ref, seq, t, lo, hi, kl_c, ent_c):
    live = w != 0
    x = torch.where(live[:, None], logits.double(), 0.0)
    p, logp, d, lp, h, spread = rows64(x, tokens, t)
    a = adv.double()[seq.long()] if seq is not None else adv.double()
    ratio = (lp - old.double()).exp() if old is not None else torch.ones_like(lp)
    held = ratio.clip(1 - lo, 1 + hi)
    cut = ratio * a > held * a
    pol = -torch.where(cut, held * a, ratio * a)
    slope = torch.where(cut, 0.0, -ratio * a)
    kl = torch.zeros_like(lp)
    bend = torch.zeros_like(lp)
    if kl_c:
        bend = (ref.double() - lp).exp()
        kl = bend - (ref.double() - lp) - 1
        slope = slope + kl_c * (1 - bend)
    loss = pol + kl_c * kl - ent_c * h
    terms = torch.stack([loss, pol, kl, h, cut.double()])
    stats = torch.where(live, terms * w.double(), 0.0).sum(1)
    e_lp = E + 2.0 ** -24 * lp.abs()
    e_loss = e_lp * ((ratio * a).abs() + abs(kl_c) * (1 + bend)) + abs(ent_c) * E * (1 + spread)
    z = lambda v: torch.where(live, v, 0.0)  # noqa: E731
    return dict(p=p, logp=logp, d=d, h=h, lp=z(lp), ent=z(h), ratio=z(ratio), kl=z(kl), pol=z(pol),
                cut=z(cut.double()), loss=z(loss), stats=stats, g=z(slope * w), gh=z(-ent_c * w.double()),
                e_loss=z(e_loss), e_lp=z(e_lp), spread=spread, live=live,
                e_g=z((ratio * a).abs() + abs(kl_c) * (1 + bend)) * e_lp * w.abs(), mass=terms.abs())


def case(dev, R, V, dtype, seed, groups=None):
    logits, tokens = logits_of(dev, R, V, dtype, seed)
    g = torch.Generator(device=dev).manual_seed(seed + 1)
    lp = torch.log_softmax(logits.float(), 1).gather(1, tokens.long()[:, None])[:, 0]
    S = groups or R
    seq = (torch.arange(R, device=dev) * S // R).to(torch.int32) if groups else None
    adv = torch.randn(S, generator=g, device=dev)
    old = lp + 0.25 * torch.randn(R, generator=g, device=dev)
    return dict(logits=logits, tokens=tokens, weights=torch.rand(R, generator=g, device=dev) / R,
                advantages=adv, old_logprobs=old, row_seq=seq,
                ref_logprobs=lp + 0.3 * torch.randn(R, generator=g, device=dev))


def check_policy(pkg, c, t=1.0, lo=0.2, hi=0.2, kl=0.04, ent=0.01, **kw):
    ref = policy64(c["logits"], c["tokens"], c["weights"], c["advantages"], c["old_logprobs"],
                   c["ref_logprobs"], c["row_seq"], t, lo, hi, kl, ent)
    r = pkg.policy_loss(**c, temperature=t, clip_low=lo, clip_high=hi, kl_coef=kl,
                        entropy_coef=ent, **kw)
    assert bool(((r.logprobs.double() - ref["lp"]).abs() <= ref["e_lp"]).all())
    assert bool(((r.entropy.double() - ref["ent"]).abs()
                 <= E * (1 + ref["spread"]) + 2.0 ** -24 * ref["ent"]).all())
    near = lambda x, y, off: bool(((x.double() - y).abs() <= off + 2.0 ** -22 * y.abs()).all())  # noqa: E731
    assert near(r.ratio, ref["ratio"], ref["e_lp"] * ref["ratio"])
    assert near(r.row_loss, ref["loss"], ref["e_loss"])
    assert torch.equal(r.clipped.double(), ref["cut"])
    w = c["weights"].double().abs()
    off = (ref["e_loss"] * w).sum() + 1e-6 * (torch.where(ref["live"], ref["mass"], 0.0) * w).sum(1)
    assert bool(((r.stats.double() - ref["stats"]).abs() <= off).all())
    if r.dlogits is not None:
        want, off = grad64(ref["p"], ref["logp"], ref["d"], ref["h"], c["tokens"], ref["g"],
                           ref["gh"], t, c["logits"].dtype)
        hit = torch.zeros_like(want).scatter_(1, c["tokens"].long()[:, None], 1.0)
        off = off + ref["e_g"][:, None] * (ref["p"] + hit) / (t if t else 1.0)
        assert bool(((r.dlogits.double() - want).abs() <= off).all())
    return r


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("R,V,groups", [(1, 1, None), (3, 17, None), (64, 1000, 4), (33, 32001, 5),
                                        (600, 32000, 75), (3, 131072, None), (3000, 601, 30)])
def test_policy_sizes(pkg, cuda, dtype, R, V, groups):
    check_policy(pkg, case(cuda, R, V, dtype, R + V, groups), t=0.8)


@pytest.mark.parametrize("kl,ent", [(0.0, 0.0), (0.1, 0.0), (0.0, 0.02), (-0.1, -0.01)])
def test_policy_terms(pkg, cuda, kl, ent):
    c = case(cuda, 40, 777, torch.float32, 20, 8)
    check_policy(pkg, c, kl=kl, ent=ent)
    check_policy(pkg, c, kl=kl, ent=ent, lo=0.0, hi=0.5)
    check_policy(pkg, c, kl=kl, ent=ent, backward=False)
    if kl == 0:
        c["ref_logprobs"] = None
        check_policy(pkg, c, kl=kl, ent=ent)
    c["old_logprobs"] = None
    r = check_policy(pkg, c, kl=kl, ent=ent)
    assert bool((r.ratio == 1).all()) and not bool(r.clipped.any())


def test_policy_of_padded_rows(pkg, cuda):
    """Rows of weight 0 are not read (here they are NaN) and give zeros; tokens and rollouts out
    of range are reported and treated the same way."""
    c = case(cuda, 30, 2003, torch.bfloat16, 21, 6)
    c["logits"][::3] = math.nan
    c["weights"][::3] = 0.0
    c["old_logprobs"][::3] = math.nan
    c["tokens"][0] = -1
    c["row_seq"][3] = 99
    error = torch.zeros(1, dtype=torch.int32, device=cuda)
    d = torch.full((30, 2003), 3.0, dtype=torch.bfloat16, device=cuda)
    r = pkg.policy_loss(**c, kl_coef=0.04, entropy_coef=0.01, error=error, dlogits=d)
    assert error.item() == 0
    assert bool((r.rows[::3] == 0).all())
    assert bool((r.dlogits[::3] == 0).all()) and bool(torch.isfinite(r.stats).all())
    c["tokens"][0], c["row_seq"][3] = 0, 0
    c["old_logprobs"][::3] = 0.0
    good = check_policy(pkg, c)
    assert torch.equal(good.dlogits, r.dlogits) and torch.equal(good.stats, r.stats)
    for name, value, code in (("tokens", 2003, 1), ("row_seq", 6, 2), ("row_seq", -1, 2)):
        bad = dict(c)
        bad[name] = c[name].clone()
        bad[name][4] = value
        error.zero_()
        r = pkg.policy_loss(**bad, kl_coef=0.04, entropy_coef=0.01, error=error)
        assert error.item() == code
        none = dict(c, weights=c["weights"].clone())
        none["weights"][4] = 0.0
        want = pkg.policy_loss(**none, kl_coef=0.04, entropy_coef=0.01)
        assert torch.equal(r.stats, want.stats) and torch.equal(r.dlogits, want.dlogits)


def test_policy_without_live_rows(pkg, cuda):
    c = case(cuda, 4, 100, torch.float32, 22)
    c["weights"].zero_()
    r = pkg.policy_loss(**c, kl_coef=0.1)
    assert bool((r.stats == 0).all()) and bool((r.dlogits == 0).all())
    none = {k: (v[:0] if torch.is_tensor(v) else v) for k, v in c.items()}
    r = pkg.policy_loss(**none, kl_coef=0.1)
    assert bool((r.stats == 0).all()) and r.dlogits.shape == (0, 100)


def test_policy_gradient_in_place_and_again(pkg, cuda):
    c = case(cuda, 50, 32000, torch.float32, 23)
    first = pkg.policy_loss(**c, kl_coef=0.04, entropy_coef=0.01)
    again = pkg.policy_loss(**c, kl_coef=0.04, entropy_coef=0.01)
    for name in ("stats", "rows", "dlogits"):                 # the same bits every time
        assert torch.equal(getattr(first, name), getattr(again, name))
    same = pkg.policy_loss(**c, kl_coef=0.04, entropy_coef=0.01, dlogits=c["logits"])
    assert same.dlogits.data_ptr() == c["logits"].data_ptr()
    assert torch.equal(same.dlogits, first.dlogits) and torch.equal(same.stats, first.stats)


def test_policy_gradient_against_differences(pkg, cuda):
    """Central differences of the kernel's own loss along the gradient and along single rows.
    With steps of s standard deviations the third derivative's share is below s^2 of the
    slope's terms; the loss's fp32 rounding, 2^-24 |loss|, is divided by the step."""
    c = case(cuda, 12, 300, torch.float32, 24, 3)
    c["weights"].fill_(1.0)
    lp = torch.log_softmax(c["logits"], 1).gather(1, c["tokens"].long()[:, None])[:, 0]
    # away from the clip's corners: ratios of 1.1, 1.5 and 0.6
    c["old_logprobs"] = lp - torch.log(torch.tensor([1.1, 1.5, 0.6] * 4, device=cuda))
    kw = dict(kl_coef=0.5, entropy_coef=0.3, temperature=0.9)
    base = pkg.policy_loss(**c, **kw)
    grad = base.dlogits.double()
    ways = [grad / grad.norm()]
    for r in (0, 5, 11):
        one = torch.zeros_like(grad)
        one[r] = grad[r] / grad[r].norm().clamp(min=1e-6)
        ways.append(one)
    step = 0.02
    for way in ways:
        loss = []
        for s in (step, -step):
            x = (c["logits"].double() + s * way).float()
            loss.append(pkg.policy_loss(**dict(c, logits=x), **kw, backward=False).stats[0].double())
        slope = ((loss[0] - loss[1]) / (2 * step)).item()
        want = (grad * way).sum().item()
        # values of order 10: 2^-24 x 10 / step < 1e-4; the curvature's share step^2 x 10
        assert abs(slope - want) <= 1e-4 + 10 * step ** 2 * max(1.0, abs(want)), (slope, want)


def test_policy_captured_and_replayed(pkg, cuda):
    c = case(cuda, 20, 5000, torch.bfloat16, 25, 4)
    kw = dict(kl_coef=0.04, entropy_coef=0.01)
    pkg.policy_loss(**c, **kw)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        r = pkg.policy_loss(**c, **kw)
    for seed in (30, 31):
        new = case(cuda, 20, 5000, torch.bfloat16, seed, 4)
        for k, v in c.items():
            v.copy_(new[k])
        graph.replay()
        torch.cuda.synchronize()
        want = pkg.policy_loss(**new, **kw)
        for name in ("stats", "rows", "dlogits"):
            assert torch.equal(getattr(r, name), getattr(want, name))


def test_rows_beyond_32_bits(pkg, cuda):
    """Rows whose element offsets pass 2^32."""
    R, V, stride = 3, 1000, 2 ** 31 + 8
    flat = torch.empty(2 * stride + V, dtype=torch.bfloat16, device=cuda)
    logits = flat.as_strided((R, V), (stride, 1))
    small, tokens = logits_of(cuda, R, V, torch.bfloat16, 26)
    logits.copy_(small)
    g = torch.ones(R, device=cuda)
    a, b = pkg.token_logprobs(logits, tokens), pkg.token_logprobs(small, tokens)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    want = pkg.token_logprobs_backward(small, tokens, g, g)
    assert torch.equal(pkg.token_logprobs_backward(logits, tokens, g, g, dlogits=logits), want)


def test_calls_of_two_threads(pkg, cuda):
    """Two host threads with rows of different lengths, each on its own stream."""
    import threading
    shapes = [(64, 32000), (64, 131077)]
    cases = [logits_of(cuda, R, V, torch.float32, V) for R, V in shapes]
    want = [pkg.token_logprobs(*c) for c in cases]
    torch.cuda.synchronize()
    wrong, streams = [], [torch.cuda.Stream() for _ in shapes]

    def work(i):
        try:
            got = [pkg.token_logprobs(*cases[i], stream=streams[i]) for _ in range(200)]
            streams[i].synchronize()
            wrong.extend(1 for a, b in got
                         if not (torch.equal(a, want[i][0]) and torch.equal(b, want[i][1])))
        except Exception as e:
            wrong.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
