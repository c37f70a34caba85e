"""The 8-bit KV cache over wide ranges: length bounds, queries and values.  References and
tolerances are those of test_kv8_gpu.py, except where a test states its own."""
import pytest
import torch

from test_kv8_gpu import KO, VO, attend, check, make, reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads,G", [(8, 4), (2, 8)])
@pytest.mark.parametrize("chunk", [0, 8])
def test_attention_bounds_above_the_page_table(pkg, cuda, heads, G, chunk):
    """A bound that no page table of P columns can hold is 16 P + 15, bit for bit; a length
    beyond that is reported and skipped."""
    lens = [1500, 0, 767, 33]
    case = make(pkg, cuda, lens, heads, G, "s8", seed=51)
    P = case[4].shape[1]
    want = attend(pkg, cuda, *case, lens, max_seq_len=16 * P + 15, chunk_pages=chunk)
    check(want, *case, lens)
    for bound in (16 * P + 16, 16 * P + 32, 4096, 2 ** 31 - 1):
        got = attend(pkg, cuda, *case, lens, max_seq_len=bound, chunk_pages=chunk)
        assert torch.equal(got, want)
    error = torch.zeros(1, dtype=torch.int32, device=cuda)
    out = torch.full_like(want, 7.0)
    far = torch.tensor([1500, 16 * P + 16, 767, 33], dtype=torch.int32, device=cuda)
    pkg.kv8_decode_attention(*case[:4], torch.from_numpy(case[4]).to(cuda), far, 4096, out=out,
                             chunk_pages=chunk, error=error)
    assert error.item() == 1 and bool((out[1] == 7.0).all())
    assert torch.equal(out[[0, 2, 3]], want[[0, 2, 3]])


@pytest.mark.parametrize("fmt", ["e4m3", "s8"])
@pytest.mark.parametrize("heads,G", [(4, 4), (2, 8)])
@pytest.mark.parametrize("pages,tail", [(1.0, 1e35), (1.0, 1e38), (1e38, 1.0), (1e38, 1e38),
                                        (1e-30, 1e38), (1e-30, 1e-30), (1e38, 1e-30), (1e20, 1e36)])
def test_attention_of_large_and_small_values(pkg, cuda, fmt, heads, G, pages, tail):
    """V up to bf16's largest, in pages, in tails and in both: a mean of finite values is finite,
    also where their sum is not, in one item, over warps, over chunks, and over both merges."""
    lens = [15, 9, 31, 40, 1, 700, 2050, 0]
    q, codes, scales, rest, table = make(pkg, cuda, lens, heads, G, fmt, seed=52)
    scales[..., 1] *= pages
    rest.clamp_(-3, 3)
    rest[:, :, 1] *= tail
    case = (q, codes, scales, rest, table)
    for chunk in (0, 8):
        out = attend(pkg, cuda, *case, lens, chunk_pages=chunk)
        assert bool(torch.isfinite(out).all())
        check(out, *case, lens)
    long = [16 * 600 + 15]
    q, codes, scales, rest, table = make(pkg, cuda, long, heads, G, fmt, seed=53)
    scales[..., 1] *= pages
    rest.clamp_(-3, 3)
    rest[:, :, 1] *= tail
    case = (q, codes, scales, rest, table)
    for chunk in (0, 2, 64):
        check(attend(pkg, cuda, *case, long, chunk_pages=chunk), *case, long)


@pytest.mark.parametrize("fmt", ["e4m3", "s8"])
@pytest.mark.parametrize("heads,G", [(3, 1), (2, 4), (2, 5), (2, 8)])
@pytest.mark.parametrize("gap", [4, 9, 13, 14, 16, 17, 20, 21, 22, 25, 40, 100])
def test_attention_of_queries_of_a_wide_range(pkg, cuda, fmt, heads, G, gap):
    """Elements 2^-gap of their row's largest, where K is 0 at the large ones: the score is the
    small elements' alone, and as accurate as theirs."""
    lens = [70, 16, 9, 160, 33]
    q, pages, scales, tail, table = make(pkg, cuda, lens, heads, G, fmt, seed=54)
    large = torch.arange(0, 128, 9, device=cuda)
    at = torch.from_numpy(KO).to(cuda)[:, large].reshape(-1)
    pages.view(torch.int8)[:, :, 0, at] = 0
    tail[:, :, 0, :, large] = 0
    small = torch.ones(128, dtype=torch.bool, device=cuda)
    small[large] = False
    q[:, :, large] = torch.where(q[:, :, large] < 0, -1.0, 1.0).bfloat16()
    q[:, :, small] = (q[:, :, small].float() * 2.0 ** -gap).clamp(-1, 1).bfloat16()
    q[1] = torch.where(small, 129 / 128 * 2.0 ** -gap, 1.0).bfloat16()
    q[2, ::2] = q[2, ::2].abs()
    case = (q, pages, scales, tail, table)
    scale = 0.08 * 2.0 ** gap
    check(attend(pkg, cuda, *case, lens, scale=scale), *case, lens, scale)
    # elements of all sizes in between, and K everywhere
    q, pages, scales, tail, table = make(pkg, cuda, lens, heads, G, fmt, seed=55)
    q *= torch.logspace(0, -gap, 128, base=2.0, device=cuda).bfloat16()
    case = (q, pages, scales, tail, table)
    check(attend(pkg, cuda, *case, lens, scale=0.3), *case, lens, 0.3)


@pytest.mark.parametrize("fmt", ["e4m3", "s8"])
@pytest.mark.parametrize("heads,G", [(2, 4), (2, 8)])
def test_attention_of_a_query_without_numbers(pkg, cuda, fmt, heads, G):
    """A NaN or an infinity in one head's query is that head's alone, also where its
    neighbours need all of bf16's range, and a skipped page counts as absent there."""
    lens = [70, 300]
    q, pages, scales, tail, table = make(pkg, cuda, lens, heads, G, fmt, seed=56)
    q[:, :, ::3] *= 2.0 ** -30
    q[0, 1, 5] = float("nan")
    q[1, G, 7] = float("inf")
    case = (q, pages, scales, tail, table)
    out = attend(pkg, cuda, *case, lens)
    want = torch.zeros(2, heads * G, dtype=torch.bool, device=cuda)
    want[0, 1] = want[1, G] = True
    assert torch.equal(torch.isnan(out).all(-1), want) and torch.equal(torch.isnan(out).any(-1), want)
    q[0, 1, 5] = q[1, G, 7] = 0
    clean = attend(pkg, cuda, *case, lens)
    check(clean, *case, lens)
    assert torch.equal(out[~want], clean[~want])
    gone = table.copy()
    gone[0, 2] = pages.shape[0]
    error = torch.zeros(1, dtype=torch.int32, device=cuda)
    got = pkg.kv8_decode_attention(*case[:4], torch.from_numpy(gone).to(cuda),
                                   torch.tensor(lens, dtype=torch.int32, device=cuda), 300,
                                   error=error)
    assert error.item() == 2 and torch.equal(got[1], clean[1])
    # the same without that page: 54 tokens, the last page one to the left
    short = table.copy()
    short[0, 2:-1] = table[0, 3:]
    check(got[:1], q[:1], pages, scales, tail[:1], short[:1], [54])


@pytest.mark.parametrize("fmt", ["e4m3", "s8"])
@pytest.mark.parametrize("heads,G", [(4, 4), (2, 8)])
@pytest.mark.parametrize("order", ["up", "down", "mixed", "one"])
@pytest.mark.parametrize("scale", [0.02, 0.5])
def test_attention_of_value_scales_of_a_wide_range(pkg, cuda, fmt, heads, G, order, scale):
    """V scales from 2^-40 to 2^40 in one sequence; where the pages of large scales hold zeros
    the small ones' values are what is left, also beside scores that are far apart."""
    lens = [16 * 37 + 5, 16 * 8, 31, 16 * 150]
    q, pages, scales, tail, table = make(pkg, cuda, lens, heads, G, fmt, seed=57)
    g = torch.Generator(device=cuda).manual_seed(58)
    some = torch.from_numpy(VO).to(cuda)[:, ::5].reshape(-1)
    for b, n in enumerate(lens):
        full = n // 16
        at = torch.from_numpy(table[b, :full]).to(cuda).long()
        power = torch.linspace(-40, 40, max(full, 2), device=cuda)[:full].round()
        if order == "down":
            power = power.flip(0)
        elif order == "mixed":
            power = power[torch.randperm(full, generator=g, device=cuda)]
        elif order == "one":
            power = torch.where(torch.arange(full, device=cuda) == full // 2, 40.0, 0.0)
        scales[at, :, 1] *= (2.0 ** power)[:, None]
        for page in at[power > power.min() + 6].tolist():
            pages.view(torch.int8)[page, :, 1, some] = 0
    tail[:, :, 1, :, ::5] *= 2.0 ** -20
    case = (q, pages, scales, tail, table)
    for chunk in (0, 8, 128):
        check(attend(pkg, cuda, *case, lens, scale=scale, chunk_pages=chunk), *case, lens, scale)


@pytest.mark.parametrize("fmt", ["e4m3", "s8"])
@pytest.mark.parametrize("heads,G", [(2, 4), (2, 8)])
@pytest.mark.parametrize("power", [-118, -105, -90, 60, 100, 115])
def test_attention_of_small_queries_and_large_keys(pkg, cuda, fmt, heads, G, power):
    """Queries around 2^power over keys around 2^-power: ordinary scores."""
    lens = [70, 16, 9, 300]
    q, pages, scales, tail, table = make(pkg, cuda, lens, heads, G, fmt, seed=59)
    q *= 2.0 ** power
    scales[:, :, 0] *= 2.0 ** -power
    tail[:, :, 0] *= 2.0 ** -power
    case = (q, pages, scales, tail, table)
    check(attend(pkg, cuda, *case, lens), *case, lens)


@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("heads,G", [(2, 4), (2, 8)])
def test_attention_of_a_tail_without_numbers(pkg, cuda, heads, G, value):
    """In V it shows in its head and dimension alone.  In K it makes a score NaN, or infinite:
    +infinity leaves NaN, -infinity is a weight of 0, the token's absence."""
    lens = [70, 300]
    q, pages, scales, tail, table = make(pkg, cuda, lens, heads, G, "s8", seed=60)
    clean = attend(pkg, cuda, q, pages, scales, tail, table, lens)
    v = tail.clone()
    v[0, 0, 1, 3, 7] = value
    out = attend(pkg, cuda, q, pages, scales, v, table, lens)
    hit = torch.zeros_like(out, dtype=torch.bool)
    hit[0, :G, 7] = True
    assert torch.equal(~torch.isfinite(out), hit) and torch.equal(out[~hit], clean[~hit])
    k = tail.clone()
    k[0, 0, 0, 3, 7] = value
    out = attend(pkg, cuda, q, pages, scales, k, table, lens)
    sign = value * q[0, :G, 7].float()
    nan = torch.zeros_like(hit)
    nan[0, :G] = ~(sign < 0)[:, None]
    assert torch.equal(torch.isnan(out), nan)
    assert torch.equal(out[0, G:], clean[0, G:]) and torch.equal(out[1], clean[1])
    short = tail.clone()
    short[0, :, :, 3:5] = tail[0, :, :, 4:6]
    ref, bound = reference(q, pages, scales, short, table, [69, 300], 0, 128 ** -0.5)
    near = (out[0, :G].double() - ref[:G]).abs() <= bound[:G]
    assert bool((near | nan[0, :G]).all())
