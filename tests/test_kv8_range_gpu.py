"""The 8-bit KV cache over wide ranges: length bounds, queries and values.  References and
tolerances are those of test_kv8_gpu.py, except where a test states its own."""
import pytest
import torch

from test_kv8_gpu import attend, check, make

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
