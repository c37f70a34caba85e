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
