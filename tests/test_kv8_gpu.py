"""The 8-bit KV cache (rt_kv8_append, rt_kv8_decode_attention) against plain
64-bit implementations.

The cache is exact: codes, scales and tail must equal the definition's bit for
bit.  Attention's tolerance counts the kernel's roundings.  With
A = scale * sum_d |q_d k_d| the fp32 accumulation of a score (8 tensor-core
steps of 16 products, each step off by at most 2^-23 of what it holds) and the
two factors' roundings are off by at most 2^-19 A, so e^s by that share; exp2
adds 2^-21.  P in two fp16 terms is off by 2^-22 of 1, the fp32 sums by
2^-24 a step, of which a worker and the merge have at most some hundreds: 2^-16
in all would be the worst case, 2^-18 covers it with the sums' roundings
independent of one another.  Both errors enter the sum and the normaliser, hence twice:
|error| <= 2 (2^-19 max A + 2^-18) sum_t p_t |v_t|."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

QMAX = {"e4m3": 448.0, "s8": 127.0}


def offsets():
    """Byte of (token, dim) in a K plane and a V plane, as kv_layout.h states them."""
    t, d = np.meshgrid(np.arange(16), np.arange(128), indexing="ij")
    k = (d // 32) * 512 + ((t % 8) * 4 + (d // 4) % 4) * 16 + (2 * ((d // 16) % 2) + t // 8) * 4 + d % 4
    v = (d // 32) * 512 + ((d % 8) * 4 + (t % 8) // 2) * 16 \
        + (2 * ((d // 16) % 2) + (d // 8) % 2) * 4 + t % 2 + 2 * (t // 8)
    return k, v


KO, VO = offsets()


def quantise(x, fmt):
    """(codes as int8 bytes, scale) of one 16 x 128 tile of bf16 values held in float64."""
    top = np.abs(x).max()
    if not np.isfinite(top):
        return np.zeros(x.shape, np.int8), np.float32(np.nan)
    scale = np.float32(top / QMAX[fmt])  # float64 quotient, then fp32: the fp32 division
    if scale == 0:
        return np.zeros(x.shape, np.int8), scale
    y = np.clip((x / np.float64(scale)).astype(np.float32), -QMAX[fmt], QMAX[fmt])
    if fmt == "s8":
        return np.rint(y).astype(np.int8), scale
    return torch.from_numpy(y).to(torch.float8_e4m3fn).view(torch.int8).numpy(), scale


class Model:
    """The cache's contents by definition: every sequence's rows, and the bytes they give."""

    def __init__(self, pages, scales, tail, fmt):
        self.fmt = fmt
        self.pages = pages.view(torch.int8).cpu().numpy().copy()
        self.scales = scales.cpu().numpy().copy()
        self.tail = tail.double().cpu().numpy().copy()

    def append(self, b, old, rows, table):
        """rows [n, heads, 2, 128] of bf16 values in float64."""
        heads = rows.shape[1]
        for i in range(rows.shape[0]):
            pos = old + i
            self.tail_next(b, pos, rows[i])
            if pos % 16 == 15:
                for h in range(heads):
                    for plane in range(2):
                        codes, s = quantise(self.work[h, plane], self.fmt)
                        at = self.pages[table[pos // 16], h, plane]
                        at[(VO if plane else KO).reshape(-1)] = codes.reshape(-1)
                        self.scales[table[pos // 16], h, plane] = s
        if rows.shape[0]:
            keep = (old + rows.shape[0]) % 16
            first = keep - min(keep, rows.shape[0])
            self.tail[b, :, :, first:keep] = self.work[:, :, first:keep]

    def tail_next(self, b, pos, row):
        if not hasattr(self, "work") or self.owner != b:
            self.work, self.owner = self.tail[b].copy(), b
        self.work[:, :, pos % 16] = row

    def check(self, pages, scales, tail):
        assert np.array_equal(scales.cpu().numpy(), self.scales, equal_nan=True)
        assert np.array_equal(pages.view(torch.int8).cpu().numpy(), self.pages)
        assert np.array_equal(tail.double().cpu().numpy(), self.tail, equal_nan=True)


def cache(pkg, dev, fmt, n_pages, B, heads, seed):
    """Buffers that hold noise everywhere, so that a write out of place shows."""
    g = torch.Generator(device=dev).manual_seed(seed)
    pages, scales, tail = pkg.kv8_cache(n_pages, B, heads, fmt, dev)
    pages.view(torch.int8).copy_(torch.randint(-100, 100, pages.shape, generator=g, device=dev,
                                               dtype=torch.int8))
    scales.uniform_(0.01, 0.03, generator=g)
    tail.normal_(generator=g)
    return pages, scales, tail


def tables(lens, n_pages, seed, spare=3):
    """A page table with exactly the full pages of `lens`, scattered; the rest is -7."""
    full = [int(n) // 16 for n in lens]
    perm = np.random.default_rng(seed).permutation(n_pages)
    t = np.full((len(lens), max(full + [1]) + spare), -7, np.int32)
    k = 0
    for b, n in enumerate(full):
        t[b, :n] = perm[k:k + n]
        k += n
    return t


def bf16(x):
    return x.to(torch.bfloat16).double().cpu().numpy()


def do_append(pkg, dev, bufs, k, v, old, new, table, **kw):
    cu = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    pkg.kv8_append(k, v, torch.from_numpy(cu).to(dev),
                   torch.tensor(old, dtype=torch.int32, device=dev),
                   torch.from_numpy(table).to(dev), *bufs, **kw)
    torch.cuda.synchronize()


@pytest.mark.parametrize("fmt", ["e4m3", "s8"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads,old,new", [
    (1, [0], [1]), (1, [15], [1]), (1, [0], [16]), (3, [10], [20]),
    (8, [0, 5, 16, 31, 40], [33, 0, 15, 1, 49]), (2, [0] * 7, [0, 0, 17, 0, 160, 1, 0]),
    (5, [14, 0, 3], [2, 16, 12])])
def test_append(pkg, cuda, fmt, dtype, heads, old, new):
    g = torch.Generator(device=cuda).manual_seed(heads + sum(new))
    n_pages = sum((a + b) // 16 for a, b in zip(old, new)) + 2
    bufs = cache(pkg, cuda, fmt, n_pages, len(old), heads, 3)
    table = tables([a + b for a, b in zip(old, new)], n_pages, 4)
    T = sum(new)
    # columns of one wider projection: token stride (heads * 2 + 1) * 128
    qkv = torch.randn(T, heads * 2 + 1, 128, generator=g, device=cuda).to(dtype)
    k, v = qkv[:, 1:heads + 1], qkv[:, heads + 1:]
    model = Model(*bufs, fmt)
    error = torch.zeros(1, dtype=torch.int32, device=cuda)
    do_append(pkg, cuda, bufs, k, v, old, new, table, error=error)
    rows = np.stack([bf16(k), bf16(v)], 2)
    at = 0
    for b, (o, n) in enumerate(zip(old, new)):
        model.append(b, o, rows[at:at + n], table[b])
        at += n
    model.check(*bufs)
    assert error.item() == 0


@pytest.mark.parametrize("fmt", ["e4m3", "s8"])
def test_append_in_parts_equals_at_once(pkg, cuda, fmt):
    g = torch.Generator(device=cuda).manual_seed(8)
    k, v = (torch.randn(2, 83, 4, 128, generator=g, device=cuda).bfloat16())
    table = tables([83], 6, 1)
    one, many = cache(pkg, cuda, fmt, 6, 1, 4, 2), cache(pkg, cuda, fmt, 6, 1, 4, 2)
    do_append(pkg, cuda, one, k, v, [0], [83], table)
    at = 0
    for n in [1, 14, 1, 1, 16, 30, 0, 20]:
        do_append(pkg, cuda, many, k[at:at + n], v[at:at + n], [at], [n], table)
        at += n
    assert at == 83
    assert torch.equal(one[0].view(torch.int8), many[0].view(torch.int8))
    assert torch.equal(one[1], many[1])
    assert torch.equal(one[2][:, :, :, :3], many[2][:, :, :, :3])


@pytest.mark.parametrize("fmt", ["e4m3", "s8"])
def test_append_of_awkward_values(pkg, cuda, fmt):
    """Zeros, a NaN, an infinity, the smallest bf16 numbers, the largest, and quotients
    that fall on and next to the border between two codes."""
    x = torch.zeros(16 * 8, 2, 128)
    g = torch.Generator().manual_seed(1)
    x[16:32] = torch.randn(16, 2, 128, generator=g)
    x[20, 0, 7] = float("nan")
    x[32:48] = torch.randn(16, 2, 128, generator=g)
    x[40, 1, 0] = float("-inf")
    x[48:64] = torch.randn(16, 2, 128, generator=g) * 2.0 ** -130
    x[64:80] = torch.randn(16, 2, 128, generator=g).clamp(-3, 3) * 1e38
    x[80:96] = (torch.arange(16 * 256).reshape(16, 2, 128) % 255 - 127) / 2  # multiples of a half
    x[80, :, 0] = 127.0
    x[96:112] = (torch.arange(16 * 256).reshape(16, 2, 128) % 449) * 2.0 ** -4
    x[96, :, 0] = 448.0
    x[112:128] = -3.0
    x = x.bfloat16().to(cuda)
    bufs = cache(pkg, cuda, fmt, 8, 1, 2, 5)
    table = tables([128], 8, 9)
    model = Model(*bufs, fmt)
    do_append(pkg, cuda, bufs, x, x.flip(0).contiguous(), [0], [128], table)
    model.append(0, 0, np.stack([bf16(x), bf16(x.flip(0))], 2), table[0])
    model.check(*bufs)
    assert torch.isnan(bufs[1]).sum().item() == 4


def test_append_reports_bad_indices(pkg, cuda):
    g = torch.Generator(device=cuda).manual_seed(2)
    k = torch.randn(96, 2, 128, generator=g, device=cuda).bfloat16()

    def run(old, cu, table, n_pages=6):
        bufs = cache(pkg, cuda, "s8", n_pages, len(old), 2, 6)
        model = Model(*bufs, "s8")
        error = torch.zeros(1, dtype=torch.int32, device=cuda)
        pkg.kv8_append(k, k, torch.tensor(cu, dtype=torch.int32, device=cuda),
                       torch.tensor(old, dtype=torch.int32, device=cuda),
                       torch.from_numpy(table).to(cuda), *bufs, error=error)
        torch.cuda.synchronize()
        return bufs, model, error.item()

    rows = np.stack([bf16(k), bf16(k)], 2)
    table = tables([48, 48], 6, 1, spare=0)
    bad = table.copy()
    bad[0, 1] = 6
    bufs, model, code = run([0, 0], [0, 48, 96], bad)   # that page alone is not written
    assert code == 2
    spare = table.copy()
    model.append(0, 0, rows[:48], table[0])
    model.append(1, 0, rows[48:], table[1])
    before = cache(pkg, cuda, "s8", 6, 2, 2, 6)
    model.pages[spare[0, 1]] = before[0].view(torch.int8).cpu().numpy()[spare[0, 1]]
    model.scales[spare[0, 1]] = before[1].cpu().numpy()[spare[0, 1]]
    model.check(*bufs)
    bufs, model, code = run([-1, 0], [0, 48, 96], table)
    assert code == 1
    model.append(1, 0, rows[48:], table[1])
    model.check(*bufs)
    _, _, code = run([17, 0], [0, 48, 96], table)       # a fourth page of a table of three
    assert code == 1
    bufs, model, code = run([0, 0], [0, 97, 96], table)
    assert code == 3
    _, _, code = run([0, 0], [-1, 48, 96], table)
    assert code == 3


# ------------------------------------------------------------------ attention
def make(pkg, dev, lens, heads, G, fmt, seed, n_pages=None, first_page=0):
    g = torch.Generator(device=dev).manual_seed(seed)
    used = sum(int(n) // 16 for n in lens)
    n_pages = n_pages or used + 2
    table = tables(lens, used, seed)
    table[table >= 0] += first_page
    pages, scales, tail = pkg.kv8_cache(n_pages, len(lens), heads, fmt, dev)
    part = slice(first_page, first_page + used)
    if used:
        code = torch.randint(-127, 128, (used, heads, 2, 2048), generator=g, device=dev)
        if fmt == "e4m3":  # a NaN code has all of its low bits set
            code = torch.where(code == 127, 126, code)
            code = torch.where(code == -1, -2, code)
        pages.view(torch.int8)[part] = code.to(torch.int8)
        scales[part].uniform_(0.5, 1.5, generator=g)
        scales[part] *= 2.0 / QMAX[fmt]
    tail.normal_(generator=g)
    q = torch.randn(len(lens), heads * G, 128, generator=g, device=dev).bfloat16()
    return q, pages, scales, tail, table


def reference(q, pages, scales, tail, table, lens, b, scale):
    """(out, bound) of sequence b in float64."""
    heads = pages.shape[1]
    n = int(lens[b])
    at = torch.from_numpy(table[b, :n // 16].astype(np.int64)).to(q.device)
    x = pages.view(torch.int8)[at].view(pages.dtype).double() * scales[at].double()[..., None]
    ko, vo = (torch.from_numpy(o.reshape(-1)).to(q.device) for o in (KO, VO))
    k = x[:, :, 0][..., ko].reshape(-1, heads, 16, 128).transpose(0, 1).reshape(heads, -1, 128)
    v = x[:, :, 1][..., vo].reshape(-1, heads, 16, 128).transpose(0, 1).reshape(heads, -1, 128)
    rest = tail[b, :, :, :n % 16].double()
    k, v = torch.cat([k, rest[:, 0]], 1), torch.cat([v, rest[:, 1]], 1)
    qq = q[b].double().reshape(heads, -1, 128)
    p = torch.softmax(qq @ k.transpose(1, 2) * scale, -1)
    size = (qq.abs() @ k.abs().transpose(1, 2) * abs(scale)).amax(-1, keepdim=True)
    out, mass = p @ v, p @ v.abs()
    return out.reshape(-1, 128), (2 * (size * 2.0 ** -19 + 2.0 ** -18) * mass).reshape(-1, 128)


def check(got, q, pages, scales, tail, table, lens, scale=128 ** -0.5):
    for b in range(len(lens)):
        if lens[b] == 0:
            assert torch.all(got[b] == 0)
            continue
        ref, bound = reference(q, pages, scales, tail, table, lens, b, scale)
        err = (got[b].double() - ref).abs()
        assert bool((err <= bound).all()), (b, lens[b], err.max().item(), bound.min().item())


def attend(pkg, dev, q, pages, scales, tail, table, lens, **kw):
    kw.setdefault("max_seq_len", max(int(max(lens)), 1))
    error = torch.zeros(1, dtype=torch.int32, device=dev)
    out = pkg.kv8_decode_attention(q, pages, scales, tail, torch.from_numpy(table).to(dev),
                                   torch.tensor(lens, dtype=torch.int32, device=dev),
                                   error=error, **kw)
    torch.cuda.synchronize()
    assert error.item() == 0
    return out


LENS = [1, 0, 15, 16, 17, 31, 32, 33, 64, 100, 257, 1039]


@pytest.mark.parametrize("fmt", ["e4m3", "s8"])
@pytest.mark.parametrize("heads,G", [(1, 1), (4, 2), (2, 3), (8, 4), (3, 5), (1, 7), (2, 8)])
def test_attention_groups(pkg, cuda, fmt, heads, G):
    case = make(pkg, cuda, LENS, heads, G, fmt, seed=G)
    check(attend(pkg, cuda, *case, LENS), *case, LENS)


@pytest.mark.parametrize("lens", [
    [16 * 130, 16 * 37 + 5, 0, 33, 2049, 15], [7000], [16 * 64] * 3, [0, 0, 5000, 0],
    list(range(0, 600, 7)), [20000] + [3] * 300, [161] * 150, [40000, 1, 40000, 17]])
@pytest.mark.parametrize("heads,G", [(4, 4), (1, 8), (7, 3)])
def test_attention_splits(pkg, cuda, lens, heads, G):
    """Batches that are cut in every way: one row over the whole GPU, many short rows, rows
    without tokens between, long rows beside short ones."""
    case = make(pkg, cuda, lens, heads, G, "s8", seed=len(lens))
    check(attend(pkg, cuda, *case, lens), *case, lens)


@pytest.mark.parametrize("chunk", [1, 2, 3, 8, 31, 64, 127, 128])
def test_attention_chunks(pkg, cuda, chunk):
    lens = [16 * 130, 16 * 37 + 5, 0, 33, 2049, 15]
    case = make(pkg, cuda, lens, 4, 4, "s8", seed=chunk)
    check(attend(pkg, cuda, *case, lens, chunk_pages=chunk), *case, lens)


@pytest.mark.parametrize("scale", [0.0, -0.05, 1.0])
def test_attention_scales(pkg, cuda, scale):
    lens = [40, 300]
    case = make(pkg, cuda, lens, 2, 4, "e4m3", seed=4)
    check(attend(pkg, cuda, *case, lens, scale=scale), *case, lens, scale)


def test_attention_bounds_above_the_lengths(pkg, cuda):
    """max_seq_len far above every length: the empty items give nothing."""
    lens = [0, 5, 700, 16]
    case = make(pkg, cuda, lens, 2, 4, "s8", seed=6)
    table = np.full((4, 600), -7, np.int32)
    table[:, :case[4].shape[1]] = case[4]
    case = (*case[:4], table)
    check(attend(pkg, cuda, *case, lens, max_seq_len=9000), *case, lens)


def test_attention_ragged_batch(pkg, cuda):
    lens = np.random.default_rng(2).integers(128, 4097, 64).tolist()
    case = make(pkg, cuda, lens, 8, 4, "e4m3", seed=2)
    a = attend(pkg, cuda, *case, lens)
    check(a, *case, lens)
    assert torch.equal(a, attend(pkg, cuda, *case, lens))  # the same bits every time


def test_attention_long_context(pkg, cuda):
    lens = [131071]
    case = make(pkg, cuda, lens, 2, 8, "s8", seed=12)
    check(attend(pkg, cuda, *case, lens), *case, lens)


def test_offsets_beyond_32_bits(pkg, cuda):
    """A cache of 4.6 GB whose used pages lie behind 4 GiB, appended to and attended to."""
    n_pages, heads = 140000, 8
    lens = [100, 33]
    bufs = pkg.kv8_cache(n_pages, 2, heads, "s8", cuda)
    table = tables(lens, sum(n // 16 for n in lens), 3)
    table[table >= 0] += n_pages - 12
    g = torch.Generator(device=cuda).manual_seed(7)
    k, v = torch.randn(2, 133, heads, 128, generator=g, device=cuda).bfloat16()
    do_append(pkg, cuda, bufs, k, v, [0, 0], lens, table)
    assert int(bufs[0][:n_pages - 12].view(torch.int64).count_nonzero()) == 0
    q = torch.randn(2, 32, 128, generator=g, device=cuda).bfloat16()
    check(attend(pkg, cuda, q, *bufs, table, lens), q, *bufs, table, lens)


def test_attention_of_extreme_queries(pkg, cuda):
    """Rows of zeros, of the smallest and of large bf16 numbers, and of a wide range: the
    power of two that brings a row into fp16 must not show."""
    lens = [70] * 6
    q, *rest = make(pkg, cuda, lens, 1, 4, "s8", seed=9)
    q[0] = 0
    q[1] *= 2.0 ** -126
    q[2] *= 2.0 ** 20
    q[3] = q[3] * torch.logspace(-12, 1, 128, device=cuda).bfloat16()
    q[4, :, 1:] *= 2.0 ** -30
    check(attend(pkg, cuda, q, *rest, lens, scale=2.0 ** -22), q, *rest, lens, 2.0 ** -22)


def test_attention_nan_stays_in_its_head(pkg, cuda):
    lens = [40, 40]
    q, pages, scales, tail, table = make(pkg, cuda, lens, 4, 2, "e4m3", seed=10)
    tail[:, :, :, 8:] = float("nan")       # behind the tail's end: not the cache's
    case = (q, pages, scales, tail, table)
    clean = attend(pkg, cuda, *case, lens)
    check(clean, *case, lens)
    scales[table[0, 1], 2, 0] = float("nan")
    scales[table[1, 0], 0, 1] = float("nan")
    out = attend(pkg, cuda, *case, lens)
    nan = torch.isnan(out).all(-1)
    want = torch.zeros(2, 8, dtype=torch.bool, device=cuda)
    want[0, 4:6] = True
    want[1, 0:2] = True
    assert torch.equal(nan, want)
    assert torch.equal(out[~want], clean[~want])


def test_attention_reports_bad_indices(pkg, cuda):
    lens = [64, 40, 32]
    q, pages, scales, tail, table = make(pkg, cuda, lens, 2, 4, "s8", seed=11)

    def run(table, lens, max_seq_len):
        error = torch.zeros(1, dtype=torch.int32, device=cuda)
        out = torch.full((3, 8, 128), 7.0, device=cuda)
        pkg.kv8_decode_attention(q, pages, scales, tail, torch.from_numpy(table).to(cuda),
                                 torch.tensor(lens, dtype=torch.int32, device=cuda), max_seq_len,
                                 out=out, error=error)
        torch.cuda.synchronize()
        return out, error.item()

    for bad in (-1, pages.shape[0], 2 ** 31 - 1):
        t = table.copy()
        t[0, 2] = bad
        out, code = run(t, lens, 64)
        assert code == 2
        check(out[1:], q[1:], pages, scales, tail[1:], table[1:], lens[1:])
    for wrong in (65, -5):
        out, code = run(table, [64, wrong, 32], 64)
        assert code == 1 and bool((out[1] == 7.0).all())
        check(out[[0, 2]], q[[0, 2]], pages, scales, tail[[0, 2]], table[[0, 2]], [64, 32])


def test_attention_of_strided_queries(pkg, cuda):
    """Queries that are columns of a wider projection."""
    lens = [20, 45, 7]
    q, *rest = make(pkg, cuda, lens, 2, 4, "e4m3", seed=13)
    wide = torch.full((3, 12, 128), float("nan"), device=cuda).bfloat16()
    wide[:, :8] = q
    assert torch.equal(attend(pkg, cuda, wide[:, :8], *rest, lens),
                       attend(pkg, cuda, q, *rest, lens))


def test_captured_steps_replay(pkg, cuda):
    """Append and attention captured once on a side stream and replayed as lengths and
    inputs change, each replay as the eager calls."""
    B, heads, G = 5, 4, 4
    g = torch.Generator(device=cuda).manual_seed(14)
    start = [0, 14, 15, 31, 200]
    table = tables([s + 8 for s in start], 40, 5)
    td = torch.from_numpy(table).to(cuda)
    state = [cache(pkg, cuda, "s8", 40, B, heads, 8) for _ in range(2)]
    # earlier contents: one appended prompt
    prompt = torch.randn(sum(start), heads, 128, generator=g, device=cuda).bfloat16()
    for s in state:
        do_append(pkg, cuda, s, prompt, prompt, [0] * B, start, table)
    lens = torch.tensor(start, dtype=torch.int32, device=cuda)
    after = lens + 1
    cu = torch.arange(B + 1, dtype=torch.int32, device=cuda)
    k, v = torch.zeros(2, B, heads, 128, device=cuda).bfloat16()
    q = torch.zeros(B, heads * G, 128, device=cuda).bfloat16()
    out = torch.zeros(B, heads * G, 128, device=cuda)

    def step(s, out):
        pkg.kv8_append(k, v, cu, lens, td, *s)
        pkg.kv8_decode_attention(q, *s, td, after, max_seq_len=250, out=out)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step(state[0], out)
    eager = torch.zeros_like(out)
    for _ in range(8):
        for t in (k, v, q):
            t.copy_(torch.randn(t.shape, generator=g, device=cuda))
        graph.replay()
        step(state[1], eager)
        torch.cuda.synchronize()
        assert torch.equal(out, eager)
        assert torch.equal(state[0][0], state[1][0]) and torch.equal(state[0][2], state[1][2])
        check(out, q, *state[0], table, after.tolist())
        lens += 1
        after += 1


def test_two_streams_at_once(pkg, cuda):
    """Calls on two streams, each with the workspace that the binding takes for it."""
    lens = [3000, 1700]
    case = make(pkg, cuda, lens, 8, 4, "s8", seed=15)
    want = attend(pkg, cuda, *case, lens)
    td, ld = torch.from_numpy(case[4]).to(cuda), torch.tensor(lens, dtype=torch.int32, device=cuda)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = [[pkg.kv8_decode_attention(*case[:4], td, ld, 3000, stream=s) for s in streams]
            for _ in range(20)]
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for pair in outs for o in pair)


@pytest.mark.parametrize("heads,G", [(1, 1), (8, 4)])
def test_what_follows_waits_for_the_whole_call(pkg, cuda, heads, G):
    """A bound that provides for splits where no sequence has any: the merge has nothing to
    do, and what the stream does next must still find the outputs done."""
    lens = [1500, 1530, 3, 1536]
    case = make(pkg, cuda, lens, heads, G, "s8", seed=21)
    table = np.full((4, 4096), -7, np.int32)
    table[:, :case[4].shape[1]] = case[4]
    case = (*case[:4], table)
    want = attend(pkg, cuda, *case, lens)
    td, ld = torch.from_numpy(table).to(cuda), torch.tensor(lens, dtype=torch.int32, device=cuda)
    out, seen = torch.zeros_like(want), []
    for _ in range(50):
        out.fill_(-1.0)
        pkg.kv8_decode_attention(*case[:4], td, ld, 65535, out=out, chunk_pages=96)
        seen.append(out.clone())
    torch.cuda.synchronize()
    check(want, *case, lens)
    for s in seen:
        check(s, *case, lens)


@pytest.mark.parametrize("fmt", ["e4m3", "s8"])
def test_sequences_without_a_page(pkg, cuda, fmt):
    """An arena of no pages and a page table of no columns: tails alone."""
    g = torch.Generator(device=cuda).manual_seed(22)
    lens = [15, 0, 1, 9]
    k, v = torch.randn(2, sum(lens), 2, 128, generator=g, device=cuda).bfloat16()
    bufs = pkg.kv8_cache(0, 4, 2, fmt, cuda)
    table = np.zeros((4, 0), np.int32)
    do_append(pkg, cuda, bufs, k, v, [0] * 4, lens, table)
    q = torch.randn(4, 8, 128, generator=g, device=cuda).bfloat16()
    got = attend(pkg, cuda, q, *bufs, table, lens)
    check(got, q, *bufs, table, lens)
    # a token more would need a page
    error = torch.zeros(1, dtype=torch.int32, device=cuda)
    pkg.kv8_append(k[:1], v[:1], torch.tensor([0, 1, 1, 1, 1], dtype=torch.int32, device=cuda),
                   torch.tensor(lens, dtype=torch.int32, device=cuda),
                   torch.from_numpy(table).to(cuda), *bufs, error=error)
    assert error.item() == 1


def test_padded_tokens_and_shared_pages(pkg, cuda):
    """Rows behind the last sequence's (NaN here) are not read; two sequences read the same
    pages of a common prefix, one of them twice."""
    g = torch.Generator(device=cuda).manual_seed(23)
    k, v = torch.full((2, 64, 2, 128), float("nan"), device=cuda).bfloat16()
    k[:40], v[:40] = torch.randn(2, 40, 2, 128, generator=g, device=cuda).bfloat16()
    bufs = cache(pkg, cuda, "s8", 4, 2, 2, 6)
    model = Model(*bufs, "s8")
    table = tables([32, 8], 4, 7)
    do_append(pkg, cuda, bufs, k, v, [0, 0], [32, 8], table)
    rows = np.stack([bf16(k), bf16(v)], 2)
    model.append(0, 0, rows[:32], table[0])
    model.append(1, 0, rows[32:40], table[1])
    model.check(*bufs)
    table[1, :3] = table[0, [0, 1, 0]]
    lens = [32, 56]
    q = torch.randn(2, 8, 128, generator=g, device=cuda).bfloat16()
    check(attend(pkg, cuda, q, *bufs, table, lens), q, *bufs, table, lens)


@pytest.mark.parametrize("chunk", [0, 8])
def test_captured_splits_replay(pkg, cuda, chunk):
    """Split rows, captured in two graphs that replay in turn and at once on two streams, as
    lengths and queries change between the replays."""
    lens = [9000, 300, 5000, 17]
    q, *rest, table = make(pkg, cuda, lens, 4, 4, "e4m3", seed=31)
    td, ld = torch.from_numpy(table).to(cuda), torch.tensor(lens, dtype=torch.int32, device=cuda)
    g = torch.Generator(device=cuda).manual_seed(32)
    kw = dict(max_seq_len=9000, chunk_pages=chunk)
    pkg.kv8_decode_attention(q, *rest, td, ld, **kw)
    graphs, outs, streams = [], [], [torch.cuda.Stream() for _ in range(2)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            outs.append([pkg.kv8_decode_attention(q, *rest, td, ld, **kw) for _ in range(2)])
        graphs.append(graph)
    for cut in (0, 1, 700, 16):
        now = [max(n - cut, 0) for n in lens]
        ld.copy_(torch.tensor(now, dtype=torch.int32))
        q.copy_(torch.randn(q.shape, generator=g, device=cuda))
        want = pkg.kv8_decode_attention(q, *rest, td, ld, **kw)
        check(want, q, *rest, table, now)
        torch.cuda.synchronize()
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, want) for pair in outs for o in pair)


@pytest.mark.parametrize("start", [1, 15, 16, 40])
def test_append_of_tokens_from_the_middle(pkg, cuda, start):
    """cu_tokens that begin and end inside the rows, and a batch of many empty sequences."""
    g = torch.Generator(device=cuda).manual_seed(start)
    new = [0] * 40 + [31, 0, 1, 16] + [0] * 40 + [50]
    old = [(7 * i) % 33 for i in range(len(new))]
    T = start + sum(new) + 9
    k, v = torch.randn(2, T, 2, 128, generator=g, device=cuda).bfloat16()
    n_pages = sum((a + b) // 16 for a, b in zip(old, new)) + 2
    bufs = cache(pkg, cuda, "s8", n_pages, len(new), 2, 6)
    table = tables([a + b for a, b in zip(old, new)], n_pages, 7)
    model = Model(*bufs, "s8")
    error = torch.zeros(1, dtype=torch.int32, device=cuda)
    cu = np.concatenate([[start], start + np.cumsum(new)]).astype(np.int32)
    pkg.kv8_append(k, v, torch.from_numpy(cu).to(cuda),
                   torch.tensor(old, dtype=torch.int32, device=cuda),
                   torch.from_numpy(table).to(cuda), *bufs, error=error)
    rows = np.stack([bf16(k), bf16(v)], 2)
    for b, n in enumerate(new):
        model.append(b, old[b], rows[cu[b]:cu[b] + n], table[b])
    model.check(*bufs)
    assert error.item() == 0
