"""What the 8-bit cache and the policy operators refuse, on the CPU: every check
runs before the first CUDA call, so the addresses here are never followed."""
import ctypes
import math

import pytest
import torch

OK = 4096      # a well-aligned address
ODD = 4098


def append_params(pkg, **kw):
    p = dict(num_seqs=2, num_kv_heads=4, num_tokens=32, max_pages_per_seq=8, arena_pages=16,
             k_stride=512, v_stride=512, format=pkg.RT_KV8_S8, dtype=pkg.RT_DTYPE_BF16)
    p.update(kw)
    return pkg.rt_kv8_append_params_t(**p)


def append(pkg, p, at=None, value=OK):
    ptrs = [OK] * 8 + [None, None]      # k v cu lens table pages scales tail error stream
    if at is not None:
        ptrs[at] = value
    return pkg.lib().rt_kv8_append(ctypes.byref(p) if p else None, *ptrs)


@pytest.mark.parametrize("kw", [dict(num_kv_heads=0), dict(format=2), dict(dtype=2),
                                dict(k_stride=511), dict(v_stride=504), dict(k_stride=516),
                                dict(num_tokens=2 ** 31)])
def test_append_refuses_params(pkg, kw):
    assert append(pkg, append_params(pkg, **kw)) == pkg.RT_EINVAL
    assert b"kv8_append" in pkg.lib().rt_last_error()


def test_append_refuses_pointers(pkg):
    assert append(pkg, None) == pkg.RT_EINVAL
    for i in range(8):
        assert append(pkg, append_params(pkg), i, None) == pkg.RT_EINVAL
        assert append(pkg, append_params(pkg), i, ODD) == pkg.RT_EINVAL
    assert append(pkg, append_params(pkg), 8, ODD) == pkg.RT_EINVAL
    assert append(pkg, append_params(pkg), 0, OK + 8) == pkg.RT_EINVAL
    # nothing to do needs no arrays
    assert append(pkg, append_params(pkg, num_tokens=0), 0, None) == pkg.RT_OK
    assert append(pkg, append_params(pkg, num_seqs=0), 0, None) == pkg.RT_OK


def attn_params(pkg, **kw):
    p = dict(num_seqs=2, num_q_heads=16, num_kv_heads=4, max_pages_per_seq=8, max_seq_len=143,
             format=pkg.RT_KV8_E4M3, arena_pages=16, q_stride=2048, scale=0.1, chunk_pages=0)
    p.update(kw)
    return pkg.rt_kv8_attn_params_t(**p)


def attend(pkg, p, at=None, value=OK, workspace=OK, size=1 << 20):
    ptrs = [OK] * 7                     # q pages scales tail table lens out
    if at is not None:
        ptrs[at] = value
    return pkg.lib().rt_kv8_decode_attention(ctypes.byref(p) if p else None, *ptrs, workspace, size,
                                             None, None)


@pytest.mark.parametrize("kw", [dict(num_kv_heads=0), dict(num_q_heads=0), dict(num_q_heads=18),
                                dict(num_q_heads=36), dict(format=2), dict(q_stride=2047),
                                dict(q_stride=2052), dict(chunk_pages=129), dict(scale=math.inf),
                                dict(scale=math.nan), dict(max_seq_len=144),
                                dict(max_seq_len=2 ** 31), dict(num_seqs=2 ** 28)])
def test_attention_refuses_params(pkg, kw):
    p = attn_params(pkg, **kw)
    assert attend(pkg, p) == pkg.RT_EINVAL
    assert b"kv8_decode_attention" in pkg.lib().rt_last_error()
    assert pkg.lib().rt_kv8_attn_workspace_bytes(ctypes.byref(p)) == 0


def test_attention_refuses_pointers_and_workspaces(pkg):
    assert attend(pkg, None) == pkg.RT_EINVAL
    for i in range(7):
        assert attend(pkg, attn_params(pkg), i, None) == pkg.RT_EINVAL
        assert attend(pkg, attn_params(pkg), i, ODD) == pkg.RT_EINVAL
    short = attn_params(pkg, max_seq_len=100)
    assert pkg.lib().rt_kv8_attn_workspace_bytes(ctypes.byref(short)) == 0
    split = attn_params(pkg, max_pages_per_seq=1000, max_seq_len=16000)
    need = pkg.lib().rt_kv8_attn_workspace_bytes(ctypes.byref(split))
    assert need > 0
    assert attend(pkg, split, size=need - 1) == pkg.RT_ENOMEM
    assert attend(pkg, split, workspace=None) == pkg.RT_ENOMEM
    assert attend(pkg, split, workspace=OK + 8, size=need) == pkg.RT_EINVAL
    assert attend(pkg, attn_params(pkg, num_seqs=0), 0, None) == pkg.RT_OK


def logprob_params(pkg, **kw):
    p = dict(num_rows=4, vocab=100, row_stride=100, grad_stride=100, dtype=pkg.RT_DTYPE_F32,
             temperature=1.0, row_enable=None)
    p.update(kw)
    return pkg.rt_logprob_params_t(**p)


BAD_ROWS = [dict(vocab=0), dict(vocab=262145, row_stride=300000, grad_stride=300000),
            dict(dtype=2), dict(row_stride=99), dict(temperature=-1.0),
            dict(temperature=1e-5), dict(temperature=2e4), dict(temperature=math.nan)]


@pytest.mark.parametrize("kw", BAD_ROWS + [dict(row_enable=ODD)])
def test_logprobs_refuse(pkg, kw):
    lib, p = pkg.lib(), logprob_params(pkg, **kw)
    assert lib.rt_token_logprobs(ctypes.byref(p), OK, OK, OK, OK, None, None) == pkg.RT_EINVAL
    assert lib.rt_token_logprobs_backward(ctypes.byref(p), OK, OK, OK, OK, 1 << 20, None,
                                          None) == pkg.RT_EINVAL
    assert b"token_logprobs_backward" in lib.rt_last_error()


def test_logprobs_refuse_pointers(pkg):
    lib, p = pkg.lib(), logprob_params(pkg)
    ref = ctypes.byref(p)
    assert lib.rt_token_logprobs(None, OK, OK, OK, OK, None, None) == pkg.RT_EINVAL
    for i in range(3):
        for bad in (None, ODD):
            a = [OK, OK, OK]
            a[i] = bad
            assert lib.rt_token_logprobs(ref, *a, None, None, None) == pkg.RT_EINVAL
    back = [OK, OK, OK, OK, 1 << 20]    # logits tokens dlogprobs dentropy dlogits
    for i in (0, 1, 2, 4):
        a = list(back)
        a[i] = None
        assert lib.rt_token_logprobs_backward(ref, *a, None, None) == pkg.RT_EINVAL
    # the gradient in the middle of the logits, or over them with another stride
    for d in (OK + 4, OK + 1596, OK - 1596):
        assert lib.rt_token_logprobs_backward(ref, *back[:4], d, None, None) == pkg.RT_EINVAL
    other = logprob_params(pkg, grad_stride=101)
    assert lib.rt_token_logprobs_backward(ctypes.byref(other), *back[:4], OK, None,
                                          None) == pkg.RT_EINVAL
    none = logprob_params(pkg, num_rows=0)
    assert lib.rt_token_logprobs(ctypes.byref(none), None, None, None, None, None, None) == pkg.RT_OK


def policy_params(pkg, **kw):
    p = dict(num_rows=4, vocab=100, num_seqs=4, dtype=pkg.RT_DTYPE_F32, row_stride=100,
             grad_stride=100, temperature=1.0, clip_low=0.2, clip_high=0.2, kl_coef=0.1,
             entropy_coef=0.0)
    p.update(kw)
    return pkg.rt_policy_params_t(**p)


def policy(pkg, p, at=None, value=None):
    # logits tokens weights advantages row_seq old ref rows stats dlogits error stream
    ptrs = [OK] * 9 + [1 << 20, None, None]
    if at is not None:
        ptrs[at] = value
    return pkg.lib().rt_policy_loss(ctypes.byref(p) if p else None, *ptrs)


@pytest.mark.parametrize("kw", BAD_ROWS + [dict(clip_low=-0.1), dict(clip_high=math.nan),
                                           dict(clip_high=math.inf), dict(kl_coef=math.inf),
                                           dict(entropy_coef=math.nan), dict(grad_stride=99)])
def test_policy_refuses_params(pkg, kw):
    assert policy(pkg, policy_params(pkg, **kw)) == pkg.RT_EINVAL
    assert b"policy_loss" in pkg.lib().rt_last_error()


def test_policy_refuses_pointers(pkg):
    assert policy(pkg, None) == pkg.RT_EINVAL
    p = policy_params(pkg)
    for i in (0, 1, 2, 3, 6, 7, 8):
        assert policy(pkg, p, i, None) == pkg.RT_EINVAL
    for i in range(11):
        assert policy(pkg, p, i, ODD) == pkg.RT_EINVAL
    assert policy(pkg, p, 7, OK + 8) == pkg.RT_EINVAL            # the rows' records: 16 bytes
    assert policy(pkg, policy_params(pkg, num_seqs=3), 4, None) == pkg.RT_EINVAL


def test_bindings_refuse_tensors(pkg):
    """Shapes, types and devices the C entry points cannot see."""
    logits, tokens = torch.zeros(4, 10), torch.zeros(4, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        pkg.token_logprobs(logits, tokens)
    with pytest.raises(ValueError, match="logits"):
        pkg.token_logprobs(logits.half(), tokens)
    with pytest.raises(ValueError, match="logits"):
        pkg.token_logprobs(logits.t(), tokens)
    with pytest.raises(ValueError, match="tokens"):
        pkg.token_logprobs(logits, tokens.long())
    with pytest.raises(ValueError, match="tokens"):
        pkg.policy_loss(logits, tokens[:3], torch.ones(4), torch.ones(4))
    with pytest.raises(ValueError, match="format"):
        pkg.kv8_cache(2, 1, 1, "fp4", device="cpu")
    pages, scales, tail = pkg.kv8_cache(2, 1, 4, device="cpu")
    assert pages.dtype == torch.float8_e4m3fn and pages.shape == (2, 4, 2, 2048)
    k = torch.zeros(3, 4, 128, dtype=torch.bfloat16)
    cu, lens = torch.tensor([0, 3], dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    table = torch.zeros(1, 2, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        pkg.kv8_append(k, k, cu, lens, table, pages, scales, tail)
