"""Cases of the 8-bit KV cache and of the policy-gradient row operators.

Four operators, each in its plain form (elementary torch operations) and, where
``own`` is true, as a user's program calls the framework's kernels:

  append     new K/V tokens into the 8-bit paged cache (full pages quantised with
             one scale per page, head and plane; the unfinished page stays bf16)
  attention  one decode step of paged GQA attention over that cache
  logprobs   log-probability and entropy of one token per row of logits
             (forward, or the gradient with respect to the logits)
  policy     clipped policy loss with KL and entropy terms over rows of logits,
             with its gradient

Run from the repository's root.
"""
import importlib.util
import math
import os
import sys

import numpy as np
import torch

own = False

PAGE, DIM = 16, 128
QMAX = {"e4m3": 448.0, "s8": 127.0}
STORE = {"e4m3": torch.float8_e4m3fn, "s8": torch.int8}
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}


def _package():
    name = "gb300_rl_runtime_b200"
    if name not in sys.modules:
        folder = os.path.join(os.getcwd(), "gb300-rl-runtime_b200")
        spec = importlib.util.spec_from_file_location(
            name, os.path.join(folder, "__init__.py"), submodule_search_locations=[folder])
        module = importlib.util.module_from_spec(spec)
        sys.modules[name] = module
        spec.loader.exec_module(module)
    return sys.modules[name]


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # every slot of a full decode batch writes its new token, some of them finish a page
        dict(name="append step 256", op="append", seqs=256, old_min=512, old_max=768, new_min=1,
             new_max=1, kv_heads=8, format="s8", dtype="fp32"),
        # ragged prompts enter the cache together
        dict(name="append prompts 64", op="append", seqs=64, old_min=0, old_max=0, new_min=64,
             new_max=1024, kv_heads=8, format="e4m3", dtype="bf16"),
        # a few long prompts: the largest append
        dict(name="append long 4", op="append", seqs=4, old_min=0, old_max=0, new_min=30001,
             new_max=32768, kv_heads=8, format="s8", dtype="bf16"),
        # the first steps of a single rollout: one page and one token, latency alone
        dict(name="attention 1x17", op="attention", seqs=1, len_min=17, len_max=17, q_heads=32,
             kv_heads=8, format="e4m3"),
        # a ragged batch, lengths uniform in [128, 4096]
        dict(name="attention 64x4096", op="attention", seqs=64, len_min=128, len_max=4096,
             q_heads=32, kv_heads=8, format="e4m3"),
        # a full batch of slots with a 512-token prompt and up to 256 new tokens
        dict(name="attention 256x768", op="attention", seqs=256, len_min=512, len_max=768,
             q_heads=32, kv_heads=8, format="s8"),
        # one very long context: the split along the sequence carries it
        dict(name="attention 1x131072", op="attention", seqs=1, len_min=131071, len_max=131071,
             q_heads=32, kv_heads=4, format="s8"),
        # behaviour log-probabilities of the tokens a decode step has sampled
        dict(name="logprobs 256", op="logprobs", rows=256, vocab=32000, dtype="fp32",
             temperature=0.8, backward=False, masked=0),
        # gradient through the log-probabilities, odd vocabulary with masked padding columns
        dict(name="logprobs back 2048", op="logprobs", rows=2048, vocab=32001, dtype="bf16",
             temperature=1.0, backward=True, masked=33),
        # the last tokens of one short rollout
        dict(name="policy 64", op="policy", rows=64, vocab=32000, dtype="fp32", temperature=0.8,
             kl=0.04, entropy=0.0, masked=0, group=1),
        # an update over a batch of rollouts, all terms on: the largest policy loss
        dict(name="policy 8192", op="policy", rows=8192, vocab=32000, dtype="fp32",
             temperature=1.0, kl=0.04, entropy=0.01, masked=0, group=256),
        # padded rollouts, a larger odd vocabulary, bf16 logits, one advantage per rollout
        dict(name="policy 1023", op="policy", rows=1023, vocab=50001, dtype="bf16",
             temperature=0.7, kl=0.0, entropy=0.001, masked=17, group=33),
    ]


def _log_uniform(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["append", "attention", "logprobs", "policy"])
    if op == "append":
        heads = rng.choice([1, 2, 4, 8])
        seqs = _log_uniform(rng, 1, 512)
        new_max = _log_uniform(rng, 1, max(1, min(32768, 120000 // seqs)))
        old_max = rng.choice([0, 1]) * _log_uniform(rng, 1, 4096)
        return dict(op="append", seqs=seqs, old_min=old_max // 2, old_max=old_max,
                    new_min=rng.choice([1, new_max, (new_max + 1) // 2]), new_max=new_max,
                    kv_heads=heads, format=rng.choice(["e4m3", "s8"]),
                    dtype=rng.choice(["bf16", "bf16", "fp32"]) if seqs * new_max < 50000
                    else "bf16")
    if op == "attention":
        heads = rng.choice([1, 2, 4, 8])
        seqs = _log_uniform(rng, 1, 512)
        len_max = _log_uniform(rng, 1, max(1, min(131072, 1000000 // (seqs * heads))))
        return dict(op="attention", seqs=seqs, len_min=rng.choice([0, 1, len_max]) if len_max > 1
                    else 1, len_max=len_max, q_heads=heads * rng.choice([1, 2, 4, 5, 8]),
                    kv_heads=heads, format=rng.choice(["e4m3", "s8"]))
    vocab = _log_uniform(rng, 100, 160000)
    rows = _log_uniform(rng, 1, max(1, min(8192, 120000000 // vocab)))
    case = dict(op=op, rows=rows, vocab=vocab, dtype=rng.choice(["fp32", "bf16"]),
                temperature=rng.choice([0.7, 0.8, 1.0, 1.3]),
                masked=rng.choice([0, 0, rng.randint(1, 40)]))
    if op == "logprobs":
        return dict(case, backward=rng.random() < 0.5)
    return dict(case, kl=rng.choice([0.0, 0.04]), entropy=rng.choice([0.0, 0.01]),
                group=rng.randint(1, max(1, rows // 2)))


def _lengths(case, low, high, count, salt):
    """Lengths of a case's sequences: they belong to the case, not to the seed."""
    state = np.random.RandomState(salt + 7 * count + high)
    return state.randint(low, high + 1, count).astype(np.int64)


def work(case):
    c = case
    if c["op"] == "append":
        old = _lengths(c, c["old_min"], c["old_max"], c["seqs"], 1)
        new = _lengths(c, c["new_min"], c["new_max"], c["seqs"], 2)
        size = 4 if c["dtype"] == "fp32" else 2
        row = c["kv_heads"] * 2 * DIM
        full = (old + new) // PAGE - old // PAGE
        kept = np.where(full > 0, (old + new) % PAGE, new)         # tokens that go to the tail
        read = new.sum() * row * size + np.where(full > 0, old % PAGE, 0).sum() * row * 2
        wrote = full.sum() * (row * PAGE + c["kv_heads"] * 8) + kept.sum() * row * 2
        # scales: a maximum, a quotient and a rounding for each value that is quantised
        return {"bytes": int(read + wrote), "flops": int(full.sum() * PAGE * row * 3)}
    if c["op"] == "attention":
        n = _lengths(c, c["len_min"], c["len_max"], c["seqs"], 3)
        full, tail = n // PAGE, n % PAGE
        kv = full.sum() * c["kv_heads"] * (2 * PAGE * DIM + 8) + tail.sum() * c["kv_heads"] * 512
        table = 4 * full.sum() + 4 * c["seqs"]
        return {"bytes": int(kv + table + c["seqs"] * c["q_heads"] * DIM * 6),
                "flops": int(n.sum() * c["q_heads"] * DIM * 4)}
    size = 4 if c["dtype"] == "fp32" else 2
    cells = c["rows"] * c["vocab"]
    if c["op"] == "logprobs":
        if c["backward"]:
            return {"bytes": 2 * cells * size + 12 * c["rows"], "flops": 12 * cells}
        return {"bytes": cells * size + 12 * c["rows"], "flops": 6 * cells}
    live = c["rows"] - _padding_rows(c)
    return {"bytes": (live + c["rows"]) * c["vocab"] * size + 32 * c["rows"],
            "flops": 14 * live * c["vocab"]}


# ------------------------------------------------------------- what a user has
def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 7919 + 17)
    return g


def _page_table(full_pages, width, pages, g):
    """Every sequence's pages, scattered over the arena; unused entries are -1."""
    order = torch.randperm(pages, generator=g, device="cuda", dtype=torch.int64).to(torch.int32)
    first = torch.cumsum(full_pages, 0) - full_pages
    column = torch.arange(width, device="cuda")
    place = (first[:, None] + column[None, :]).clamp(max=pages - 1)
    return torch.where(column[None, :] < full_pages[:, None], order[place], -1).contiguous()


def _padding_rows(case):
    """Rows behind the rollouts' ends: the last seventh of each group of rows."""
    if not case["masked"]:
        return 0
    return int((np.arange(case["rows"]) % case["group"] >= case["group"] - case["group"] // 7).sum())


def prepare(case, seed):
    c, g = case, _generator(seed)
    randn = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    state = {"case": c}
    if c["op"] == "append":
        old = torch.from_numpy(_lengths(c, c["old_min"], c["old_max"], c["seqs"], 1)).cuda()
        new = torch.from_numpy(_lengths(c, c["new_min"], c["new_max"], c["seqs"], 2)).cuda()
        tokens, h = int(new.sum()), c["kv_heads"]
        after = (old + new) // PAGE
        # one page more than the sequences need: it belongs to none of them
        used = int(after.sum())
        table = _page_table(after, max(1, int(after.max())), used + 1, g)
        named = torch.zeros(used + 1, dtype=torch.bool, device="cuda")
        named[table[table >= 0].long()] = True
        state["page_table"], state["spare"] = table, (~named).nonzero()[:1, 0]
        cu = torch.zeros(c["seqs"] + 1, dtype=torch.int32, device="cuda")
        cu[1:] = torch.cumsum(new, 0)
        state["cu_tokens"], state["seq_lens"] = cu, old.to(torch.int32)
        gain = torch.exp(0.5 * randn(1, h, 1))                    # heads differ in their range
        state["k"] = (randn(tokens, h, DIM) * gain).to(TYPES[c["dtype"]])
        state["v"] = (randn(tokens, h, DIM) * gain).to(TYPES[c["dtype"]])
        state["pages"] = torch.zeros(used + 1, h, 2, PAGE * DIM, dtype=torch.int8,
                                     device="cuda").view(STORE[c["format"]])
        state["scales"] = torch.zeros(used + 1, h, 2, device="cuda")
        state["tail"] = randn(c["seqs"], h, 2, PAGE, DIM).to(torch.bfloat16)
        return state
    if c["op"] == "attention":
        lens = torch.from_numpy(_lengths(c, c["len_min"], c["len_max"], c["seqs"], 3)).cuda()
        full, h = lens // PAGE, c["kv_heads"]
        used = max(1, int(full.sum()))
        state["page_table"] = _page_table(full, max(1, int(full.max())), used, g)
        values = randn(used, h, 2, PAGE, DIM) * torch.exp(0.3 * randn(used, h, 2, 1, 1))
        codes, state["scales"] = _quantise(values.to(torch.bfloat16), c["format"])
        del values
        state["pages"] = _to_page_order(codes)
        state["tail"] = randn(c["seqs"], h, 2, PAGE, DIM).to(torch.bfloat16)
        state["q"] = randn(c["seqs"], c["q_heads"], DIM).to(torch.bfloat16)
        state["seq_lens"] = lens.to(torch.int32)
        return state
    rows, vocab = c["rows"], c["vocab"]
    logits = (2.0 * randn(rows, vocab)).to(TYPES[c["dtype"]])
    if c["masked"]:
        logits[:, vocab - c["masked"]:] = -math.inf               # padding of the vocabulary
    z = logits.float() / c["temperature"]
    noise = torch.empty(rows, vocab, device="cuda").exponential_(generator=g)
    tokens = (z - torch.log(noise)).argmax(1)                     # sampled from the softmax
    del noise
    lp = z.gather(1, tokens[:, None])[:, 0] - torch.logsumexp(z, 1)
    del z
    state.update(logits=logits, tokens=tokens.to(torch.int32))
    if c["op"] == "logprobs":
        if c["backward"]:
            state["dlogprobs"], state["dentropy"] = randn(rows) / rows, 0.01 * randn(rows) / rows
        return state
    group = torch.arange(rows, device="cuda") // c["group"]
    seqs = -(-rows // c["group"])
    state["row_seq"] = group.to(torch.int32)
    state["advantages"] = randn(seqs)
    state["weights"] = torch.full((rows,), 1.0 / rows, device="cuda")
    if c["masked"]:
        at = torch.arange(rows, device="cuda") % c["group"]
        padding = at >= c["group"] - c["group"] // 7
        state["weights"][padding] = 0.0
        state["logits"][padding] = math.nan                       # whatever the buffer held
        lp = torch.where(padding, torch.zeros_like(lp), lp)
    state["old"] = lp + 0.1 * randn(rows)
    state["ref"] = lp + 0.2 * randn(rows) if c["kl"] else None
    return state


# ------------------------------------------------------------ the plain forms
def _quantise(x, form):
    """Codes and scales of bf16 tiles [..., 16, 128]."""
    x = x.float()
    top = x.abs().amax((-1, -2))
    scale = top / torch.full_like(top, QMAX[form])
    scale = torch.where(torch.isfinite(top), scale, math.nan)
    y = torch.where(scale[..., None, None] > 0, x / scale[..., None, None], 0.0)
    y = y.clamp(-QMAX[form], QMAX[form])
    return (y.round() if form == "s8" else y).to(STORE[form]), scale


def _to_page_order(codes):
    """[n, heads, 2, 16 tokens, 128 dims] as the cache stores it: [n, heads, 2, 2048]."""
    n, h = codes.shape[:2]
    raw = codes.view(torch.int8)
    #                      t: high, low   d: j  s  c  e    ->  j  low  c  s  high  e
    k = raw[:, :, 0].reshape(n, h, 2, 8, 4, 2, 4, 4).permute(0, 1, 4, 3, 6, 5, 2, 7)
    #                      t: high, c, low   d: j  s  half  r    ->  j  r  c  s  half  high  low
    v = raw[:, :, 1].reshape(n, h, 2, 4, 2, 4, 2, 2, 8).permute(0, 1, 5, 8, 3, 6, 7, 2, 4)
    return torch.stack([k.reshape(n, h, 2048), v.reshape(n, h, 2048)], 2).view(codes.dtype)


def _from_page_order(pages):
    n, h = pages.shape[:2]
    raw = pages.view(torch.int8)
    k = raw[:, :, 0].reshape(n, h, 4, 8, 4, 2, 2, 4).permute(0, 1, 6, 3, 2, 5, 4, 7)
    v = raw[:, :, 1].reshape(n, h, 4, 8, 4, 2, 2, 2, 2).permute(0, 1, 7, 4, 8, 2, 5, 6, 3)
    return torch.stack([k.reshape(n, h, PAGE, DIM), v.reshape(n, h, PAGE, DIM)], 2).view(
        pages.dtype)


def _append_plain(s):
    form, tail = s["case"]["format"], s["tail"]
    old, cu = s["seq_lens"].long(), s["cu_tokens"].long()
    tokens, seqs, width = s["k"].shape[0], old.shape[0], s["page_table"].shape[1]
    dev = old.device
    kv = torch.stack([s["k"], s["v"]], 2).to(torch.bfloat16)              # [T, h, 2, 128]
    new = cu[1:] - cu[:-1]
    # units: more than enough (sequence, page) pairs; sequence b has those from first[b] on
    units = torch.arange(tokens // PAGE + 2 * seqs, device=dev)
    first = cu[:-1] // PAGE + 2 * torch.arange(seqs, device=dev)
    b = torch.searchsorted(first, units, right=True) - 1
    page = old[b] // PAGE + units - first[b]
    place = page[:, None] * PAGE + torch.arange(PAGE, device=dev)          # token positions
    full = (page + 1) * PAGE <= (old + new)[b]
    full &= new[b] > 0
    fresh = kv[(cu[b][:, None] + place - old[b][:, None]).clamp(0, tokens - 1)].permute(
        0, 2, 3, 1, 4)                                                     # [U, h, 2, 16, 128]
    values = torch.where((place >= old[b][:, None])[:, None, None, :, None], fresh, tail[b])
    codes, scales = _quantise(values, form)
    # units without a full page land on the spare page, which is cleared again
    to = torch.where(full, s["page_table"][b, page.clamp(max=width - 1)].long(), s["spare"])
    raw = s["pages"].view(torch.int8)
    raw[to] = _to_page_order(codes).view(torch.int8)
    s["scales"][to] = scales
    raw[s["spare"]] = 0
    s["scales"][s["spare"]] = 0.0
    last = (old + new) // PAGE * PAGE
    place = last[:, None] + torch.arange(PAGE, device=dev)                 # [B, 16]
    write = (place >= old[:, None]) & (place < (old + new)[:, None])
    fresh = kv[(cu[:-1, None] + place - old[:, None]).clamp(0, tokens - 1)].permute(0, 2, 3, 1, 4)
    tail.copy_(torch.where(write[:, None, None, :, None], fresh, tail))
    return {"pages": s["pages"], "scales": s["scales"], "tail": tail}


def _attention_plain(s):
    q, lens = s["q"].float(), s["seq_lens"].long()
    seqs, heads = q.shape[:2]
    kv_heads, width = s["pages"].shape[1], s["page_table"].shape[1]
    values = _from_page_order(s["pages"]).float() * s["scales"][..., None, None]
    cache = values[s["page_table"].clamp(min=0).long()]                    # [B, P, h, 2, 16, 128]
    cache = cache.permute(0, 2, 3, 1, 4, 5).reshape(seqs, kv_heads, 2, width * PAGE, DIM)
    cache = torch.cat([cache, s["tail"].float()], 3)
    place = torch.arange(width * PAGE, device=q.device)
    full = lens // PAGE * PAGE
    live = torch.cat([place < full[:, None],
                      torch.arange(PAGE, device=q.device) < (lens - full)[:, None]], 1)
    live = live[:, None, None, :]
    keys, vals = cache[:, :, 0], cache[:, :, 1]
    vals = torch.where(live[:, :, 0, :, None], vals, 0.0)
    score = (q.reshape(seqs, kv_heads, -1, DIM) * DIM ** -0.5) @ keys.transpose(2, 3)
    score = torch.where(live, score, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    out = (p @ vals) / torch.where(total == 0, 1.0, total)
    return out.reshape(seqs, heads, DIM)


def _rows_plain(logits, tokens, temperature):
    """Shifted logits, softmax, log of its sum, the token's log-probability (64 bits), entropy."""
    z = logits.float() / temperature
    z = z - z.amax(1, keepdim=True)
    e = torch.exp(z)
    total = e.sum(1, keepdim=True)
    log_total = torch.log(total.double())
    lp = z.gather(1, tokens.long()[:, None]).double() - log_total
    z = torch.where(e == 0, 0.0, z)
    entropy = log_total - ((e * z).sum(1, keepdim=True) / total).double()
    return z, e.div_(total), log_total, lp, entropy


def _gradient_plain(z, p, log_total, entropy, tokens, dlp, dh, temperature, dtype):
    """dlp (1[v = token] - p) - dh p (log p + entropy), over the temperature."""
    inner = dlp[:, None] + dh[:, None] * (z + (entropy - log_total).float())
    grad = p.mul_(inner).neg_()
    grad.scatter_add_(1, tokens.long()[:, None], dlp[:, None])
    return grad.div_(temperature).to(dtype)


def _logprobs_plain(s):
    c, t = s["case"], s["case"]["temperature"]
    z, p, log_total, lp, entropy = _rows_plain(s["logits"], s["tokens"], t)
    if not c["backward"]:
        return {"logprobs": lp[:, 0].float(), "entropy": entropy[:, 0].float()}
    return _gradient_plain(z, p, log_total, entropy, s["tokens"], s["dlogprobs"], s["dentropy"],
                           t, s["logits"].dtype)


CLIP = 0.2


def _policy_plain(s):
    c, t, w = s["case"], s["case"]["temperature"], s["weights"]
    live = w != 0
    logits = torch.where(live[:, None], s["logits"], 0.0) if c["masked"] else s["logits"]
    z, p, log_total, lp, entropy = _rows_plain(logits, s["tokens"], t)
    lp, h = lp[:, 0], entropy[:, 0]
    a = s["advantages"][s["row_seq"].long()].double()
    ratio = torch.exp(lp - s["old"].double())
    bound = ratio.clamp(1 - CLIP, 1 + CLIP)
    clipped = ratio * a > bound * a
    policy = -torch.minimum(ratio * a, bound * a)
    dlp = torch.where(clipped, 0.0, -ratio * a)
    kl = torch.zeros_like(lp)
    if c["kl"]:
        gap = s["ref"].double() - lp
        kl = torch.exp(gap) - gap - 1
        dlp = dlp + c["kl"] * (1 - torch.exp(gap))
    loss = policy + c["kl"] * kl - c["entropy"] * h
    terms = torch.stack([loss, policy, kl, h, clipped.double()])
    stats = torch.where(live, terms * w.double(), 0.0).sum(1).float()
    rows = [torch.where(live, x, 0.0).float() for x in (loss, lp, h)]
    # rows of weight 0 have no gradient
    grad = _gradient_plain(z, p, log_total, entropy, s["tokens"], (dlp * w).float(),
                           (-c["entropy"] * w.double()).float(), t, s["logits"].dtype)
    return {"stats": stats, "row_loss": rows[0], "logprobs": rows[1], "entropy": rows[2],
            "dlogits": grad}


def run(state):
    s, c = state, state["case"]
    if not own:
        return {"append": _append_plain, "attention": _attention_plain,
                "logprobs": _logprobs_plain, "policy": _policy_plain}[c["op"]](s)
    rt = _package()
    if c["op"] == "append":
        rt.kv8_append(s["k"], s["v"], s["cu_tokens"], s["seq_lens"], s["page_table"], s["pages"],
                      s["scales"], s["tail"])
        return {"pages": s["pages"], "scales": s["scales"], "tail": s["tail"]}
    if c["op"] == "attention":
        return rt.kv8_decode_attention(s["q"], s["pages"], s["scales"], s["tail"],
                                       s["page_table"], s["seq_lens"], max_seq_len=c["len_max"])
    if c["op"] == "logprobs":
        if c["backward"]:
            return rt.token_logprobs_backward(s["logits"], s["tokens"], s["dlogprobs"],
                                              s["dentropy"], temperature=c["temperature"])
        lp, h = rt.token_logprobs(s["logits"], s["tokens"], temperature=c["temperature"])
        return {"logprobs": lp, "entropy": h}
    r = rt.policy_loss(s["logits"], s["tokens"], s["weights"], s["advantages"], s["old"],
                       s["ref"], s["row_seq"], temperature=c["temperature"], clip_low=CLIP,
                       clip_high=CLIP, kl_coef=c["kl"], entropy_coef=c["entropy"])
    return {"stats": r.stats, "row_loss": r.row_loss, "logprobs": r.logprobs,
            "entropy": r.entropy, "dlogits": r.dlogits}


# ----------------------------------------------------- the definitions, 64 bits
def _page_offsets():
    """Byte of (token, dim) in a page's K plane and V plane."""
    t, d = torch.meshgrid(torch.arange(PAGE), torch.arange(DIM), indexing="ij")
    k = (d // 32) * 512 + ((t % 8) * 4 + (d // 4) % 4) * 16 + (2 * ((d // 16) % 2) + t // 8) * 4 \
        + d % 4
    v = (d // 32) * 512 + ((d % 8) * 4 + (t % 8) // 2) * 16 \
        + (2 * ((d // 16) % 2) + (d // 8) % 2) * 4 + t % 2 + 2 * (t // 8)
    return k.cuda(), v.cuda()


def _nearest_code(y, form):
    """The values that 8 bits can hold, nearest to y, ties to the even code."""
    if form == "s8":
        low = torch.floor(y)
        up = (y - low > 0.5) | ((y - low == 0.5) & (low % 2 != 0))
        return (low + up).clamp(-127, 127)
    grid = torch.tensor([m / 8 * 2.0 ** -6 for m in range(8)]
                        + [(1 + m / 8) * 2.0 ** (e - 7) for e in range(1, 16) for m in range(8)
                           if (e, m) != (15, 7)], dtype=torch.float64, device=y.device)
    a = y.abs().clamp(max=448.0)
    i = (torch.searchsorted(grid, a, right=True) - 1).clamp(max=grid.numel() - 2)
    gap, step = a - grid[i], grid[i + 1] - grid[i]
    up = (gap > step / 2) | ((gap == step / 2) & (i % 2 == 1))
    return torch.copysign(grid[i + up.long()], y)


def _append_exact(s):
    form, tail = s["case"]["format"], s["tail"].clone()
    pages = torch.zeros(s["pages"].shape, dtype=torch.float64, device="cuda")
    scales = torch.zeros(s["scales"].shape, dtype=torch.float64, device="cuda")
    ko, vo = _page_offsets()
    old, cu, table = s["seq_lens"].tolist(), s["cu_tokens"].tolist(), s["page_table"]
    for b, n0 in enumerate(old):
        fresh = torch.stack([s["k"][cu[b]:cu[b + 1]], s["v"][cu[b]:cu[b + 1]]], 2).bfloat16()
        if not fresh.shape[0]:
            continue
        kept = n0 % PAGE
        seq = torch.cat([tail[b, :, :, :kept].permute(2, 0, 1, 3), fresh])   # from the old page on
        full = seq.shape[0] // PAGE
        x = seq[:full * PAGE].double().reshape(full, PAGE, *seq.shape[1:]).permute(0, 2, 3, 1, 4)
        if full:
            at = table[b, n0 // PAGE:n0 // PAGE + full].long()
            scale = (x.abs().amax((-1, -2)) / QMAX[form]).float().double()
            codes = _nearest_code((x / scale[..., None, None]).float().double(), form)
            out = torch.zeros(full, x.shape[1], 2, PAGE * DIM, dtype=torch.float64, device="cuda")
            out[:, :, 0, ko.reshape(-1)] = codes[:, :, 0].reshape(full, -1, PAGE * DIM)
            out[:, :, 1, vo.reshape(-1)] = codes[:, :, 1].reshape(full, -1, PAGE * DIM)
            pages[at], scales[at] = out, scale
        first = 0 if full else kept
        rest = seq[full * PAGE + first:]
        tail[b, :, :, first:first + rest.shape[0]] = rest.permute(1, 2, 0, 3)
    return {"pages": pages if form == "e4m3" else None, "scales": scales, "tail": tail.double()}


def _attention_exact(s):
    ko, vo = _page_offsets()
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    heads = s["pages"].shape[1]
    for b, n in enumerate(s["seq_lens"].tolist()):
        if not n:
            continue
        at = s["page_table"][b, :n // PAGE].long()
        codes = s["pages"].view(torch.int8)[at].view(s["pages"].dtype)
        codes = codes.float().double() * s["scales"][at].double()[..., None]
        k = codes[:, :, 0][..., ko.reshape(-1)].reshape(-1, heads, PAGE, DIM)
        v = codes[:, :, 1][..., vo.reshape(-1)].reshape(-1, heads, PAGE, DIM)
        rest = s["tail"][b, :, :, :n % PAGE].double()
        k = torch.cat([k.transpose(0, 1).reshape(heads, -1, DIM), rest[:, 0]], 1)
        v = torch.cat([v.transpose(0, 1).reshape(heads, -1, DIM), rest[:, 1]], 1)
        q = s["q"][b].double().reshape(heads, -1, DIM)
        p = torch.softmax(torch.einsum("hgd,htd->hgt", q, k) / math.sqrt(DIM), -1)
        out[b] = torch.einsum("hgt,htd->hgd", p, v).reshape(-1, DIM)
    return out


def _rows_exact(s):
    """By blocks of rows: (rows, log-softmax, token's value, entropy)."""
    step = max(1, 40_000_000 // s["logits"].shape[1])
    for i in range(0, s["logits"].shape[0], step):
        r = slice(i, i + step)
        logp = torch.log_softmax(s["logits"][r].double() / s["case"]["temperature"], 1)
        p = logp.exp()
        logp = torch.where(p == 0, 0.0, logp)
        token = s["tokens"][r].long()[:, None]
        yield r, p, logp, token, logp.gather(1, token)[:, 0], -(p * logp).sum(1)


def _grad_exact(p, logp, token, h, dlp, dh, temperature):
    hit = torch.zeros_like(p).scatter_(1, token, 1.0)
    return (dlp[:, None] * (hit - p) - dh[:, None] * p * (logp + h[:, None])) / temperature


def exact(case, seed):
    s, c = prepare(case, seed), case
    if c["op"] == "append":
        return _append_exact(s)
    if c["op"] == "attention":
        return _attention_exact(s)
    t, lps, hs, losses, grads, stats = c["temperature"], [], [], [], [], 0.0
    if c["op"] == "policy" and c["masked"]:
        s["logits"][s["weights"] == 0] = 0.0
    for r, p, logp, token, lp, h in _rows_exact(s):
        if c["op"] == "logprobs":
            if c["backward"]:
                grads.append(_grad_exact(p, logp, token, h, s["dlogprobs"][r].double(),
                                         s["dentropy"][r].double(), t))
            lps.append(lp)
            hs.append(h)
            continue
        w = s["weights"][r].double()
        a = s["advantages"].double()[s["row_seq"][r].long()]
        ratio = (lp - s["old"][r].double()).exp()
        free, held = ratio * a, ratio.clip(1 - CLIP, 1 + CLIP) * a
        cut = free > held
        policy, dlp = -torch.where(cut, held, free), torch.where(cut, 0.0, -free)
        kl = torch.zeros_like(lp)
        if c["kl"]:
            back = (s["ref"][r].double() - lp).exp()
            kl = back - (s["ref"][r].double() - lp) - 1
            dlp = dlp + c["kl"] * (1 - back)
        loss = policy + c["kl"] * kl - c["entropy"] * h
        on = (w != 0).double()
        stats = stats + (torch.stack([loss, policy, kl, h, cut.double()]) * w).sum(1)
        losses.append(loss * on)
        lps.append(lp * on)
        hs.append(h * on)
        grads.append(_grad_exact(p, logp, token, h, dlp * w, -c["entropy"] * w, t))
    if c["op"] == "logprobs":
        if c["backward"]:
            return torch.cat(grads)
        return {"logprobs": torch.cat(lps), "entropy": torch.cat(hs)}
    return {"stats": stats, "row_loss": torch.cat(losses), "logprobs": torch.cat(lps),
            "entropy": torch.cat(hs), "dlogits": torch.cat(grads)}
