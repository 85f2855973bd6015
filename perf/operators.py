"""Cases of the decode-step operators: what they compute, in elementary torch operations, and the calls a user makes.

Four operators that follow one another in a decode step of the deterministic engine:

* ``qk_norm_rope``   per-head fixed-point RMSNorm of queries and keys with the rotary position in the same pass;
* ``rope_append``    rotary position (and optionally that norm) with the new keys and values written into the paged cache;
* ``prefix_attn``    paged attention of a batch whose requests share a long prefix;
* ``verify``         drafted tokens checked against the target's probabilities from given random numbers.

Fixed point: ``F2X(x) = rint(clamp(x * 2^f))``, integer sums, ``X2F(n) = n * 2^-f``. Every sum below stays far inside the
accumulator's range, so its wrap-around is never reached; an integer sum is taken in float64, where it is exact.
"""

import math
import sys

import torch

own = False

_DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_ES = {"bf16": 2, "fp16": 2, "fp32": 4}
RCP_LN2 = 1.4426950408889634


# ------------------------------------------------------------------------------------------------ cases
def _norm(name, tokens, heads, kv_heads, dim, rot, dtype, table, neox, bits, span):
    return {"name": name, "op": "qk_norm_rope", "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "dim": dim, "rot": rot,
            "dtype": dtype, "table": table, "neox": neox, "bits": bits, "span": span}


def _append(name, tokens, pad, heads, kv_heads, dim, rot, dtype, cache, page, table, neox, norm, bits, span):
    return {"name": name, "op": "rope_append", "tokens": tokens, "pad": pad, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "rot": rot, "dtype": dtype, "cache": cache, "page": page, "table": table, "neox": neox, "norm": norm, "bits": bits,
            "span": span}


def _prefix(name, requests, queries, prefix, suffix, heads, kv_heads, dim, dtype, page, bits, window, softcap, alibi):
    return {"name": name, "op": "prefix_attn", "requests": requests, "queries": queries, "prefix": prefix, "suffix": suffix,
            "heads": heads, "kv_heads": kv_heads, "dim": dim, "dtype": dtype, "page": page, "bits": bits, "window": window,
            "softcap": softcap, "alibi": alibi}


def _verify(name, requests, drafts, vocab, dtype, with_q, frac):
    return {"name": name, "op": "verify", "requests": requests, "drafts": drafts, "vocab": vocab, "dtype": dtype,
            "with_q": with_q, "frac": frac}


def listed():
    return [
        # one new token of one request: only latency counts
        _norm("norm_rope_one", 1, 32, 8, 128, 128, "bf16", "fp32", True, 32, 32768),
        # a ragged prefill chunk with half of each head rotated in interleaved pairs, 64-bit accumulators
        _norm("norm_rope_ragged", 509, 32, 8, 64, 32, "fp16", "fp32", False, 64, 8192),
        # a full prefill step
        _norm("norm_rope_prefill", 8192, 32, 8, 128, 128, "bf16", "bf16", True, 32, 8192),
        # a decode step of 64 requests
        _append("append_decode", 64, 0, 32, 8, 128, 128, "bf16", "bf16", 16, "bf16", True, False, 32, 8192),
        # a mixed step padded to its graph's size, keys normed on the way, another type in the cache
        _append("append_padded_norm", 777, 55, 32, 8, 64, 64, "bf16", "fp16", 16, "fp32", True, True, 32, 8192),
        # a full prefill step
        _append("append_prefill", 8192, 0, 32, 8, 128, 128, "bf16", "bf16", 16, "bf16", True, False, 32, 8192),
        # a few requests behind a short system prompt
        _prefix("prefix_few", 8, 1, 512, 64, 32, 8, 128, "bf16", 16, 32, 0, 0.0, False),
        # a decode batch behind a long system prompt
        _prefix("prefix_decode", 64, 1, 4096, 256, 32, 8, 128, "bf16", 16, 32, 0, 0.0, False),
        # drafted tokens verified (up to 5 queries a request) behind a long document, 64-bit accumulators
        _prefix("prefix_verify", 24, 5, 8191, 130, 32, 8, 64, "fp16", 16, 64, 0, 0.0, False),
        # one request, four drafted tokens
        _verify("verify_one", 1, 4, 128256, "fp32", True, 30),
        # up to eight tokens from an n-gram drafter (no draft probabilities), an odd vocabulary
        _verify("verify_ngram", 33, 8, 50257, "bf16", False, 24),
        # a full batch
        _verify("verify_batch", 128, 4, 128256, "fp32", True, 30),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    op = rng.choice(["qk_norm_rope", "rope_append", "prefix_attn", "verify"])
    if op in ("qk_norm_rope", "rope_append"):
        dim = rng.choice([64, 80, 96, 128, 128, 256])
        rot = rng.choice([dim, dim, dim // 2])
        kv_heads = rng.choice([1, 2, 4, 8])
        heads = kv_heads * rng.choice([1, 2, 4, 5, 8])
        most = max(1, min(8192, 8192 * 40 * 128 // ((heads + 2 * kv_heads) * dim)))
        tokens = _log(rng, 1, most)
        dtype = rng.choice(["bf16", "fp16"])
        table, neox, bits = rng.choice(["bf16", "fp32"]), rng.random() < 0.7, rng.choice([32, 64])
        if op == "qk_norm_rope":
            case = _norm("", tokens, heads, kv_heads, dim, rot, dtype, table, neox, bits, 32768)
        else:
            pad = rng.randrange(0, tokens) // 4
            case = _append("", tokens, pad, heads, kv_heads, dim, rot, dtype, rng.choice(["bf16", "fp16"]),
                           rng.choice([1, 16, 16, 24, 64]), table, neox, rng.random() < 0.5, bits, 32768)
    elif op == "prefix_attn":
        dim = rng.choice([64, 128])
        kv_heads = rng.choice([1, 2, 4, 8])
        heads = kv_heads * rng.choice([1, 2, 4, 4, 7, 8])
        queries = rng.choice([1, 1, 2, 5, 9])
        requests = _log(rng, 2, 96)
        most = 64 * 4096 * 32 * 128 // (requests * (queries + 1) // 2 * heads * dim)
        prefix = _log(rng, 33, max(40, min(12000, most)))
        suffix = _log(rng, queries, 512)
        case = _prefix("", requests, queries, prefix, suffix, heads, kv_heads, dim, rng.choice(["bf16", "fp16"]),
                       rng.choice([16, 16, 32, 24]), rng.choice([32, 64]), rng.choice([0, 0, 0, _log(rng, 16, 4096)]),
                       rng.choice([0.0, 0.0, 0.0, 30.0]), rng.random() < 0.2)
    else:
        requests = _log(rng, 1, 128)
        case = _verify("", requests, rng.randrange(1, 9), _log(rng, 1000, 151936 if requests < 100 else 120000),
                       rng.choice(["fp32", "fp32", "bf16"]), rng.random() < 0.6, rng.choice([24, 30]))
        case["drafts"] = max(1, min(case["drafts"], 128 * 4 // requests))
    del case["name"]
    return case


def _query_lens(case):
    """Queries of each request: from 1 to case["queries"]."""
    return [1 + (3 * r + case["queries"] - 1) % case["queries"] for r in range(case["requests"])]


def _suffix_lens(case):
    """Each request's own keys (its queries are the last of them): up to case["suffix"]."""
    return [max(n, 1 + (r * 7919 + case["suffix"] - 1) % case["suffix"]) for r, n in enumerate(_query_lens(case))]


def _draft_lens(case):
    return [(5 * r + case["drafts"]) % (case["drafts"] + 1) if case["requests"] > 1 else case["drafts"] for r in range(case["requests"])]


# ------------------------------------------------------------------------------------------------ inputs
def _table(case, dev):
    """cos and sin of every position, [span, rot]: the angles in float64."""
    half = case["rot"] // 2
    inv = 500000.0 ** (-torch.arange(half, dtype=torch.float64, device=dev) * 2 / case["rot"])
    ang = torch.arange(case["span"], dtype=torch.float64, device=dev)[:, None] * inv
    return torch.cat([ang.cos(), ang.sin()], -1).to(_DT[case["table"]])


def _qkv(case, g, dev):
    """Queries, keys and values as the fused projection leaves them: views into one matrix. Some heads run larger than others."""
    h, kh, d, t = case["heads"], case["kv_heads"], case["dim"], case["tokens"]
    x = torch.randn(t, h + 2 * kh, d, generator=g, device=dev) * (0.25 + 2 * torch.rand(1, h + 2 * kh, 1, generator=g, device=dev))
    x = x.to(_DT[case["dtype"]])
    return x[:, :h], x[:, h:h + kh], x[:, h + kh:]


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    s = {"case": case}
    if case["op"] in ("qk_norm_rope", "rope_append"):
        s["q"], s["k"], s["v"] = _qkv(case, g, dev)
        dt = _DT[case["dtype"]]
        s["qw"] = (1 + 0.2 * torch.randn(case["dim"], generator=g, device=dev)).to(dt)
        s["kw"] = (1 + 0.2 * torch.randn(case["dim"], generator=g, device=dev)).to(dt)
        s["positions"] = torch.randint(0, case["span"], (case["tokens"],), generator=g, device=dev)
        s["table"] = _table(case, dev)
        if case["op"] == "rope_append":
            used = case["tokens"] - case["pad"]
            blocks = (used + used // 4) // case["page"] + 2
            s["cache"] = torch.randn(blocks, 2, case["page"], case["kv_heads"], case["dim"], generator=g, device=dev).to(_DT[case["cache"]])
            s["slots"] = torch.randperm(blocks * case["page"], generator=g, device=dev)[:case["tokens"]]
            if s["slots"].numel() < case["tokens"]:
                s["slots"] = torch.cat([s["slots"], s["slots"].new_full((case["tokens"] - s["slots"].numel(),), -1)])
            s["slots"][used:] = -1
    elif case["op"] == "prefix_attn":
        ql, sl = _query_lens(case), _suffix_lens(case)
        page, pre, reqs = case["page"], case["prefix"], case["requests"]
        shared = pre // page  # whole pages in common; the rest of the prefix is a copy in each request's own page
        total = [pre + n for n in sl]
        cols = max(-(-n // page) for n in total)
        blocks = shared + reqs * (cols - shared) + 3
        perm = torch.randperm(blocks, generator=g, device=dev).to(torch.int32)
        bt = torch.empty(reqs, cols, dtype=torch.int32, device=dev)
        bt[:, :shared] = perm[:shared]
        bt[:, shared:] = perm[shared:shared + reqs * (cols - shared)].view(reqs, cols - shared)
        dt = _DT[case["dtype"]]
        kv = torch.randn(blocks, 2, page, case["kv_heads"], case["dim"], generator=g, device=dev).to(dt)
        if pre % page:
            kv[bt[1:, shared].long(), :, :pre % page] = kv[bt[0, shared].long(), :, :pre % page]
        s["kv"], s["bt"] = kv, bt
        s["q"] = (1.5 * torch.randn(sum(ql), case["heads"], case["dim"], generator=g, device=dev)).to(dt)
        s["o"] = torch.empty_like(s["q"])
        s["qsl"] = torch.tensor([0] + [sum(ql[:i + 1]) for i in range(reqs)], dtype=torch.int32, device=dev)
        s["seq"] = torch.tensor(total, dtype=torch.int32, device=dev)
        s["req"] = torch.tensor([r for r, n in enumerate(ql) for _ in range(n)], device=dev)
        s["pos"] = torch.tensor([total[r] - n + i for r, n in enumerate(ql) for i in range(n)], device=dev)
        s["max_q"], s["max_seq"] = max(ql), max(total)
        s["slopes"] = None
        if case["alibi"]:  # per-head slopes, scaled by 1/ln 2 as the attention operators take them
            s["slopes"] = (2.0 ** (-8.0 * torch.arange(1, case["heads"] + 1, device=dev) / case["heads"]) * RCP_LN2).float()
    else:
        n, lens, vocab, reqs = sum(_draft_lens(case)), _draft_lens(case), case["vocab"], case["requests"]
        dt = _DT[case["dtype"]]
        logits = 2.5 * torch.randn(n, vocab, generator=g, device=dev)
        s["p"] = torch.softmax(logits, -1).to(dt)
        if case["with_q"]:  # the drafter: close to the target, its tokens drawn from its own distribution
            s["q"] = torch.softmax(logits + 0.6 * torch.randn(n, vocab, generator=g, device=dev), -1).to(dt)
            race = s["q"].float() / torch.empty(n, vocab, device=dev).exponential_(generator=g)
            s["drafts"] = race.argmax(-1).to(torch.int32) if n else torch.empty(0, dtype=torch.int32, device=dev)
        else:  # a token that the target finds likely, half the time its likeliest
            s["q"] = None
            s["drafts"] = torch.randint(0, vocab, (n,), generator=g, device=dev).to(torch.int32)
            if n:
                top = s["p"].float().argmax(-1).to(torch.int32)
                s["p"][torch.arange(n, device=dev), top.long()] += 0.6
                s["drafts"] = torch.where(torch.rand(n, generator=g, device=dev) < 0.8, top, s["drafts"])
        s["start"] = torch.tensor([sum(lens[:i]) for i in range(reqs + 1)], dtype=torch.int32, device=dev)
        s["bonus"] = torch.randint(0, vocab, (reqs,), generator=g, device=dev).to(torch.int32)
        s["u"] = torch.rand(n, generator=g, device=dev)
        s["r"] = torch.rand(reqs, generator=g, device=dev)
    return s


# ------------------------------------------------------------------------------------------------ plain forms
def _f2x(x, frac, bits):
    """Scaled, clamped and rounded, as whole numbers in x's own type."""
    top = 2.0 ** 31 - 2.0 ** 8 if bits == 32 else 2.0 ** 63 - 2.0 ** 40
    return torch.round((x * 2.0 ** frac).clamp_(-2.0 ** (bits - 1), top))


def _rms(x, w, bits, eps=1e-6, frac=16):
    """x [.., dim] in 32 bits, normed over its last dim."""
    mean = _f2x(x * x, frac, bits).sum(-1, keepdim=True, dtype=torch.float64).float() * 2.0 ** -frac / x.shape[-1]
    return (x * w.float()) * torch.rsqrt(mean.clamp_min(0) + eps)


def _rope(x, positions, table, rot, neox):
    """x [tokens, heads, dim] in 32 bits: the first `rot` dims turned by their position's angles."""
    cs = table[positions].float()[:, None]
    c, s = cs[..., :rot // 2], cs[..., rot // 2:]
    if neox:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        turned = torch.cat([a * c - b * s, b * c + a * s], -1)
    else:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        turned = torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2)
    return torch.cat([turned, x[..., rot:]], -1)


def _plain_norm_rope(s, case):
    out = []
    for x, w in ((s["q"], s["qw"]), (s["k"], s["kw"])):
        y = _rms(x.float(), w, case["bits"])
        out.append(_rope(y, s["positions"], s["table"], case["rot"], case["neox"]).to(x.dtype))
    return out


def _plain_append(s, case):
    q, k = s["q"].float(), s["k"].float()
    if case["norm"]:
        q, k = _rms(q, s["qw"], case["bits"]), _rms(k, s["kw"], case["bits"])
    q = _rope(q, s["positions"], s["table"], case["rot"], case["neox"])
    k = _rope(k, s["positions"], s["table"], case["rot"], case["neox"])
    n = case["tokens"] - case["pad"]
    block, off = s["slots"][:n] // case["page"], s["slots"][:n] % case["page"]
    s["cache"][block, 0, off] = k[:n].to(s["cache"].dtype)
    s["cache"][block, 1, off] = s["v"][:n].to(s["cache"].dtype)
    return [q.to(s["q"].dtype), s["cache"]]


def _plain_prefix(s, case, frac=16):
    d, kh, page, pre = case["dim"], case["kv_heads"], case["page"], case["prefix"]
    grp, bits, tokens = case["heads"] // kh, case["bits"], s["q"].shape[0]
    q = s["q"].float().view(tokens, kh, grp, 1, d)
    j = torch.arange(s["max_seq"], device=q.device)
    # the prefix from the first request's pages, once for all; then each request's own keys, padded to the longest
    kv = s["kv"][s["bt"][0, j[:pre] // page].long(), :, j[:pre] % page]
    own_kv = s["kv"][s["bt"][:, j[pre:] // page].long(), :, j[pre:] % page][s["req"]]
    limit = s["seq"][s["req"]][:, None]
    pos = s["pos"][:, None]
    seen = (j < limit) & (j <= pos)
    if case["window"]:
        seen &= j > pos - case["window"]

    def dots(keys):
        return _f2x(q * keys, frac, bits).sum(-1, dtype=torch.float64)

    score = torch.cat([dots(kv[:, 0].float().transpose(0, 1)[None, :, None]),
                       dots(own_kv[:, :, 0].float().transpose(1, 2)[:, :, None])], -1)
    score = score.float() * 2.0 ** -frac * torch.tensor(RCP_LN2 / math.sqrt(d), device=q.device)
    if case["softcap"]:
        score = case["softcap"] * RCP_LN2 * torch.tanh(score / (case["softcap"] * RCP_LN2))
    if case["alibi"]:
        score = score + s["slopes"].view(1, kh, grp, 1) * (j - pos).float()[:, None, None]
    score = score.masked_fill(~seen[:, None, None], -math.inf)
    p = torch.exp2(score - score.amax(-1, keepdim=True))
    den = _f2x(p, frac, bits).sum(-1, dtype=torch.float64)

    def sums(w, values):
        return _f2x(w[..., None] * values.half().float(), frac, bits).sum(-2, dtype=torch.float64)

    acc = sums(p[..., :pre], kv[:, 1].transpose(0, 1)[None, :, None])
    acc += sums(p[..., pre:], own_kv[:, :, 1].transpose(1, 2)[:, :, None])
    out = acc.float() / den.float()[..., None].clamp_min(1e-6 * 2.0 ** frac)
    s["o"].copy_(out.reshape(s["o"].shape))
    return s["o"]


def _plain_verify(s, case):
    f, reqs, most = case["frac"], case["requests"], case["drafts"]
    one = 1 << f
    whole = lambda x: torch.round(x.float().clamp(0, 1) * 2.0 ** f).to(torch.int64)  # noqa: E731
    start = s["start"].long()
    length = start[1:] - start[:-1]
    at = start[:-1, None] + torch.arange(most, device=start.device)
    row = at.clamp_max(max(0, s["drafts"].numel() - 1))
    i = torch.arange(most, device=start.device)
    out = torch.full((reqs, most + 1), -1, dtype=torch.int32, device=start.device)
    if s["drafts"].numel():
        tok = s["drafts"].long()[row]
        p = whole(s["p"][row, tok])
        q = whole(s["q"][row, tok]) if case["with_q"] else torch.full_like(p, one)
        u = torch.floor(s["u"][row].double() * 2 ** 24).to(torch.int64)
        ok = (u * q < (p << 24)) & (i < length[:, None])
        taken = ok.long().cumprod(-1).sum(-1)
        last = row.gather(1, taken.clamp_max(most - 1)[:, None])[:, 0]
        w = whole(s["p"][last])
        if case["with_q"]:
            left = (w - whole(s["q"][last])).clamp_min(0)
        else:
            left = w.scatter(1, s["drafts"].long()[last][:, None], 0)
        left = torch.where(left.sum(-1, keepdim=True) > 0, left, w)
        cum = left.cumsum(-1)
        all_ = cum[:, -1]
        r = torch.floor(s["r"].double() * 2 ** 24).to(torch.int64)
        at_ = (all_ >> 24) * r + (((all_ & 0xFFFFFF) * r) >> 24)
        drawn = torch.where(all_ > 0, (cum <= at_[:, None]).sum(-1), -1)
        out[:, :most] = torch.where(i < taken[:, None], tok, -1).int()
        final = torch.where(taken < length, drawn, s["bonus"].long())
    else:
        taken, final = length, s["bonus"].long()
    out.scatter_(1, taken[:, None], final[:, None].int())
    return [out, taken.int()]


# ------------------------------------------------------------------------------------------------ the passes
def _ops():
    if "fixed-point-reductions-for-vllm_b200" not in sys.path:
        sys.path.insert(0, "fixed-point-reductions-for-vllm_b200")
    import fxpr_vllm.library_ops  # noqa: F401

    return torch.ops.fxpr


def run(state):
    s, case = state, state["case"]
    if case["op"] == "qk_norm_rope":
        if own:
            return list(_ops().qk_norm_rope_fxp(s["q"], s["k"], s["qw"], s["kw"], s["positions"], s["table"], case["neox"], 1e-6,
                                                16, case["bits"]))
        return _plain_norm_rope(s, case)
    if case["op"] == "rope_append":
        if own:
            w = (s["qw"], s["kw"]) if case["norm"] else (None, None)
            q = _ops().rope_append_kv_fxp(s["q"], s["k"], s["v"], s["cache"], s["slots"], s["positions"], s["table"], case["neox"],
                                          *w, 1e-6, 16, case["bits"])
            return [q, s["cache"]]
        return _plain_append(s, case)
    if case["op"] == "prefix_attn":
        if own:
            _ops().shared_prefix_attention_fxp(s["q"], s["kv"], s["o"], s["qsl"], s["seq"], s["bt"], case["prefix"], s["max_q"],
                                               s["slopes"], case["bits"], True, None, 16, case["softcap"], case["window"],
                                               s["max_seq"])
            return s["o"]
        return _plain_prefix(s, case)
    if own:
        return list(_ops().verify_draft_fxp(s["p"], s["q"], s["drafts"], s["start"], s["bonus"], s["u"], s["r"], case["drafts"],
                                            case["frac"]))
    return _plain_verify(s, case)


def work(case):
    if case["op"] in ("qk_norm_rope", "rope_append"):
        t, d, es = case["tokens"], case["dim"], _ES[case["dtype"]]
        table = min(t, case["span"]) * case["rot"] * _ES[case["table"]] + 8 * t
        q, k = t * case["heads"] * d, t * case["kv_heads"] * d
        if case["op"] == "qk_norm_rope":
            return {"bytes": 2 * (q + k) * es + table, "flops": 6 * (q + k)}
        new = k * (t - case["pad"]) // t
        return {"bytes": 2 * q * es + 2 * new * (es + _ES[case["cache"]]) + table + 8 * t, "flops": (6 if case["norm"] else 3) * (q + k)}
    if case["op"] == "prefix_attn":
        ql, sl, d, es = _query_lens(case), _suffix_lens(case), case["dim"], _ES[case["dtype"]]
        keys = case["prefix"] + sum(sl)
        pairs = case["heads"] * sum(n * (case["prefix"] + m) for n, m in zip(ql, sl))
        return {"bytes": 2 * keys * case["kv_heads"] * d * es + 2 * sum(ql) * case["heads"] * d * es, "flops": 4 * pairs * d}
    lens, v, es = _draft_lens(case), case["vocab"], _ES[case["dtype"]]
    # about three drafted tokens in four are taken; a request whose drafts are not all taken has its row(s) read
    rows = sum(1 - 0.75 ** n for n in lens) * (2 if case["with_q"] else 1)
    return {"bytes": rows * v * es + 16 * sum(lens) + 4 * len(lens) * (case["drafts"] + 4), "flops": 3 * rows * v}


# ------------------------------------------------------------------------------------------------ the same in 64 bits
def _exact_head(x, w, cs, rot, neox, norm, bits, eps=1e-6):
    x = x.double()
    if norm:
        top = 2 ** 31 - 2 ** 8 if bits == 32 else 2 ** 62
        n = torch.minimum((x.square() * 65536).round(), torch.tensor(float(top), dtype=torch.float64, device=x.device)).sum(-1, keepdim=True)
        x = x * w.double() / torch.sqrt(n / 65536 / x.shape[-1] + eps)
    y = x.clone()
    half = rot // 2
    first = torch.arange(half, device=x.device) if neox else torch.arange(0, rot, 2, device=x.device)
    second = first + (half if neox else 1)
    z = torch.complex(x[..., first], x[..., second]) * torch.complex(cs[:, None, :half], cs[:, None, half:])
    y[..., first], y[..., second] = z.real, z.imag
    return y


def _exact_prefix(s, case):
    d, page, grp = case["dim"], case["page"], case["heads"] // case["kv_heads"]
    one = 65536.0
    out = torch.empty(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    starts, totals = s["qsl"].tolist(), s["seq"].tolist()
    for r, total in enumerate(totals):
        ids = s["bt"][r, :-(-total // page)].long()
        k = s["kv"][ids, 0].reshape(-1, case["kv_heads"], d)[:total].double()
        v = s["kv"][ids, 1].reshape(-1, case["kv_heads"], d)[:total].half().double()
        where = torch.arange(total, device=k.device)
        for t in range(starts[r], starts[r + 1]):
            at = total - starts[r + 1] + t
            mask = where > at
            if case["window"]:
                mask |= where <= at - case["window"]
            for h in range(case["kv_heads"]):
                x = s["q"][t, h * grp:(h + 1) * grp].double()
                z = (x[:, None] * k[None, :, h] * one).round().sum(-1) / one / math.sqrt(d)
                if case["softcap"]:
                    z = case["softcap"] * torch.tanh(z / case["softcap"])
                z = z * RCP_LN2
                if case["alibi"]:
                    z = z + s["slopes"][h * grp:(h + 1) * grp, None].double() * (where - at)
                z[:, mask] = -math.inf
                w = 2.0 ** (z - z.max(-1, keepdim=True).values)
                den = (w * one).round().sum(-1, keepdim=True)
                out[t, h * grp:(h + 1) * grp] = (w[..., None] * v[None, :, h] * one).round().sum(1) / den
    return out


def _exact_verify(s, case):
    scale = float(2 ** case["frac"])
    starts, drafts = s["start"].tolist(), s["drafts"].tolist()
    u, r, bonus = s["u"].double().tolist(), s["r"].double().tolist(), s["bonus"].tolist()
    reqs = case["requests"]
    tokens = torch.full((reqs, case["drafts"] + 1), -1, dtype=torch.int32)
    taken = torch.zeros(reqs, dtype=torch.int32)
    for n in range(reqs):
        a, b = starts[n], starts[n + 1]
        last = bonus[n]
        for i in range(a, b):
            p = s["p"][i].double()
            q = s["q"][i].double() if case["with_q"] else torch.nn.functional.one_hot(s["drafts"][i].long(), case["vocab"]).double()
            p, q = (p.clamp(0, 1) * scale).round().long(), (q * scale).round().long()
            if int(u[i] * 2 ** 24) * int(q[drafts[i]]) < int(p[drafts[i]]) * 2 ** 24:
                tokens[n, i - a] = drafts[i]
                taken[n] += 1
                continue
            left = (p - q).clamp_min(0)
            left = left if int(left.sum()) else p
            goal = int(left.sum()) * int(r[n] * 2 ** 24) // 2 ** 24
            last = int(torch.searchsorted(left.cumsum(0), torch.tensor(goal, device=left.device), right=True))
            break
        tokens[n, int(taken[n])] = last
    return [tokens, taken]


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "prefix_attn":
        return _exact_prefix(s, case) if s["q"].shape[0] * case["kv_heads"] < 6000 else None
    if case["op"] == "verify":
        return _exact_verify(s, case)
    cs = s["table"][s["positions"]].double()
    norm = case["op"] == "qk_norm_rope" or case["norm"]
    q = _exact_head(s["q"], s["qw"], cs, case["rot"], case["neox"], norm, case["bits"])
    k = _exact_head(s["k"], s["kw"], cs, case["rot"], case["neox"], norm, case["bits"])
    if case["op"] == "qk_norm_rope":
        return [q, k]
    cache = s["cache"].double()
    n = case["tokens"] - case["pad"]
    block, off = s["slots"][:n] // case["page"], s["slots"][:n] % case["page"]
    cache[block, 0, off], cache[block, 1, off] = k[:n], s["v"][:n].double()
    return [q, cache]
