"""The text-generation operators: what is measured, and their plain forms.

Three operators carry one token of a text decoder through the framework:

  append   norms of queries and keys for each head, the position rotation, and
           the new keys and values into a paged cache that holds 8 bits a value
           with a power-of-two scale for each page and head
  attend   attention of the rotated queries over that cache
  sample   the next token of every row by temperature, top-k, top-p and min-p
           from given random numbers

`run` computes them with elementary torch operations where `own` is false, and
through bark3_b200 where it is true.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
E4M3_MAX = 448.0
EXP_LO, EXP_HI = -40, 40     # exponents a page's scale may have
WEIGHT_ONE = 2.0 ** 31       # the largest weight of a sampled row, in whole numbers


# ─────────────────────────────── the cases ───────────────────────────────

def listed():
    return [
        # one live utterance takes one more token: everything is latency
        dict(name="append_one", op="append", dtype="f16", batch=1, q_heads=8, kv_heads=8, head_dim=128, page=64,
             past_min=379, past_max=379, q_min=1, q_max=1, norm=True, rot=128, interleaved=False),
        # one decode step of a full batch: 256 sequences of ragged lengths, shared key heads
        dict(name="append_step", op="append", dtype="bf16", batch=256, q_heads=32, kv_heads=8, head_dim=128, page=64,
             past_min=15, past_max=1879, q_min=1, q_max=1, norm=True, rot=128, interleaved=False),
        # the prompts of eight utterances (30 s to 150 s of frames) into an empty cache, straight from f32 projections
        dict(name="append_prompts", op="append", dtype="f32", batch=8, q_heads=12, kv_heads=4, head_dim=64, page=16,
             past_min=0, past_max=0, q_min=379, q_max=1879, norm=False, rot=64, interleaved=True),
        # a long prompt's chunk behind a part-filled page
        dict(name="append_chunk", op="append", dtype="bf16", batch=1, q_heads=32, kv_heads=8, head_dim=128, page=64,
             past_min=1001, past_max=1001, q_min=16384, q_max=16384, norm=True, rot=128, interleaved=False),
        # one utterance, one token over 30 s of frames
        dict(name="attend_one", op="attend", dtype="f16", batch=1, q_heads=8, kv_heads=8, head_dim=128, page=64,
             past_min=378, past_max=378, q_min=1, q_max=1, causal=True, window=0),
        # one decode step of a batch with lengths from a few tokens to ten minutes of frames
        dict(name="attend_step", op="attend", dtype="bf16", batch=128, q_heads=32, kv_heads=8, head_dim=128, page=64,
             past_min=15, past_max=7503, q_min=1, q_max=1, causal=True, window=0),
        # one very long sequence: the work has to be split along its length
        dict(name="attend_long", op="attend", dtype="bf16", batch=1, q_heads=32, kv_heads=8, head_dim=128, page=64,
             past_min=100002, past_max=100002, q_min=1, q_max=1, causal=True, window=0),
        # the prompts of eight utterances over themselves, small heads in groups of three, small pages
        dict(name="attend_prompts", op="attend", dtype="f16", batch=8, q_heads=12, kv_heads=4, head_dim=64, page=16,
             past_min=0, past_max=0, q_min=379, q_max=1879, causal=True, window=0),
        # a chunk of a long prompt over what is cached already: the arithmetic bounds it
        dict(name="attend_chunk", op="attend", dtype="bf16", batch=1, q_heads=32, kv_heads=8, head_dim=128, page=64,
             past_min=14336, past_max=14336, q_min=2048, q_max=2048, causal=True, window=0),
        # one row over the decoder's 8192 tokens and the blank
        dict(name="sample_one", op="sample", dtype="f32", rows=1, vocab=8193, mix="all"),
        # a batch's rows over the same vocabulary, every row with its own settings
        dict(name="sample_step", op="sample", dtype="f32", rows=256, vocab=8193, mix="all"),
        # a large vocabulary in 16 bits
        dict(name="sample_wide", op="sample", dtype="bf16", rows=256, vocab=131072, mix="all"),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "sample"])
    if op == "sample":
        vocab = _log_int(rng, 1025, 131072)
        rows = _log_int(rng, 1, 256)
        return dict(op=op, dtype=rng.choice(["f32", "f16", "bf16"]), rows=rows, vocab=vocab,
                    mix=rng.choice(["all", "plain", "top_k", "top_p", "min_p"]))
    head_dim = rng.choice([64, 128])
    group = rng.choice([1, 2, 3, 4, 5, 7, 8])
    kv_heads = rng.choice([1, 2, 3, 4, 8])
    case = dict(op=op, batch=_log_int(rng, 1, 128), q_heads=group * kv_heads, kv_heads=kv_heads, head_dim=head_dim,
                page=rng.choice([16, 32, 64, 128]))
    if op == "append":
        case["dtype"] = rng.choice(["f32", "f16", "bf16"])
        most = 16384 * 48 // ((group + 2) * kv_heads * case["batch"])
        q_max = 1 if rng.random() < 0.5 else _log_int(rng, 2, max(2, min(4096, most)))
        case.update(past_min=0, past_max=_log_int(rng, 1, 1879), q_min=1, q_max=q_max, norm=rng.random() < 0.5,
                    rot=rng.choice([0, 32, head_dim, head_dim]), interleaved=rng.random() < 0.5)
        return case
    case["dtype"] = rng.choice(["f16", "bf16"])
    case["causal"] = rng.random() < 0.75
    case["window"] = rng.choice([0, 0, 0, 100, 512]) if case["causal"] else 0
    if rng.random() < 0.5:      # decode: one or a few tokens a sequence
        past = _log_int(rng, 16, min(32768, 524288 // case["batch"]))
        case.update(past_min=rng.choice([0, past // 8]), past_max=past, q_min=1, q_max=rng.choice([1, 1, 1, 2, 4]))
    else:                       # prompts, alone or behind cached tokens
        q = _log_int(rng, 8, 2048)
        past = rng.choice([0, _log_int(rng, 1, 4096)])
        case["batch"] = max(1, min(case["batch"], 16, 2 ** 29 // (case["q_heads"] * q * (q + past))))
        case.update(past_min=past // 2, past_max=past, q_min=max(1, q // 4), q_max=q)
    return case


def _spread(lo, hi, n, turn):
    """n lengths over [lo, hi], even over the logarithm: the same ones for every seed."""
    out = []
    for i in range(n):
        f = math.modf((i + 0.5) * turn)[0] if n > 1 else 1.0
        out.append(min(hi, max(lo, int(round((lo + 1) * ((hi + 1) / (lo + 1)) ** f)) - 1)))
    return out


def _lengths(case):
    n = case["batch"]
    past = _spread(case["past_min"], case["past_max"], n, 0.6180339887)
    new = _spread(case["q_min"], case["q_max"], n, 0.7548776662)
    return past, new


# ──────────────────────────────── inputs ────────────────────────────────

def _rotation(positions, rot):
    """cos and sin of position * 10000^(-2 i / rot), as a model's table holds them."""
    freq = 10000.0 ** (-torch.arange(0, rot, 2, device="cuda", dtype=torch.float64) / rot)
    angle = torch.arange(positions, device="cuda", dtype=torch.float64)[:, None] * freq
    return angle.cos().float(), angle.sin().float()


def _features(g, shape):
    """Keys or values as a model makes them: some channels much larger than the rest."""
    x = torch.randn(shape, generator=g, device="cuda")
    gain = 0.5 + torch.rand(shape[-1], generator=g, device="cuda")
    gain[torch.randint(shape[-1], (max(1, shape[-1] // 32),), generator=g, device="cuda")] *= 8.0
    return x.mul_(gain)


def _cache(g, case, kv_lens):
    """A paged cache with every sequence's pages filled, in an order of its own, and its page table."""
    page, heads, dim = case["page"], case["kv_heads"], case["head_dim"]
    need = [(n + page - 1) // page for n in kv_lens]
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    width = max(need)
    first = torch.tensor([sum(need[:i]) for i in range(len(need))], device="cuda")[:, None]
    at = torch.arange(width, device="cuda")[None, :]
    held = at < torch.tensor(need, device="cuda")[:, None]
    table = torch.where(held, order[(first + at).clamp(max=pages - 1)], -1).to(torch.int32)
    pools = []
    for _ in range(2):
        x = _features(g, (pages, heads, page, dim))
        exp = _exponent(x.abs().amax(dim=(2, 3)))
        codes = (x * torch.exp2(-exp.float())[..., None, None]).clamp_(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
        pools.append((codes, torch.exp2(exp.float())))
        del x
    return pools, table


def _exponent(amax):
    """The least exponent e with amax <= 448 * 2^e, within what a page's scale may have."""
    frac, exp = torch.frexp(amax)
    exp = exp - 9 + (frac > 0.875).to(exp.dtype)
    return torch.where(amax > 0, exp.clamp(EXP_LO, EXP_HI), EXP_LO).to(torch.int32)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    if case["op"] == "sample":
        return _prepare_sample(case, g)
    past, new = _lengths(case)
    kv = [a + b for a, b in zip(past, new)]
    (k_pool, v_pool), table = _cache(g, case, kv)
    s = {"case": case, "table": table, "max_q": max(new), "max_kv": max(kv),
         "kv_lens": torch.tensor(kv, device="cuda", dtype=torch.int32),
         "cu_q": torch.tensor([sum(new[:i]) for i in range(len(new) + 1)], device="cuda", dtype=torch.int32),
         "k": k_pool[0], "k_scale": k_pool[1], "v": v_pool[0], "v_scale": v_pool[1]}
    tokens, dtype, dim = sum(new), DTYPES[case["dtype"]], case["head_dim"]
    if case["op"] == "append":
        # one projection's output: queries, keys and values side by side
        rows = _features(g, (tokens, case["q_heads"] + 2 * case["kv_heads"], dim)).to(dtype)
        s["new_q"], s["new_k"], s["new_v"] = rows.split([case["q_heads"], case["kv_heads"], case["kv_heads"]], dim=1)
        s["q_norm"] = s["k_norm"] = s["cos"] = s["sin"] = None
        if case["norm"]:
            s["q_norm"] = 0.5 + torch.rand(dim, generator=g, device="cuda")
            s["k_norm"] = 0.5 + torch.rand(dim, generator=g, device="cuda")
        if case["rot"]:
            s["cos"], s["sin"] = _rotation(max(kv), case["rot"])
    else:
        s["new_q"] = (torch.randn(tokens, case["q_heads"], dim, generator=g, device="cuda") * 1.5).to(dtype)
        s["scale"] = dim ** -0.5
        # what stands behind a sequence's end in its last page is no number
        page = case["page"]
        for pool in (s["k"], s["v"]):
            last = table.gather(1, ((s["kv_lens"] - 1) // page)[:, None].long())[:, 0].long()
            tail = torch.arange(page, device="cuda")[None, :] > ((s["kv_lens"] - 1) % page)[:, None]
            rows = pool.view(torch.uint8)[last]
            pool.view(torch.uint8)[last] = torch.where(tail[:, None, :, None], 0x7F, rows)
    if own:
        s["cache"] = _package().KvCache.over(s["k"], s["v"], s["k_scale"], s["v_scale"])
    return s


def _prepare_sample(case, g):
    rows, vocab, mix = case["rows"], case["vocab"], case["mix"]
    logits = torch.randn(rows, vocab, generator=g, device="cuda") * 1.5
    # a few dozen likely tokens in each row, as a trained model's head gives
    top = torch.randint(vocab, (rows, 48), generator=g, device="cuda")
    logits.scatter_reduce_(1, top, 8.0 + 2.5 * torch.randn(rows, 48, generator=g, device="cuda"), "amax")
    logits[:, vocab // 3] = -math.inf      # a token that may not be taken
    s = {"case": case, "logits": logits.to(DTYPES[case["dtype"]]),
         "uniform": torch.rand(rows, generator=g, device="cuda"),
         "temperature": None, "top_k": None, "top_p": None, "min_p": None}
    pick = torch.rand(4, rows, generator=g, device="cuda")
    if mix != "plain":
        s["temperature"] = torch.where(pick[0] < 0.125, 0.0, 0.5 + pick[0])
    if mix in ("all", "top_k"):
        s["top_k"] = torch.where(pick[1] < 0.3, 0, (1 + 80 * pick[1]).int()).to(torch.int32)
    if mix in ("all", "top_p"):
        s["top_p"] = torch.where(pick[2] < 0.3, 1.0, 0.5 + 0.49 * pick[2])
    if mix in ("all", "min_p"):
        s["min_p"] = torch.where(pick[3] < 0.5, 0.0, 0.1 * pick[3])
    return s


# ─────────────────────────────── the calls ───────────────────────────────

def _package():
    from __graft_entry__ import load_package

    return load_package()


def run(s):
    op = s["case"]["op"]
    if own:
        if op == "append":
            q = s["cache"].append(s["new_q"], s["new_k"], s["new_v"], s["cu_q"], s["kv_lens"], s["table"],
                                  q_norm=s["q_norm"], k_norm=s["k_norm"], eps=1e-6, cos=s["cos"], sin=s["sin"],
                                  interleaved=s["case"]["interleaved"])
            return {"q": q, "k": s["k"], "v": s["v"], "k_scale": s["k_scale"], "v_scale": s["v_scale"]}
        if op == "attend":
            out, lse = s["cache"].attend(s["new_q"], s["cu_q"], s["kv_lens"], s["table"], max_q=s["max_q"],
                                         scale=s["scale"], causal=s["case"]["causal"], window=s["case"]["window"],
                                         return_lse=True)
            return {"out": out, "lse": lse}
        ids, logprob = _package().sample(s["logits"], s["uniform"], temperature=s["temperature"], top_k=s["top_k"],
                                         top_p=s["top_p"], min_p=s["min_p"])
        return {"ids": ids, "logprob": logprob}
    return {"append": _append, "attend": _attend, "sample": _sample}[op](s)


# ────────────────────────────── plain: append ──────────────────────────────

def _rotate(x, cos, sin, interleaved):
    half = cos.shape[-1]
    rot, rest = x[..., : 2 * half], x[..., 2 * half:]
    a, b = (rot[..., 0::2], rot[..., 1::2]) if interleaved else (rot[..., :half], rot[..., half:])
    c, d = cos[:, None, :], sin[:, None, :]
    lo, hi = a * c - b * d, b * c + a * d
    rot = torch.stack([lo, hi], dim=-1).flatten(-2) if interleaved else torch.cat([lo, hi], dim=-1)
    return torch.cat([rot, rest], dim=-1)


def _append(s):
    case, page = s["case"], s["case"]["page"]
    tokens = s["new_q"].shape[0]
    # where each token goes
    at = torch.arange(tokens, device="cuda", dtype=torch.int32)
    seq = torch.searchsorted(s["cu_q"], at, right=True) - 1
    begin = s["kv_lens"] - (s["cu_q"][1:] - s["cu_q"][:-1])
    pos = (begin[seq] + at - s["cu_q"][seq]).long()
    to, slot = s["table"][seq, pos // page].long(), pos % page

    q, k, v = s["new_q"].float(), s["new_k"].float(), s["new_v"].float()
    if s["q_norm"] is not None:
        q = q * torch.rsqrt(q.square().mean(-1, keepdim=True) + 1e-6) * s["q_norm"]
        k = k * torch.rsqrt(k.square().mean(-1, keepdim=True) + 1e-6) * s["k_norm"]
    if s["cos"] is not None:
        cos, sin = s["cos"][pos], s["sin"][pos]
        q, k = _rotate(q, cos, sin, case["interleaved"]), _rotate(k, cos, sin, case["interleaved"])

    first, held = s["table"].gather(1, (begin // page)[:, None].long())[:, 0].long(), (begin % page)
    _into(s["k"], s["k_scale"], k, to, slot, first, held)
    _into(s["v"], s["v_scale"], v, to, slot, first, held)
    out = q.to(torch.float16 if s["new_q"].dtype == torch.float32 else s["new_q"].dtype)
    return {"q": out, "k": s["k"], "v": s["v"], "k_scale": s["k_scale"], "v_scale": s["v_scale"]}


def _into(pool, scale, x, to, slot, first, held):
    """Tokens x into the pages `to`; a page that held tokens keeps the larger scale, and those tokens follow it."""
    pages, heads, page, dim = pool.shape
    amax = torch.zeros(pages, heads, device="cuda")
    amax.scatter_reduce_(0, to[:, None].expand(-1, heads), x.abs().amax(-1), "amax")
    new = _exponent(amax)
    old = torch.frexp(scale[first])[1] - 1
    grown = torch.where((held > 0)[:, None], torch.maximum(new[first], old), new[first])
    new[first] = grown
    # tokens of the first page that were there before
    codes = pool[first].float() * torch.exp2((old - grown).float())[..., None, None]
    keep = (torch.arange(page, device="cuda")[None, :] < held[:, None])[:, None, :, None]
    raw = pool.view(torch.uint8)
    raw[first] = torch.where(keep, codes.to(torch.float8_e4m3fn).view(torch.uint8), raw[first])
    scale[to] = torch.exp2(new[to].float())
    codes = (x * torch.exp2(-new[to].float())[..., None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
    raw[to, :, slot] = codes.view(torch.uint8)


# ────────────────────────────── plain: attend ──────────────────────────────

def _attend(s):
    case, page = s["case"], s["case"]["page"]
    heads, dim, batch = case["kv_heads"], case["head_dim"], case["batch"]
    group = case["q_heads"] // heads
    length = s["table"].shape[1] * page
    table = s["table"].clamp(min=0).long()

    def dense(pool, scale):
        return (pool[table].float() * scale[table][..., None, None]).transpose(1, 2).reshape(batch, heads, length, dim)

    counts = s["cu_q"][1:] - s["cu_q"][:-1]
    at = torch.arange(s["max_q"], device="cuda")
    rows = (s["cu_q"][:-1, None] + at).clamp(max=s["new_q"].shape[0] - 1).long()
    q = s["new_q"][rows].float()                                             # [batch, max_q, q_heads, dim]
    q = q.reshape(batch, s["max_q"], heads, group, dim).permute(0, 2, 3, 1, 4).reshape(batch, heads, -1, dim)
    key = torch.arange(length, device="cuda")
    pos = (s["kv_lens"] - counts)[:, None] + at                              # of each query
    seen = (key < s["kv_lens"][:, None])[:, None, :].expand(-1, s["max_q"], -1)
    if case["causal"]:
        seen = seen & (key <= pos[..., None])
        if case["window"]:
            seen = seen & (key > pos[..., None] - case["window"])
    seen = seen[:, None, None]                                               # [batch, 1, 1, max_q, length]

    scores = (q @ dense(s["k"], s["k_scale"]).transpose(2, 3)).mul_(s["scale"])
    scores = scores.reshape(batch, heads, group, s["max_q"], length).masked_fill_(~seen, -math.inf)
    peak = scores.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    scores = scores.sub_(peak).exp_()
    total = scores.sum(-1, keepdim=True)
    held = (key < s["kv_lens"][:, None])[:, None, :, None]
    v = dense(s["v"], s["v_scale"]).masked_fill_(~held, 0.0)
    out = (scores.reshape(batch, heads, -1, length) @ v).reshape(batch, heads, group, s["max_q"], dim)
    out = torch.where(total > 0, out / total, 0.0)
    lse = (peak + total.log())[..., 0]
    # back to one row a token
    token = torch.arange(s["new_q"].shape[0], device="cuda", dtype=torch.int32)
    seq = torch.searchsorted(s["cu_q"], token, right=True) - 1
    at = (token - s["cu_q"][seq]).long()
    return {"out": out[seq, :, :, at].reshape(-1, case["q_heads"], dim).to(s["new_q"].dtype),
            "lse": lse[seq, :, :, at].reshape(-1, case["q_heads"])}


# ────────────────────────────── plain: sample ──────────────────────────────

def _sample(s):
    x = s["logits"].float()
    rows, vocab = x.shape
    temperature = s["temperature"] if s["temperature"] is not None else torch.ones(rows, device="cuda")
    peak = x.amax(-1, keepdim=True)
    best = (x == peak).int().argmax(-1)
    z = (x - peak) / torch.where(temperature > 0, temperature, 1.0)[:, None]
    w = z.exp()
    # weights are whole numbers of 2^-31 of the row's largest, so that a sum
    # does not depend on the order of its terms and a token is taken or not on
    # every machine alike
    whole = (w * WEIGHT_ONE).to(torch.int64)
    order = torch.sort(x, dim=-1, descending=True, stable=True).indices
    place = torch.arange(vocab, device="cuda")
    sorted_w = whole.gather(1, order)
    keep = torch.ones_like(sorted_w, dtype=torch.bool)
    if s["top_k"] is not None:
        keep = (place < s["top_k"][:, None]) | (s["top_k"] <= 0)[:, None]
    if s["top_p"] is not None:
        sorted_w = torch.where(keep, sorted_w, 0)
        total = sorted_w.sum(-1, keepdim=True)
        before = sorted_w.cumsum(-1) - sorted_w
        mass = s["top_p"].double()[:, None] * total.double()
        keep = keep & ((before < mass) | (place == 0) | (s["top_p"] >= 1)[:, None])
    keep = torch.zeros_like(keep).scatter_(1, order, keep)
    if s["min_p"] is not None:
        keep = keep & (w >= s["min_p"][:, None])
    whole = torch.where(keep, whole, 0)
    sums = whole.cumsum(-1)
    total = sums[:, -1:]
    mark = s["uniform"].double()[:, None] * total.double()
    ids = (sums.double() > mark).int().argmax(-1)
    logprob = z.gather(1, ids[:, None])[:, 0] - (total[:, 0].float() / WEIGHT_ONE).log()
    greedy = temperature <= 0
    return {"ids": torch.where(greedy, best, ids).to(torch.int32), "logprob": torch.where(greedy, 0.0, logprob)}


# ───────────────────────── the definition in 64 bits ─────────────────────────

def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "attend": _exact_attend, "sample": _exact_sample}[case["op"]](s)


def _exact_heads(x, norm, s, begin, case):
    x = x.double()
    if norm is not None:
        x = x / (x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + 1e-6).sqrt() * norm.double()
    if s["cos"] is not None:
        n, half = x.shape[0], case["rot"] // 2
        turn = torch.complex(s["cos"][begin:begin + n].double(), s["sin"][begin:begin + n].double())[:, None]
        part = x[..., : 2 * half]
        if case["interleaved"]:
            z = torch.view_as_complex(part.reshape(*part.shape[:-1], half, 2).contiguous()) * turn
            part = torch.view_as_real(z).flatten(-2)
        else:
            z = torch.complex(part[..., :half].contiguous(), part[..., half:].contiguous()) * turn
            part = torch.cat([z.real, z.imag], -1)
        x = torch.cat([part, x[..., 2 * half:]], -1)
    return x


def _exact_append(s):
    case, page = s["case"], s["case"]["page"]
    cu, kv, table = s["cu_q"].tolist(), s["kv_lens"].tolist(), s["table"].tolist()
    out_q = []
    pools = {n: (s[n].double(), s[n + "_scale"].double()) for n in ("k", "v")}
    for b in range(case["batch"]):
        lo, hi = cu[b], cu[b + 1]
        begin = kv[b] - (hi - lo)
        out_q.append(_exact_heads(s["new_q"][lo:hi], s["q_norm"], s, begin, case))
        new = {"k": _exact_heads(s["new_k"][lo:hi], s["k_norm"], s, begin, case), "v": s["new_v"][lo:hi].double()}
        for p in range(begin // page, (kv[b] - 1) // page + 1):
            a, z = max(begin, p * page), min(kv[b], (p + 1) * page)
            to, held = table[b][p], a - p * page
            for n, (codes, scale) in pools.items():
                x = new[n][a - begin:z - begin].transpose(0, 1)                # [heads, tokens, dim]
                step = torch.clamp(torch.ceil(torch.log2(x.abs().amax((1, 2)) / E4M3_MAX)), EXP_LO, EXP_HI).exp2()
                if held:
                    step = torch.maximum(step, scale[to])
                    old = codes[to, :, :held] * (scale[to] / step)[:, None, None]
                    codes[to, :, :held] = old.float().to(torch.float8_e4m3fn).double()
                scale[to] = step
                x = (x / step[:, None, None]).clamp(-E4M3_MAX, E4M3_MAX)
                codes[to, :, held:held + x.shape[1]] = x.float().to(torch.float8_e4m3fn).double()
    return {"q": torch.cat(out_q), "k": pools["k"][0], "v": pools["v"][0], "k_scale": pools["k"][1],
            "v_scale": pools["v"][1]}


def _exact_attend(s):
    case, page = s["case"], s["case"]["page"]
    heads, group = case["kv_heads"], case["q_heads"] // case["kv_heads"]
    cu, kv = s["cu_q"].tolist(), s["kv_lens"].tolist()
    out = torch.zeros(cu[-1], case["q_heads"], case["head_dim"], device="cuda", dtype=torch.float64)
    lse = torch.zeros(cu[-1], case["q_heads"], device="cuda", dtype=torch.float64)
    for b in range(case["batch"]):
        n, length = cu[b + 1] - cu[b], kv[b]
        pages = s["table"][b, : (length + page - 1) // page].long()
        at = length - n + torch.arange(n, device="cuda")[:, None]
        key = torch.arange(length, device="cuda")[None, :]
        hidden = torch.zeros(n, length, device="cuda", dtype=torch.bool)
        if case["causal"]:
            hidden = key > at
            if case["window"]:
                hidden = hidden | (key <= at - case["window"])
        for h in range(heads):
            k, v = ((s[m][pages, h].double() * s[m + "_scale"][pages, h].double()[:, None, None])
                    .flatten(0, 1)[:length] for m in ("k", "v"))
            for j in range(h * group, (h + 1) * group):
                x = s["new_q"][cu[b]:cu[b + 1], j].double() @ k.T * s["scale"]
                x.masked_fill_(hidden, -math.inf)
                lse[cu[b]:cu[b + 1], j] = torch.logsumexp(x, -1)
                out[cu[b]:cu[b + 1], j] = torch.nan_to_num(torch.softmax(x, -1)) @ v
    return {"out": out, "lse": lse}


def _exact_sample(s):
    logprob = []
    setting = {n: s[n].tolist() if s[n] is not None else None for n in ("temperature", "top_k", "top_p", "min_p")}
    for r, u in enumerate(s["uniform"].tolist()):
        value = {n: v[r] if v is not None else None for n, v in setting.items()}
        if value["temperature"] is not None and value["temperature"] <= 0:
            logprob.append(torch.zeros((), device="cuda", dtype=torch.float64))
            continue
        x = s["logits"][r].double()
        z = (x - x.max()) / (value["temperature"] or 1.0)
        z, index = torch.sort(z, descending=True, stable=True)
        if value["top_k"]:
            z, index = z[: value["top_k"]], index[: value["top_k"]]
        w = z.exp()
        if value["top_p"] is not None and value["top_p"] < 1:
            count = 1 + int((w.cumsum(0)[:-1] < value["top_p"] * w.sum()).sum())
            z, index, w = z[:count], index[:count], w[:count]
        if value["min_p"]:
            held = w >= value["min_p"]
            z, index, w = z[held], index[held], w[held]
        by_index = torch.argsort(index)
        z, sums = z[by_index], w[by_index].cumsum(0)
        logprob.append(z[int((sums <= u * sums[-1]).sum().clamp(max=z.numel() - 1))] - sums[-1].log())
    return {"ids": None, "logprob": torch.stack(logprob)}


# ──────────────────────── what a pass cannot do without ────────────────────────

def work(case):
    if case["op"] == "sample":
        size = 4 if case["dtype"] == "f32" else 2
        n = case["rows"] * case["vocab"]
        return {"bytes": n * size + case["rows"] * 28, "flops": 4 * n}
    past, new = _lengths(case)
    tokens, dim, heads, q_heads = sum(new), case["head_dim"], case["kv_heads"], case["q_heads"]
    size = 4 if case["dtype"] == "f32" else 2
    pages = sum((a + b - 1) // case["page"] - a // case["page"] + 1 for a, b in zip(past, new))
    if case["op"] == "append":
        read = tokens * (q_heads + 2 * heads) * dim * size + tokens * case["rot"] * 4
        written = tokens * q_heads * dim * 2 + 2 * tokens * heads * dim
        return {"bytes": read + written + 16 * pages * heads + 8 * case["batch"],
                "flops": 10 * tokens * (q_heads + 2 * heads) * dim}
    pairs = keys = 0
    for a, n in zip(past, new):
        reach = [min(a + i + 1, case["window"] or a + n) if case["causal"] else a + n for i in range(n)]
        pairs += sum(reach)
        keys += min(a + n, (n + reach[0] - 1) if case["window"] else a + n)
    read = tokens * q_heads * dim * 2 + 2 * keys * heads * dim + 8 * heads * (keys // case["page"] + case["batch"])
    return {"bytes": read + tokens * q_heads * (dim * 2 + 4), "flops": 4 * pairs * q_heads * dim}
