"""Text generation at sizes where the work of a call is cut up: warps that go
through many steps and several sequences, blocks that take item after item,
more sequences and tiles than one pass of a kernel's bookkeeping holds.

The references are float64 on the GPU, by the definitions in
include/bark3_b200.h.  Tolerances are those of test_gpu_textgen.py: out moves by
half a unit of its type, by 2^-11 of sum p |v| (probabilities are f16) and
2^-24 of the largest value for each key (where they are subnormal), by 1e-5 for
f32 sums and 4e-6 of the scores' size for f32 scores; lse by 1e-5 of that size.
"""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from test_gpu_textgen import HALF_UNIT, check_pages, make_batch, normed, random_cache, rotate  # noqa: E402


def shared_batch(rng, page, past, new, pages):
    """Sequences that hold `past` tokens and receive `new`, over a pool of pages that they share."""
    kv = [a + b for a, b in zip(past, new)]
    width = max(1, max(-(-n // page) for n in kv))
    table = rng.integers(0, pages, (len(kv), width)).astype(np.int32)
    for i, n in enumerate(kv):
        table[i, -(-n // page):] = -1
    cu = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    dev = dict(cu_q=torch.from_numpy(cu).cuda(), kv_lens=torch.tensor(kv, dtype=torch.int32).cuda(),
               page_table=torch.from_numpy(table).cuda())
    return dev, cu, kv


def reference(cache, q, dev, cu, kv, scale, causal, window):
    """out, lse and the bound of out's error, float64 on the GPU."""
    heads, dim, page = cache.kv_heads, cache.head_dim, cache.page_tokens
    group = q.shape[1] // heads
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    bound = torch.zeros_like(out)
    lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device="cuda")
    size = torch.ones_like(lse)
    for i in range(len(kv)):
        n, length = int(cu[i + 1] - cu[i]), kv[i]
        if not n or not length:
            continue
        pages = dev["page_table"][i, :-(-length // page)].long()
        k, v = ((codes[pages].double() * s[pages].double()[..., None, None]).transpose(0, 1).reshape(heads, -1, dim)[:, :length]
                for codes, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)))
        x = q[cu[i]:cu[i + 1]].double().reshape(n, heads, group, dim).permute(1, 0, 2, 3).reshape(heads, n * group, dim)
        s = x @ k.transpose(1, 2) * scale
        largest = s.abs().amax(-1)
        if causal:
            pos = (length - n + torch.arange(n, device="cuda")).repeat_interleave(group)[:, None]
            key = torch.arange(length, device="cuda")[None]
            hidden = key > pos
            if window:
                hidden |= key <= pos - window
            s.masked_fill_(hidden, -math.inf)
        m = s.amax(-1, keepdim=True)
        p = torch.exp(s - torch.where(m > -math.inf, m, 0.0))
        seen = (s > -math.inf).sum(-1, keepdim=True)
        total = p.sum(-1, keepdim=True)
        live = total > 0
        inv = torch.where(live, 1 / total, 0.0)
        o = (p @ v) * inv
        a = (p @ v.abs()) * inv
        b = v.abs().amax(1, keepdim=True) * seen * inv
        sz = 1 + largest[..., None]
        e = HALF_UNIT[q.dtype] * o.abs() + (2.0 ** -11 + 1e-5 + 4e-6 * sz) * a + 2.0 ** -24 * b + 1e-30
        put = lambda t: t.reshape(heads, n, group, -1).permute(1, 0, 2, 3).reshape(n, heads * group, -1)
        rows = slice(int(cu[i]), int(cu[i + 1]))
        out[rows], bound[rows] = put(o), put(e)
        lse[rows] = put(torch.where(live, torch.where(m > -math.inf, m, 0.0) + total.log(), -math.inf))[..., 0]
        size[rows] = put(sz)[..., 0]
    return out, lse, bound, size


def check(cache, q, dev, cu, kv, max_q, scale, causal=True, window=0):
    out, lse = cache.attend(q, **dev, max_q=max_q, scale=scale, causal=causal, window=window, return_lse=True)
    cache.check()
    ref, ref_lse, bound, size = reference(cache, q, dev, cu, kv, scale, causal, window)
    worst = ((out.double() - ref).abs() / bound).max().item()
    assert worst <= 1, worst
    empty = ref_lse == -math.inf
    assert torch.equal(lse == -math.inf, empty) and not out[empty].any()
    assert ((lse.double() - ref_lse)[~empty].abs() <= 1e-5 * size[~empty]).all()
    return out, lse


def ragged(rng, n, lo, hi):
    return np.exp(rng.uniform(math.log(lo), math.log(hi + 1), n)).astype(int).tolist()


# dtype, q_heads, kv_heads, dim, page, sequences, longest, new tokens, causal, window
DECODE = [
    (torch.bfloat16, 32, 8, 128, 16, 128, 6000, [1], True, 0),
    (torch.float16, 8, 8, 128, 64, 128, 20000, [1], True, 0),
    (torch.bfloat16, 16, 8, 64, 128, 96, 60000, [1], True, 0),          # pages past the first 32 of a run
    (torch.float16, 16, 1, 128, 32, 300, 9000, [1], True, 0),           # 16 heads share a key head
    (torch.bfloat16, 16, 4, 64, 16, 150, 7000, [1, 4, 2, 0, 3], True, 0),
    (torch.float16, 8, 4, 128, 64, 200, 9000, [5, 1, 8], True, 700),
    (torch.bfloat16, 6, 2, 64, 32, 170, 9000, [2, 1], False, 0),
    (torch.float16, 3, 1, 64, 16, 1, 90000, [1], True, 0),
]


@pytest.mark.parametrize("case", DECODE)
def test_few_rows_in_long_runs(pkg, case):
    dtype, q_heads, kv_heads, dim, page, n, longest, pattern, causal, window = case
    rng = np.random.default_rng(longest + dim)
    new = [pattern[i % len(pattern)] for i in range(n)]
    past = ragged(rng, n, max(1, longest // 200), longest) if n > 1 else [longest]
    pages = 400
    dev, cu, kv = shared_batch(rng, page, past, new, pages)
    cache = random_cache(pkg, rng, pages, kv_heads, page, dim)
    q = torch.from_numpy(rng.normal(0, 1, (int(cu[-1]), q_heads, dim)).astype(np.float32)).to(dtype).cuda()
    check(cache, q, dev, cu, kv, max(new), 0.02, causal, window)


# dtype, q_heads, kv_heads, dim, page, sequences, past up to, new from, to, causal, window
PROMPTS = [
    (torch.bfloat16, 32, 8, 128, 64, 24, 3000, 1, 900, True, 0),
    (torch.float16, 12, 4, 64, 16, 60, 1500, 1, 700, True, 0),          # three heads a group: tokens split between tiles
    (torch.bfloat16, 8, 8, 128, 32, 40, 2000, 1, 400, True, 300),
    (torch.float16, 16, 8, 64, 128, 30, 2500, 20, 500, False, 0),
    (torch.bfloat16, 20, 1, 128, 16, 200, 4000, 1, 1, True, 0),         # one token, 20 rows a key head
    (torch.float16, 32, 8, 64, 64, 3, 16000, 300, 1900, True, 0),
    (torch.bfloat16, 14, 2, 128, 128, 50, 0, 1, 600, True, 0),
]


@pytest.mark.parametrize("case", PROMPTS)
def test_tiles_item_after_item(pkg, case):
    dtype, q_heads, kv_heads, dim, page, n, longest, lo, hi, causal, window = case
    rng = np.random.default_rng(longest + 7 * dim + n)
    new = ragged(rng, n, lo, hi)
    past = ragged(rng, n, max(1, longest // 100), longest) if longest else [0] * n
    pages = 300
    dev, cu, kv = shared_batch(rng, page, past, new, pages)
    cache = random_cache(pkg, rng, pages, kv_heads, page, dim)
    q = torch.from_numpy(rng.normal(0, 1, (int(cu[-1]), q_heads, dim)).astype(np.float32)).to(dtype).cuda()
    first = check(cache, q, dev, cu, kv, max(new), 0.02, causal, window)
    again = cache.attend(q, **dev, max_q=max(new), scale=0.02, causal=causal, window=window, return_lse=True)
    assert all(torch.equal(a, b) for a, b in zip(first, again))


@pytest.mark.parametrize("max_q,dim", [(2, 64), (2, 128), (24, 64), (24, 128)])
def test_attend_more_sequences_than_a_pass_holds(pkg, max_q, dim):
    """2,500 sequences: three launches of the kernel for few rows, three passes of the other one's plan."""
    rng = np.random.default_rng(max_q + dim)
    n = 2500
    new = rng.integers(0, max_q + 1, n).tolist()
    past = rng.integers(0, 90, n).tolist()
    new[0], past[5], new[5], new[-1] = 0, 0, 0, max_q
    dev, cu, kv = shared_batch(rng, 16, past, new, 200)
    cache = random_cache(pkg, rng, 200, 2, 16, dim)
    q = torch.from_numpy(rng.normal(0, 1, (int(cu[-1]), 6, dim)).astype(np.float32)).half().cuda()
    check(cache, q, dev, cu, kv, max_q, 0.02)


@pytest.mark.parametrize("n,most,page,dim", [(1100, 2, 16, 64), (1100, 30, 16, 128), (40, 200, 64, 128), (300, 9, 128, 64)])
def test_append_many_sequences(pkg, n, most, page, dim):
    """Ragged new tokens, none for some sequences, over more sequences than one round of a search."""
    rng = np.random.default_rng(n + most)
    new = rng.integers(0, most + 1, n).tolist()
    past = rng.integers(0, 2 * page + 3, n).tolist()
    new[0], new[n // 2], new[-1] = 0, most, 1
    dev, cu, kv, table, pages = make_batch(rng, page, past, new)
    cache = random_cache(pkg, rng, pages, 2, page, dim)
    cache.k_scale.fill_(2.0 ** -40), cache.v_scale.fill_(2.0 ** -40)
    tokens = int(cu[-1])
    qkv = torch.from_numpy(rng.normal(0, 2, (tokens, 8, dim)).astype(np.float32)).bfloat16().cuda()
    q, k, v = qkv.split([4, 2, 2], dim=1)
    wq, wk = (torch.from_numpy(rng.uniform(0.5, 1.5, dim).astype(np.float32)).cuda() for _ in range(2))
    angle = np.arange(max(kv))[:, None] * 10000.0 ** (-np.arange(0, dim, 2) / dim)
    cos, sin = (torch.from_numpy(f(angle).astype(np.float32)).cuda() for f in (np.cos, np.sin))
    got = cache.append(q, k, v, **dev, q_norm=wq, k_norm=wk, cos=cos, sin=sin)
    cache.check()
    pos = np.concatenate([np.arange(b, b + m) for b, m in zip(past, new)])
    turned = [rotate(normed(t.double().cpu().numpy(), w.double().cpu().numpy(), 1e-6), cos.double().cpu().numpy()[pos],
                     sin.double().cpu().numpy()[pos], False) for t, w in ((q, wq), (k, wk))]
    d = np.abs(got.double().cpu().numpy() - turned[0])
    assert (d <= 2.0 ** -8 * np.abs(turned[0]) + 2e-6 * (1 + np.abs(turned[0]).max())).all()
    check_pages(cache, "k", turned[1], cu, kv, table, past)
    check_pages(cache, "v", v.double().cpu().numpy(), cu, kv, table, past)
