"""Text generation on the GPU (bark3_b200.KvCache, bark3_b200.sample) against
plain float64 restatements of the definitions in include/bark3_b200.h.

Tolerances, from the arithmetic:
  q_out   f32 arithmetic (about 20 operations: 2e-6 relative), then one
          rounding to 16 bits: half a unit, 2^-11 (f16, 11 significant
          bits) or 2^-8 (bf16, 8 of them)
  codes   e4m3 keeps 4 significant bits: half a unit is at most 2^-4 of the
          value, or half a subnormal step, 2^-10 scales; a second rounding
          (a page's scale grew) can only add as much again below the normal
          range, where a step is a step of the larger scale
  out     every probability is rounded to f16 (2^-11 of itself, or 2^-25 of the
          largest where it is subnormal), sums are f32 (1e-5 is generous for a
          few thousand terms), then one rounding to 16 bits
  lse     f32: 1e-5 relative to the scores' magnitudes
"""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

HALF_UNIT = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def make_batch(rng, page, past, new, extra_pages=2, width=None):
    """Page table of sequences that hold `past` tokens and receive `new`; entries past the end are -1."""
    kv = [a + b for a, b in zip(past, new)]
    need = [-(-n // page) for n in kv]
    pages = sum(need) + extra_pages
    order = rng.permutation(pages).astype(np.int32)
    table = np.full((len(kv), width or max(max(need), 1)), -1, np.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    cu = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    dev = dict(cu_q=torch.from_numpy(cu).cuda(), kv_lens=torch.tensor(kv, dtype=torch.int32).cuda(),
               page_table=torch.from_numpy(table).cuda())
    return dev, cu, kv, table, pages


def e4m3_exponent(amax):
    if amax == 0:
        return -40
    return int(min(max(math.ceil(math.log2(amax / 448.0)), -40), 40))


def rotate(x, cos, sin, interleaved):
    """x (tokens, heads, dim) f64, cos / sin (tokens, rot / 2)."""
    half = cos.shape[1]
    y = x.copy()
    a, b = (x[..., 0:2 * half:2], x[..., 1:2 * half:2]) if interleaved else (x[..., :half], x[..., half:2 * half])
    c, s = cos[:, None], sin[:, None]
    lo, hi = a * c - b * s, b * c + a * s
    if interleaved:
        y[..., 0:2 * half:2], y[..., 1:2 * half:2] = lo, hi
    else:
        y[..., :half], y[..., half:2 * half] = lo, hi
    return y


def normed(x, w, eps):
    return x / np.sqrt((x ** 2).mean(-1, keepdims=True) + eps) * w


def dequantised(cache, which):
    codes, scale = (cache.k, cache.k_scale) if which == "k" else (cache.v, cache.v_scale)
    return (codes.float() * scale[..., None, None]).cpu().numpy().astype(np.float64)


def random_cache(pkg, rng, pages, heads, page, dim, spread=4.0):
    """A full cache of random codes and scales 2^-spread .. 2^spread times 2^-8."""
    c = pkg.KvCache(pages, heads, dim, page)
    g = torch.Generator(device="cuda").manual_seed(int(rng.integers(1 << 30)))
    for pool, scale in ((c.k, c.k_scale), (c.v, c.v_scale)):
        x = (torch.randn(pool.shape, generator=g, device="cuda") * 120).clamp(-448, 448)
        pool.copy_(x.to(torch.float8_e4m3fn))
        scale.copy_(torch.exp2(torch.randint(int(-8 - spread), int(-8 + spread) + 1, scale.shape, generator=g,
                                             device="cuda").float()))
    return c


# ─────────────────────────────── append ───────────────────────────────

def check_pages(cache, which, want, cu, kv, table, begin):
    """want (tokens, heads, dim) f64 is what the new tokens of the sequences should hold; the codes of a fresh page."""
    page = cache.page_tokens
    codes, scale = (cache.k, cache.k_scale) if which == "k" else (cache.v, cache.v_scale)
    got, scale = dequantised(cache, which), scale.cpu().numpy()
    for i in range(len(kv)):
        for p in range(begin[i] // page, -(-kv[i] // page)):
            lo, hi = max(begin[i], p * page), min(kv[i], (p + 1) * page)
            if lo >= hi:
                continue
            x = want[cu[i] + lo - begin[i]:cu[i] + hi - begin[i]]               # tokens, heads, dim
            for h in range(cache.kv_heads):
                v = x[:, h]
                if lo % page == 0:
                    finite = np.abs(v)[np.isfinite(v)]
                    assert scale[table[i, p], h] == 2.0 ** e4m3_exponent(finite.max() if finite.size else 0.0)
                s = float(scale[table[i, p], h])
                stored = got[table[i, p], h, lo % page:lo % page + hi - lo]
                clipped = np.clip(v, -448 * s, 448 * s)
                bound = 2.0 ** -4 * np.abs(clipped) + s * 2.0 ** -10 + 1e-5 * np.abs(clipped).max(initial=0.0)
                assert (np.abs(stored - clipped) <= bound).all(), (which, i, p, h)


APPEND_CASES = [
    # dtype, q_heads, kv_heads, dim, page, past, new, rot, interleaved, norm
    (torch.float16, 8, 8, 128, 64, [0], [1], 128, False, True),
    (torch.bfloat16, 8, 2, 128, 64, [63, 64, 0, 5], [1, 1, 1, 1], 128, False, True),
    (torch.float32, 12, 4, 64, 16, [0, 3, 16], [37, 0, 130], 64, True, False),
    (torch.bfloat16, 4, 4, 64, 32, [1, 31, 32, 90], [3, 70, 1, 0], 32, False, True),
    (torch.float16, 7, 1, 128, 128, [100], [300], 48, True, True),
    (torch.float32, 6, 2, 128, 16, [7, 0], [1, 200], 0, False, True),
    (torch.float16, 40, 8, 128, 32, list(range(33)), [1] * 33, 128, False, False),
    (torch.bfloat16, 5, 5, 64, 128, [0, 0], [1, 513], 64, False, False),
]


@pytest.mark.parametrize("case", APPEND_CASES)
def test_append_matches_float64(pkg, case):
    dtype, q_heads, kv_heads, dim, page, past, new, rot, interleaved, norm = case
    rng = np.random.default_rng(q_heads * 1000 + dim + page)
    dev, cu, kv, table, pages = make_batch(rng, page, past, new)
    cache = random_cache(pkg, rng, pages, kv_heads, page, dim)
    cache.k_scale.fill_(2.0 ** -40), cache.v_scale.fill_(2.0 ** -40)   # what pages held before is far below the new
    tokens = int(cu[-1])
    qkv = torch.from_numpy(rng.normal(0, 2, (tokens, q_heads + 2 * kv_heads, dim)).astype(np.float32)).to(dtype).cuda()
    q, k, v = qkv.split([q_heads, kv_heads, kv_heads], dim=1)
    wq, wk = (torch.from_numpy(rng.uniform(0.5, 1.5, dim).astype(np.float32)).cuda() for _ in range(2))
    cos = sin = None
    if rot:
        angle = np.arange(max(kv))[:, None] * 10000.0 ** (-np.arange(0, rot, 2) / rot)
        cos, sin = (torch.from_numpy(f(angle).astype(np.float32)).cuda() for f in (np.cos, np.sin))
    before = qkv.clone()
    got = cache.append(q, k, v, **dev, q_norm=wq if norm else None, k_norm=wk if norm else None, eps=1e-5, cos=cos,
                       sin=sin, interleaved=interleaved)
    cache.check()
    assert torch.equal(qkv.view(torch.uint8), before.view(torch.uint8))
    begin = [a for a in past]
    pos = np.concatenate([np.arange(b, b + n) for b, n in zip(begin, new)])
    ref = {}
    for name, t, w in (("q", q, wq), ("k", k, wk)):
        x = t.double().cpu().numpy()
        if norm:
            x = normed(x, w.double().cpu().numpy(), 1e-5)
        if rot:
            x = rotate(x, cos.double().cpu().numpy()[pos], sin.double().cpu().numpy()[pos], interleaved)
        ref[name] = x
    out_dtype = torch.float16 if dtype is torch.float32 else dtype
    assert got.dtype is out_dtype and got.shape == q.shape
    d = np.abs(got.double().cpu().numpy() - ref["q"])
    size = np.abs(ref["q"])
    assert (d <= HALF_UNIT[out_dtype] * size + 2e-6 * (1 + size.max())).all()
    check_pages(cache, "k", ref["k"], cu, kv, table, begin)
    check_pages(cache, "v", v.double().cpu().numpy(), cu, kv, table, begin)


@pytest.mark.parametrize("dim,page", [(64, 16), (128, 64)])
def test_append_one_by_one_is_as_at_once(pkg, dim, page):
    """Tokens of rising magnitude, one at a time and all at once: the same
    scales, and codes that differ only where the once larger codes were
    rounded below e4m3's normal range."""
    rng = np.random.default_rng(5)
    n, heads = page + page // 2, 2
    dev, cu, kv, table, pages = make_batch(rng, page, [0], [n])
    x = rng.normal(0, 1, (n, 2 * heads + 2, dim)) * 2.0 ** (np.arange(n) / 5.0)[:, None, None]
    x = torch.from_numpy(x.astype(np.float32)).cuda()
    q, k, v = x.split([2, heads, heads], dim=1)
    once, steps = (random_cache(pkg, rng, pages, heads, page, dim) for _ in range(2))
    once.append(q, k, v, **dev)
    for i in range(n):
        steps.append(q[i:i + 1], k[i:i + 1], v[i:i + 1], torch.tensor([0, 1], dtype=torch.int32).cuda(),
                     torch.tensor([i + 1], dtype=torch.int32).cuda(), dev["page_table"])
    once.check(), steps.check()
    for which in ("k", "v"):
        s = getattr(once, which + "_scale").cpu().numpy()
        used = table[0]
        assert np.array_equal(s[used], getattr(steps, which + "_scale").cpu().numpy()[used])
        a, b = (dequantised(c, which)[used] for c in (once, steps))
        a, b = (t.transpose(0, 2, 1, 3).reshape(-1, heads, dim)[:n] for t in (a, b))
        step = np.repeat(s[used], page, 0)[:n][..., None] * 2.0 ** -9
        normal = np.abs(a) >= 8 * step                       # 2^-6 scales
        assert np.array_equal(a[normal], b[normal])
        assert (np.abs(a - b) <= step + 1e-30).all()


def test_append_nonfinite_values(pkg):
    """NaN stays NaN, infinities are held as the page's largest, and neither costs the other tokens their scale."""
    rng = np.random.default_rng(6)
    dev, cu, kv, table, pages = make_batch(rng, 16, [0], [8])
    cache = pkg.KvCache(pages, 1, 64, 16)
    x = rng.normal(0, 1, (8, 3, 64)).astype(np.float32)
    clean = x.copy()
    x[2, 1:, 5], x[3, 1:, 6], x[4, 1:, 7] = np.nan, np.inf, -np.inf
    x[5, 1:, 8] = 3e38
    x = torch.from_numpy(x).cuda()
    cache.append(x[:, :1], x[:, 1:2], x[:, 2:], **dev)
    for which in ("k", "v"):
        scale = float(getattr(cache, which + "_scale")[table[0, 0], 0])
        assert scale == 2.0 ** 40                            # 3e38 is past 448 * 2^40: held as that
        got = dequantised(cache, which)[table[0, 0], 0]
        assert np.isnan(got[2, 5]) and np.isnan(got).sum() == 1
        assert got[3, 6] == 448 * scale and got[4, 7] == -448 * scale and got[5, 8] == 448 * scale
    x[5, 1:, 8] = 1.0
    cache.append(x[:, :1], x[:, 1:2], x[:, 2:], **dev)
    for i, which in ((1, "k"), (2, "v")):
        scale = float(getattr(cache, which + "_scale")[table[0, 0], 0])
        finite = clean[:, i].copy()
        finite[2, 5] = finite[3, 6] = finite[4, 7] = 0
        finite[5, 8] = 1.0
        assert scale == 2.0 ** e4m3_exponent(np.abs(finite).max())


def test_append_zero_page_then_values(pkg):
    """A page of zeros has the least scale; the first real values raise it."""
    rng = np.random.default_rng(7)
    dev, cu, kv, table, pages = make_batch(rng, 16, [0], [2])
    cache = pkg.KvCache(pages, 1, 64, 16)
    z = torch.zeros(2, 3, 64, dtype=torch.float16, device="cuda")
    cache.append(z[:, :1], z[:, 1:2], z[:, 2:], **dev)
    assert float(cache.k_scale[table[0, 0], 0]) == 2.0 ** -40
    assert torch.isfinite(cache.k[table[0, 0]].float()[:, :2]).all() and not cache.k[table[0, 0]].float()[:, :2].any()
    one = torch.ones(1, 3, 64, dtype=torch.float16, device="cuda")
    cache.append(one[:, :1], one[:, 1:2], one[:, 2:], torch.tensor([0, 1], dtype=torch.int32).cuda(),
                 torch.tensor([3], dtype=torch.int32).cuda(), dev["page_table"])
    got = dequantised(cache, "v")[table[0, 0], 0]
    assert not got[:2].any() and (got[2] == 1.0).all()


def test_append_strided_unaligned_and_positions(pkg):
    """Rows at odd element offsets, heads last-but-one in memory, and given positions."""
    rng = np.random.default_rng(8)
    dev, cu, kv, table, pages = make_batch(rng, 32, [0, 9], [40, 3])
    raw = torch.from_numpy(rng.normal(0, 1, (5 * 64 * 43 + 3,)).astype(np.float32)).cuda().half()
    x = raw[3:].as_strided((43, 5, 64), (64, 43 * 64, 1), 3)      # heads outermost, off by three elements
    q, k, v = x[:, :3], x[:, 3:4], x[:, 4:]
    pos = torch.from_numpy(rng.permutation(100)[:43].astype(np.int32)).cuda()
    angle = np.arange(100)[:, None] * 10000.0 ** (-np.arange(0, 64, 2) / 64)
    cos, sin = (torch.from_numpy(f(angle).astype(np.float32)).cuda() for f in (np.cos, np.sin))
    a, b = pkg.KvCache(pages, 1, 64, 32), pkg.KvCache(pages, 1, 64, 32)
    got = a.append(q, k, v, **dev, cos=cos, sin=sin, positions=pos)
    want = b.append(q.contiguous(), k.contiguous(), v.contiguous(), **dev, cos=cos, sin=sin, positions=pos)
    assert torch.equal(got, want) and torch.equal(a.k.view(torch.uint8), b.k.view(torch.uint8))
    ref = rotate(q.double().cpu().numpy(), *(t.double().cpu().numpy()[pos.cpu().numpy()] for t in (cos, sin)), False)
    assert (np.abs(got.double().cpu().numpy() - ref) <= 2.0 ** -11 * np.abs(ref) + 1e-5).all()


def test_append_reports_what_only_the_gpu_sees(pkg):
    cache = pkg.KvCache(4, 1, 64, 16)
    x = torch.ones(2, 3, 64, dtype=torch.float16, device="cuda")
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")
    good = dict(cu_q=i32(0, 2), kv_lens=i32(2), page_table=i32(1, 2).reshape(1, 2))
    call = lambda **kw: cache.append(x[:, :1], x[:, 1:2], x[:, 2:], **{**good, **kw})
    call()
    cache.check()
    keep = cache.k.view(torch.uint8).clone()
    for bad, text in ((dict(page_table=i32(4, 0).reshape(1, 2)), "page number"),
                      (dict(page_table=i32(-1, 0).reshape(1, 2)), "page number"),
                      (dict(kv_lens=i32(1)), "out of range"),
                      (dict(kv_lens=i32(33)), "out of range")):
        call(**bad)
        with pytest.raises(pkg.B3Error, match=text) as ei:
            cache.check()
        assert ei.value.code == pkg.B3_EINVAL
        assert torch.equal(cache.k.view(torch.uint8), keep)
    t = torch.ones(1, 32, device="cuda")
    call(cos=t, sin=t)
    with pytest.raises(pkg.B3Error, match="position"):
        cache.check()
    cache.check()


# ─────────────────────────────── attend ───────────────────────────────

def attend_f64(cache, q, cu, kv, table, scale, causal, window):
    """out, lse, and the sums that bound the rounding: A = sum p |v|, B = sum |v| exp(-largest score) / sum."""
    K, V = dequantised(cache, "k"), dequantised(cache, "v")
    page, group = cache.page_tokens, q.shape[1] // cache.kv_heads
    x = q.double().cpu().numpy()
    out, A, B = (np.zeros(x.shape) for _ in range(3))
    lse = np.full(x.shape[:2], -np.inf)
    size = np.ones(x.shape[:2])
    for i in range(len(kv)):
        n, L = cu[i + 1] - cu[i], kv[i]
        if not n or not L:
            continue
        pages = table[i, :-(-L // page)]
        pos = L - n + np.arange(n)[:, None]
        key = np.arange(L)[None, :]
        seen = np.ones((n, L), bool)
        if causal:
            seen = (key <= pos) & ((key > pos - window) if window else True)
        for h in range(q.shape[1]):
            k = K[pages, h // group].reshape(-1, cache.head_dim)[:L]
            v = V[pages, h // group].reshape(-1, cache.head_dim)[:L]
            s = x[cu[i]:cu[i + 1], h] @ k.T * scale
            size[cu[i]:cu[i + 1], h] += np.abs(s).max(initial=0.0)
            s = np.where(seen, s, -np.inf)
            m = s.max(1, initial=-np.inf)
            live = m > -np.inf
            p = np.exp(s[live] - m[live, None])
            l = p.sum(1)
            rows = np.arange(cu[i], cu[i + 1])[live]
            out[rows, h] = p @ v / l[:, None]
            A[rows, h] = p @ np.abs(v) / l[:, None]
            B[rows, h] = (np.abs(v).max(0) * 1.0)[None] * (seen[live].sum(1) / l)[:, None]
            lse[rows, h] = m[live] + np.log(l)
    return out, lse, A, B, size


def check_attend(cache, q, dev, cu, kv, table, max_q, scale=None, causal=True, window=0):
    out, lse = cache.attend(q, **dev, max_q=max_q, scale=scale, causal=causal, window=window, return_lse=True)
    cache.check()
    ref, ref_lse, A, B, size = attend_f64(cache, q, cu, kv, table, scale or cache.head_dim ** -0.5, causal, window)
    d = np.abs(out.double().cpu().numpy() - ref)
    # scores are f32: 2e-6 of their magnitude moves a probability by as much
    bound = HALF_UNIT[q.dtype] * np.abs(ref) + (2.0 ** -11 + 1e-5 + 4e-6 * size[..., None]) * A + 2.0 ** -24 * B + 1e-30
    assert (d <= bound).all(), float((d / bound).max())
    got = lse.double().cpu().numpy()
    empty = np.isneginf(ref_lse)
    assert np.array_equal(np.isneginf(got), empty)
    assert (np.abs(got[~empty] - ref_lse[~empty]) <= 1e-5 * size[~empty]).all()
    assert not out.cpu().numpy()[empty].any() if q.dtype is torch.float16 else not out.float().cpu().numpy()[empty].any()
    return out, lse


ATTEND_CASES = [
    # dtype, q_heads, kv_heads, dim, page, past, new, causal, window
    (torch.float16, 8, 8, 128, 64, [0], [1], True, 0),
    (torch.bfloat16, 32, 8, 128, 64, [378, 0, 63, 64, 65, 1000, 15, 127], [1] * 8, True, 0),
    (torch.bfloat16, 16, 1, 64, 16, [15, 16, 17, 0, 200], [1] * 5, True, 0),
    (torch.float16, 10, 2, 128, 32, [33, 7, 0], [3, 1, 2], True, 0),
    (torch.float16, 14, 2, 64, 128, [1, 300, 129], [1, 0, 1], True, 64),
    (torch.bfloat16, 40, 2, 128, 16, [77, 5], [1, 1], True, 0),        # 20 heads share a key head
    (torch.float16, 6, 2, 64, 16, [0, 0, 0], [1, 37, 300], True, 0),
    (torch.bfloat16, 12, 4, 128, 64, [100, 0, 64], [70, 129, 64], True, 0),
    (torch.float16, 8, 1, 128, 32, [513], [200], True, 100),
    (torch.bfloat16, 5, 5, 64, 64, [40, 0, 9], [33, 128, 300], False, 0),
    (torch.float16, 4, 4, 128, 128, [600, 2], [1, 1], False, 0),
    (torch.float16, 4, 4, 128, 64, [0, 70, 0], [0, 130, 65], True, 0),
    (torch.bfloat16, 8, 8, 64, 32, [2500], [1], True, 0),              # one long row: split along the keys
    (torch.float16, 4, 1, 128, 64, [4000, 10], [260, 5], True, 0),
]


@pytest.mark.parametrize("case", ATTEND_CASES)
def test_attend_matches_float64(pkg, case):
    dtype, q_heads, kv_heads, dim, page, past, new, causal, window = case
    rng = np.random.default_rng(q_heads * 100 + dim + page + len(past))
    dev, cu, kv, table, pages = make_batch(rng, page, past, new)
    cache = random_cache(pkg, rng, pages, kv_heads, page, dim)
    # behind the last token of each sequence, and in pages no sequence has, nothing is a number
    for i, n in enumerate(kv):
        if n % page:
            for pool in (cache.k, cache.v):
                pool.view(torch.uint8)[table[i, n // page], :, n % page:] = 0x7F
    free = np.setdiff1d(np.arange(pages), table[table >= 0])
    cache.k_scale[free], cache.v_scale[free] = math.nan, math.nan
    scale = 0.02                                     # codes of 120 x 2^-8 x 2^4 with unit queries: scores of a few units
    q = torch.from_numpy(rng.normal(0, 1, (int(cu[-1]), q_heads, dim)).astype(np.float32)).to(dtype).cuda()
    check_attend(cache, q, dev, cu, kv, table, max(new), scale, causal, window)
    # a looser bound on the new tokens changes nothing that matters
    if max(new) <= 2:
        check_attend(cache, q, dev, cu, kv, table, 64, scale, causal, window)


@pytest.mark.parametrize("max_q", [1, 32])
def test_attend_no_keys_at_all(pkg, max_q):
    """Rows that see nothing: an empty sequence, more new tokens than cached ones; zeros and -inf."""
    rng = np.random.default_rng(1)
    page, dim = 16, 64
    cache = random_cache(pkg, rng, 4, 2, page, dim)
    new = [1, 1] if max_q == 1 else [1, 20, 3]
    kv = [0, 5] if max_q == 1 else [0, 5, 0]
    cu = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    table = np.array([[-1], [2], [-1]], np.int32)[:len(kv)]
    dev = dict(cu_q=torch.from_numpy(cu).cuda(), kv_lens=torch.tensor(kv, dtype=torch.int32).cuda(),
               page_table=torch.from_numpy(table).cuda())
    q = torch.from_numpy(rng.normal(0, 1, (int(cu[-1]), 4, dim)).astype(np.float32)).half().cuda()
    out, lse = check_attend(cache, q, dev, cu, kv, table, max_q, 0.02)
    assert torch.isneginf(lse[0]).all() and not out[0].any()


@pytest.mark.parametrize("max_q", [1, 128])
def test_attend_extreme_values(pkg, max_q):
    """Scores far apart, tiny and huge page scales side by side, large and tiny queries."""
    rng = np.random.default_rng(2)
    page, dim, heads = 16, 64, 2
    n = 1 if max_q == 1 else 70
    dev, cu, kv, table, pages = make_batch(rng, page, [150, 40], [n, n])
    cache = random_cache(pkg, rng, pages, heads, page, dim)
    cache.v_scale.copy_(torch.exp2(torch.from_numpy(rng.integers(-40, 41, cache.v_scale.shape)).float()).cuda())
    cache.k_scale.copy_(torch.exp2(torch.from_numpy(rng.integers(-20, -3, cache.k_scale.shape)).float()).cuda())
    q = rng.normal(0, 1, (int(cu[-1]), 4, dim)) * 2.0 ** rng.integers(-18, 6, (int(cu[-1]), 4, 1))
    q[0] = 0
    for dtype in (torch.float16, torch.bfloat16):
        t = torch.from_numpy(q.astype(np.float32)).to(dtype).cuda()
        out, lse = cache.attend(t, **dev, max_q=max_q, scale=0.05, return_lse=True)
        ref, ref_lse, A, B, size = attend_f64(cache, t, cu, kv, table, 0.05, True, 0)
        # values as large as 448 * 2^40 pass f16: held as infinity there, as everywhere
        with np.errstate(over="ignore"):
            want = torch.from_numpy(ref).to(dtype).double().numpy()
        got = out.double().cpu().numpy()
        bound = 2 * HALF_UNIT[dtype] * np.abs(ref) + (2.0 ** -11 + 1e-5 + 4e-6 * size[..., None]) * A + 2.0 ** -24 * B
        near_max = np.isinf(want) | np.isinf(got)
        assert (np.abs(got - ref)[~near_max] <= bound[~near_max] + 1e-7).all()
        assert (np.abs(ref)[near_max] + bound[near_max] >= 65504).all()
        assert (np.abs(lse.double().cpu().numpy() - ref_lse) <= 1e-5 * size).all()


@pytest.mark.parametrize("max_q", [1, 128])
def test_attend_nan_reaches_only_who_sees_it(pkg, max_q):
    rng = np.random.default_rng(3)
    page, dim = 32, 128
    n = 1 if max_q == 1 else 100
    dev, cu, kv, table, pages = make_batch(rng, page, [200, 200], [n, n])
    cache = random_cache(pkg, rng, pages, 2, page, dim)
    cache.v.view(torch.uint8)[table[0, 1], 1, 3, 7] = 0x7F
    q = torch.from_numpy(rng.normal(0, 1, (int(cu[-1]), 4, dim)).astype(np.float32)).bfloat16().cuda()
    out = cache.attend(q, **dev, max_q=max_q, scale=0.02).float().cpu().numpy()
    bad = np.isnan(out)
    assert bad[cu[0]:cu[1], 2:, 7].all() and bad.sum() == 2 * n
    cache.v.view(torch.uint8)[table[0, 1], 1, 3, 7] = 0
    cache.k.view(torch.uint8)[table[1, 2], 0, 0, 0] = 0x7F
    out = cache.attend(q, **dev, max_q=max_q, scale=0.02).float().cpu().numpy()
    bad = np.isnan(out)
    assert bad[cu[1]:cu[2], :2].all() and bad.sum() == n * 2 * dim


@pytest.mark.parametrize("n,q_heads,window", [(4, 4, 0), (3, 10, 8), (100, 4, 0), (300, 6, 20)])
def test_attend_masked_nan_stays_masked(pkg, n, q_heads, window):
    """A NaN value (and a NaN key) of a new token: the tokens before it, and those whose window is past it, do not see it."""
    rng = np.random.default_rng(n)
    page, dim, kv_heads = 16, 64, 2
    dev, cu, kv, table, pages = make_batch(rng, page, [50, 3], [n, n])
    q = torch.from_numpy(rng.normal(0, 1, (int(cu[-1]), q_heads, dim)).astype(np.float32)).half().cuda()
    clean = random_cache(pkg, rng, pages, kv_heads, page, dim)
    at = kv[0] - n + n // 2                     # the middle one of the new tokens of sequence 0
    want, want_lse = clean.attend(q, **dev, max_q=n, scale=0.02, window=window, return_lse=True)
    for pool in (clean.v, clean.k):
        cell = pool.view(torch.uint8)[table[0, at // page], 1, at % page]
        keep = cell.clone()
        cell[5] = 0x7F
        out, lse = clean.attend(q, **dev, max_q=n, scale=0.02, window=window, return_lse=True)
        cell.copy_(keep)
        clean.check()
        sees = np.zeros(int(cu[-1]), bool)
        sees[n // 2:n if not window else min(n, n // 2 + window)] = True
        group = q_heads // kv_heads
        bad = torch.isnan(out).cpu().numpy()
        if pool is clean.v:
            assert bad[sees][:, group:, 5].all() and bad.sum() == sees.sum() * group
        else:
            assert bad[sees][:, group:].all() and bad.sum() == sees.sum() * group * dim
        # who does not see it: as before, but for the order in which rows taken again add up (f32, probabilities not rounded)
        d = (out.float() - want.float()).abs().cpu().numpy()
        assert (d[~bad] <= 2.0 ** -9 * np.abs(want.float().cpu().numpy()).max()).all()
        fine = ~np.isnan(lse.cpu().numpy())
        assert np.allclose(lse.cpu().numpy()[fine], want_lse.cpu().numpy()[fine], rtol=1e-5, atol=1e-5)


def test_attend_strides_streams_and_repeats(pkg):
    """Query views, a side stream, and the same bits every time."""
    rng = np.random.default_rng(4)
    dev, cu, kv, table, pages = make_batch(rng, 64, [700, 3, 64], [1, 1, 1], width=20)
    cache = random_cache(pkg, rng, pages, 4, 64, 128)
    wide = torch.from_numpy(rng.normal(0, 1, (3, 25, 129)).astype(np.float32)).half().cuda()
    view = wide[:, 1:17, 1:]
    dev["page_table"] = dev["page_table"].repeat(1, 2)[:, :20]      # rows 40 apart
    a, la = cache.attend(view, **dev, max_q=1, scale=0.02, return_lse=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b, lb = cache.attend(view.contiguous(), **dev, max_q=1, scale=0.02, return_lse=True)
    side.synchronize()
    assert torch.equal(a, b) and torch.equal(la, lb)
    for _ in range(5):
        assert torch.equal(a, cache.attend(view, **dev, max_q=1, scale=0.02))
    check_attend(cache, view, dev, cu, kv, table, 1, 0.02)


@pytest.mark.parametrize("max_q", [1, 64])
def test_attend_far_pages(pkg, max_q):
    """Codes more than 2^32 bytes into the cache."""
    rng = np.random.default_rng(9)
    page, heads, dim = 128, 8, 128
    pages = (1 << 32) // (page * heads * dim) + 40
    cache = pkg.KvCache(pages, heads, dim, page)
    far = pages - 5
    g = torch.Generator(device="cuda").manual_seed(1)
    for pool, scale in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        pool[far:far + 2] = (torch.randn(2, heads, page, dim, generator=g, device="cuda") * 100).clamp(-448, 448).to(torch.float8_e4m3fn)
        scale[far:far + 2] = 2.0 ** -7
    n = 1 if max_q == 1 else 40
    table = np.array([[far, far + 1]], np.int32)
    dev = dict(cu_q=torch.tensor([0, n], dtype=torch.int32).cuda(), kv_lens=torch.tensor([200], dtype=torch.int32).cuda(),
               page_table=torch.from_numpy(table).cuda())
    q = torch.randn(n, heads, dim, generator=g, device="cuda").half()
    out = cache.attend(q, **dev, max_q=max_q, scale=0.02)
    cache.check()
    small = pkg.KvCache.over(cache.k[far:far + 2].clone(), cache.v[far:far + 2].clone(),
                             cache.k_scale[far:far + 2].clone(), cache.v_scale[far:far + 2].clone())
    dev["page_table"] = torch.tensor([[0, 1]], dtype=torch.int32).cuda()
    assert torch.equal(out, small.attend(q, **dev, max_q=max_q, scale=0.02))
    check_attend(small, q, dev, np.array([0, n]), [200], np.array([[0, 1]]), max_q, 0.02)
    x = torch.randn(n, 3 * heads, dim, generator=g, device="cuda").half()
    dev["page_table"] = torch.from_numpy(table).cuda()
    cache.append(x[:, :heads], x[:, heads:2 * heads], x[:, 2 * heads:], **dev)
    cache.check()
    page_at, slot = table[0, 199 // page], 199 % page
    got = cache.values(int(page_at))[1][:, slot].cpu().numpy()
    want = x[-1, 2 * heads:].float().cpu().numpy()
    assert (np.abs(got - want) <= 2.0 ** -4 * np.abs(want) + 2.0 ** -10 * cache.v_scale[page_at].cpu().numpy()[:, None]).all()


@pytest.mark.parametrize("max_q", [1, 64])
def test_attend_reports_what_only_the_gpu_sees(pkg, max_q):
    cache = pkg.KvCache(4, 1, 64, 16)
    n = 1 if max_q == 1 else 10
    q = torch.ones(n, 2, 64, dtype=torch.float16, device="cuda")
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")
    good = dict(cu_q=i32(0, n), kv_lens=i32(20), page_table=i32(1, 2).reshape(1, 2))
    call = lambda **kw: cache.attend(q, **{**good, **kw}, max_q=max_q)
    call()
    cache.check()
    for bad, text in ((dict(page_table=i32(1, 4).reshape(1, 2)), "page number"),
                      (dict(page_table=i32(-7, 0).reshape(1, 2)), "page number"),
                      (dict(kv_lens=i32(-1)), "out of range"),
                      (dict(kv_lens=i32(33)), "out of range")):
        call(**bad)
        with pytest.raises(pkg.B3Error, match=text):
            cache.check()
    # more new tokens than max_q says
    q3 = torch.ones(3 * n, 2, 64, dtype=torch.float16, device="cuda")
    if max_q == 1:
        cache.attend(q3, i32(0, 3), i32(20), good["page_table"], max_q=1)
        with pytest.raises(pkg.B3Error, match="out of range"):
            cache.check()


def test_decode_step_replays_in_a_graph(pkg):
    """append + attend + sample captured once, replayed with new lengths and inputs in the same tensors."""
    rng = np.random.default_rng(10)
    page, dim, heads = 16, 64, 2
    cache, plain = pkg.KvCache(16, heads, dim, page), pkg.KvCache(16, heads, dim, page)
    table = torch.arange(16, dtype=torch.int32, device="cuda").reshape(2, 8)
    cu = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
    lens = torch.tensor([0, 0], dtype=torch.int32, device="cuda")
    x = torch.zeros(2, 8, dim, device="cuda", dtype=torch.float16)
    head = torch.from_numpy(rng.normal(0, 0.3, (4 * dim, 500)).astype(np.float32)).half().cuda()
    u = torch.zeros(2, device="cuda")

    def step(c):
        lens.add_(1)
        q = c.append(x[:, :4], x[:, 4:6], x[:, 6:], cu, lens, table)
        o = c.attend(q, cu, lens, table, max_q=1)
        return o, *pkg.sample(o.reshape(2, -1) @ head, u)

    step(cache)
    lens.zero_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(cache)
    lens.zero_()
    inputs = [(torch.from_numpy(rng.normal(0, 1, (2, 8, dim)).astype(np.float32)).half().cuda(),
               torch.from_numpy(rng.uniform(0, 1, 2).astype(np.float32)).cuda()) for _ in range(40)]
    kept = []
    for a, b in inputs:
        x.copy_(a), u.copy_(b)
        graph.replay()
        kept.append([t.clone() for t in got])
    lens.zero_()
    for (a, b), want in zip(inputs, kept):
        x.copy_(a), u.copy_(b)
        for t, w in zip(step(plain), want):
            assert torch.equal(t, w)
    cache.check()


# ─────────────────────────────── sample ───────────────────────────────

def sample_by_definition(x, u, t, top_k, top_p, min_p):
    """One row by the definition, the weights in f32 (torch's exp on the same GPU), the sums in Python integers."""
    x = x.float()
    x = torch.where(torch.isnan(x), -math.inf, x)
    peak = x.max()
    if peak == -math.inf:
        return -1, math.nan
    if not t > 0:
        return int((x == peak).int().argmax()), 0.0
    w = torch.where(x == peak, 1.0, ((x - peak) / torch.tensor(t, device=x.device)).exp())
    whole = (w * 2.0 ** 31).to(torch.int64).cpu().numpy()
    order = torch.sort(x, descending=True, stable=True).indices.cpu().numpy()
    if top_k is not None and top_k > 0:
        order = order[:top_k]
    if top_p is not None and top_p < 1:
        sums = np.cumsum(whole[order])
        mass = float(np.float32(top_p)) * float(sums[-1])
        order = order[:1 + int((sums[:-1] < mass).sum())]
    kept = np.sort(order)
    if min_p is not None and min_p > 0:
        kept = kept[(w >= torch.tensor(min_p, device=x.device)).cpu().numpy()[kept]]
    if not len(kept):
        return -1, math.nan
    sums = np.cumsum(whole[kept])
    i = min(int((sums.astype(np.float64) <= float(np.float32(u)) * float(sums[-1])).sum()), len(kept) - 1)
    z = (x[kept[i]].double() - peak.double()).item() / t if x[kept[i]] != peak else 0.0
    return int(kept[i]), z - math.log(float(sums[-1]) / 2.0 ** 31)


def check_sample(pkg, x, u, t=None, top_k=None, top_p=None, min_p=None):
    rows = x.shape[0]
    f32 = lambda v: None if v is None else torch.tensor(v, dtype=torch.float32).cuda()
    i32 = lambda v: None if v is None else torch.tensor(v, dtype=torch.int32).cuda()
    ids, logprob = pkg.sample(x, f32(u), temperature=f32(t), top_k=i32(top_k), top_p=f32(top_p), min_p=f32(min_p))
    ids, logprob = ids.cpu().numpy(), logprob.cpu().numpy()
    row = lambda v, r: None if v is None else float(np.float32(v[r]))
    for r in range(rows):
        want, lp = sample_by_definition(x[r], u[r], 1.0 if t is None else row(t, r),
                                        None if top_k is None else top_k[r], row(top_p, r), row(min_p, r))
        assert ids[r] == want, (r, ids[r], want)
        if math.isnan(lp):
            assert math.isnan(logprob[r])
        else:
            assert abs(logprob[r] - lp) <= 4e-6 * (1 + abs(lp))
    return ids


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("vocab", [1, 2, 31, 1025, 8193, 16384, 16385, 50001, 131072, 262144])
def test_sample_matches_the_definition(pkg, dtype, vocab):
    rng = np.random.default_rng(vocab)
    rows = 6
    x = rng.normal(0, 2.5, (rows, vocab)).astype(np.float32)
    x[:, rng.integers(0, vocab, max(1, vocab // 1000))] += 6
    x = torch.from_numpy(x).to(dtype).cuda()
    u = rng.uniform(0, 1, rows).astype(np.float32)
    u[0] = 0.0
    u[1] = np.float32(1.0 - 2.0 ** -24)
    k = [0, 1, 5, 40, vocab, 2 * vocab]
    check_sample(pkg, x, u)
    check_sample(pkg, x, u, t=[0.0, 0.3, 1.0, 1.7, 30.0, 1.0])
    check_sample(pkg, x, u, top_k=k)
    check_sample(pkg, x, u, top_p=[0.0, 0.1, 0.5, 0.9, 0.999, 1.0])
    check_sample(pkg, x, u, min_p=[0.0, 0.001, 0.05, 0.3, 1.0, 1e-6])
    check_sample(pkg, x, u, t=[0.7] * 6, top_k=k[::-1], top_p=[0.95, 0.2, 0.8, 1.0, 0.6, 0.99],
                 min_p=[0.0, 0.02, 0.1, 0.0, 0.01, 0.2])


@pytest.mark.parametrize("vocab", [7, 300, 20000, 70000])
def test_sample_equal_logits(pkg, vocab):
    """Rows of one value, of two, of few: top-k and top-p cut among equals by index."""
    rng = np.random.default_rng(vocab)
    flat = np.full((3, vocab), -3.25, np.float32)
    flat[1, ::2] = 1.5
    flat[2] = rng.integers(0, 3, vocab)
    x = torch.from_numpy(flat).cuda()
    for u in (0.0, 0.37, 0.5, 0.9999):
        us = [u] * 3
        check_sample(pkg, x, us)
        check_sample(pkg, x, us, top_k=[3, vocab // 2 + 1, vocab // 3])
        check_sample(pkg, x, us, top_p=[0.5, 0.3, 0.7])
        check_sample(pkg, x, us, top_k=[vocab - 1, 5, 6], top_p=[0.25, 0.5, 0.9], min_p=[0.5, 0.0, 0.3])
    assert check_sample(pkg, x, [0.5] * 3, t=[0.0] * 3)[0] == 0


def test_sample_masked_rows(pkg):
    """-inf, NaN, +inf, signed zeros, the type's lowest value, and rows with nothing to take."""
    v = 9000
    x = np.full((8, v), -np.inf, np.float32)
    x[1, 17] = -5.0
    x[2, :] = np.nan
    x[3, [4, 400, 8999]] = [1.0, np.nan, 1.0]
    x[4, [3, 70, 800]] = [np.inf, 5.0, np.inf]
    x[5, :] = np.finfo(np.float32).min
    x[6, [10, 20]] = [0.0, -0.0]
    x[7, :] = -65504.0
    x[7, 5000] = -65503.0
    x = torch.from_numpy(x).cuda()
    for u in (0.0, 0.5, 0.99):
        ids = check_sample(pkg, x, [u] * 8, top_p=[0.9] * 8, top_k=[50] * 8)
        assert ids[0] == ids[2] == -1 and ids[1] == 17
        check_sample(pkg, x, [u] * 8)
        check_sample(pkg, x, [u] * 8, t=[0.0] * 8)
        check_sample(pkg, x, [u] * 8, min_p=[1.5] * 8)
    check_sample(pkg, x.half(), [0.3] * 8)


def test_sample_strided_rows_and_any_uniform(pkg):
    rng = np.random.default_rng(3)
    wide = torch.from_numpy(rng.normal(0, 2, (5, 4111)).astype(np.float32)).cuda()
    for dtype in (torch.float32, torch.bfloat16):
        view = wide.to(dtype)[:, 3:4004]
        check_sample(pkg, view, [0.1, 0.3, 0.5, 0.7, 0.9], top_k=[9] * 5)
    ids, _ = pkg.sample(wide, torch.tensor([1.0, 2.0, -1.0, math.nan, math.inf]).cuda(),
                        top_k=torch.full((5,), 4, dtype=torch.int32).cuda())
    top = torch.topk(wide, 4).indices.sort(dim=1).values.cpu().numpy()
    ids = ids.cpu().numpy()
    assert ids[0] == top[0, 3] and ids[1] == top[1, 3] and ids[4] == top[4, 3]     # at or past 1: the last kept token
    assert ids[2] == top[2, 0] and ids[3] == top[3, 0]                             # below 0 or no number: the first


def test_sample_frequencies(pkg):
    """20,000 draws from a small distribution: each count within five standard deviations."""
    p = np.array([0.5, 0.05, 0.2, 0.25])
    n = 20000
    x = torch.from_numpy(np.log(p).astype(np.float32)).cuda().repeat(n, 1)
    u = torch.rand(n, generator=torch.Generator(device="cuda").manual_seed(3), device="cuda")
    ids, logprob = pkg.sample(x, u)
    count = np.bincount(ids.cpu().numpy(), minlength=4)
    assert (np.abs(count - n * p) <= 5 * np.sqrt(n * p * (1 - p))).all()
    assert np.allclose(np.exp(logprob.cpu().numpy()), p[ids.cpu().numpy()], rtol=1e-5)


# ────────────────────────────── refusals ──────────────────────────────

def test_bad_arguments_are_refused(pkg):
    torch.cuda.synchronize()
    cache = pkg.KvCache(4, 2, 64, 16)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")
    x = torch.zeros(1, 4, 64, dtype=torch.float16, device="cuda")
    q, k, v = x, x[:, :2], x[:, 2:]
    good = dict(cu_q=i32(0, 1), kv_lens=i32(1), page_table=i32(0).reshape(1, 1))
    table = torch.zeros(4, 24, device="cuda")
    weight = torch.ones(64, device="cuda")

    def refused(f, *a, **kw):
        with pytest.raises(pkg.B3Error) as ei:
            f(*a, **kw)
        assert ei.value.code == pkg.B3_EINVAL

    for dim, page in ((96, 16), (64, 24), (32, 16), (64, 256)):
        c = pkg.KvCache(2, 1, dim, page)
        t = torch.zeros(1, 1, dim, dtype=torch.float16, device="cuda")
        refused(c.append, t, t, t, **good)
        refused(c.attend, t, **good, max_q=1)
    refused(pkg.KvCache, 0, 2, 64, 16)
    refused(pkg.KvCache.over, cache.k.float(), cache.v, cache.k_scale, cache.v_scale)
    refused(pkg.KvCache.over, cache.k, cache.v[:2], cache.k_scale, cache.v_scale)
    refused(pkg.KvCache.over, cache.k, cache.v, cache.k_scale.double(), cache.v_scale)
    refused(cache.append, q[:, :3], k, v, **good)                              # 3 heads over 2
    refused(cache.append, q, k[:, :1], v, **good)
    refused(cache.append, q, k.float(), v, **good)
    refused(cache.append, q.double(), k.double(), v.double(), **good)
    refused(cache.append, q[..., :32], k, v, **good)
    refused(cache.append, q, k, v, **{**good, "cu_q": torch.tensor([0, 1]).cuda()})
    refused(cache.append, q, k, v, **{**good, "cu_q": i32(0, 1, 2)})
    refused(cache.append, q, k, v, **{**good, "kv_lens": i32(1).cpu()})
    refused(cache.append, q, k, v, **{**good, "page_table": i32(0)})
    refused(cache.append, q, k, v, **good, q_norm=weight[:32])
    refused(cache.append, q, k, v, **good, cos=table)
    refused(cache.append, q, k, v, **good, cos=table[:, :20].contiguous(), sin=table[:, :20].contiguous())   # 40 channels
    refused(cache.append, q, k, v, **good, cos=torch.zeros(4, 40, device="cuda"), sin=torch.zeros(4, 40, device="cuda"))
    refused(cache.append, q, k, v, **good, positions=i32(0, 1))
    refused(cache.append, q, k, v, **good, out=torch.zeros(1, 4, 64, device="cuda"))
    refused(cache.attend, q.float(), **good, max_q=1)
    refused(cache.attend, q[:, :3], **good, max_q=1)
    refused(cache.attend, q, **good, max_q=0)
    refused(cache.attend, q, **good, max_q=1, window=-1)
    refused(cache.attend, q, **good, max_q=1, window=4, causal=False)
    refused(cache.attend, q, **good, max_q=1, out=q.float())
    logits, u = torch.zeros(2, 100, device="cuda"), torch.zeros(2, device="cuda")
    refused(pkg.sample, logits, None)
    refused(pkg.sample, logits, u[:1])
    refused(pkg.sample, logits.double(), u)
    refused(pkg.sample, logits[0], u)
    refused(pkg.sample, logits.cpu(), u.cpu())
    refused(pkg.sample, logits, u, top_k=u)
    refused(pkg.sample, logits, u, temperature=u.double())
    refused(pkg.sample, torch.zeros(1, 262145, device="cuda"), u[:1])
    cache.check()


def test_nothing_to_do(pkg):
    """No new tokens, no rows: the calls return empty tensors."""
    cache = pkg.KvCache(4, 2, 64, 16)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")
    x = torch.zeros(0, 4, 64, dtype=torch.float16, device="cuda")
    b = dict(cu_q=i32(0, 0), kv_lens=i32(3), page_table=i32(0).reshape(1, 1))
    assert cache.append(x, x[:, :2], x[:, 2:], **b).shape == (0, 4, 64)
    assert cache.attend(x, **b, max_q=1).shape == (0, 4, 64)
    ids, lp = pkg.sample(torch.zeros(0, 9, device="cuda"), torch.zeros(0, device="cuda"))
    assert ids.shape == lp.shape == (0,)
