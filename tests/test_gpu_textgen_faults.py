"""Text generation where calls once answered wrongly or out of what they were given."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from test_gpu_textgen import check_sample, make_batch, random_cache  # noqa: E402


def i32(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


# ─────────────────────── expanded and overlapping rows ───────────────────────

@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("offset", [0, 3])
def test_sample_one_row_many_times(pkg, dtype, offset):
    """Many draws from one row of logits, given as an expanded tensor."""
    rng = np.random.default_rng(11)
    row = torch.from_numpy(rng.normal(0, 2, (1, 5003 + offset)).astype(np.float32)).to(dtype).cuda()[:, offset:]
    n = 40
    u = rng.uniform(0, 1, n).astype(np.float32)
    many = row.expand(n, -1)
    assert many.stride(0) == 0
    check_sample(pkg, many, u, t=[0.8] * n, top_k=[0, 30] * (n // 2), top_p=[0.9] * n)


def test_rows_that_overlap_are_refused(pkg):
    logits = torch.zeros(400, device="cuda").as_strided((4, 100), (50, 1))
    with pytest.raises(pkg.B3Error, match="row stride 50") as ei:
        pkg.sample(logits, torch.zeros(4, device="cuda"))
    assert ei.value.code == pkg.B3_EINVAL
    cache = pkg.KvCache(8, 1, 64, 16)
    x = torch.zeros(2, 3, 64, dtype=torch.float16, device="cuda")
    table = torch.arange(8, dtype=torch.int32, device="cuda").as_strided((2, 4), (2, 1))
    b = dict(cu_q=i32(0, 1, 2), kv_lens=i32(60, 60), page_table=table)
    for f in (lambda: cache.append(x[:, :1], x[:, 1:2], x[:, 2:], **b), lambda: cache.attend(x, **b, max_q=1)):
        with pytest.raises(pkg.B3Error, match="stride 2") as ei:
            f()
        assert ei.value.code == pkg.B3_EINVAL
    cache.check()
    # a single row's stride means nothing, whatever it is
    one = torch.zeros(100, device="cuda").as_strided((1, 100), (7, 1))
    assert pkg.sample(one, torch.zeros(1, device="cuda"))[0].tolist() == [0]


@pytest.mark.parametrize("max_q", [1, 40])
def test_one_page_table_row_for_all(pkg, max_q):
    """Several queries over one cached sequence: a page table of one row, expanded."""
    rng = np.random.default_rng(12)
    page, n = 16, 5
    dev, cu, kv, table, pages = make_batch(rng, page, [150], [max_q])
    cache = random_cache(pkg, rng, pages, 2, page, 64)
    q = torch.from_numpy(rng.normal(0, 1, (n * max_q, 4, 64)).astype(np.float32)).half().cuda()
    lens = i32(*[kv[0] - 7 * i for i in range(n)])
    cu_q = i32(*[max_q * i for i in range(n + 1)])
    wide = dev["page_table"].expand(n, -1)
    assert wide.stride(0) == 0
    got = cache.attend(q, cu_q, lens, wide, max_q=max_q, scale=0.02, return_lse=True)
    want = cache.attend(q, cu_q, lens, wide.contiguous(), max_q=max_q, scale=0.02, return_lse=True)
    cache.check()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    # append: the second sequence has no new tokens, the row is its too
    a, b = (pkg.KvCache(pages, 2, 64, page) for _ in range(2))
    x = torch.from_numpy(rng.normal(0, 1, (3, 8, 64)).astype(np.float32)).half().cuda()
    for c, t in ((a, wide[:2]), (b, wide[:2].contiguous())):
        c.append(x[:, :4], x[:, 4:6], x[:, 6:], i32(0, 3, 3), i32(20, 150), t)
        c.check()
    assert torch.equal(a.k.view(torch.uint8), b.k.view(torch.uint8)) and torch.equal(a.v_scale, b.v_scale)


# ───────────────────────────── NaN in the cache ─────────────────────────────

def ms(f, n=5):
    f()
    a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    a.record()
    for _ in range(n):
        f()
    b.record()
    b.synchronize()
    return a.elapsed_time(b) / n


# dtype, q_heads, kv_heads, dim, page, past, new, causal, window
NAN_CASES = [
    (torch.float16, 8, 2, 128, 64, [1900, 30], [300, 500], True, 0),
    (torch.bfloat16, 6, 2, 64, 16, [700, 0, 90], [200, 333, 1], True, 90),
    (torch.float16, 2, 2, 128, 32, [100, 1000], [400, 130], True, 300),
    (torch.bfloat16, 4, 4, 64, 128, [500, 3], [100, 60], False, 0),
    (torch.float16, 8, 2, 128, 64, [4000, 70, 0, 200], [4, 3, 2, 1], True, 0),
    (torch.bfloat16, 6, 2, 64, 16, [3000, 5, 90], [5, 2, 4], True, 40),
    (torch.float16, 16, 1, 128, 32, [900, 20], [1, 1], True, 0),
    (torch.float16, 4, 2, 64, 32, [900, 20], [6, 8], False, 0),
]


@pytest.mark.parametrize("case", NAN_CASES)
def test_nan_values_reach_exactly_who_sees_them(pkg, case):
    """NaN codes of V all over the cache, many among the new tokens: a channel of a
    row is NaN where a key that it sees has NaN there, everything else keeps its bits."""
    dtype, q_heads, kv_heads, dim, page, past, new, causal, window = case
    rng = np.random.default_rng(dim + page + sum(past))
    dev, cu, kv, table, pages = make_batch(rng, page, past, new)
    cache = random_cache(pkg, rng, pages, kv_heads, page, dim)
    q = torch.from_numpy(rng.normal(0, 1, (int(cu[-1]), q_heads, dim)).astype(np.float32)).to(dtype).cuda()
    call = lambda: cache.attend(q, **dev, max_q=max(new), scale=0.02, causal=causal, window=window, return_lse=True)
    want, want_lse = call()
    raw = cache.v.view(torch.uint8)
    nan_at = [np.zeros((n, kv_heads, dim), bool) for n in kv]
    for i, n in enumerate(kv):
        at = np.concatenate([rng.integers(0, n, 3), n - 1 - rng.integers(0, min(n, new[i] + 5), 6)])
        for j in at:
            h, c = rng.integers(kv_heads), rng.integers(dim)
            nan_at[i][j, h, c] = True
            raw[table[i, j // page], h, j % page, c] = 0x7F if rng.random() < 0.5 else 0xFF
    got, lse = call()
    cache.check()
    expect = np.zeros((int(cu[-1]), q_heads, dim), bool)
    for i in range(len(kv)):
        for t in range(new[i]):
            pos = kv[i] - new[i] + t
            hi = pos + 1 if causal else kv[i]
            lo = max(0, pos + 1 - window) if causal and window else 0
            expect[cu[i] + t] = np.repeat(nan_at[i][lo:hi].any(0), q_heads // kv_heads, 0)
    bad = torch.isnan(got).cpu().numpy()
    assert np.array_equal(bad, expect)
    assert torch.equal(got[~torch.isnan(got)], want[~torch.isnan(got)])
    assert torch.equal(lse, want_lse)


@pytest.mark.parametrize("n,past", [(2048, 14336), (4, 30000)])
def test_nan_costs_no_more_than_numbers(pkg, n, past):
    """NaN that rows do see (an early value, a whole padded query) leaves a call's time as it is."""
    rng = np.random.default_rng(n)
    page, dim, kv_heads, q_heads = 64, 128, 2, 8
    dev, cu, kv, table, pages = make_batch(rng, page, [past, 500], [n, n])
    cache = random_cache(pkg, rng, pages, kv_heads, page, dim)
    q = torch.from_numpy(rng.normal(0, 1, (int(cu[-1]), q_heads, dim)).astype(np.float32)).half().cuda()
    call = lambda: cache.attend(q, **dev, max_q=n, scale=0.02)
    clean = ms(call)
    want = call()
    cache.v.view(torch.uint8)[table[0, 0], 1, 3, 7] = 0x7F
    q[1] = math.nan
    slow = ms(call)
    got = call()
    cache.check()
    bad = torch.isnan(got)
    group = q_heads // kv_heads
    assert bad[1].all() and bad[:n, group:, 7].all()
    expect = torch.zeros_like(bad)
    expect[1] = True
    expect[:n, group:, 7] = True
    assert torch.equal(bad, expect) and torch.equal(got[~bad], want[~bad])
    assert slow <= 3 * clean + 0.05, (slow, clean)


# ──────────────────────────────── gradients ────────────────────────────────

def test_a_gradient_that_would_be_lost_is_refused(pkg):
    cache = pkg.KvCache(2, 1, 64, 16)
    x = torch.ones(1, 3, 64, dtype=torch.float16, device="cuda")
    w, t = torch.ones(64, device="cuda"), torch.ones(4, 32, device="cuda")
    b = dict(cu_q=i32(0, 1), kv_lens=i32(1), page_table=i32(0).reshape(1, 1))
    logits, u = torch.zeros(1, 100, device="cuda"), torch.zeros(1, device="cuda")
    leaf = lambda a: a.clone().requires_grad_()

    def calls(f):
        yield "q requires", lambda: cache.append(f(x[:, :1]), x[:, 1:2], x[:, 2:], **b)
        yield "k requires", lambda: cache.append(x[:, :1], f(x[:, 1:2]), x[:, 2:], **b)
        yield "v requires", lambda: cache.append(x[:, :1], x[:, 1:2], f(x[:, 2:]), **b)
        yield "k_norm requires", lambda: cache.append(x[:, :1], x[:, 1:2], x[:, 2:], **b, q_norm=w, k_norm=f(w))
        yield "cos requires", lambda: cache.append(x[:, :1], x[:, 1:2], x[:, 2:], **b, cos=f(t), sin=t)
        yield "q requires", lambda: cache.attend(f(x), **b, max_q=1)
        yield "logits requires", lambda: pkg.sample(f(logits), u)

    for text, call in calls(leaf):
        with pytest.raises(pkg.B3Error, match=text) as ei:
            call()
        assert ei.value.code == pkg.B3_EINVAL
        with torch.no_grad():
            call()
    for _, call in calls(lambda a: leaf(a).detach()):
        call()
    cache.check()


# ──────────────────────────────── the status ────────────────────────────────

def test_check_waits_for_other_streams(pkg):
    """A call that is still waiting on another stream is in what check() reports."""
    cache = pkg.KvCache(2, 1, 64, 16)
    x = torch.ones(1, 3, 64, dtype=torch.float16, device="cuda")
    b = dict(cu_q=i32(0, 1), kv_lens=i32(1), page_table=i32(5).reshape(1, 1))
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(400_000_000)
        cache.append(x[:, :1], x[:, 1:2], x[:, 2:], **b)
    with pytest.raises(pkg.B3Error, match="page number"):
        cache.check()
    cache.check()


@pytest.mark.parametrize("max_q", [1, 40])
@pytest.mark.parametrize("cu", [(1, 2, 3), (0, 1, 2), (0, 2, 1, 3), (0, 0, 0)])
def test_rows_of_no_sequence_are_reported(pkg, cu, max_q):
    """Three rows, and a cu_q that leaves some of them out, or steps back: their outputs are not written."""
    cache = pkg.KvCache(8, 1, 64, 16)
    x = torch.ones(3, 3, 64, dtype=torch.float16, device="cuda")
    n = len(cu) - 1
    b = dict(cu_q=i32(*cu), kv_lens=i32(*[20] * n), page_table=torch.arange(2 * n, dtype=torch.int32, device="cuda").reshape(n, 2))
    cache.attend(x, **b, max_q=max_q)
    with pytest.raises(pkg.B3Error, match="cu_q"):
        cache.check()
    if list(cu) == sorted(cu):
        cache.append(x[:, :1], x[:, 1:2], x[:, 2:], **b)
        with pytest.raises(pkg.B3Error, match="cu_q"):
            cache.check()


@pytest.mark.parametrize("length", [-1, 0, -(1 << 31), 1 - (1 << 31), (1 << 31) - 1])
def test_append_lengths_far_out_of_range(pkg, length):
    cache = pkg.KvCache(4, 1, 64, 16)
    x = torch.ones(2, 3, 64, dtype=torch.float16, device="cuda")
    cache.append(x[:, :1], x[:, 1:2], x[:, 2:], i32(0, 2), i32(length), i32(0, 1).reshape(1, 2))
    with pytest.raises(pkg.B3Error, match="kv_lens"):
        cache.check()
    assert not cache.k.float().any() and not cache.v.float().any()


# ──────────────────────────────── errors ────────────────────────────────

def test_out_of_memory_is_torchs(pkg):
    """An allocation that fails inside a call raises what torch raises for it, and the cache goes on."""
    cache = pkg.KvCache(2, 1, 64, 16)
    n = 4_000_000
    x = torch.zeros(1, 1, 64, dtype=torch.float16, device="cuda").expand(n, 1, 64)   # an output of half a gigabyte
    b = dict(cu_q=i32(0, n), kv_lens=i32(3), page_table=i32(0).reshape(1, 1))
    torch.cuda.empty_cache()
    torch.cuda.set_per_process_memory_fraction(0.001)
    try:
        with pytest.raises(torch.OutOfMemoryError):
            cache.attend(x, **b, max_q=n)
    finally:
        torch.cuda.set_per_process_memory_fraction(1.0)
    out = cache.attend(x[:2], **{**b, "cu_q": i32(0, 2)}, max_q=2)
    cache.check()
    assert out.shape == (2, 1, 64)
