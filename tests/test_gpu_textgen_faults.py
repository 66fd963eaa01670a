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
