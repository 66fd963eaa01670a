"""Sampling rows held by several blocks, started beside other work.

A block stores into the shared memory of the others of its cluster; each has to
be running by then, whatever kept it.  The calls here start while other
kernels hold most of the GPU, so that a cluster's blocks get their
multiprocessors at different times and behind one another."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from test_gpu_textgen import check_sample  # noqa: E402


@pytest.mark.parametrize("rows,vocab", [(1, 8193), (1, 262144), (3, 40000), (37, 131072)])
def test_clusters_that_start_unevenly(pkg, rows, vocab):
    rng = np.random.default_rng(vocab + rows)
    x = torch.from_numpy(rng.normal(0, 2.5, (rows, vocab)).astype(np.float32)).cuda()
    u = torch.from_numpy(rng.uniform(0, 1, rows).astype(np.float32)).cuda()
    settings = [dict(), dict(top_k=torch.full((rows,), 40, dtype=torch.int32, device="cuda")),
                dict(top_p=torch.full((rows,), 0.9, device="cuda")), dict(temperature=torch.zeros(rows, device="cuda"))]
    want = [pkg.sample(x, u, **s) for s in settings]
    for i, s in enumerate(settings):
        host = {k: v.cpu().tolist() for k, v in s.items()}
        check_sample(pkg, x, u.cpu().numpy(), t=host.get("temperature"), top_k=host.get("top_k"), top_p=host.get("top_p"))
    load = torch.randn(4096, 4096, device="cuda")
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    got = []
    for turn in range(20):
        with torch.cuda.stream(streams[0]):
            load @ load
        for st in streams[1:]:
            with torch.cuda.stream(st):
                (load[:97] * turn).exp_()
                got.append([pkg.sample(x, u, **s) for s in settings])
    torch.cuda.synchronize()
    for run in got:
        for (a, b), (c, d) in zip(run, want):
            assert torch.equal(a, c) and torch.equal(b, d)
