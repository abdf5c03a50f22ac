"""PagedKVCache.keep on the GPU against the CPU, bit for bit.  Every case prints
its name before touching the GPU."""
import random

import pytest
import torch

from santa_amd.paged import PagedKVCache

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("layers, page, KVH, D, dtype, seqs, T", [
    (1, 8, 1, 16, torch.bfloat16, 1, 8), (2, 16, 8, 128, torch.bfloat16, 5, 30), (33, 8, 2, 64, torch.float16, 3, 12),
    (2, 8, 3, 5, torch.float32, 4, 9), (1, 16, 1, 4, torch.float16, 2, 6),  # rows that are no 16-byte pieces
    (2, 64, 32, 128, torch.bfloat16, 2, 70), (1, 256, 4, 64, torch.float32, 40, 40),  # more moves than a launch holds
    (1, 8, 1, 16, torch.int16, 1, 600),
])
def test_keep(layers, page, KVH, D, dtype, seqs, T):
    print(f"\n[case] keep layers={layers} page={page} KVH={KVH} D={D} {dtype} seqs={seqs} T={T}", flush=True)
    r = random.Random(T)
    kw = dict(kv_heads=KVH, head_dim=D, max_seqs=seqs + 1, max_len=2 * T + 400, dtype=dtype)
    pages = 2 * sum(-(-(T + 400) // page) for _ in range(seqs + 1))
    host, dev = (PagedKVCache(layers, pages, page, device=d, **kw) for d in ("cpu", "cuda"))
    for a, b in zip((*host.k, *host.v), (*dev.k, *dev.v)):
        a.copy_((torch.rand(a.shape) * 8000).to(dtype))
        b.copy_(a)
    lens = [r.randint(0, 100) for _ in range(seqs)]
    paths = lambda: [sorted(r.sample(range(T), r.randint(0, T))) for _ in range(seqs)]  # noqa: E731
    for kept in ([list(range(T))] * seqs, paths(), [[T - 1]] * seqs, [list(range(1, T))] * seqs, paths(), [[]] * seqs):
        for c in (host, dev):
            ids = c.add(lens)
            c.extend(ids, T)
            c.keep(ids, T, kept)
        assert host.lengths(ids) == dev.lengths(ids) == [n + len(k) for n, k in zip(lens, kept)]
        assert all(torch.equal(a, b.cpu()) for a, b in zip((*host.k, *host.v), (*dev.k, *dev.v)))
        assert torch.equal(host.block_table, dev.block_table.cpu())
        for c in (host, dev):
            c.free(ids)


def test_refused_while_captured():
    print("\n[case] keep while a graph is captured", flush=True)
    cache = PagedKVCache(1, 9, 8, kv_heads=1, head_dim=16, max_seqs=2, max_len=64)
    a, = cache.add([9])
    x = torch.zeros(4, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        x.add_(1)
        with pytest.raises(RuntimeError, match="while a graph is captured"):
            cache.keep([a], 2, [[1]])
    assert cache.lengths([a]) == [9]
