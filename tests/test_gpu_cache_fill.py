"""A cache that has room for every page keeps every page: nothing is evicted while there are unused slots."""
import pytest

pytestmark = pytest.mark.gpu
SEC = 1_000_000_000
M64 = (1 << 64) - 1


@pytest.mark.parametrize("pages, page", [(40000, 4096), (9000, 4096), (500, 4096), (3000, 16384)])
def test_cache_of_the_size_of_the_data_holds_all_of_it(cuda, bam, orc, pages, page):
    torch = cuda
    n = pages * page // 8
    ctrl = bam.Controller(n * 8, 0, queue_depth=256, num_queues=32)
    ctrl.configure(spin_timeout_ns=5 * SEC)
    ctrl.fill_store(9)
    cache = bam.PageCache(ctrl, page, pages)
    arr = bam.Array(cache, n)
    want = int(orc.fill_store(9, 0, n).sum(dtype="uint64")) & M64
    for again in range(3):
        cache.stats(reset=True)
        out = torch.zeros(1, dtype=torch.int64, device="cuda")
        arr.page_scan(pages, out)
        assert ctrl.status() == (0, "none", 0)
        assert (int(out.item()) & M64) == want
        assert cache.stats()["read_ios"] == (0 if again else pages)
        assert cache.audit() == 0
    # the same after every page was dropped
    cache.invalidate_async()
    cache.stats(reset=True)
    for _ in range(2):
        out = torch.zeros(1, dtype=torch.int64, device="cuda")
        arr.page_scan(pages, out)
    assert ctrl.status() == (0, "none", 0) and (int(out.item()) & M64) == want
    assert cache.stats()["read_ios"] == pages
    arr.close(); cache.close(); ctrl.close()
