"""The slots of a cache lie on controller pages, whatever was allocated before it."""
import ctypes as C

import pytest

pytestmark = pytest.mark.gpu
SEC = 1_000_000_000


@pytest.mark.parametrize("page, slots", [(4096, 1), (4096, 37), (4096, 260), (4096, 300), (512, 9), (8192, 5), (16384, 3)])
def test_cache_base_is_page_aligned(cuda, bam, orc, page, slots):
    torch = cuda
    lib = bam.load()
    n = 64 * page // 8
    ctrl = bam.Controller(max(n * 8, 4096), 0, queue_depth=16, num_queues=2)
    ctrl.configure(ctrl_blocks=1, spin_timeout_ns=5 * SEC)
    ctrl.set_max_grid(2)
    ctrl.fill_store(5)
    # caches of odd sizes before it move the place the allocator hands out next
    others = [bam.PageCache(ctrl, 512, 1 + i) for i in range(3)]
    for cache in others + [bam.PageCache(ctrl, page, slots)]:
        d = (C.c_uint8 * 4096)()
        assert lib.bam_cache_descriptor(cache.h, d, 4096) == 0
        base = int.from_bytes(bytes(d[:8]), "little")              # base_addr is the descriptor's first member
        assert base and base % 4096 == 0
    arr = bam.Array(cache, n)
    out = torch.zeros(1, dtype=torch.int64, device="cuda")
    if slots >= 37:                                               # room for what eight warps pin at once
        idx = torch.arange(0, n, 3, device="cuda")
        arr.read(idx.numel(), 1, out, idx=idx)
        assert ctrl.status() == (0, "none", 0)
        want = orc.fill_store(5, 0, n)[::3].sum(dtype="uint64")
        assert (int(out.item()) & ((1 << 64) - 1)) == int(want)
    arr.close()
    for c in others + [cache]:
        c.close()
    ctrl.close()
