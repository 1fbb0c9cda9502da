"""GPU tests of handles that go in another order than they should: what is collected together is closed in any order."""
import gc
import itertools

import pytest

pytestmark = pytest.mark.gpu


def objects(bam, torch, n_ctrls=1):
    ctrls = [bam.Controller(1 << 20, 0, queue_depth=64, num_queues=4) for _ in range(n_ctrls)]
    cache = bam.PageCache(ctrls if n_ctrls > 1 else ctrls[0], 4096, 64)
    kv = bam.KvCache(cache, 8, 2, 64)
    return [*ctrls, cache, kv]


def works(bam, torch):
    """A new set does what it should: nothing is left behind, no pending error among it."""
    *ctrls, cache, kv = objects(bam, torch)
    rows = torch.randn(5, 2, 64, device="cuda").bfloat16()
    kv.append(rows, rows, torch.arange(5, device="cuda"))
    assert torch.equal(kv.gather(torch.arange(5, device="cuda"))[0], rows)
    assert ctrls[0].status() == (0, "none", 0)
    for x in (kv, cache, *ctrls):
        x.close()


@pytest.mark.parametrize("n_ctrls", [1, 2])
def test_handles_close_in_any_order(cuda, bam, n_ctrls):
    torch = cuda
    for order in itertools.permutations(range(n_ctrls + 2)):
        x = objects(bam, torch, n_ctrls)
        for i in order:
            x[i].close()
    torch.cuda.synchronize()
    works(bam, torch)


def test_what_is_collected_together(cuda, bam):
    """A cycle holds them all, as a traceback does that an exception leaves behind."""
    torch = cuda
    for n_ctrls in (1, 2, 1):
        cycle = {"x": objects(bam, torch, n_ctrls)}
        cycle["self"] = cycle
        del cycle
        gc.collect()
    torch.cuda.synchronize()
    works(bam, torch)
