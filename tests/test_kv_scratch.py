"""CPU tests of who gets which scratch memory: the launches of a key/value cache must never share it while they run."""
import ctypes as C

import pytest


class _Lib:
    """Stands in for the library: streams have the numbers of `ids`; set-ups of scratch memory are counted."""

    def __init__(self):
        self.ids, self.made = {}, []

    def bam_kv_stream_id(self, stream):
        return self.ids.get(stream, (1 << 64) - 1)

    def bam_kv_scratch_init(self, array, at, size, stream):
        self.made.append((at, size, stream))
        return 0


class _Array:
    h, closed = None, 0

    def close(self):
        self.closed += 1


@pytest.fixture()
def caches(bam, monkeypatch):
    """A maker of caches without a GPU; the module's scratch memory is the test's own."""
    import torch
    from bam_b200 import kv as module
    lib, waits = _Lib(), []
    monkeypatch.setattr(module, "_scratch", {})
    monkeypatch.setattr(module, "_open", type(module._open)())
    monkeypatch.setattr(torch.cuda, "synchronize", lambda device=None: waits.append(device))

    def make(size=256):
        k = bam.KvCache.__new__(bam.KvCache)
        k.lib, k.array, k.device, k._scratch_bytes = lib, _Array(), torch.device("cpu"), size
        module._open.add(k)
        return k
    make.lib, make.waits, make.module = lib, waits, module
    return make


def test_scratch_belongs_to_the_stream_and_not_to_its_handle(caches):
    kv, lib = caches(), caches.lib
    lib.ids = {0x500: 7, 0x600: 8}
    first = kv._scratch_of(0x500)
    assert first.numel() == 256 and lib.made == [(first.data_ptr(), 256, 0x500)]
    assert kv._scratch_of(0x500) is first                        # the stream's launches run one after the other
    other = kv._scratch_of(0x600)
    assert other.data_ptr() != first.data_ptr() and len(lib.made) == 2
    assert caches.waits == []
    # the stream is gone and a new one has its handle: the last launch of the old one may still run
    lib.ids[0x500] = 9
    again = kv._scratch_of(0x500)
    assert len(caches.waits) == 1 and lib.made[2] == (again.data_ptr(), 256, 0x500)
    assert kv._scratch_of(0x500) is again and kv._scratch_of(0x600) is other and len(caches.waits) == 1
    # a cache with wider heads wants more
    wide = caches(1024)
    large = wide._scratch_of(0x600)
    assert large.numel() == 1024 and kv._scratch_of(0x600) is large and len(caches.waits) == 1


def test_a_stream_that_is_none_is_an_error(caches):
    with pytest.raises(RuntimeError):
        caches()._scratch_of(0x700)


@pytest.mark.parametrize("call", ["append", "gather", "attend"])
def test_the_per_thread_stream_is_refused(bam, caches, call):
    """Its handle is the same number in every thread and another stream in each."""
    import torch
    kv = caches()
    kv.dtype, kv.n_kv_heads, kv.head_dim, kv.n_layers, kv.block_tokens, kv.n_blocks, kv._layouts = torch.bfloat16, 2, 64, 1, 16, 8, [None]
    rows, slots = torch.zeros(3, 2, 64, dtype=torch.bfloat16), torch.zeros(3, dtype=torch.int64)
    args = {"append": (rows, rows, slots), "gather": (slots,),
            "attend": (rows, torch.zeros(3, 1, dtype=torch.int32), torch.zeros(3, dtype=torch.int32))}[call]
    for handle in (2, C.c_void_p(2)):
        with pytest.raises(ValueError, match="per-thread"):
            getattr(kv, call)(*args, stream=handle)
    assert caches.module._scratch == {} and caches.lib.made == []


def test_the_per_thread_stream_is_refused_as_the_current_one(caches):
    caches.lib.ids = {2: 5}
    with pytest.raises(ValueError, match="per-thread"):
        caches()._scratch_of(2)


def test_scratch_goes_with_the_last_cache_of_its_device(caches):
    import torch
    one, two, lib = caches(), caches(), caches.lib
    lib.ids = {0x500: 7}
    far = torch.zeros(8)
    caches.module._scratch[3, 0x500] = 9, far                   # another device's
    one._scratch_of(0x500)
    one.close()
    assert len(caches.module._scratch) == 2                      # `two` may want it
    one.close()
    assert one.array.closed == 2 and len(caches.module._scratch) == 2
    two.close()
    assert list(caches.module._scratch) == [(3, 0x500)]
    # a cache that is made later starts anew, and one that nobody closes goes when it is collected
    three = caches()
    assert three._scratch_of(0x500).numel() == 256 and len(lib.made) == 2
    array = three.array
    del three
    assert array.closed == 1 and list(caches.module._scratch) == [(3, 0x500)]
