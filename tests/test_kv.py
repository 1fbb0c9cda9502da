"""CPU tests of the key/value cache: what its entry points refuse before anything reaches a GPU."""
import ctypes as C

import pytest

EINVAL = 22


def test_c_entries_refuse_missing_handles(bam):
    from bam_b200 import _lib
    lib = bam.load()
    layout = _lib.KvLayout(0, 64, 2, 16, 8, 0)
    two = (C.c_int64 * 2)(0, 0)
    assert lib.bam_kv_scratch_bytes(None, C.byref(layout)) == 0
    assert lib.bam_kv_scratch_init(None, None, 0, None) == EINVAL
    assert lib.bam_launch_kv_append(None, C.byref(layout), C.byref(_lib.KvAppend()), None, 0, None) == EINVAL
    assert lib.bam_launch_kv_gather(None, C.byref(layout), 1, None, None, None, two, two, None, 0, None) == EINVAL
    assert lib.bam_launch_kv_attend(None, C.byref(layout), C.byref(_lib.KvAttend()), None, 0, None) == EINVAL


def test_struct_sizes_match_the_header(bam, tmp_path):
    """The ctypes mirrors have the layout the C compiler gives the structs of the header."""
    import os
    import subprocess
    from bam_b200 import _lib
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    src = tmp_path / "s.c"
    fields = [("bam_kv_layout_t", _lib.KvLayout), ("bam_kv_append_t", _lib.KvAppend), ("bam_kv_attend_t", _lib.KvAttend)]
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "bam_abi.h"', "int main(void) {"]
    for name, t in fields:
        lines.append(f'printf("{name} %zu\\n", sizeof({name}));')
        lines += [f'printf("{name}.{f[0]} %zu\\n", offsetof({name}, {f[0]}));' for f in t._fields_]
    src.write_text("\n".join(lines + ["return 0; }"]))
    subprocess.run(["gcc", "-I" + os.path.join(root, "include"), str(src), "-o", str(tmp_path / "s")], check=True)
    said = dict(x.split() for x in subprocess.run([str(tmp_path / "s")], capture_output=True, text=True, check=True).stdout.splitlines())
    for name, t in fields:
        assert int(said[name]) == C.sizeof(t)
        for f in t._fields_:
            assert int(said[f"{name}.{f[0]}"]) == getattr(t, f[0]).offset, f[0]


class _Pages:
    """Stands in for a page cache: only its page size is looked at before the arguments are checked."""

    def __init__(self, page_size):
        self.page_size = page_size


@pytest.mark.parametrize("page, dim, tokens", [(4096, 128, None), (4096, 64, 32), (8192, 128, 24), (8192, 72, None),
                                               (65536, 272, None), (4096, 8, None), (4096, 64, 0)])
def test_refuses_geometries(bam, page, dim, tokens):
    with pytest.raises(ValueError):
        bam.KvCache(_Pages(page), 4, 2, dim, block_tokens=tokens)


def test_refuses_types_and_counts(bam):
    import torch
    with pytest.raises(ValueError):
        bam.KvCache(_Pages(8192), 4, 2, 64, dtype=torch.float32)
    for blocks, heads, layers in ((0, 1, 1), (1, 0, 1), (1, 1, 0), (1 << 31, 1, 1), (1, 65537, 1)):
        with pytest.raises(ValueError):
            bam.KvCache(_Pages(8192), blocks, heads, 64, n_layers=layers)


@pytest.fixture()
def kv(bam):
    """A cache whose checks of arguments run on CPU tensors; nothing is launched."""
    import torch
    k = bam.KvCache.__new__(bam.KvCache)
    k.device, k.dtype, k.n_kv_heads, k.head_dim, k.n_layers, k.block_tokens, k.n_blocks = torch.device("cpu"), torch.bfloat16, 2, 64, 1, 16, 8
    k._layouts = [None]
    return k


def test_append_refuses(kv):
    import torch
    n = 5
    k, v, q = (torch.zeros(n, h, 64, dtype=torch.bfloat16) for h in (2, 2, 4))
    slots, pos = torch.zeros(n, dtype=torch.int64), torch.zeros(n, dtype=torch.int64)
    cos = torch.zeros(10, 32)
    w = torch.zeros(64, dtype=torch.bfloat16)
    rope = dict(positions=pos, rope=(cos, cos))
    bad = [
        dict(k=k.float()), dict(v=v[:4]), dict(k=k[:, :1]), dict(v=v[..., :32]), dict(k=k.transpose(1, 2).contiguous().transpose(1, 2)),
        dict(slots=slots.int()), dict(slots=slots[:4]), dict(slots=torch.zeros(2 * n, dtype=torch.int64)[::2]),
        dict(rope=(cos, cos)), dict(rope=(cos, cos[:, :16]), positions=pos), dict(rope=(cos.double(), cos.double()), positions=pos),
        dict(rope=(cos[:, :4], cos[:, :4]), positions=pos), dict(rope=(torch.zeros(10, 40),) * 2, positions=pos),
        dict(rope=(cos[:0], cos[:0]), positions=pos), dict(rope_style="other", **rope), dict(rope=(cos, cos), positions=pos.int()),
        dict(k_norm=w[:32]), dict(k_norm=w.float()), dict(q_norm=w), dict(q_out=q), dict(q=q[:, :0]), dict(q=q[:4]),
        dict(q=q, q_out=q[:, :2]), dict(q=q.half()), dict(layer=1), dict(layer=-1, q=q),
    ]
    for change in bad:
        args = dict(k=k, v=v, slots=slots)
        args.update(change)
        if "layer" in change:                                    # checked after the tensors: the empty call reaches it
            args.update(k=k[:0], v=v[:0], slots=slots[:0], **({"q": q[:0]} if "q" in change else {}))
        with pytest.raises(ValueError):
            kv.append(**args)


def test_gather_refuses(kv):
    import torch
    slots = torch.zeros(3, dtype=torch.int64)
    good = torch.zeros(3, 2, 64, dtype=torch.bfloat16)
    for args in (dict(slots=slots.int()), dict(slots=slots[None]), dict(slots=slots, out=(good, good[:2])),
                 dict(slots=slots, out=(good.float(), good)), dict(slots=slots, layer=3)):
        with pytest.raises(ValueError):
            kv.gather(**args)


def test_attend_refuses(kv):
    import torch
    q = torch.zeros(3, 4, 64, dtype=torch.bfloat16)
    table, lens = torch.zeros(3, 5, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    bad = [dict(q=q[0]), dict(q=q[:, :3]), dict(q=q[:, :0]), dict(q=q.half()), dict(q=q[..., :32]), dict(block_table=table.long()),
           dict(block_table=table[:2]), dict(block_table=table[:, :0]), dict(block_table=table.t().contiguous().t()),
           dict(seq_lens=lens.long()), dict(seq_lens=lens[:2]), dict(window=-1), dict(window=4, sinks=-1),
           dict(out=q[:, :2]), dict(out=q.float()), dict(layer=1)]
    for change in bad:
        args = dict(q=q, block_table=table, seq_lens=lens)
        args.update(change)
        with pytest.raises(ValueError):
            kv.attend(**args)
