"""CPU tests of what the key/value cache refuses to write to."""
import pytest

from test_kv import kv  # noqa: F401


def test_outputs_whose_rows_lie_on_one_another_are_refused(kv):  # noqa: F811
    """Heads or tokens that share elements, as expanded tensors do, would hold whatever was written last."""
    import torch
    n, heads = 3, 4
    q = torch.zeros(n, heads, 64, dtype=torch.bfloat16)
    k, slots = q[:, :2], torch.zeros(n, dtype=torch.int64)
    table, lens = torch.zeros(n, 5, dtype=torch.int32), torch.zeros(n, dtype=torch.int32)
    flat = torch.zeros(4096, dtype=torch.bfloat16)
    same = [torch.zeros(1, heads, 64, dtype=torch.bfloat16).expand(n, -1, -1), torch.zeros(n, 1, 64, dtype=torch.bfloat16).expand(-1, heads, -1),
            flat.as_strided((n, heads, 64), (heads * 64, 63, 1)), flat.as_strided((n, heads, 64), (1, 64 * n, 1))]
    for out in same:
        with pytest.raises(ValueError, match="one another"):
            kv.append(k, k, slots, q=q, q_out=out)
        with pytest.raises(ValueError, match="one another"):
            kv.attend(q, table, lens, out=out)
        with pytest.raises(ValueError, match="one another"):
            kv.gather(slots, out=(out[:, :2], k))
        with pytest.raises(ValueError, match="one another"):
            kv.gather(slots, out=(k, out[:, :2]))


def test_inputs_may_be_expanded_and_single_rows_have_any_stride(kv):  # noqa: F811
    import torch
    calls = []
    kv._call = lambda *a: calls.append(a)

    class _Lib:
        bam_launch_kv_append = bam_launch_kv_gather = None
    kv.lib = _Lib
    row = torch.zeros(1, 1, 64, dtype=torch.bfloat16)
    slots = torch.zeros(3, dtype=torch.int64)
    kv.append(row.expand(3, 2, -1), row.expand(3, 2, -1), slots, q=row.expand(3, 4, -1))
    flat = torch.zeros(64, dtype=torch.bfloat16).as_strided((1, 1, 64), (0, 0, 1))
    kv.n_kv_heads = 1
    kv.gather(slots[:1], out=(flat, flat))
    interleaved = torch.zeros(3 * 4 * 64, dtype=torch.bfloat16).as_strided((3, 4, 64), (64, 3 * 64, 1))
    kv.append(row.expand(3, 1, -1), row.expand(3, 1, -1), slots, q=interleaved, q_out=interleaved)
    assert len(calls) == 3


def test_writes_in_place_count_as_changes(kv):  # noqa: F811
    """A tensor that autograd has saved and a call then overwrites is found to have changed."""
    import torch
    kv._call = lambda *a: None

    class _Lib:
        bam_launch_kv_append = bam_launch_kv_gather = bam_launch_kv_attend = None
    kv.lib = _Lib
    q = torch.zeros(3, 2, 64, dtype=torch.bfloat16)
    slots, table, lens = torch.zeros(3, dtype=torch.int64), torch.zeros(3, 1, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    out, k, v, mine = (torch.zeros_like(q) for _ in range(4))
    for call, written in ((lambda: kv.append(k, v, slots, q=q, q_out=q), [q]), (lambda: kv.append(k, v, slots, q=q, q_out=mine), [mine]),
                          (lambda: kv.gather(slots, out=(k, v)), [k, v]), (lambda: kv.attend(q, table, lens, out=out), [out])):
        before = [t._version for t in (q, out, k, v, mine)]
        call()
        for t, was in zip((q, out, k, v, mine), before):
            assert (t._version > was) == any(t is w for w in written)
    w = torch.ones(64, dtype=torch.bfloat16, requires_grad=True)
    y = (q * w).sum()
    kv.attend(q, table, lens, out=q)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    with torch.inference_mode():
        t = torch.zeros_like(q)
        assert kv.attend(t, table, lens, out=t) is t
