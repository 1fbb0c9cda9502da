"""GPU tests of the key/value cache where its attention's numbers get hard."""
import pytest

from test_gpu_kv import done, fill, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("scale", [1.0, 0.3, -0.7])
@pytest.mark.parametrize("top", [2.0 ** 27, 2.0 ** 33, 2.0 ** 50, -2.0 ** 40, 2.0 ** 100])
def test_scores_far_beyond_the_exponential(cuda, bam, scale, top):
    """Scores whose distance from the next number is itself far beyond the exponential's range.  The largest has the weight
    one; equal ones share it."""
    torch = cuda
    g = torch.Generator(device="cuda").manual_seed(22)
    lens = [400, 130]
    kv = make(bam, torch, sum(-(-n // 16) for n in lens) + 4, 1, 64, torch.bfloat16, page=4096)
    _, v, table = fill(torch, g, kv, lens)
    T = kv.block_tokens
    # the score of token j is top * (1 + m / 128) with m = 0 .. 127, exact in every type here; two tokens have the largest
    m = torch.randint(0, 120, (len(v),), generator=g, device="cuda").float()
    best = []
    for b, n in enumerate(lens):
        two = [table[b].long()[j // T] * T + j % T for j in (n // 4, n - 2)]
        for i in two:
            m[i] = 127.0 if top * scale > 0 else -1.0                    # nearest to zero where all are negative
        best.append(two)
    k = torch.zeros_like(v)
    k[:, 0, 0] = ((1 + m / 128) * 2.0 ** 13).bfloat16()
    kv.append(k, v, torch.arange(len(k), device="cuda"))
    q = torch.zeros(2, 5, 64, dtype=torch.bfloat16, device="cuda")
    q[..., 0] = top / 2.0 ** 13
    out, lse = kv.attend(q, table, torch.tensor(lens, dtype=torch.int32, device="cuda"), scale=scale, return_lse=True)
    for b, two in enumerate(best):
        want = (v[two[0], 0].double() + v[two[1], 0].double()) / 2
        assert ((out[b].double() - want).abs() <= torch.finfo(torch.bfloat16).eps / 2 * want.abs() + 2.0 ** -20 * v.double().abs().max()).all()
        s = float(k[two[0], 0, 0].double()) * float(q[b, 0, 0].double()) * scale
        # products with the scale and the logarithm's base: three roundings and the rounded constants
        assert ((lse[b].double() - s).abs() <= 6 * 2.0 ** -24 * abs(s) + 1).all()
    done(kv)
