"""GPU tests of the key/value cache where its attention's numbers get hard.

Tolerances beyond those of test_gpu_kv: the weights of an fp16 product are kept to 2^-40 of the largest, or to 2^-16 of
themselves where that is more, so n of them with values up to V are off by n * 2^-40 * V in all."""
import pytest

from test_gpu_kv import attend64, check_attend, done, fill, make, rand

pytestmark = pytest.mark.gpu


def led(torch, g, kv, lens, table, lead, below, spread, v):
    """Keys whose scores against the query `8, 0, 0, ...` at scale 1 are 0 at token `lead(n)` of each sequence and between
    -below and -below - spread nats elsewhere; they are exact in 64 bits and in 32."""
    T = kv.block_tokens
    k = torch.zeros_like(v)
    x = -(below + spread * torch.rand(len(k), kv.n_kv_heads, generator=g, device="cuda")) / 8
    k[..., 0] = x.to(kv.dtype)
    at = [table[b].long()[lead(n) // T] * T + lead(n) % T for b, n in enumerate(lens)]
    for i in at:
        k[i] = 0
    return k, at


def close_led(torch, got, ref, lens, dtype, vmax):
    """Scores and their differences are single products, rounded once or twice: 2^-22 of their size; a weight is kept to
    2^-16 of itself or 2^-40 of the largest; sums as in test_gpu_kv.  The rounding to the type comes last."""
    out, a, smax = ref
    n = torch.tensor(lens, dtype=torch.float64, device="cuda")[:, None, None]
    rel = 2 * smax * 2.0 ** -22 + 2.0 ** -16 + n.clamp(max=1024) * 2.0 ** -22
    tol = a * rel + n * 2.0 ** -40 * vmax
    tol = tol + torch.finfo(dtype).eps / 2 * (out.abs() + tol) + (2.0 ** -25 if dtype == torch.float16 else 0)
    err = (got.double() - out).abs()
    assert torch.isfinite(got).all() and (err <= tol).all(), f"worst {float((err / tol).max())} x the tolerance"


def weighted64(torch, q, k, v, table, lens, T):
    """(out, sum of the magnitudes, largest score) at scale 1, in 64 bits."""
    B, HQ, D = q.shape
    H = k.shape[1]
    out, a = torch.zeros(B, HQ, D, dtype=torch.float64, device="cuda"), torch.zeros(B, HQ, D, dtype=torch.float64, device="cuda")
    smax = torch.zeros(B, HQ, 1, dtype=torch.float64, device="cuda")
    for b, n in enumerate(lens):
        j = torch.arange(n, device="cuda")
        rows = table[b].long()[j // T] * T + j % T
        s = torch.einsum("hgd,nhd->hgn", q[b].double().view(H, HQ // H, D), k[rows].double())
        p = torch.softmax(s, -1)
        out[b] = torch.einsum("hgn,nhd->hgd", p, v[rows].double()).reshape(HQ, D)
        a[b] = torch.einsum("hgn,nhd->hgd", p, v[rows].double().abs()).reshape(HQ, D)
        smax[b] = s.abs().amax(-1).reshape(HQ, 1)
    return out, a, smax


@pytest.mark.parametrize("dtype_name", ["float16", "bfloat16"])
@pytest.mark.parametrize("dim, group, where, below, spread", [
    (64, 4, "first", 15.5, 0.4), (128, 8, "first", 17.4, 0.0), (128, 9, "middle", 16.0, 3.0), (256, 2, "first", 11.0, 9.0),
    (48, 3, "last", 17.0, 1.5), (96, 1, "last", 14.0, 6.0),
])
def test_small_weights_beside_a_large_one(cuda, bam, dtype_name, dim, group, where, below, spread):
    """One token leads by 11 to 20 nats and has a value of zero, as the first token of a sequence often does: the output is
    what thousands of small weights make of their values.  Few workers, so that one run holds the leader and many others."""
    torch = cuda
    dtype = getattr(torch, dtype_name)
    g = torch.Generator(device="cuda").manual_seed(dim + group)
    lens = [8000, 1500, 33]
    kv = make(bam, torch, sum(-(-n // 16) for n in lens) + 4, 1, dim, dtype, tokens=16, max_grid=3)
    _, v, table = fill(torch, g, kv, lens)
    v = (v.float().abs() + 0.5).to(dtype)
    lead = {"first": lambda n: 0, "middle": lambda n: n // 2, "last": lambda n: n - 1}[where]
    k, at = led(torch, g, kv, lens, table, lead, below, spread, v)
    for i in at:
        v[i] = 0
    kv.append(k, v, torch.arange(len(k), device="cuda"))
    q = torch.zeros(len(lens), group, dim, dtype=dtype, device="cuda")
    q[..., 0] = 8
    got = kv.attend(q, table, torch.tensor(lens, dtype=torch.int32, device="cuda"), scale=1.0)
    close_led(torch, got, weighted64(torch, q, k, v, table, lens, 16), lens, dtype, float(v.abs().max()))
    done(kv)


@pytest.mark.parametrize("dtype_name, below", [("bfloat16", 0.0), ("bfloat16", 3.0), ("bfloat16", 60.0), ("bfloat16", 80.0),
                                               ("float16", 0.0), ("float16", 5.0), ("float16", 16.0), ("float16", 40.0), ("float16", 80.0)])
@pytest.mark.parametrize("dim, group", [(64, 2), (128, 11), (256, 3), (48, 1)])
def test_values_that_are_infinite_in_visible_rows(cuda, bam, dtype_name, below, dim, group):
    """An infinite value of a visible token makes its element of the output infinite, whether the token's weight is one or
    e^-80; two of different sign, or a NaN, make it NaN; the other elements, heads and sequences do not notice."""
    torch = cuda
    dtype = getattr(torch, dtype_name)
    g = torch.Generator(device="cuda").manual_seed(dim)
    lens = [300, 90, 45, 200]
    kv = make(bam, torch, sum(-(-n // 16) for n in lens) + 4, 2, dim, dtype, tokens=16)
    _, v, table = fill(torch, g, kv, lens)
    k, at = led(torch, g, kv, lens, table, lambda n: n // 3, below, 0.0 if below else 4.0, v)
    inf, nan = float("inf"), float("nan")
    row = lambda b, j: table[b].long()[j // 16] * 16 + j % 16           # noqa: E731
    for j, d, x in ((5, 0, inf), (299, 1, -inf), (100, 2, inf), (100, 3, -inf), (7, 4, inf), (200, 4, -inf), (8, 5, inf), (250, 5, inf),
                    (299, dim - 1, nan)):                               # token 100 is the leader, of weight one
        v[row(0, j), 0, d] = x
    for j in range(90):
        v[row(1, j), 1, dim - 2] = -inf
    kv.append(k, v, torch.arange(len(k), device="cuda"))
    q = torch.zeros(len(lens), 2 * group, dim, dtype=dtype, device="cuda")
    q[..., 0] = 8
    got, lse = kv.attend(q, table, torch.tensor(lens, dtype=torch.int32, device="cuda"), scale=1.0, return_lse=True)
    want = torch.zeros(len(lens), 2 * group, dim, device="cuda")
    want[0, :group, 0] = want[0, :group, 2] = want[0, :group, 5] = inf
    want[0, :group, 1] = want[0, :group, 3] = -inf
    want[0, :group, 4] = want[0, :group, dim - 1] = nan
    want[1, group:, dim - 2] = -inf
    odd = want != 0
    assert torch.equal(got[odd].float().nan_to_num(123.0), want[odd].nan_to_num(123.0))
    v = torch.where(torch.isfinite(v), v, torch.zeros_like(v))
    out, a, smax = weighted64(torch, q, k, v, table, lens, 16)
    got = torch.where(odd, torch.zeros_like(got), got)
    close_led(torch, got, (out.masked_fill(odd, 0), a.masked_fill(odd, 0), smax), lens, dtype, float(v.abs().max()))
    assert torch.isfinite(lse).all()
    done(kv)


@pytest.mark.parametrize("lens", [[1], [700, 1, 20]])
def test_rows_whose_every_score_is_nan(cuda, bam, lens):
    """The maximum of no number at all must not turn into an empty sequence's: lse is NaN like the output."""
    torch = cuda
    g = torch.Generator(device="cuda").manual_seed(21)
    kv = make(bam, torch, sum(-(-n // 16) for n in lens) + 4, 1, 64, torch.bfloat16, page=4096)
    k, v, table = fill(torch, g, kv, lens)
    k.fill_(float("nan"))
    kv.append(k, v, torch.arange(len(k), device="cuda"))
    q = rand(torch, g, len(lens), 3, 64, dtype=torch.bfloat16)
    out, lse = kv.attend(q, table, torch.tensor(lens, dtype=torch.int32, device="cuda"), return_lse=True)
    assert torch.isnan(out).all() and torch.isnan(lse).all()
    done(kv)


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


@pytest.mark.parametrize("rising", [6.0, -6.0, 200.0])
def test_a_sequence_shared_by_more_workers_than_join_at_once(cuda, bam, rising):
    """40000 tokens of one key/value head are more than 128 workers' parts: the join takes them in rounds, and the maximum
    moves between the rounds."""
    torch = cuda
    g = torch.Generator(device="cuda").manual_seed(23)
    lens, dim = [40000, 37001], 64
    kv = make(bam, torch, sum(-(-n // 256) for n in lens) + 4, 1, dim, torch.bfloat16, page=65536)
    k, v, table = fill(torch, g, kv, lens)
    T = kv.block_tokens
    q = rand(torch, g, 2, 3, dim, dtype=torch.bfloat16)
    q[..., 0] = 8
    for b, n in enumerate(lens):
        j = torch.arange(n, device="cuda")
        k[table[b].long()[j // T] * T + j % T, 0, 0] = (rising * j / n / (8 * dim ** -0.5)).bfloat16()
    kv.append(k, v, torch.arange(len(k), device="cuda"))
    out, lse = kv.attend(q, table, torch.tensor(lens, dtype=torch.int32, device="cuda"), return_lse=True)
    check_attend(torch, out, lse, attend64(torch, q, k, v, table, lens, T, dim ** -0.5), torch.bfloat16)
    done(kv)


def test_more_sequences_than_a_scan_of_the_lengths(cuda, bam):
    """5000 sequences, many of them empty: each thread that lays out the list counts more than 32."""
    torch = cuda
    g = torch.Generator(device="cuda").manual_seed(24)
    B, dim = 5000, 64
    kv = make(bam, torch, 64, 2, dim, torch.bfloat16, page=4096)
    T = kv.block_tokens
    k, v = rand(torch, g, 64 * T, 2, dim, dtype=torch.bfloat16), rand(torch, g, 64 * T, 2, dim, dtype=torch.bfloat16)
    kv.append(k, v, torch.arange(64 * T, device="cuda"))
    table = torch.randint(0, 64, (B, 3), generator=g, device="cuda", dtype=torch.int32)
    lens = torch.randint(0, 3 * T + 1, (B,), generator=g, device="cuda", dtype=torch.int32)
    lens[torch.rand(B, generator=g, device="cuda") < 0.4] = 0
    lens[1000:1100] = 0
    q = rand(torch, g, B, 4, dim, dtype=torch.bfloat16, scale=2.0)
    out, lse = kv.attend(q, table, lens, return_lse=True)
    check_attend(torch, out, lse, attend64(torch, q, k, v, table, lens.tolist(), T, dim ** -0.5), torch.bfloat16)
    done(kv)


@pytest.mark.parametrize("dim, page, slots, grid", [(128, 16384, 60, 4), (256, 16384, 700, 0), (48, 4096, 50, 3)])
def test_fp16_attention_from_the_store(cuda, bam, dim, page, slots, grid):
    torch = cuda
    g = torch.Generator(device="cuda").manual_seed(25)
    lens = [1300, 3, 0, 700]
    T = page // (4 * dim) // 16 * 16
    kv = make(bam, torch, sum(-(-n // T) for n in lens) + 3, 2, dim, torch.float16, page=page, slots=slots, max_grid=grid)
    k, v, table = fill(torch, g, kv, lens)
    kv.append(k, v, torch.arange(len(k), device="cuda"))
    kv.cache.flush()
    kv.cache.invalidate()
    q = rand(torch, g, len(lens), 6, dim, dtype=torch.float16, scale=2.0)
    ls = torch.tensor(lens, dtype=torch.int32, device="cuda")
    for window, sinks in ((0, 0), (200, 5)):
        out, lse = kv.attend(q, table, ls, window=window, sinks=sinks, return_lse=True)
        check_attend(torch, out, lse, attend64(torch, q, k, v, table, lens, T, dim ** -0.5, window, sinks), torch.float16)
    assert kv.cache.ctrl.status() == (0, "none", 0)
    assert kv.cache.stats()["read_ios"] > 0
    done(kv)


def test_streams_that_come_and_go(cuda, bam):
    """Streams that are destroyed behind a call, whose handles come back: each has a number of its own, and no two launches
    that run at once have the same scratch memory."""
    torch = cuda
    g = torch.Generator(device="cuda").manual_seed(26)
    lens = [900, 20, 400]
    kv = make(bam, torch, 90, 2, 64, torch.bfloat16, page=4096)
    k, v, table = fill(torch, g, kv, lens)
    kv.append(k, v, torch.arange(len(k), device="cuda"))
    q = rand(torch, g, 3, 8, 64, dtype=torch.bfloat16, scale=2.0)
    ls = torch.tensor(lens, dtype=torch.int32, device="cuda")
    ref = attend64(torch, q, k, v, table, lens, kv.block_tokens, 0.125)
    torch.cuda.synchronize()
    rt, at = torch.cuda.cudart(), torch.zeros(1, dtype=torch.int64)
    outs, numbers = [], set()
    for _ in range(40):
        assert int(rt.cudaStreamCreate(at.data_ptr())) == 0
        handle = int(at)
        numbers.add(kv.lib.bam_kv_stream_id(handle))
        outs.append(kv.attend(q, table, ls, stream=handle))
        outs.append(kv.attend(q, table, ls))                     # at the same time on the current stream
        assert int(rt.cudaStreamDestroy(handle)) == 0
    torch.cuda.synchronize()
    assert len(numbers) == 40 and (1 << 64) - 1 not in numbers
    assert kv.lib.bam_kv_stream_id(0) not in numbers
    for o in outs:
        check_attend(torch, o, None, ref, torch.bfloat16)
    with pytest.raises(ValueError, match="per-thread"):
        kv.attend(q, table, ls, stream=2)
    assert kv.cache.ctrl.status() == (0, "none", 0)
    done(kv)


def test_scratch_is_given_back(cuda, bam):
    """The streams' scratch memory goes with the last cache of the device; a captured graph keeps its own."""
    torch = cuda
    g = torch.Generator(device="cuda").manual_seed(27)
    lens = [200, 3]

    def cache():
        kv = make(bam, torch, 24, 2, 64, torch.bfloat16, page=4096)
        k, v, table = fill(torch, g, kv, lens)
        kv.append(k, v, torch.arange(len(k), device="cuda"))
        return kv, k, v, table
    q = rand(torch, g, 2, 4, 64, dtype=torch.bfloat16)
    ls = torch.tensor(lens, dtype=torch.int32, device="cuda")
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    for _ in range(2):
        one, two = cache(), cache()
        size = one[0]._scratch_bytes
        held = torch.cuda.memory_allocated()
        kept = one[0].attend(q, one[3], ls, stream=side)
        assert torch.cuda.memory_allocated() - held >= size      # the side stream's
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = one[0].attend(q, one[3], ls)
        graph.replay()
        done(two[0])
        ref = attend64(torch, q, one[1], one[2], one[3], lens, one[0].block_tokens, 0.125)
        for o in (kept, out, one[0].attend(q, one[3], ls)):
            check_attend(torch, o, None, ref, torch.bfloat16)
        torch.cuda.synchronize()
        del graph, out, o, kept, ref
        done(one[0])
        del one, two
        assert torch.cuda.memory_allocated() - before < size


@pytest.mark.parametrize("slots, page, grid", [(1, 4096, 3), (1, 8192, 3), (2, 4096, 3), (3, 4096, 3), (5, 8192, 3), (3, 4096, 5), (6, 4096, 0)])
def test_caches_of_a_few_slots(cuda, bam, slots, page, grid):
    """Blocks of 16 tokens are read in pairs, which takes two slots; a single one is refused and not waited for."""
    torch = cuda
    g = torch.Generator(device="cuda").manual_seed(28)
    lens = [100, 1, 33]
    kv = make(bam, torch, 16, 2, 64, torch.bfloat16, page=page, slots=slots, max_grid=grid)
    kv.cache.ctrl.configure(spin_timeout_ns=2_000_000_000)
    k, v, table = fill(torch, g, kv, lens)
    kv.append(k, v, torch.arange(len(k), device="cuda"))
    bk, bv = kv.gather(torch.arange(len(k), device="cuda"))
    assert torch.equal(bk, k) and torch.equal(bv, v)
    q = rand(torch, g, len(lens), 4, 64, dtype=torch.bfloat16)
    ls = torch.tensor(lens, dtype=torch.int32, device="cuda")
    if slots == 1 and kv.block_tokens == 16:
        with pytest.raises(RuntimeError, match="bam_launch_kv_attend"):
            kv.attend(q, table, ls)
    else:
        out, lse = kv.attend(q, table, ls, return_lse=True)
        assert kv.cache.ctrl.status() == (0, "none", 0)
        check_attend(torch, out, lse, attend64(torch, q, k, v, table, lens, kv.block_tokens, 0.125), torch.bfloat16)
    done(kv)


@pytest.mark.parametrize("page, dim, tokens", [(1024, 16, 16), (2048, 32, 16), (2048, 16, 32), (4096, 16, 48)])
def test_pages_smaller_than_the_controllers(cuda, bam, page, dim, tokens):
    """Pages of 1 and 2 KiB: several slots, and several blocks of the store, in one page of the controller."""
    torch = cuda
    g = torch.Generator(device="cuda").manual_seed(29)
    lens = [500, 0, 31, 90]
    kv = make(bam, torch, sum(-(-n // tokens) for n in lens) + 5, 3, dim, torch.float16, page=page, slots=40, tokens=tokens, max_grid=4)
    k, v, table = fill(torch, g, kv, lens)
    order = torch.randperm(len(k), generator=g, device="cuda")
    kv.append(k[order], v[order], order)
    bk, bv = kv.gather(order)
    assert torch.equal(bk, k[order]) and torch.equal(bv, v[order])
    q = rand(torch, g, len(lens), 6, dim, dtype=torch.float16, scale=2.0)
    out, lse = kv.attend(q, table, torch.tensor(lens, dtype=torch.int32, device="cuda"), return_lse=True)
    assert kv.cache.ctrl.status() == (0, "none", 0)
    check_attend(torch, out, lse, attend64(torch, q, k, v, table, lens, tokens, dim ** -0.5), torch.float16)
    done(kv)


def test_a_bad_index_leaves_the_other_rows_right(cuda, bam):
    """What an index outside its range concerns is undefined, and nothing else: other tokens, sequences and pages."""
    torch = cuda
    g = torch.Generator(device="cuda").manual_seed(30)
    lens = [300, 77, 150, 40]
    kv = make(bam, torch, sum(-(-n // 16) for n in lens) + 4, 2, 64, torch.bfloat16, page=4096)
    k, v, table = fill(torch, g, kv, lens)
    total = len(k)
    kv.append(k, v, torch.arange(total, device="cuda"))
    q = rand(torch, g, 4, 8, 64, dtype=torch.bfloat16, scale=2.0)
    ls = torch.tensor(lens, dtype=torch.int32, device="cuda")
    out, lse, tol, ltol = attend64(torch, q, k, v, table, lens, 16, 0.125)
    for what in ("block", "length"):
        bad_t, bad_l = table.clone(), ls.clone()
        if what == "block":
            bad_t[1, 2] = kv.n_blocks
        else:
            bad_l[1] = 1 << 30
        o, s = kv.attend(q, bad_t, bad_l, return_lse=True)
        assert kv.cache.ctrl.status(clear=True)[:2] == (34, "range")
        rest = torch.tensor([0, 2, 3], device="cuda")
        check_attend(torch, o[rest], s[rest], (out[rest], lse[rest], tol[rest], ltol[rest]), torch.bfloat16)
    # append: token 5 has no such slot, token 9 no such position
    n = 40
    nk, nv, nq = (rand(torch, g, n, h, 64, dtype=torch.bfloat16) for h in (2, 2, 4))
    slots = torch.randperm(total, generator=g, device="cuda")[:n]
    was, pos = slots.clone(), torch.arange(n, device="cuda")
    cos, sin = torch.ones(n, 32, device="cuda"), torch.zeros(n, 32, device="cuda")
    slots[5], pos[9] = total, n
    got = kv.append(nk, nv, slots, positions=pos, rope=(cos, sin), q=nq)
    assert kv.cache.ctrl.status(clear=True)[:2] == (34, "range")
    good = torch.tensor([i for i in range(n) if i not in (5, 9)], device="cuda")
    assert torch.equal(got[good], nq[good])
    k[was[good]], v[was[good]] = nk[good], nv[good]
    every = torch.arange(total, device="cuda")
    kept = every != was[9]                                       # the row whose position is none
    bk, bv = kv.gather(every)
    assert torch.equal(bk[kept], k[kept]) and torch.equal(bv[kept], v[kept])
    every[3] = -total
    every[7] = total + 5
    bk, bv = kv.gather(every)
    assert kv.cache.ctrl.status(clear=True)[:2] == (34, "range")
    kept[7] = kept[3] = False
    assert torch.equal(bk[kept], k[kept]) and torch.equal(bv[kept], v[kept]) and not bk[3].any() and not bv[3].any()
    done(kv)
