"""GPU tests of the key/value cache against plain computations in 64 bits.

Tolerances.  eps(t) / 2 is the relative error of the one rounding to the 16-bit type.  Sums of n products in 32 bits,
in any order and with the truncating adds that matrix instructions may use, are off by at most n * 2^-22 of the sum of
the magnitudes (a truncated add loses 2^-23 of its result, the running magnitude is below the total; the factor 2
covers the rounding of the factors)."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
SEC = 1_000_000_000
MS = 1_000_000


def make(bam, torch, blocks, heads, dim, dtype, page=None, slots=None, layers=1, tokens=None, max_grid=0, ctrls=1, dist=0, queues=16):
    """A cache over one or several controllers; slots None: every page fits."""
    if page is None:
        page = 512
        while page < 16 * dim * 4:
            page *= 2
        page = max(page, 4096)
    pages = blocks * heads * layers
    cs = []
    for _ in range(ctrls):
        c = bam.Controller(max(pages // (ctrls if dist else 1) + 1, 1) * page, 0, queue_depth=64, num_queues=queues)
        c.configure(spin_timeout_ns=5 * SEC)
        if max_grid:
            c.configure(ctrl_blocks=2)
            c.set_max_grid(max_grid)
        cs.append(c)
    cache = bam.PageCache(cs if ctrls > 1 else cs[0], page, slots or pages + 8)
    return bam.KvCache(cache, blocks, heads, dim, dtype=dtype, n_layers=layers, block_tokens=tokens, dist=dist)


def done(kv, clean=True):
    if clean:
        assert kv.cache.ctrl.status() == (0, "none", 0)
    assert kv.cache.audit() == 0
    kv.close(); kv.cache.close()
    for c in kv.cache.ctrls:
        c.close()


def store_rows(kv, torch, layer=0):
    """K and V [n_blocks * block_tokens, heads, dim] decoded from the store of one controller by the documented layout."""
    kv.cache.flush()
    assert kv.cache.ctrl.status() == (0, "none", 0)
    page, T, D, H = kv.cache.page_size, kv.block_tokens, kv.head_dim, kv.n_kv_heads
    n = kv.n_blocks * H
    raw = kv.cache.ctrl.store_numpy("uint8")[layer * n * page:(layer + 1) * n * page].reshape(n, page)
    rows = raw[:, :T * D * 4].copy().view("int16").reshape(kv.n_blocks, H, 2, T, D // 8, 8)
    nc = D // 8
    a, b = (0, 7) if nc % 8 == 0 else (1, 3) if nc % 8 == 4 else (2, 1)
    out = np.empty_like(rows)
    for r in range(T):
        for c in range(nc):
            out[:, :, :, r, c] = rows[:, :, :, r, c ^ ((r >> a) & b)]
    t = torch.from_numpy(out.reshape(kv.n_blocks, H, 2, T, D)).cuda().view(kv.dtype)
    k, v = (t[:, :, i].transpose(1, 2).reshape(kv.n_blocks * T, H, D) for i in (0, 1))
    return k, v


def rand(torch, g, *shape, dtype=None, scale=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def transform64(torch, x, norm, eps, cos, sin, style):
    """(result, magnitude that bounds its rounding errors) of norm and rotation in 64 bits."""
    y = x.double()
    if norm is not None:
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + eps) * norm.double()
    mag = y.abs()
    if cos is not None:
        half = cos.shape[-1]
        i = torch.arange(half, device=x.device)
        a, b = (i, i + half) if style == "half" else (2 * i, 2 * i + 1)
        c, s = cos.double()[:, None], sin.double()[:, None]
        z, mag = y.clone(), mag.clone()
        z[..., a], z[..., b] = y[..., a] * c - y[..., b] * s, y[..., b] * c + y[..., a] * s
        mag[..., a] = y[..., a].abs() * c.abs() + y[..., b].abs() * s.abs()
        mag[..., b] = y[..., b].abs() * c.abs() + y[..., a].abs() * s.abs()
        y = z
    return y, mag


def close_transform(torch, got, want, mag, dim, dtype):
    """One rounding to the type; before it the sum of squares (dim terms of one sign: dim * 2^-24 relative, halved by the
    root), the root, the products and the rotation: (dim / 2 + 12) * 2^-24 of the magnitudes."""
    tol = torch.finfo(dtype).eps / 2 * want.abs() + (dim / 2 + 12) * 2.0 ** -24 * mag * 1.01
    if dtype == torch.float16:
        tol = tol + 2.0 ** -25                                   # half a step of the subnormal range
    bad = (got.double() - want).abs() > tol
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst {float(((got.double() - want).abs() / tol).max())} x the tolerance"


@pytest.mark.parametrize("dim, dtype_name, heads, qheads, rotary, style, norm, n, page", [
    (64, "bfloat16", 2, 8, 64, "half", False, 1, 4096),
    (64, "bfloat16", 1, 1, 32, "pairs", True, 3, 8192),
    (128, "bfloat16", 8, 32, 128, "half", True, 65, 16384),
    (128, "float16", 3, 3, 64, "half", True, 500, 8192),
    (256, "bfloat16", 2, 10, 256, "pairs", False, 40, 32768),
    (256, "float16", 1, 7, 256, "half", True, 33, 16384),
    (80, "bfloat16", 5, 10, 80, "half", True, 77, 8192),
    (96, "float16", 4, 8, 48, "pairs", True, 130, 8192),
    (16, "bfloat16", 2, 2, 16, "half", True, 31, 4096),
    (112, "bfloat16", 2, 2, 96, "half", False, 64, 16384),
    (240, "float16", 2, 4, 16, "pairs", True, 20, 16384),
    (128, "bfloat16", 2, 2, 0, "half", False, 20, 16384),
])
def test_append_store_and_gather(cuda, bam, dim, dtype_name, heads, qheads, rotary, style, norm, n, page):
    torch = cuda
    dtype = getattr(torch, dtype_name)
    g = torch.Generator(device="cuda").manual_seed(dim * 1000 + n)
    blocks = n // 16 + 6
    kv = make(bam, torch, blocks, heads, dim, dtype, page=page, layers=2)
    total = blocks * kv.block_tokens
    # the rows that are not written stay as they were
    old_k, old_v = rand(torch, g, total, heads, dim, dtype=dtype), rand(torch, g, total, heads, dim, dtype=dtype)
    kv.append(old_k, old_v, torch.arange(total, device="cuda"), layer=1)
    qkv = rand(torch, g, n, qheads + 2 * heads, dim, dtype=dtype, scale=2.0)
    q, k, v = qkv.split([qheads, heads, heads], dim=1)
    slots = torch.randperm(total, generator=g, device="cuda")[:n]
    if n > 2:
        slots[1::7] = -1
    npos = 5000
    pos = torch.randint(0, npos, (n,), generator=g, device="cuda")
    args, cos, sin = {}, None, None
    if rotary:
        ang = torch.rand(npos, rotary // 2, generator=g, device="cuda", dtype=torch.float64) * 6.3
        cos, sin = ang.cos().float(), ang.sin().float()
        args.update(positions=pos, rope=(cos, sin), rope_style=style)
        cos, sin = cos[pos], sin[pos]
    qw = kw = None
    if norm:
        qw, kw = (1 + rand(torch, g, dim, dtype=torch.float32, scale=0.3)).to(dtype), (1 + rand(torch, g, dim, dtype=torch.float32, scale=0.3)).to(dtype)
        args.update(q_norm=qw, k_norm=kw, norm_eps=1e-5)
    before = qkv.clone()
    got_q = kv.append(k, v, slots, layer=1, q=q, **args)
    assert kv.cache.ctrl.status() == (0, "none", 0)
    assert torch.equal(qkv, before)                              # the inputs are left alone
    want_q, mag_q = transform64(torch, q, qw, 1e-5, cos, sin, style)
    want_k, mag_k = transform64(torch, k, kw, 1e-5, cos, sin, style)
    close_transform(torch, got_q, want_q, mag_q, dim, dtype)
    live = slots >= 0
    back_k, back_v = kv.gather(slots, layer=1)
    close_transform(torch, back_k[live], want_k[live], mag_k[live], dim, dtype)
    assert torch.equal(back_v[live], v[live])
    assert not back_k[~live].any() and not back_v[~live].any()
    # the store has the same rows, and the old ones everywhere else; the other layer is untouched
    sk, sv = store_rows(kv, torch, 1)
    assert torch.equal(sk[slots[live]], back_k[live]) and torch.equal(sv[slots[live]], back_v[live])
    rest = torch.ones(total, dtype=torch.bool, device="cuda")
    rest[slots[live]] = False
    assert torch.equal(sk[rest], old_k[rest]) and torch.equal(sv[rest], old_v[rest])
    # in place, and into rows of a wider tensor that lie on no 16-byte boundary
    wide = torch.zeros(n, qheads, dim + 6, dtype=dtype, device="cuda")
    odd = wide[..., 3:3 + dim]
    odd.copy_(q)
    assert kv.append(k, v, slots, layer=1, q=odd, q_out=odd, **args) is odd
    assert torch.equal(odd, got_q) and not wide[..., :3].any() and not wide[..., 3 + dim:].any()
    wk = torch.zeros(n, heads, dim + 2, dtype=dtype, device="cuda")
    wv = torch.zeros(n, heads, dim + 2, dtype=dtype, device="cuda")
    kv.gather(slots, layer=1, out=(wk[..., 1:1 + dim], wv[..., 1:1 + dim]))
    assert torch.equal(wk[..., 1:1 + dim], back_k) and torch.equal(wv[..., 1:1 + dim], back_v)
    assert not wk[..., 0].any() and not wk[..., -1].any()
    done(kv)


def test_append_and_gather_with_constant_eviction(cuda, bam):
    """A cache of 48 pages in front of 640: dirty pages leave through the write path and come back."""
    torch = cuda
    g = torch.Generator(device="cuda").manual_seed(4)
    kv = make(bam, torch, 160, 4, 64, torch.bfloat16, page=4096, slots=48, max_grid=3)
    total = 160 * kv.block_tokens
    k, v = rand(torch, g, total, 4, 64, dtype=torch.bfloat16), rand(torch, g, total, 4, 64, dtype=torch.bfloat16)
    order = torch.randperm(total, generator=g, device="cuda")
    kv.append(k[order], v[order], order)
    assert kv.cache.ctrl.status() == (0, "none", 0)
    other = torch.randperm(total, generator=g, device="cuda")
    bk, bv = kv.gather(other)
    assert torch.equal(bk, k[other]) and torch.equal(bv, v[other])
    sk, sv = store_rows(kv, torch)
    assert torch.equal(sk, k) and torch.equal(sv, v)
    done(kv)


def fill(torch, g, kv, lens, spare=3, layer=0):
    """Random rows everywhere and a random block table for sequences of these lengths; entries behind a sequence are
    no blocks at all."""
    T = kv.block_tokens
    need = [-(-n // T) for n in lens]
    assert sum(need) + spare <= kv.n_blocks
    order = torch.randperm(kv.n_blocks, generator=g, device="cuda")
    table = torch.full((len(lens), max(1, max(need))), -7, dtype=torch.int32, device="cuda")
    at = 0
    for i, m in enumerate(need):
        table[i, :m] = order[at:at + m]
        at += m
    total = kv.n_blocks * T
    k = rand(torch, g, total, kv.n_kv_heads, kv.head_dim, dtype=kv.dtype)
    v = rand(torch, g, total, kv.n_kv_heads, kv.head_dim, dtype=kv.dtype)
    return k, v, table


def attend64(torch, q, k, v, table, lens, T, scale, window=0, sinks=0):
    """(out, lse, tolerance of out without the last rounding, tolerance of lse) in 64 bits."""
    B, HQ, D = q.shape
    H = k.shape[1]
    out = torch.zeros(B, HQ, D, dtype=torch.float64, device="cuda")
    tol = torch.zeros_like(out)
    lse = torch.full((B, HQ), -float("inf"), dtype=torch.float64, device="cuda")
    ltol = torch.zeros_like(lse)
    for b, n in enumerate(lens):
        j = torch.arange(n, device="cuda")
        if window > 0:
            j = j[(j >= n - window) | (j < sinks)]
        if not len(j):
            continue
        rows = table[b].long()[j // T] * T + j % T
        kk, vv = k[rows].double(), v[rows].double()
        qq = q[b].double().view(H, HQ // H, D)
        s = torch.einsum("hgd,nhd->hgn", qq, kk) * scale
        p = torch.softmax(s, -1)
        out[b] = torch.einsum("hgn,nhd->hgd", p, vv).reshape(HQ, D)
        lse[b] = torch.logsumexp(s, -1).reshape(HQ)
        # a score is off by ds; a weight by 2 ds (its own and the denominator's), by the exponential's error (2^-21
        # with the argument's rounding at |s| < 32 counted in ds) and by what it is rounded to for the product
        ds = (torch.einsum("hgd,nhd->hgn", qq.abs(), kk.abs()).amax(-1) * abs(scale)) * (D + 4) * 2.0 ** -22 + s.abs().amax(-1) * 2.0 ** -22
        a = torch.einsum("hgn,nhd->hgd", p, vv.abs())
        rel = 2 * ds + 2.0 ** -16 + min(len(j), 1024) * 2.0 ** -22 + len(j) * 2.0 ** -24
        tol[b] = (a * rel[..., None]).reshape(HQ, D)
        ltol[b] = (ds + 2.0 ** -20 + len(j) * 2.0 ** -24 + lse[b].view(H, -1).abs() * 2.0 ** -22).reshape(HQ)
    return out, lse, tol, ltol


def check_attend(torch, got, lse, ref, dtype):
    out, want_lse, tol, ltol = ref
    tol = tol + torch.finfo(dtype).eps / 2 * (out.abs() + tol) + (2.0 ** -25 if dtype == torch.float16 else 0)
    err = (got.double() - out).abs()
    assert torch.isfinite(got).all()
    assert (err <= tol).all(), f"worst {float((err / tol.clamp(min=1e-30)).max())} x the tolerance at {divmod(int((err - tol).argmax()), got.shape[1] * got.shape[2])}"
    if lse is not None:
        none = want_lse == -float("inf")
        assert torch.equal(lse == -float("inf"), none)
        assert ((lse.double() - want_lse).abs()[~none] <= ltol[~none]).all()


LENS = {
    "short": [1, 0, 2, 15, 16, 17, 31, 32, 33, 0, 5],
    "edges": [63, 64, 65, 127, 128, 129, 255, 256, 257, 1, 0],
    "mixed": [700, 3, 0, 1111, 90, 16],
    "one": [1],
    "long": [9000],
    "twolong": [5001, 4097],
}


@pytest.mark.parametrize("dim, dtype_name, heads, group, page, lens, window, sinks", [
    (64, "bfloat16", 2, 4, 4096, "short", 0, 0),
    (64, "bfloat16", 2, 4, 8192, "edges", 0, 0),
    (128, "bfloat16", 8, 4, 16384, "mixed", 0, 0),
    (128, "float16", 2, 8, 8192, "edges", 0, 0),
    (128, "bfloat16", 1, 1, 16384, "one", 0, 0),
    (128, "bfloat16", 1, 16, 65536, "long", 0, 0),
    (128, "bfloat16", 1, 20, 16384, "twolong", 0, 0),
    (64, "float16", 1, 71, 4096, "mixed", 0, 0),
    (256, "bfloat16", 2, 5, 16384, "mixed", 0, 0),
    (256, "float16", 1, 16, 32768, "edges", 0, 0),
    (80, "bfloat16", 3, 1, 8192, "edges", 0, 0),
    (96, "float16", 2, 3, 16384, "mixed", 0, 0),
    (112, "bfloat16", 1, 2, 8192, "short", 0, 0),
    (16, "bfloat16", 2, 2, 4096, "mixed", 0, 0),
    (48, "bfloat16", 2, 2, 4096, "edges", 0, 0),
    (192, "bfloat16", 1, 8, 16384, "mixed", 0, 0),
    (240, "float16", 1, 3, 16384, "short", 0, 0),
    (128, "bfloat16", 2, 4, 16384, "edges", 1, 0),
    (128, "bfloat16", 2, 4, 8192, "mixed", 100, 4),
    (64, "bfloat16", 1, 8, 8192, "long", 1024, 17),
    (64, "bfloat16", 1, 8, 4096, "edges", 64, 300),
    (256, "float16", 1, 4, 16384, "mixed", 33, 1),
    (128, "bfloat16", 1, 4, 32768, "twolong", 4990, 12),
])
def test_attend_matches_64_bits(cuda, bam, dim, dtype_name, heads, group, page, lens, window, sinks):
    torch = cuda
    dtype, lens = getattr(torch, dtype_name), LENS[lens]
    g = torch.Generator(device="cuda").manual_seed(dim + group + len(lens))
    T = page // (4 * dim) // 16 * 16
    blocks = sum(-(-n // T) for n in lens) + 4
    kv = make(bam, torch, blocks, heads, dim, dtype, page=page, layers=2)
    k, v, table = fill(torch, g, kv, lens)
    # what no sequence may see: rows behind the lengths and, with a window, those before it
    seen = torch.zeros(blocks * T, dtype=torch.bool, device="cuda")
    for b, n in enumerate(lens):
        j = torch.arange(n, device="cuda")
        if window:
            j = j[(j >= n - window) | (j < sinks)]
        seen[table[b].long()[j // T] * T + j % T] = True
    hidden = (~seen).nonzero()[:, 0]
    pk, pv = k.clone(), v.clone()
    for value, part in ((float("nan"), hidden[0::3]), (float("inf"), hidden[1::3]), (-torch.finfo(dtype).max, hidden[2::3])):
        pk[part], pv[part] = value, value
    kv.append(pk, pv, torch.arange(blocks * T, device="cuda"), layer=1)
    if window:                                                   # blocks without a visible token need no table entry
        for b, n in enumerate(lens):
            for i in range(-(-n // T)):
                if i * T >= sinks and min(n, (i + 1) * T) <= n - window:
                    table[b, i] = 1 << 30
    q = rand(torch, g, len(lens), heads * group, dim, dtype=dtype, scale=3.0)
    ls = torch.tensor(lens, dtype=torch.int32, device="cuda")
    ref = attend64(torch, q, k, v, table.clamp(0, blocks - 1), lens, T, dim ** -0.5, window, sinks)
    out, lse = kv.attend(q, table, ls, layer=1, window=window, sinks=sinks, return_lse=True)
    assert kv.cache.ctrl.status() == (0, "none", 0)
    check_attend(torch, out, lse, ref, dtype)
    assert torch.equal(kv.attend(q, table, ls, layer=1, window=window, sinks=sinks), out)      # the same bits again
    # heads of a wider tensor on no boundary, an output with gaps, a table that is a part of a wider one
    wq = torch.zeros(len(lens), heads * group, dim + 3, dtype=dtype, device="cuda")
    wq[..., 1:1 + dim] = q
    wo = torch.full((len(lens), heads * group, dim + 5), 7.0, dtype=dtype, device="cuda")
    wt = torch.cat([table, torch.full_like(table, -3)], 1)[:, :table.shape[1]]
    o2 = kv.attend(wq[..., 1:1 + dim], wt, ls, layer=1, window=window, sinks=sinks, out=wo[..., 3:3 + dim])
    assert torch.equal(o2, out)
    assert (wo[..., :3] == 7).all() and (wo[..., 3 + dim:] == 7).all()
    done(kv)


@pytest.mark.parametrize("scale", [0.0, 1.0, -0.25])
def test_attend_scales(cuda, bam, scale):
    torch = cuda
    g = torch.Generator(device="cuda").manual_seed(3)
    lens = [40, 100, 1]
    kv = make(bam, torch, 14, 2, 64, torch.bfloat16, page=4096)
    k, v, table = fill(torch, g, kv, lens)
    kv.append(k, v, torch.arange(len(k), device="cuda"))
    q = rand(torch, g, 3, 4, 64, dtype=torch.bfloat16)
    out, lse = kv.attend(q, table, torch.tensor(lens, dtype=torch.int32, device="cuda"), scale=scale, return_lse=True)
    check_attend(torch, out, lse, attend64(torch, q, k, v, table, lens, kv.block_tokens, scale), torch.bfloat16)
    done(kv)


def test_attend_shared_blocks_and_many_sequences(cuda, bam):
    """300 sequences over one prefix: the same pages pinned by many at once; more sequences than worker blocks."""
    torch = cuda
    g = torch.Generator(device="cuda").manual_seed(8)
    kv = make(bam, torch, 320, 2, 64, torch.bfloat16, page=4096)
    T = kv.block_tokens
    k, v = rand(torch, g, 320 * T, 2, 64, dtype=torch.bfloat16), rand(torch, g, 320 * T, 2, 64, dtype=torch.bfloat16)
    kv.append(k, v, torch.arange(320 * T, device="cuda"))
    table = torch.empty(300, 5, dtype=torch.int32, device="cuda")
    table[:, :4] = torch.tensor([310, 2, 311, 2], dtype=torch.int32, device="cuda")          # one block twice
    table[:, 4] = torch.arange(300, device="cuda")
    lens = [(7 * i) % (5 * T + 1) for i in range(300)]
    q = rand(torch, g, 300, 8, 64, dtype=torch.bfloat16, scale=2.0)
    out, lse = kv.attend(q, table, torch.tensor(lens, dtype=torch.int32, device="cuda"), return_lse=True)
    check_attend(torch, out, lse, attend64(torch, q, k, v, table, lens, T, 0.125), torch.bfloat16)
    done(kv)


@pytest.mark.parametrize("ctrls, dist, slots, grid", [(1, 0, 40, 3), (1, 0, 700, 0), (2, 1, 60, 4), (2, 0, 600, 0)])
def test_attend_from_the_store(cuda, bam, ctrls, dist, slots, grid):
    """Contexts larger than the cache, over one controller, striped and replicated: pages are fetched and evicted while
    the attention runs."""
    torch = cuda
    g = torch.Generator(device="cuda").manual_seed(5)
    lens = [2000, 7, 1600, 0, 900]
    T = 16
    blocks = sum(-(-n // T) for n in lens) + 4
    kv = make(bam, torch, blocks, 3, 64, torch.bfloat16, page=4096, slots=slots, max_grid=grid, ctrls=ctrls, dist=dist)
    k, v, table = fill(torch, g, kv, lens)
    kv.append(k, v, torch.arange(len(k), device="cuda"))
    kv.cache.flush()
    q = rand(torch, g, len(lens), 6, 64, dtype=torch.bfloat16, scale=3.0)
    ls = torch.tensor(lens, dtype=torch.int32, device="cuda")
    ref = attend64(torch, q, k, v, table, lens, T, 0.125)
    kv.cache.stats(reset=True)
    for _ in range(3):
        out, lse = kv.attend(q, table, ls, return_lse=True)
        check_attend(torch, out, lse, ref, torch.bfloat16)
    assert kv.cache.ctrl.status() == (0, "none", 0)
    assert kv.cache.stats()["read_ios"] > 3 * (blocks * 3 - slots) // 2
    # a window leaves all but its own pages alone
    kv.cache.invalidate()
    kv.cache.stats(reset=True)
    out = kv.attend(q, table, ls, window=20, sinks=3)
    check_attend(torch, out, None, attend64(torch, q, k, v, table, lens, T, 0.125, 20, 3), torch.bfloat16)
    assert kv.cache.stats()["read_ios"] <= 4 * 3 * 4             # at most three pages of the window and one of the first tokens
    done(kv)


@pytest.mark.parametrize("what", ["block", "negative", "length", "minus"])
def test_bad_indices_are_reported_and_not_followed(cuda, bam, what):
    torch = cuda
    g = torch.Generator(device="cuda").manual_seed(6)
    lens = [50, 33]
    kv = make(bam, torch, 10, 2, 64, torch.bfloat16, page=4096)
    k, v, table = fill(torch, g, kv, lens)
    every = torch.arange(len(k), device="cuda")
    kv.append(k, v, every)
    q = rand(torch, g, 2, 4, 64, dtype=torch.bfloat16)
    ls = torch.tensor(lens, dtype=torch.int32, device="cuda")
    bad_t, bad_l = table.clone(), ls.clone()
    if what == "block":
        bad_t[0, 1] = 10
    elif what == "negative":
        bad_t[1, 0] = -1
    elif what == "length":
        bad_l[0] = table.shape[1] * kv.block_tokens + 1
    else:
        bad_l[1] = -1
    kv.attend(q, bad_t, bad_l)
    code, where, _ = kv.cache.ctrl.status(clear=True)
    assert (code, where) == (34, "range")
    assert kv.cache.audit() == 0
    out, lse = kv.attend(q, table, ls, return_lse=True)           # the cache works on
    check_attend(torch, out, lse, attend64(torch, q, k, v, table, lens, kv.block_tokens, 0.125), torch.bfloat16)
    slots = every[:3].clone()
    slots[1] = 10 * kv.block_tokens
    kv.gather(slots)
    assert kv.cache.ctrl.status(clear=True)[:2] == (34, "range")
    kv.append(k[:3], v[:3], slots)
    assert kv.cache.ctrl.status(clear=True)[:2] == (34, "range")
    cos = torch.ones(4, 32, device="cuda")
    for p in (4, -1):
        pos = torch.tensor([0, p, 1], device="cuda")
        kv.append(k[:3], v[:3], every[:3], positions=pos, rope=(cos, cos))
        assert kv.cache.ctrl.status(clear=True)[:2] == (34, "range")
    done(kv)


def test_c_entries_refuse(cuda, bam):
    import ctypes as C
    from bam_b200 import _lib
    torch = cuda
    kv = make(bam, torch, 10, 2, 64, torch.bfloat16, page=4096)
    lib, h = kv.lib, kv.array.h
    EINVAL, ERANGE = 22, 34
    scratch = torch.empty(kv._scratch_bytes + 256, dtype=torch.uint8, device="cuda")
    sp, sb = scratch.data_ptr(), kv._scratch_bytes
    assert lib.bam_kv_scratch_init(None, sp, sb, None) == EINVAL and lib.bam_kv_scratch_init(h, None, sb, None) == EINVAL
    assert lib.bam_kv_scratch_init(h, sp + 64, sb, None) == EINVAL and lib.bam_kv_scratch_init(h, sp, 64, None) == EINVAL
    assert lib.bam_kv_scratch_init(h, sp, sb, None) == 0
    t = torch.zeros(4096, dtype=torch.bfloat16, device="cuda")
    i64, i32, f = (torch.zeros(64, dtype=d, device="cuda") for d in (torch.int64, torch.int32, torch.float32))
    good = dict(dtype=0, head_dim=64, n_kv_heads=2, block_tokens=16, n_blocks=10, first_page=0)
    L = lambda **c: C.byref(_lib.KvLayout(**{**good, **c}))       # noqa: E731
    two = (C.c_int64 * 2)(128, 64)
    for c, code in ((dict(dtype=2), EINVAL), (dict(head_dim=72), EINVAL), (dict(head_dim=272), EINVAL), (dict(block_tokens=8), EINVAL),
                    (dict(block_tokens=32), EINVAL), (dict(n_kv_heads=0), EINVAL), (dict(n_blocks=0), EINVAL),
                    (dict(n_blocks=11), ERANGE), (dict(first_page=1), ERANGE), (dict(first_page=1 << 63), ERANGE)):
        assert lib.bam_kv_scratch_bytes(h, L(**c)) == 0
        assert lib.bam_launch_kv_gather(h, L(**c), 1, i64.data_ptr(), t.data_ptr(), t.data_ptr(), two, two, sp, sb, None) == code
    ap = dict(k=t.data_ptr(), v=t.data_ptr(), k_stride=(128, 64), v_stride=(128, 64), n_tokens=1, slots=i64.data_ptr())
    rope = dict(cos=f.data_ptr(), sin=f.data_ptr(), positions=i64.data_ptr(), n_positions=1, rope_stride=32, rotary_dim=64)

    def append(scratch=sp, size=sb, **c):
        a = _lib.KvAppend()
        for name, value in {**ap, **c}.items():
            if isinstance(value, tuple):
                getattr(a, name)[:] = value
            else:
                setattr(a, name, value)
        return lib.bam_launch_kv_append(h, L(), C.byref(a), scratch, size, None)
    assert append() == 0 and append(**rope) == 0 and append(n_tokens=0) == 0
    for c in (dict(k=None), dict(v=None), dict(slots=None), dict(n_tokens=1 << 31), dict(q=t.data_ptr()), dict(scratch=None), dict(scratch=sp + 64),
              dict(size=sb - 1), dict(rope, sin=None), dict(rope, positions=None), dict(rope, n_positions=0), dict(rope, rotary_dim=24),
              dict(rope, rotary_dim=80), dict(rope, rope_stride=-1), dict(rope, rope_style=2), dict(k_norm=t.data_ptr(), norm_eps=-1.0),
              dict(k_norm=t.data_ptr(), norm_eps=float("nan")), dict(q=t.data_ptr(), q_out=t.data_ptr(), n_q_heads=0),
              dict(k=t.data_ptr() + 1), dict(v=t.data_ptr() + 1), dict(slots=i64.data_ptr() + 4), dict(rope, cos=f.data_ptr() + 2),
              dict(rope, positions=i64.data_ptr() + 4), dict(q=t.data_ptr(), q_out=t.data_ptr() + 1, n_q_heads=2)):
        assert append(**c) == EINVAL, c
    at = dict(q=t.data_ptr(), out=t.data_ptr(), q_stride=(128, 64), out_stride=(128, 64), block_table=i32.data_ptr(), seq_lens=i32.data_ptr(),
              table_stride=1, batch=1, n_q_heads=2, table_width=1, scale=0.1)

    def attend(scratch=sp, size=sb, **c):
        a = _lib.KvAttend()
        for name, value in {**at, **c}.items():
            if isinstance(value, tuple):
                getattr(a, name)[:] = value
            else:
                setattr(a, name, value)
        return lib.bam_launch_kv_attend(h, L(), C.byref(a), scratch, size, None)
    assert attend() == 0 and attend(batch=0) == 0
    for c in (dict(q=None), dict(out=None), dict(block_table=None), dict(seq_lens=None), dict(n_q_heads=3), dict(n_q_heads=0), dict(table_width=0),
              dict(window=-1), dict(sinks=-1), dict(scale=float("nan")), dict(scale=float("inf")), dict(batch=(1 << 20) + 1), dict(size=0), dict(scratch=None),
              dict(q=t.data_ptr() + 1), dict(out=t.data_ptr() + 1), dict(lse=f.data_ptr() + 2), dict(block_table=i32.data_ptr() + 2),
              dict(seq_lens=i32.data_ptr() + 2)):
        assert attend(**c) == EINVAL, c
    for c in ((i64.data_ptr() + 4, t.data_ptr(), t.data_ptr()), (i64.data_ptr(), t.data_ptr() + 1, t.data_ptr()), (i64.data_ptr(), t.data_ptr(), t.data_ptr() + 1)):
        assert lib.bam_launch_kv_gather(h, L(), 1, *c, two, two, sp, sb, None) == EINVAL
    # an array that starts inside a page is refused
    a2 = bam.Array.from_ranges(kv.cache, 512, [(0, 512, 0, 64)])
    assert lib.bam_kv_scratch_bytes(a2.h, L(n_blocks=1, n_kv_heads=1)) == 0
    a2.close()
    torch.cuda.synchronize()
    done(kv)


def test_captured_graphs(cuda, bam):
    """Append and attend of a decode step in two graphs that are replayed in turn and over new inputs, the second on
    another stream; eager calls in between."""
    torch = cuda
    g = torch.Generator(device="cuda").manual_seed(7)
    B, T = 6, 16
    lens = [100, 1, 300, 17, 0, 64]
    kv = make(bam, torch, 64, 2, 64, torch.bfloat16, page=4096)
    k, v, table = fill(torch, g, kv, [n + 4 for n in lens])
    kv.append(k, v, torch.arange(len(k), device="cuda"))
    cos = torch.rand(400, 32, generator=g, device="cuda")
    sin = torch.rand(400, 32, generator=g, device="cuda")
    qkv = torch.zeros(B, 8 + 4, 64, dtype=torch.bfloat16, device="cuda")
    slots, pos = torch.zeros(B, dtype=torch.int64, device="cuda"), torch.zeros(B, dtype=torch.int64, device="cuda")
    ls = torch.zeros(B, dtype=torch.int32, device="cuda")

    def step():
        q, kk, vv = qkv.split([8, 2, 2], dim=1)
        q2 = kv.append(kk, vv, slots, positions=pos, rope=(cos, sin), q=q)
        return q2, kv.attend(q2, table, ls)
    slots.fill_(-1)
    step()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            res = step()
        graphs.append((gr, res))
    side = torch.cuda.Stream()
    now = list(lens)
    for it in range(4):
        fresh = rand(torch, g, *qkv.shape, dtype=torch.bfloat16)
        qkv.copy_(fresh)
        at = torch.tensor(now, device="cuda")
        pos.copy_(at)
        slots.copy_(table.long().gather(1, (at // T)[:, None])[:, 0] * T + at % T)
        ls.copy_(at + 1)
        now = [n + 1 for n in now]
        gr, (q2, out) = graphs[it % 2]
        if it % 2:
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                gr.replay()
            torch.cuda.current_stream().wait_stream(side)
        else:
            gr.replay()
        q, kk, vv = fresh.split([8, 2, 2], dim=1)
        c, s = cos[pos], sin[pos]
        wq, mq = transform64(torch, q, None, 0, c, s, "half")
        close_transform(torch, q2, wq, mq, 64, torch.bfloat16)
        bk, bv = kv.gather(slots)                                # an eager call on the same cache
        wk, mk = transform64(torch, kk, None, 0, c, s, "half")
        close_transform(torch, bk, wk, mk, 64, torch.bfloat16)
        assert torch.equal(bv, vv)
        k[slots], v[slots] = bk, bv
        check_attend(torch, out, None, attend64(torch, q2, k, v, table, now, T, 0.125), torch.bfloat16)
    assert kv.cache.ctrl.status() == (0, "none", 0)
    del graphs, gr, res
    done(kv)


def test_two_streams_and_caches_at_once(cuda, bam):
    """Calls that run at the same time: two streams on one cache."""
    torch = cuda
    g = torch.Generator(device="cuda").manual_seed(9)
    lens = [800, 30, 400]
    kv = make(bam, torch, 90, 2, 64, torch.bfloat16, page=4096)
    k, v, table = fill(torch, g, kv, lens)
    kv.append(k, v, torch.arange(len(k), device="cuda"))
    q = rand(torch, g, 3, 8, 64, dtype=torch.bfloat16, scale=2.0)
    ls = torch.tensor(lens, dtype=torch.int32, device="cuda")
    ref = attend64(torch, q, k, v, table, lens, kv.block_tokens, 0.125)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = []
    for i in range(20):
        outs.append(kv.attend(q, table, ls, stream=streams[i % 2] if i % 3 else streams[i % 2].cuda_stream))
    torch.cuda.synchronize()
    for o in outs:
        check_attend(torch, o, None, ref, torch.bfloat16)
    with pytest.raises(ValueError):
        kv.attend(q.cpu(), table, ls)
    done(kv)


def test_decode_loop_matches_plain(cuda, bam):
    """The operators as they are used together: a prompt is appended, its context gathered, then tokens are decoded one
    by one through two layers with normed and rotated heads, in a cache that does not hold all pages."""
    torch = cuda
    g = torch.Generator(device="cuda").manual_seed(10)
    B, H, HQ, D, T = 3, 2, 6, 64, 16
    prompt = [90, 1, 200]
    blocks = sum(-(-(n + 8) // T) for n in prompt) + 2
    kv = make(bam, torch, blocks, H, D, torch.bfloat16, page=4096, slots=70, layers=2, max_grid=4)
    order = torch.randperm(blocks, generator=g, device="cuda").int()
    table = torch.full((B, 14), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(prompt):
        m = -(-(n + 8) // T)
        table[b, :m] = order[at:at + m]
        at += m
    cos, sin = torch.rand(256, 16, generator=g, device="cuda"), torch.rand(256, 16, generator=g, device="cuda")
    w = (1 + rand(torch, g, 4, D, dtype=torch.float32, scale=0.2)).bfloat16()
    mirror = [[torch.zeros(blocks * T, H, D, dtype=torch.bfloat16, device="cuda") for _ in range(2)] for _ in range(2)]

    def slots_of(b, p):
        return table[b].long()[p // T] * T + p % T
    for layer in range(2):
        slots = torch.cat([slots_of(b, torch.arange(n, device="cuda")) for b, n in enumerate(prompt)])
        pos = torch.cat([torch.arange(n, device="cuda") for n in prompt])
        x = rand(torch, g, len(pos), HQ + 2 * H, D, dtype=torch.bfloat16)
        q, k, v = x.split([HQ, H, H], dim=1)
        kv.append(k, v, slots, layer=layer, positions=pos, rope=(cos, sin), q=q, q_norm=w[2 * layer], k_norm=w[2 * layer + 1])
        wk, mk = transform64(torch, k, w[2 * layer + 1], 1e-6, cos[pos], sin[pos], "half")
        bk, bv = kv.gather(slots, layer=layer)
        close_transform(torch, bk, wk, mk, D, torch.bfloat16)
        mirror[layer][0][slots], mirror[layer][1][slots] = bk, v
    now = torch.tensor(prompt, device="cuda")
    for step in range(6):
        for layer in range(2):
            x = rand(torch, g, B, HQ + 2 * H, D, dtype=torch.bfloat16)
            q, k, v = x.split([HQ, H, H], dim=1)
            slots = torch.stack([slots_of(b, now[b]) for b in range(B)])
            q2 = kv.append(k, v, slots, layer=layer, positions=now, rope=(cos, sin), q=q, q_norm=w[2 * layer], k_norm=w[2 * layer + 1])
            wk, mk = transform64(torch, k, w[2 * layer + 1], 1e-6, cos[now], sin[now], "half")
            bk, bv = kv.gather(slots, layer=layer)
            close_transform(torch, bk, wk, mk, D, torch.bfloat16)
            mirror[layer][0][slots], mirror[layer][1][slots] = bk, v
            window = 0 if layer == 0 else 50
            out, lse = kv.attend(q2, table, (now + 1).int(), layer=layer, window=window, sinks=2, return_lse=True)
            ref = attend64(torch, q2, mirror[layer][0], mirror[layer][1], table, (now + 1).tolist(), T, D ** -0.5, window, 2)
            check_attend(torch, out, lse, ref, torch.bfloat16)
        now = now + 1
    done(kv)


def test_lost_completion_ends_the_call_with_a_status(cuda, bam):
    """The controller swallows a completion (host-configured): the waits run out, the launch drains and says so."""
    torch = cuda
    g = torch.Generator(device="cuda").manual_seed(11)
    lens = [600, 600]
    kv = make(bam, torch, 80, 1, 64, torch.bfloat16, page=4096)
    k, v, table = fill(torch, g, kv, lens)
    kv.append(k, v, torch.arange(len(k), device="cuda"))
    kv.cache.flush()
    kv.cache.invalidate()
    ctrl = kv.cache.ctrl
    ctrl.configure(spin_timeout_ns=300 * MS)
    ctrl.inject_fault(1, nth=20)
    q = rand(torch, g, 2, 4, 64, dtype=torch.bfloat16)
    ls = torch.tensor(lens, dtype=torch.int32, device="cuda")
    kv.attend(q, table, ls)
    assert ctrl.status(clear=True)[0] in (110, 5)
    ctrl.inject_fault(0)
    ctrl.configure(spin_timeout_ns=5 * SEC)
    ctrl.reset_queues()
    kv.cache.invalidate()
    out = kv.attend(q, table, ls)
    check_attend(torch, out, None, attend64(torch, q, k, v, table, lens, kv.block_tokens, 0.125), torch.bfloat16)
    done(kv)


def test_empty_calls(cuda, bam):
    torch = cuda
    kv = make(bam, torch, 4, 2, 64, torch.float16, page=4096)
    e = torch.zeros(0, 2, 64, dtype=torch.float16, device="cuda")
    none = torch.zeros(0, dtype=torch.int64, device="cuda")
    assert kv.append(e, e, none) is None
    assert kv.append(e, e, none, q=e).shape == (0, 2, 64)
    assert [x.shape[0] for x in kv.gather(none)] == [0, 0]
    out, lse = kv.attend(e, torch.zeros(0, 3, dtype=torch.int32, device="cuda"), torch.zeros(0, dtype=torch.int32, device="cuda"), return_lse=True)
    assert out.shape == (0, 2, 64) and lse.shape == (0, 2)
    # nothing but empty and padding rows
    z = torch.zeros(3, dtype=torch.int32, device="cuda")
    q = torch.ones(3, 2, 64, dtype=torch.float16, device="cuda")
    out, lse = kv.attend(q, torch.full((3, 1), -1, dtype=torch.int32, device="cuda"), z, return_lse=True)
    assert not out.any() and (lse == -float("inf")).all()
    pads = torch.full((3,), -1, dtype=torch.int64, device="cuda")
    kv.append(q, q, pads)
    assert kv.cache.stats()["accesses"] == 0
    done(kv)


def test_more_heads_than_lanes_and_angles_of_one_row(cuda, bam):
    """40 key/value heads; angles that are one row for all positions; a page that its block does not fill; windows and
    numbers of first tokens beyond any length."""
    torch = cuda
    g = torch.Generator(device="cuda").manual_seed(12)
    H, D = 40, 32
    kv = make(bam, torch, 9, H, D, torch.bfloat16, page=8192, tokens=48)
    T = 48
    lens = [100, 48, 5, 0, 47]
    k, v, table = fill(torch, g, kv, lens, spare=0)
    n = len(k)
    row = torch.rand(1, D // 2, generator=g, device="cuda")
    cos, sin = row.expand(n, -1), row.expand(n, -1)
    q = rand(torch, g, n, H, D, dtype=torch.bfloat16)
    at = torch.arange(n, device="cuda")
    got = kv.append(k, v, at, positions=at, rope=(cos, sin), q=q)
    wq, mq = transform64(torch, q, None, 0, cos, sin, "half")
    close_transform(torch, got, wq, mq, D, torch.bfloat16)
    wk, mk = transform64(torch, k, None, 0, cos, sin, "half")
    bk, bv = kv.gather(at)
    close_transform(torch, bk, wk, mk, D, torch.bfloat16)
    assert torch.equal(bv, v)
    q = rand(torch, g, len(lens), 2 * H, D, dtype=torch.bfloat16, scale=2.0)
    ls = torch.tensor(lens, dtype=torch.int32, device="cuda")
    ref = attend64(torch, q, bk, bv, table, lens, T, D ** -0.5)
    for window, sinks in ((0, 0), (1 << 70, 0), (3, 1 << 70), (100, 0)):
        out, lse = kv.attend(q, table, ls, window=window, sinks=sinks, return_lse=True)
        check_attend(torch, out, lse, ref, torch.bfloat16)
    assert kv.cache.ctrl.status() == (0, "none", 0)
    done(kv)


def test_values_that_are_not_finite_in_visible_rows(cuda, bam):
    """A score of +infinity or NaN makes its row NaN, as the formula has it; -infinity hides its token; other sequences and
    heads do not notice."""
    torch = cuda
    g = torch.Generator(device="cuda").manual_seed(13)
    lens = [70, 70, 70, 40]
    kv = make(bam, torch, 24, 1, 64, torch.bfloat16, page=4096)
    k, v, table = fill(torch, g, kv, lens)
    T = kv.block_tokens
    k = k.abs()
    at = lambda b, j: table[b].long()[j // T] * T + j % T           # noqa: E731
    k[at(0, 33), 0, 5] = float("inf")
    k[at(1, 69), 0, 5] = float("nan")
    k[at(2, 10), 0, 5] = float("-inf")
    v[at(2, 10)] = 3.0
    kv.append(k, v, torch.arange(len(k), device="cuda"))
    q = rand(torch, g, 4, 2, 64, dtype=torch.bfloat16).abs() + 0.25
    out, lse = kv.attend(q.bfloat16(), table, torch.tensor(lens, dtype=torch.int32, device="cuda"), return_lse=True)
    assert torch.isnan(out[:2]).all() and torch.isnan(lse[:2]).all()
    k[at(2, 10), 0, 5] = -1e30                                         # hidden all the same, and finite in 64 bits
    ref = attend64(torch, q.bfloat16()[2:], k, v, table[2:], lens[2:], T, 0.125)
    err = (out[2:].double() - ref[0]).abs()
    assert (err <= 2.0 ** -7 * ref[0].abs() + 2.0 ** -7).all()
    done(kv)


def test_offsets_beyond_32_bits(cuda, bam):
    """More than 4 GiB of cache memory and of store: one token in every page of a megabyte, read back and attended to."""
    torch = cuda
    g = torch.Generator(device="cuda").manual_seed(14)
    blocks, D, page = 4400, 256, 1 << 20
    kv = make(bam, torch, blocks, 1, D, torch.bfloat16, page=page)
    T = kv.block_tokens
    assert T == 1024
    first = torch.arange(blocks, device="cuda") * T
    k, v = rand(torch, g, blocks, 1, D, dtype=torch.bfloat16), rand(torch, g, blocks, 1, D, dtype=torch.bfloat16)
    kv.append(k, v, first)
    assert kv.cache.ctrl.status() == (0, "none", 0)
    bk, bv = kv.gather(first.flip(0))
    assert torch.equal(bk, k.flip(0)) and torch.equal(bv, v.flip(0))
    table = torch.tensor([[blocks - 1], [blocks - 2], [0]], dtype=torch.int32, device="cuda")
    q = rand(torch, g, 3, 2, D, dtype=torch.bfloat16)
    out = kv.attend(q, table, torch.ones(3, dtype=torch.int32, device="cuda"))
    assert torch.equal(out, v[table[:, 0].long()].expand(3, 2, D))     # one visible token: its value
    assert kv.cache.ctrl.status() == (0, "none", 0)
    done(kv)


def test_attend_in_place_and_slots_that_repeat(cuda, bam):
    """`out` is q: the warps that share a sequence write its rows when all of them have read q.  A slot may be gathered
    more than once."""
    torch = cuda
    g = torch.Generator(device="cuda").manual_seed(15)
    lens = [3000, 5, 0, 700]
    kv = make(bam, torch, 240, 2, 64, torch.bfloat16, page=4096)
    k, v, table = fill(torch, g, kv, lens)
    kv.append(k, v, torch.arange(len(k), device="cuda"))
    ls = torch.tensor(lens, dtype=torch.int32, device="cuda")
    for width in (64, 67):                                       # rows that share 32-byte sectors, too
        q = torch.zeros(4, 24, width, dtype=torch.bfloat16, device="cuda")[..., width - 64:]
        q.copy_(rand(torch, g, 4, 24, 64, dtype=torch.bfloat16, scale=2.0))
        want = kv.attend(q, table, ls)
        assert kv.attend(q, table, ls, out=q) is q
        assert torch.equal(q, want)
    slots = torch.randint(0, 40, (500,), generator=g, device="cuda")
    bk, bv = kv.gather(slots)
    assert torch.equal(bk, k[slots]) and torch.equal(bv, v[slots])
    done(kv)


def test_launches_that_fetch_at_once(cuda, bam):
    """Attention over one cache and a gather from a second one, both with more pages than slots, and a page scan through a
    third, on three streams over one controller: each launch's controller blocks serve the others' commands, too."""
    torch = cuda
    g = torch.Generator(device="cuda").manual_seed(16)
    lens, page, blocks = [1500, 700, 900], 4096, 200
    c = bam.Controller(blocks * 4 * page, 0, queue_depth=64, num_queues=16)
    c.configure(ctrl_blocks=2, spin_timeout_ns=5 * SEC)
    c.set_launch_timeout(30 * SEC)
    c.set_max_grid(24)
    caches = [bam.PageCache(c, page, slots) for slots in (150, 150, 2 * blocks + 8)]
    kvs = [bam.KvCache(caches[i], blocks, 2, 64, store_byte_offset=i * blocks * 2 * page) for i in range(2)]
    k, v, table = fill(torch, g, kvs[0], lens)
    every = torch.arange(len(k), device="cuda")
    kvs[0].append(k, v, every)
    kvs[1].append(v, k, every)
    for cache in caches:
        cache.flush()
    scanned = bam.Array(caches[2], blocks * 2 * page // 8)
    assert c.status() == (0, "none", 0)
    words = int(torch.from_numpy(c.store_numpy("int64")[:blocks * 2 * page // 8].copy()).sum())
    q = rand(torch, g, 3, 8, 64, dtype=torch.bfloat16, scale=2.0)
    ls = torch.tensor(lens, dtype=torch.int32, device="cuda")
    ref = attend64(torch, q, k, v, table, lens, kvs[0].block_tokens, 0.125)
    order = [torch.randperm(len(k), generator=g, device="cuda") for _ in range(4)]
    sums = torch.zeros(4, dtype=torch.int64, device="cuda")
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    outs, rows = [], []
    for i in range(4):
        outs.append(kvs[0].attend(q, table, ls, stream=streams[0]))
        rows.append(kvs[1].gather(order[i], stream=streams[1]))
        scanned.page_scan(blocks * 2, sums[i:], stream=streams[2].cuda_stream)
    torch.cuda.synchronize()
    assert c.status() == (0, "none", 0)
    for i in range(4):
        check_attend(torch, outs[i], None, ref, torch.bfloat16)
        assert torch.equal(rows[i][0], v[order[i]]) and torch.equal(rows[i][1], k[order[i]])
        assert int(sums[i]) == words
    for x, cache in zip((*kvs, scanned), caches):
        assert cache.audit() == 0
        x.close(); cache.close()
    c.close()
