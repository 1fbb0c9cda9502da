"""The operators of the paged key/value cache, in cases of their real range.

  append   new keys and values go into the pages of the cache, normed and rotated on the way, and the queries take the same pass;
           the rows are then read back, as a prompt that is worked off in chunks reads its context
  gather   the rows of whole sequences are read back from their pages
  attend   one new token per sequence attends over its paged keys and values, whole or through a window with first tokens

`run` computes them in plain torch operations, in 32 bits and rounded once; with `own` set it makes the framework's calls.
"""
import math
import random

import numpy as np
import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # one short conversation on a small model: what counts is the time of a call
        dict(name="attend one short", op="attend", batch=1, q_heads=8, kv_heads=2, head_dim=64, dtype="bf16", page=4096,
             shortest=37, longest=37, window=0, sinks=0, empty=0, resident=True),
        # a serving batch of ordinary lengths
        dict(name="attend batch", op="attend", batch=32, q_heads=32, kv_heads=8, head_dim=128, dtype="bf16", page=16384,
             shortest=130, longest=1700, window=0, sinks=0, empty=0, resident=True),
        # two long documents, few key heads: the length itself has to be split
        dict(name="attend long", op="attend", batch=2, q_heads=16, kv_heads=2, head_dim=128, dtype="bf16", page=8192,
             shortest=60000, longest=70001, window=0, sinks=0, empty=0, resident=True),
        # the largest: a full batch of long contexts
        dict(name="attend full", op="attend", batch=64, q_heads=64, kv_heads=8, head_dim=128, dtype="bf16", page=16384,
             shortest=2500, longest=4100, window=0, sinks=0, empty=0, resident=True),
        # wide heads, odd head counts, 16-bit floats, a batch padded with empty rows
        dict(name="attend wide padded", op="attend", batch=23, q_heads=15, kv_heads=3, head_dim=256, dtype="fp16", page=16384,
             shortest=1, longest=2000, window=0, sinks=0, empty=5, resident=True),
        # long contexts of which a window and the first tokens are visible
        dict(name="attend window", op="attend", batch=48, q_heads=16, kv_heads=2, head_dim=128, dtype="bf16", page=8192,
             shortest=3000, longest=9000, window=1024, sinks=4, empty=0, resident=True),
        # contexts four times the size of the cache: the pages come from the store in host memory
        dict(name="attend from store", op="attend", batch=4, q_heads=16, kv_heads=4, head_dim=64, dtype="bf16", page=4096,
             shortest=12000, longest=20000, window=0, sinks=0, empty=0, resident=False),
        # the new token of one sequence
        dict(name="append one token", op="append", tokens=1, sequences=1, q_heads=8, kv_heads=2, head_dim=64, dtype="bf16", page=4096,
             rotary=64, style="half", norm=False, context=100, padded=0),
        # the new tokens of a serving batch, with normed heads
        dict(name="append batch", op="append", tokens=200, sequences=200, q_heads=32, kv_heads=8, head_dim=128, dtype="bf16", page=16384,
             rotary=128, style="half", norm=True, context=1500, padded=0),
        # chunks of prompts, ragged, padded, a part of each head rotated in pairs
        dict(name="append chunks", op="append", tokens=777, sequences=3, q_heads=15, kv_heads=3, head_dim=256, dtype="fp16", page=16384,
             rotary=64, style="pairs", norm=False, context=300, padded=9),
        # a long prompt at once
        dict(name="append prompt", op="append", tokens=16000, sequences=2, q_heads=32, kv_heads=8, head_dim=128, dtype="bf16", page=16384,
             rotary=128, style="half", norm=True, context=0, padded=0),
        # the context of a prompt's next chunk, read back
        dict(name="gather context", op="gather", tokens=30001, sequences=3, kv_heads=8, head_dim=128, dtype="bf16", page=16384),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "append", "append", "gather"])
    dim = rng.choice([64, 64, 80, 96, 128, 128, 256])
    page = rng.choice([p for p in (4096, 8192, 16384, 32768) if p // (4 * dim) >= 16])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    kv = rng.choice([1, 2, 3, 4, 8])
    group = rng.choice([1, 2, 4, 5, 7, 8, 16])
    if op == "attend":
        batch = _log(rng, 1, 96)
        most = max(2, min(70000, (1 << 29) // (batch * kv * dim * 4)))
        longest = _log(rng, 1, most)
        window = rng.choice([0, 0, _log(rng, 1, 2 * longest)])
        return dict(op=op, batch=batch, q_heads=kv * group, kv_heads=kv, head_dim=dim, dtype=dtype, page=page,
                    shortest=rng.randint(1, longest), longest=longest, window=window, sinks=rng.choice([0, 1, 4, 17]) if window else 0,
                    empty=rng.choice([0, 0, 3]), resident=rng.random() < 0.85 or batch * longest * kv * dim > 1 << 24)
    tokens = _log(rng, 1, max(1, min(20000, (1 << 26) // (kv * (group + 2) * dim))))
    if op == "append":
        style = rng.choice(["half", "half", "pairs"])
        return dict(op=op, tokens=tokens, sequences=min(tokens, _log(rng, 1, 200)), q_heads=kv * group, kv_heads=kv, head_dim=dim,
                    dtype=dtype, page=page, rotary=rng.choice([dim, dim, dim // 32 * 16]), style=style, norm=rng.random() < 0.5,
                    context=rng.randint(0, 2000), padded=rng.choice([0, 0, 7]))
    return dict(op=op, tokens=tokens, sequences=min(tokens, _log(rng, 1, 64)), kv_heads=kv, head_dim=dim, dtype=dtype, page=page)


def _lengths(case, seed):
    """The lengths of a case's sequences: whole numbers on the host."""
    rng = random.Random(seed * 7919 + 11)
    if case["op"] == "attend":
        got = [rng.randint(case["shortest"], case["longest"]) for _ in range(case["batch"])]
        return [0 if case["empty"] and i % case["empty"] == 1 else n for i, n in enumerate(got)]
    n, left = case["sequences"], case["tokens"]
    cuts = sorted(rng.sample(range(1, left), n - 1)) if n > 1 else []
    return [b - a for a, b in zip([0] + cuts, cuts + [left])]


def _block_tokens(case):
    return case["page"] // (4 * case["head_dim"]) // 16 * 16


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rng = np.random.default_rng(seed + 1)
    dt, dim, kv, bt = TYPES[case["dtype"]], case["head_dim"], case["kv_heads"], _block_tokens(case)
    lens = _lengths(case, seed)
    context = case.get("context", 0)
    total = [n + context if case["op"] == "append" else n for n in lens]
    need = [-(-n // bt) for n in total]
    blocks = sum(need) + 3
    order = rng.permutation(blocks).astype(np.int64)
    table = np.full((len(lens), max(1, max(need))), -1, dtype=np.int64)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    s = dict(case=dict(case), bt=bt, blocks=blocks)

    def rand(*shape):
        return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(dt)

    s["pool_k"], s["pool_v"] = rand(blocks, bt, kv, dim), rand(blocks, bt, kv, dim)
    if case["op"] == "attend":
        s["q"] = (torch.randn((case["batch"], case["q_heads"], dim), generator=g, device="cuda") * 3).to(dt)
        s["table"] = torch.from_numpy(table.astype(np.int32)).cuda()
        s["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
        s["most"] = max(_visible(case, n) for n in lens)
        if not case["resident"]:
            s["table_host"], s["lens_host"] = torch.from_numpy(table), torch.tensor(lens)
    else:
        first = context if case["op"] == "append" else 0
        slots, positions = [], []
        for i, n in enumerate(lens):
            p = np.arange(first, first + n, dtype=np.int64)
            positions.append(p)
            slots.append(table[i, p // bt] * bt + p % bt)
        slots, positions = np.concatenate(slots), np.concatenate(positions)
        if case["op"] == "append":
            if case["padded"]:
                slots[case["padded"] - 1::case["padded"]] = -1
            heads = case["q_heads"] + 2 * kv
            qkv = rand(case["tokens"], heads * dim).view(case["tokens"], heads, dim)       # what one projection gives
            s["q"], s["k"], s["v"] = qkv.split([case["q_heads"], kv, kv], dim=1)
            half = case["rotary"] // 2
            angle = torch.arange(int(positions.max()) + 1, device="cuda", dtype=torch.float64)[:, None] * \
                torch.pow(torch.tensor(10000.0, dtype=torch.float64, device="cuda"),
                          -torch.arange(half, device="cuda", dtype=torch.float64) / half)
            s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
            s["positions"] = torch.from_numpy(positions).cuda()
            s["q_norm"], s["k_norm"] = (1 + 0.2 * rand(dim).float()).to(dt), (1 + 0.2 * rand(dim).float()).to(dt)
        s["slots"] = torch.from_numpy(slots).cuda()
    if own:
        s["kv"] = _cache(case, s)
    elif case["op"] == "attend" and not case["resident"]:
        s["pool_k"], s["pool_v"] = s["pool_k"].cpu().pin_memory(), s["pool_v"].cpu().pin_memory()
    return s


def _cache(case, s):
    """The framework's cache over a store, holding the rows of the pools: a program has it from its earlier calls."""
    import bam_b200
    pages = s["blocks"] * case["kv_heads"]
    ctrl = bam_b200.Controller(pages * case["page"], 0, queue_depth=256, num_queues=64)
    warm = case.get("resident", True)
    cache = bam_b200.PageCache(ctrl, case["page"], pages + 64 if warm else max(1024, pages // 4))
    kv = bam_b200.KvCache(cache, s["blocks"], case["kv_heads"], case["head_dim"], dtype=TYPES[case["dtype"]])
    every = torch.arange(s["blocks"] * s["bt"], device="cuda")
    kv.append(s["pool_k"].flatten(0, 1), s["pool_v"].flatten(0, 1), every)
    if not warm:
        cache.flush()
    ctrl.check_status()
    return kv


def _visible(case, n):
    return n if case["window"] <= 0 else min(n, min(case["sinks"], n) + case["window"])


def run(state):
    case = state["case"]
    if own:
        kv = state["kv"]
        if case["op"] == "attend":
            return kv.attend(state["q"], state["table"], state["lens"], window=case["window"], sinks=case["sinks"])
        if case["op"] == "append":
            norm = dict(q_norm=state["q_norm"], k_norm=state["k_norm"], norm_eps=1e-6) if case["norm"] else {}
            q = kv.append(state["k"], state["v"], state["slots"], positions=state["positions"], rope=(state["cos"], state["sin"]),
                          rope_style=case["style"], q=state["q"], **norm)
            k, v = kv.gather(state["slots"])
            return {"q": q, "k": k, "v": v}
        k, v = kv.gather(state["slots"])
        return {"k": k, "v": v}
    if case["op"] == "attend":
        return _attend(state, case)
    rows_k, rows_v, slots = state["pool_k"].flatten(0, 1), state["pool_v"].flatten(0, 1), state["slots"]
    if case["op"] == "gather":
        return {"k": rows_k[slots], "v": rows_v[slots]}
    at = state["positions"]
    cos, sin = state["cos"][at][:, None], state["sin"][at][:, None]
    q = _rotated(_normed(state["q"].float(), state["q_norm"], case), cos, sin, case).to(state["q"].dtype)
    k = _rotated(_normed(state["k"].float(), state["k_norm"], case), cos, sin, case).to(state["k"].dtype)
    if case["padded"]:
        kept = (slots >= 0).nonzero()[:, 0]
        rows_k[slots[kept]], rows_v[slots[kept]] = k[kept], state["v"][kept]
        pad = (slots < 0)[:, None, None]
        return {"q": q, "k": rows_k[slots].masked_fill(pad, 0), "v": rows_v[slots].masked_fill(pad, 0)}
    rows_k[slots], rows_v[slots] = k, state["v"]
    return {"q": q, "k": rows_k[slots], "v": rows_v[slots]}


def _normed(x, weight, case):
    if not case["norm"]:
        return x
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * weight.float()


def _rotated(x, cos, sin, case):
    r = case["rotary"]
    if case["style"] == "half":
        a, b = x[..., :r // 2], x[..., r // 2:r]
        return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., r:]], -1)
    a, b = x[..., 0:r:2], x[..., 1:r:2]
    return torch.cat([torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2), x[..., r:]], -1)


def _attend(state, case):
    bt, heads, dim = state["bt"], case["kv_heads"], case["head_dim"]
    far = not case["resident"]
    table, lens = (state["table_host"], state["lens_host"]) if far else (state["table"].long(), state["lens"].long())
    seen = torch.arange(state["most"], device=lens.device)[None]
    if case["window"] > 0:
        first = lens.clamp(max=case["sinks"])[:, None]
        begin = torch.maximum(lens[:, None] - case["window"], first)
        seen = torch.where(seen < first, seen, seen - first + begin)
    else:
        seen = seen.expand(len(lens), -1)
    valid = seen < lens[:, None]
    rows = table.gather(1, (seen // bt).clamp(max=table.shape[1] - 1)).clamp(min=0) * bt + seen % bt
    k, v = state["pool_k"].flatten(0, 1)[rows], state["pool_v"].flatten(0, 1)[rows]           # batch, tokens, heads, dim
    if far:
        k, v, valid = k.cuda(), v.cuda(), valid.cuda()
    q = state["q"].float().unflatten(1, (heads, -1))
    scores = torch.matmul(q, k.permute(0, 2, 3, 1).float()) * dim ** -0.5
    scores = scores.masked_fill(~valid[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, v.transpose(1, 2).float()) / torch.where(total == 0, 1.0, total)
    return out.flatten(1, 2).to(state["q"].dtype)


def exact(case, seed):
    s = prepare(case, seed)
    k_rows, v_rows = s["pool_k"].flatten(0, 1), s["pool_v"].flatten(0, 1)
    if case["op"] == "gather":
        return {"k": k_rows[s["slots"]].double(), "v": v_rows[s["slots"]].double()}
    if case["op"] == "append":
        r, half = case["rotary"], case["rotary"] // 2
        i = torch.arange(half, device="cuda")
        one, two = (i, i + half) if case["style"] == "half" else (2 * i, 2 * i + 1)
        turn = torch.complex(s["cos"].double(), s["sin"].double())[s["positions"]][:, None]

        def through(x, w):
            x = x.double()
            if case["norm"]:
                x = x / torch.sqrt(x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + 1e-6) * w.double()
            z = torch.complex(x[..., one], x[..., two]) * turn
            y = x.clone()
            y[..., one], y[..., two] = z.real, z.imag
            return y

        live = (s["slots"] >= 0)[:, None, None].double()
        return {"q": through(s["q"], s["q_norm"]), "k": through(s["k"], s["k_norm"]) * live, "v": s["v"].double() * live}
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    group = case["q_heads"] // case["kv_heads"]
    table = s["table"].long().cpu()
    for b, n in enumerate(s["lens"].tolist()):
        j = torch.arange(n)
        if case["window"] > 0:
            j = j[(j >= n - case["window"]) | (j < case["sinks"])]
        if not len(j):
            continue
        rows = (table[b, j // s["bt"]] * s["bt"] + j % s["bt"]).to(k_rows.device)
        k, v = k_rows[rows].cuda().double(), v_rows[rows].cuda().double()
        q = s["q"][b].double().reshape(case["kv_heads"], group, -1)
        weight = torch.softmax(torch.einsum("hgd,nhd->hgn", q, k) / math.sqrt(case["head_dim"]), -1)
        out[b] = torch.einsum("hgn,nhd->hgd", weight, v).reshape(-1, case["head_dim"])
    return out


def work(case):
    dim, kv = case["head_dim"], case["kv_heads"]
    if case["op"] == "attend":
        # the lengths are drawn from the seed; their mean stands for them
        mean = (case["shortest"] + case["longest"]) / 2
        rows = case["batch"] - (len(range(1, case["batch"], case["empty"])) if case["empty"] else 0)
        seen = rows * _visible(case, mean)
        return {"bytes": seen * kv * dim * 4 + 4 * case["batch"] * case["q_heads"] * dim, "flops": 4 * seen * case["q_heads"] * dim}
    row = case["tokens"] * kv * dim * 4                     # a key and a value of two bytes each
    if case["op"] == "gather":
        return {"bytes": 2 * row, "flops": 0}
    q = case["tokens"] * case["q_heads"] * dim
    return {"bytes": 4 * row + 4 * q + case["tokens"] * case["rotary"] * 4, "flops": 10 * (q + row // 4)}
