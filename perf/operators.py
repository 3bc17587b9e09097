"""Measured cases: the cache side of a step that serves several sequences.

Four operators, each through the public device entry points of rdlquant.attention:
* "plan": block tables, row starts, positions and slots of a step from the
  lengths of its requests (rdl_kv_plan_dev);
* "store": rotary positions applied to the q and k rows of a step, its k and v
  rows written into the cache's pages (rdl_kv_store_dev);
* "paged": attention of the step's new rows over the paged cache, sequences
  with one new token beside sequences with a chunk (rdl_attention_paged_dev);
* "packed": causal attention of whole prompts packed one behind the other, read
  from the step's own k and v rows (rdl_attention_packed_dev).

Activations are f32 as the Linears give and take them, the cache f16 or f32 as
the decoder keeps it.  Shapes are the 7B ones of the repository's benchmark (32
query and 8 KV heads of 128, pages of 64 positions) and generic ones around
them.  Lengths belong to the case, values to the seed.
"""
import math
import os
import random
import sys

import torch

own = False

sys.path.insert(0, os.path.join(os.getcwd(), "rust-deeplearning_amd"))

TYPES = {"f16": torch.float16, "f32": torch.float32}
GGML = {"f16": 1, "f32": 0}  # GGML type ids
LARGEST = 0.6e12  # flops of the largest case, about


def plan(name, n_seq, chunks, cached, page=64, pad=0, ragged=1):
    """chunks: share of the sequences with more than one new token, in percent; pad: rows of the batch behind the last sequence."""
    return {"name": name, "kind": "plan", "n_seq": n_seq, "chunks": chunks, "most_new": 96, "cached": cached,
            "page": page, "pad": pad, "ragged": ragged}


def store(name, n_seq, rows, cached, heads=32, kv_heads=8, head_dim=128, kv="f16", page=64, layout="heads", ragged=1):
    return {"name": name, "kind": "store", "n_seq": n_seq, "rows": rows, "cached": cached, "heads": heads,
            "kv_heads": kv_heads, "head_dim": head_dim, "kv": kv, "page": page, "layout": layout, "ragged": ragged}


def paged(name, n_seq, chunks, rows, cached, heads=32, kv_heads=8, head_dim=128, kv="f16", page=64, layout="heads",
          ragged=1):
    """The first `chunks` sequences bring up to `rows` new rows, the others one; up to `cached` positions before them."""
    return {"name": name, "kind": "paged", "n_seq": n_seq, "chunks": chunks, "rows": rows, "cached": cached,
            "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim, "kv": kv, "page": page, "layout": layout,
            "ragged": ragged}


def packed(name, n_seq, rows, heads=32, kv_heads=8, head_dim=128, kv="f32", ragged=1):
    """n_seq prompts of up to `rows` rows."""
    return {"name": name, "kind": "packed", "n_seq": n_seq, "rows": rows, "heads": heads, "kv_heads": kv_heads,
            "head_dim": head_dim, "kv": kv, "ragged": ragged}


def listed():
    return [
        # a decode step of sixteen sequences: the shortest call of a serving loop
        plan("plan_16_sequences", 16, 0, 2000),
        # a step of a large server: decoding sequences and prompt chunks, in a padded batch
        plan("plan_1500_mixed", 1500, 30, 6000, pad=300),
        # the rows of a decode step of 24 sequences
        store("store_24_tokens", 24, 1, 3000),
        # prompt chunks, 4096 rows of a step
        store("store_prompt_rows", 8, 512, 1500),
        # an f32 cache with positions outside heads, small heads, odd chunks
        store("store_f32_positions", 7, 301, 900, heads=16, kv_heads=4, head_dim=64, kv="f32", layout="positions"),
        # one user's next token: the shortest attention
        paged("paged_one_token", 1, 0, 1, 777),
        # a decode step of 48 sequences of very different lengths: the cache is read once
        paged("paged_decode_48", 48, 0, 1, 8192),
        # a step that mixes the chunks of four prompts with twelve decoding sequences
        paged("paged_mixed_step", 16, 4, 300, 3000),
        # the f32 cache (the decoder's exact one) with small heads, short chunks
        paged("paged_f32_short_chunks", 9, 6, 17, 1900, heads=16, kv_heads=4, head_dim=64, kv="f32", page=16),
        # a chunk of a long document: 2048 rows that see about 15000 positions
        paged("paged_long_chunk", 1, 1, 2048, 14000),
        # a few short questions scored without a cache
        packed("packed_short", 5, 60, heads=12, kv_heads=12, head_dim=64),
        # prompts of very different lengths in one pass
        packed("packed_prompts", 7, 3500),
    ]


def lengths(case):
    """[(positions cached before, new rows)] of the case's sequences."""
    r = random.Random(case["ragged"])
    n, kind = case["n_seq"], case["kind"]
    got = []
    for i in range(n):
        if kind == "packed":
            got.append((0, case["rows"] if i == 0 else max(1, int(case["rows"] * r.random() ** 2))))
            continue
        before = case["cached"] if i == 0 else int(case["cached"] * r.random())
        if kind == "plan":
            new = r.randint(2, case["most_new"]) if r.randrange(100) < case["chunks"] else 1
        elif kind == "store":
            new = case["rows"]
        else:
            new = 1 if i >= case["chunks"] else case["rows"] if i == 0 else r.randint(1, case["rows"])
        got.append((before, new))
    return got


def log_int(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    kind = rng.choice(["plan", "store", "paged", "paged", "paged", "packed", "packed"])
    ragged = rng.randrange(1 << 20)
    page = rng.choice([16, 32, 64, 64, 128, 256])
    if kind == "plan":
        return {"kind": kind, "n_seq": log_int(rng, 1, 1500), "chunks": rng.choice([0, 0, 20, 60]),
                "most_new": log_int(rng, 4, 96), "cached": log_int(rng, 16, 6000), "page": page,
                "pad": rng.choice([0, 0, 1, 300]), "ragged": ragged}
    kv_heads = rng.choice([1, 2, 4, 8, 8])
    head_dim = rng.choice([64, 128, 128, 128, 80, 96, 256])
    shape = {"heads": kv_heads * rng.choice([1, 2, 3, 4, 4, 7, 8]), "kv_heads": kv_heads, "head_dim": head_dim,
             "kv": rng.choice(["f16", "f16", "f32"]), "ragged": ragged}
    while shape["heads"] * head_dim > 8192:
        shape["heads"] -= kv_heads
    where = {"page": page, "layout": rng.choice(["heads", "heads", "positions"])}
    if kind == "store":
        n = log_int(rng, 1, 48)
        return {"kind": kind, "n_seq": n, "rows": log_int(rng, 1, 4096 // n), "cached": log_int(rng, 1, 4000), **shape,
                **where}
    while True:
        if kind == "packed":
            case = {"kind": kind, "n_seq": log_int(rng, 1, 24), "rows": log_int(rng, 1, 4096), **shape}
        else:
            n = log_int(rng, 1, 64)
            chunks = 0 if rng.random() < 0.4 else rng.randint(1, min(n, 8))
            case = {"kind": kind, "n_seq": n, "chunks": chunks, "rows": log_int(rng, 2, 2048) if chunks else 1,
                    "cached": log_int(rng, 1, 16000), **shape, **where}
        lens = lengths(case)
        longest, widest = max(n for _, n in lens), max(c + n for c, n in lens)
        padded = case["n_seq"] * longest * widest * case["heads"]
        held = case["n_seq"] * widest * case["kv_heads"] * head_dim
        if 4 * padded * head_dim <= LARGEST and padded <= 1.1e9 and held <= 4e8:
            return case


def work(case):
    lens = lengths(case)
    rows = sum(n for _, n in lens)
    if case["kind"] == "plan":
        page = case["page"]
        taken = sum(-(-(c + n) // page) - -(-c // page) for c, n in lens)
        return {"bytes": 16 * len(lens) + 8 * taken + 12 * (rows + case["pad"]), "flops": 8 * rows}
    hd, heads, kvh = case["head_dim"], case["heads"], case["kv_heads"]
    elem = 2 if case["kv"] == "f16" else 4
    if case["kind"] == "store":
        table = min(rows, max(c + n for c, n in lens)) * hd * 4
        return {"bytes": rows * hd * (8 * heads + kvh * (8 + 2 * elem)) + table + 8 * rows,
                "flops": 3 * rows * hd * (heads + kvh)}
    seen = sum(n * c + n * (n + 1) // 2 for c, n in lens)
    return {"bytes": rows * heads * hd * 8 + sum(c + n for c, n in lens) * kvh * hd * 2 * elem + 12 * len(lens),
            "flops": 4 * hd * heads * seen}


def prepare(case, seed):
    dev = torch.device("cuda" if torch.cuda.is_available() else "cpu")
    g = torch.Generator(device=dev).manual_seed(seed)
    lens = lengths(case)
    n_seq, kind = len(lens), case["kind"]

    def ints(values):
        return torch.tensor(values, dtype=torch.int32, device=dev)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=dev)

    s = {"case": case, "n_seq": n_seq, "max_new": max(n for _, n in lens), "max_kv": max(c + n for c, n in lens),
         "rows": sum(n for _, n in lens)}
    if kind == "plan":
        # the seed moves the lengths a little: other requests in the same number
        r = random.Random("%d %d" % (seed, case["ragged"]))
        lens = [(max(0, c - r.randint(0, case["page"])), n) for c, n in lens]
    starts = [0]
    for _, n in lens:
        starts.append(starts[-1] + n)
    s["row_start"], s["kv_len"] = ints(starts), ints([c + n for c, n in lens])
    if kind != "packed":
        page = case["page"]
        pages = [-(-(c + n) // page) for c, n in lens]
        pool = sum(pages) + 5
        order = torch.randperm(pool, generator=g, device=dev).int()
        width = -(-s["max_kv"] // page)
        table = torch.full((n_seq, width), -1, dtype=torch.int32, device=dev)
        had = [-(-c // page) for c, _ in lens] if kind == "plan" else pages
        first = torch.tensor([sum(had[:b]) for b in range(n_seq)], device=dev)
        at = torch.arange(width, device=dev)
        has = at < torch.tensor(had, device=dev)[:, None]
        s["table"] = torch.where(has, order[(first[:, None] + at).clamp_(max=pool - 1)], table)
        s["page"], s["pages"] = page, pool
    if kind == "plan":
        s["cached"], s["new"] = ints([c for c, _ in lens]), ints([n for _, n in lens])
        s["free"] = order[sum(had):].contiguous()
        s["m"] = m = s["rows"] + case["pad"]
        s["out"] = [torch.zeros(n, dtype=torch.int32, device=dev) for n in (n_seq + 1, n_seq, m, m, m, 4)]
        return s
    hd, heads, kvh = case["head_dim"], case["heads"], case["kv_heads"]
    rows, kv = s["rows"], TYPES[case["kv"]]
    # q, k and v as the q/k/v product leaves them: one row a token
    qkv = randn(rows, heads + 2 * kvh, hd)
    s["q"], s["k"], s["v"] = qkv[:, :heads], qkv[:, heads:heads + kvh], qkv[:, heads + kvh:]
    s["out"] = torch.zeros(rows, heads, hd, device=dev)
    s["scale"] = 1.0 / math.sqrt(hd)
    if kind == "packed":
        if kv != torch.float32:  # k and v kept in the cache's type for the cache write
            s["k"], s["v"] = s["k"].to(kv), s["v"].to(kv)
        return s
    # the pool as [pages, kv heads, positions, head dim], in either order in memory
    shape = (2, pool, kvh, page, hd) if case["layout"] == "heads" else (2, pool, page, kvh, hd)
    both = randn(*shape).to(kv)
    s["kc"], s["vc"] = both if case["layout"] == "heads" else both.transpose(2, 3)
    if kind == "store":
        half = hd // 2
        angle = (torch.arange(s["max_kv"], device=dev, dtype=torch.float64)[:, None] *
                 10000.0 ** (-torch.arange(half, device=dev, dtype=torch.float64) / half))
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
        seq = torch.repeat_interleave(torch.arange(n_seq, device=dev), ints([n for _, n in lens]).long())
        pos = torch.arange(rows, device=dev) - s["row_start"].long()[seq] + ints([c for c, _ in lens]).long()[seq]
        s["positions"] = pos.int()
        s["slots"] = (s["table"].long()[seq, pos // page] * page + pos % page).int()
    return s


# ---- the plain forms -------------------------------------------------------------------


def plain_plan(s):
    page, m, dev = s["page"], s["m"], s["cached"].device
    cached, new = s["cached"].long(), s["new"].long()
    kv_len = cached + new
    have = (cached + page - 1) // page
    need = (kv_len + page - 1) // page - have
    first = need.cumsum(0) - need
    ends = new.cumsum(0)
    at = torch.arange(s["table"].shape[1], device=dev) - have[:, None]
    fresh = (at >= 0) & (at < need[:, None])
    table = torch.where(fresh, s["free"][(first[:, None] + at).clamp(0, s["free"].numel() - 1)], s["table"])
    r = torch.arange(m, device=dev)
    seq = torch.searchsorted(ends, r, right=True)
    live = seq < s["n_seq"]
    b = seq.clamp(max=s["n_seq"] - 1)
    pos = cached[b] + r - (ends - new)[b]
    page_at = (pos // page).clamp(0, table.shape[1] - 1)
    slot = table[b, page_at].long() * page + pos % page
    summary = torch.stack([ends[-1], need.sum(), torch.zeros_like(ends[-1]), kv_len.max()])
    start = torch.cat([torch.zeros_like(ends[:1]), ends])
    got = (start, kv_len, torch.where(live, b, -1), torch.where(live, pos, 0), torch.where(live, slot, -1), summary)
    return [table] + [v.int() for v in got]


def rotate(x, cos, sin):
    a, b = x.chunk(2, -1)
    return torch.cat([a * cos - b * sin, a * sin + b * cos], -1)


def plain_store(s):
    pos, slot, page = s["positions"].long(), s["slots"].long(), s["page"]
    cos, sin = s["cos"][pos][:, None], s["sin"][pos][:, None]
    s["kc"][slot // page, :, slot % page] = rotate(s["k"], cos, sin).to(s["kc"].dtype)
    s["vc"][slot // page, :, slot % page] = s["v"].to(s["vc"].dtype)
    return [rotate(s["q"], cos, sin), s["kc"], s["vc"]]


def softmax_sum(q, k, v, sees, scale):
    """q [b, kv heads, rows, hd], k and v [b, kv heads, keys, hd], sees [b, 1, rows, keys]: rows that see nothing give zeros."""
    score = torch.matmul(q, k.transpose(-1, -2).contiguous()).mul_(scale).masked_fill_(~sees, -math.inf)
    top = score.amax(-1, keepdim=True)
    weight = score.sub_(torch.where(top > -math.inf, top, 0.0)).exp_()
    total = weight.sum(-1, keepdim=True)
    return torch.matmul(weight, v) / torch.where(total > 0, total, 1.0)


def plain_attention(s):
    case, dev = s["case"], s["q"].device
    heads, kvh, hd = case["heads"], case["kv_heads"], case["head_dim"]
    group, n_seq, most, keys = heads // kvh, s["n_seq"], s["max_new"], s["max_kv"]
    start = s["row_start"].long()
    n, t = start[1:] - start[:-1], s["kv_len"].long()
    i, j = torch.arange(most, device=dev), torch.arange(keys, device=dev)
    rows = (start[:-1, None] + i).clamp(max=s["rows"] - 1)
    q = s["q"][rows].reshape(n_seq, most, kvh, group, hd).permute(0, 2, 1, 3, 4).reshape(n_seq, kvh, most * group, hd)
    if case["kind"] == "packed":
        at = (start[:-1, None] + j).clamp(max=s["rows"] - 1)
        k, v = s["k"][at], s["v"][at]
    else:
        at = s["table"].long()[:, j // s["page"]].clamp(min=0)
        k, v = s["kc"][at, :, j % s["page"]], s["vc"][at, :, j % s["page"]]
    k, v = k.float().transpose(1, 2).contiguous(), v.float().transpose(1, 2).contiguous()
    sees = (j <= (t - n)[:, None, None] + i[:, None]) & (i < n[:, None])[:, :, None]
    sees = sees[:, None, :, None].expand(n_seq, 1, most, group, keys).reshape(n_seq, 1, most * group, keys)
    o = softmax_sum(q, k, v, sees, s["scale"])
    o = o.view(n_seq, kvh, most, group, hd).permute(0, 2, 1, 3, 4).reshape(n_seq, most, heads, hd)
    r = torch.arange(s["rows"], device=dev)
    b = torch.searchsorted(start[1:], r, right=True)
    return o[b, r - start[b]]


# ---- the framework's operators -----------------------------------------------------------


def pool_of(A, s):
    k = s["kc"]
    return A.KvPool(k.data_ptr(), s["vc"].data_ptr(), GGML[s["case"]["kv"]], k.shape[0], s["page"], k.shape[1],
                    k.shape[3], k.stride(0), k.stride(1), k.stride(2))


def own_run(s):
    from rdlquant import attention as A

    stream, case = torch.cuda.current_stream().cuda_stream if torch.cuda.is_available() else 0, s["case"]
    if case["kind"] == "plan":
        start, kv_len, seq, pos, slot, summary = s["out"]
        A.plan_dev(s["cached"].data_ptr(), s["new"].data_ptr(), s["n_seq"], s["free"].data_ptr(), s["free"].numel(),
                   s["page"], s["table"].data_ptr(), s["table"].shape[1], start.data_ptr(), kv_len.data_ptr(), s["m"],
                   seq.data_ptr(), pos.data_ptr(), slot.data_ptr(), summary.data_ptr(), stream)
        return [s["table"]] + s["out"]
    q, out = s["q"], s["out"]
    if case["kind"] == "store":
        A.store_dev(pool_of(A, s), s["rows"], q.data_ptr(), q.stride(0), out.data_ptr(), out.stride(0), case["heads"],
                    s["k"].data_ptr(), s["k"].stride(0), s["v"].data_ptr(), s["v"].stride(0),
                    s["positions"].data_ptr(), s["slots"].data_ptr(), s["cos"].data_ptr(), s["sin"].data_ptr(),
                    s["cos"].shape[0], stream)
        return [out, s["kc"], s["vc"]]
    if case["kind"] == "paged":
        A.attention_paged_dev(pool_of(A, s), q.data_ptr(), q.stride(0), case["heads"], s["rows"],
                              s["row_start"].data_ptr(), s["kv_len"].data_ptr(), s["n_seq"], s["table"].data_ptr(),
                              s["table"].shape[1], s["scale"], out.data_ptr(), out.stride(0), s["max_new"],
                              s["max_kv"], stream)
        return out
    A.attention_packed_dev(q.data_ptr(), q.stride(0), case["heads"], s["k"].data_ptr(), s["k"].stride(0),
                           s["v"].data_ptr(), s["v"].stride(0), GGML[case["kv"]], case["kv_heads"], case["head_dim"],
                           s["rows"], s["row_start"].data_ptr(), s["n_seq"], s["scale"], out.data_ptr(),
                           out.stride(0), s["max_new"], stream)
    return out


def run(state):
    if own:
        return own_run(state)
    kind = state["case"]["kind"]
    return plain_plan(state) if kind == "plan" else plain_store(state) if kind == "store" else plain_attention(state)


# ---- 64 bits --------------------------------------------------------------------------------


def exact(case, seed):
    """One sequence after the other, from the definitions, in 64 bits."""
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "plan":
        return None  # whole numbers
    hd, heads, kvh = case["head_dim"], case["heads"], case["kv_heads"]
    group = heads // kvh
    if kind == "store":
        pos = s["positions"].tolist()
        half = hd // 2
        c, n = s["cos"].double()[pos], s["sin"].double()[pos]
        turned = []
        for x in (s["q"].double(), s["k"].double()):
            y = torch.empty_like(x)
            for h in range(x.shape[1]):
                re, im = x[:, h, :half], x[:, h, half:]
                y[:, h, :half], y[:, h, half:] = c * re - n * im, n * re + c * im
            turned.append(y)
        kc, vc = s["kc"].double(), s["vc"].double()
        for r, slot in enumerate(s["slots"].tolist()):
            kc[slot // s["page"], :, slot % s["page"]] = turned[1][r]
            vc[slot // s["page"], :, slot % s["page"]] = s["v"][r].double()
        return [turned[0], kc, vc]
    start, kv_len = s["row_start"].tolist(), s["kv_len"].tolist()
    out = torch.zeros(s["rows"], heads, hd, dtype=torch.float64, device=s["q"].device)
    for b in range(s["n_seq"]):
        r0, r1, t = start[b], start[b + 1], kv_len[b]
        if kind == "packed":
            k, v = s["k"][r0:r1].double(), s["v"][r0:r1].double()
        else:
            ids = s["table"][b, :-(-t // s["page"])].long()
            k, v = (x[ids].double().permute(0, 2, 1, 3).reshape(-1, kvh, hd)[:t] for x in (s["kc"], s["vc"]))
        step = max(1, (1 << 26) // (heads * t))
        for a in range(r0, r1, step):
            z = min(r1, a + step)
            last = torch.arange(a, z, device=out.device) - r1 + t
            behind = torch.arange(t, device=out.device) > last[:, None]
            for h in range(heads):
                p = (s["q"][a:z, h].double() @ k[:, h // group].T.contiguous()) * s["scale"]
                p = torch.softmax(p.masked_fill(behind, -math.inf), -1)
                out[a:z, h] = p @ v[:, h // group].contiguous()
    return out
