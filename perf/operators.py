"""The paged-cache operators of the decode path as measured cases: attention of a few new
tokens over a paged key/value cache (`attn`), eviction from that cache by accumulated
attention weight (`evict`), and the device-side bookkeeping of the next tokens' cache rows
(`advance`).

`run` with `own` false computes them in elementary torch operations; with `own` true it
makes the calls of `iquestrt_b200.ops`."""

import math
import random

import torch

own = False

E4M3 = torch.float8_e4m3fn
_KV = {"bf16": torch.bfloat16, "e4m3": E4M3}


def listed():
    def attn(name, batch, q_len, q_heads, kv_heads, dim, kv, length, page, window=0,
             ragged=0, weights=False):
        return dict(name=name, op="attn", batch=batch, q_len=q_len, q_heads=q_heads,
                    kv_heads=kv_heads, dim=dim, kv=kv, length=length, page=page, window=window,
                    ragged=ragged, weights=weights)

    def evict(name, batch, kv_heads, dim, kv, length, page, budget, first, last, ragged=0):
        return dict(name=name, op="evict", batch=batch, kv_heads=kv_heads, dim=dim, kv=kv,
                    length=length, page=page, budget=budget, first=first, last=last,
                    ragged=ragged)

    return [
        # one rank's heads of eight at batch 1, a sliding-window layer: latency is all
        attn("attn shard window 4096", 1, 1, 8, 1, 128, "e4m3", 32001, 64, window=4096),
        # the same rank's full-attention layer at 32k
        attn("attn shard 32k", 1, 1, 8, 1, 128, "e4m3", 32768, 64),
        # four rows of a draft being verified, all heads on one GPU
        attn("attn verify 4 rows 32k", 1, 4, 64, 8, 128, "e4m3", 32749, 64),
        # the longest context, all heads on one GPU
        attn("attn 128k", 1, 1, 64, 8, 128, "e4m3", 131071, 64),
        # a server's batch: ragged lengths (some empty), bf16 cache, small pages
        attn("attn ragged batch bf16", 48, 1, 32, 8, 128, "bf16", 8192, 16, ragged=3),
        # heads of 64 without grouping, two rows a sequence, a window that is no round number
        attn("attn mha d64 window", 16, 2, 16, 16, 64, "bf16", 2047, 32, window=1000, ragged=5),
        # attention that also accumulates each cache row's weight, for eviction
        attn("attn weights 32k", 1, 1, 64, 8, 128, "e4m3", 32768, 64, weights=True),
        # one row over the budget after a step: latency again
        evict("evict one step", 1, 8, 128, "e4m3", 4097, 64, 4096, 4, 512),
        # a long prompt cut down to a budget
        evict("evict 32k to 8k", 1, 8, 128, "e4m3", 32768, 64, 8192, 4, 1024),
        # a ragged batch cut down, bf16
        evict("evict ragged batch bf16", 24, 8, 128, "bf16", 8192, 16, 2048, 16, 255, ragged=7),
        # the bookkeeping of one sequence's step, and of a server's batch of drafts
        dict(name="advance 1", op="advance", batch=1, q_len=1, length=32768, page=64),
        dict(name="advance 256 x 4", op="advance", batch=256, q_len=4, length=8191, page=16),
    ]


# Most cache bytes (rows x heads x channels, K and V) and products a drawn case has: the
# listed ragged batch and the listed long contexts have about as many.
_CAP, _CAP_FLOPS = 500e6, 4e9


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attn", "attn", "attn", "evict", "evict", "advance"])
    page = rng.choice([1, 8, 16, 24, 32, 64, 128, 256])
    ragged = rng.randint(1, 1 << 20) if rng.random() < 0.7 else 0
    if op == "advance":
        return dict(op=op, batch=_log(rng, 1, 512), q_len=rng.randint(1, 8),
                    length=_log(rng, 1, 16384), page=page, ragged=ragged)
    kv = rng.choice(["bf16", "e4m3"])
    dim = rng.choice([48, 64, 80, 96, 128, 128, 192, 256])
    kv_heads = rng.choice([1, 2, 3, 4, 8, 16])
    row = 2 * kv_heads * dim * (2 if kv == "bf16" else 1)
    length = _log(rng, 1, 131072)
    length = max(1, min(length, int(_CAP / row)))
    batch = max(1, min(_log(rng, 1, 128), int(_CAP / (row * length))))
    case = dict(op=op, batch=batch, kv_heads=kv_heads, dim=dim, kv=kv, length=length, page=page,
                ragged=ragged)
    if op == "attn":
        case.update(q_len=rng.choice([1, 1, 1, 2, 3, 4, 6, 8]),
                    q_heads=kv_heads * rng.choice([1, 2, 4, 5, 8, 16]),
                    window=rng.choice([0, 0, rng.randint(1, length)]),
                    weights=rng.random() < 0.3)
        each = 4 * dim * case["q_heads"] * case["q_len"]
        case["batch"] = max(1, min(batch, int(_CAP_FLOPS / (each * length))))
        case["length"] = max(1, min(length, int(_CAP_FLOPS / each)))
        case["window"] = min(case["window"], case["length"])
    else:
        budget = _log(rng, 1, max(1, length))
        first = rng.randint(0, min(8, budget))
        case.update(budget=budget, first=first, last=rng.randint(0, budget - first))
    return case


def _lengths(case):
    """Rows each sequence holds: all `length`, or (ragged) the first `length` and the others
    spread below it, empty and one-row sequences among them."""
    n, batch = case["length"], case["batch"]
    if not case.get("ragged"):
        return [n] * batch
    r = random.Random(case["ragged"])
    out = [n]
    for i in range(batch - 1):
        out.append(min(i, n) if i < 2 else r.randint(max(1, n // 8), n))
    return out


def _tables(case, lengths, rows, gen):
    """A page table `[batch, pages]` whose pages lie in any order (entries no sequence has
    reached are -1), and the cache's number of rows."""
    page = case["page"]
    width = -(-rows // page)
    need = [-(-n // page) for n in lengths]
    total = sum(need) + 3
    ids = torch.randperm(total, generator=gen, device="cuda").to(torch.int32)
    table = torch.full((case["batch"], width), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = ids[at:at + n]
        at += n
    return table, total * page


def _cache(capacity, case, gen):
    shape = (capacity, case["kv_heads"], case["dim"])
    out = torch.empty(shape, dtype=_KV[case["kv"]], device="cuda")
    step = max(1, (1 << 26) // (shape[1] * shape[2]))
    for i in range(0, capacity, step):
        part = out[i:i + step]
        part.copy_(torch.randn(part.shape, generator=gen, device="cuda"))
    return out


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed * 7919 + 17)
    lengths = _lengths(case)
    batch, page = case["batch"], case["page"]
    s = dict(case=case, lengths=torch.tensor(lengths, dtype=torch.int32, device="cuda"))
    if case["op"] == "advance":
        s["table"], s["capacity"] = _tables(case, [n + case["q_len"] for n in lengths],
                                            max(lengths) + case["q_len"], gen)
        s["seen"] = s["lengths"] + torch.randint(0, 1000, (batch,), generator=gen, device="cuda",
                                                 dtype=torch.int32)
        n = batch * case["q_len"]
        s["slot"] = torch.zeros(n, dtype=torch.int64, device="cuda")
        s["pos"] = torch.zeros(n, dtype=torch.int64, device="cuda")
        s["lengths_out"], s["seen_out"] = torch.zeros_like(s["lengths"]), torch.zeros_like(s["seen"])
        if own:
            from iquestrt_b200 import ops
            s["scratch"] = ops.Scratch("cuda")
        return s
    s["table"], capacity = _tables(case, lengths, max(lengths), gen)
    rows = s["table"].shape[1] * page
    s["k"], s["v"] = _cache(capacity, case, gen), _cache(capacity, case, gen)
    hk = case["kv_heads"]
    if case["op"] == "attn":
        shape = (batch, case["q_len"], case["q_heads"], case["dim"])
        # normalised heads against normalised keys, sharp enough that a few keys lead
        s["q"] = (2.5 * torch.randn(shape, generator=gen, device="cuda")).to(torch.bfloat16)
        s["out"] = torch.zeros(shape, dtype=torch.bfloat16, device="cuda")
        s["lse"] = torch.zeros(shape[:3], dtype=torch.float32, device="cuda")
        if case["weights"]:
            s["weights"] = torch.rand(batch, hk, rows, generator=gen, device="cuda")
            s["positions"] = torch.randint(0, 1 << 20, (batch, hk, rows), generator=gen,
                                           device="cuda", dtype=torch.int32)
            s["seen"] = s["lengths"] + 1000
        if own:
            from iquestrt_b200 import ops
            s["scratch"] = ops.Scratch("cuda")
            s["work"] = ops.AttnWork(batch=batch, q_len=case["q_len"], q_heads=case["q_heads"],
                                     kv_heads=hk, head_dim=case["dim"], rows=rows,
                                     weights=case["weights"], device="cuda")
    else:
        # accumulated weights: a few rows hold most of it, some were never looked at
        u = torch.rand(batch, hk, rows, generator=gen, device="cuda")
        s["weights"] = torch.where(u < 0.05, 0.0, (1.0 / u.clamp_min(1e-6)).pow(1.5))
        order = torch.rand(batch, hk, rows, generator=gen, device="cuda").argsort(dim=-1)
        s["positions"] = (2 * order).to(torch.int32)
        s["seen"] = torch.full((batch,), 2 * rows, dtype=torch.int32, device="cuda")
        s["weights_out"] = torch.zeros_like(s["weights"])
        s["positions_out"] = torch.zeros_like(s["positions"])
        s["lengths_out"] = torch.zeros_like(s["lengths"])
        if own:
            from iquestrt_b200 import ops
            s["scratch"] = ops.Scratch("cuda")
            s["work"] = ops.EvictWork(batch=batch, kv_heads=hk, rows=rows, device="cuda")
    return s


def run(s):
    return {"attn": _attn, "evict": _evict, "advance": _advance}[s["case"]["op"]](s)


def _cache_rows(s):
    """`[batch, rows]`: the cache row of each row of each sequence."""
    page = s["case"]["page"]
    table = s["table"].long().clamp_min(0)
    inside = torch.arange(page, device=table.device)
    return (table[:, :, None] * page + inside).reshape(table.shape[0], -1)


def _attn(s):
    c = s["case"]
    if own:
        from iquestrt_b200 import ops
        more = {}
        if c["weights"]:
            more = dict(weights=s["weights"], positions=s["positions"], seen=s["seen"])
        ops.attn_decode(s["q"], s["k"], s["v"], s["table"], s["lengths"], page_size=c["page"],
                        window=c["window"], out=s["out"], lse=s["lse"], work=s["work"],
                        scratch=s["scratch"], **more)
    else:
        q, n = s["q"].float(), s["lengths"].long()
        batch, q_len, q_heads, dim = q.shape
        hk = c["kv_heads"]
        group = q_heads // hk
        rows = _cache_rows(s)
        j = torch.arange(rows.shape[1], device=q.device)
        at = n[:, None] - q_len + torch.arange(q_len, device=q.device)          # [batch, q_len]
        seen = j <= at[:, :, None]
        if c["window"]:
            seen &= j > at[:, :, None] - c["window"]
        some = seen.any(1)[:, None, :, None]
        k = torch.where(some, s["k"][rows].float().transpose(1, 2), 0.0)        # [b, hk, rows, d]
        v = torch.where(some, s["v"][rows].float().transpose(1, 2), 0.0)
        q = q.view(batch, q_len, hk, group, dim).permute(0, 2, 1, 3, 4)
        sc = (q.reshape(batch, hk, q_len * group, dim) @ k.transpose(2, 3)) / math.sqrt(dim)
        sc = sc.view(batch, hk, q_len, group, -1)
        sc = torch.where(seen[:, None, :, None, :], sc, -math.inf)
        m = sc.amax(-1, keepdim=True)
        p = torch.exp(sc - torch.where(m == -math.inf, 0.0, m))
        total = p.sum(-1, keepdim=True)
        p = p / torch.where(total == 0, 1.0, total)
        o = p.reshape(batch, hk, q_len * group, -1) @ v
        o = o.view(batch, hk, q_len, group, dim).permute(0, 2, 1, 3, 4)
        s["out"].copy_(o.reshape(s["out"].shape))
        s["lse"].copy_((m + total.log())[..., 0].permute(0, 2, 1, 3).reshape(s["lse"].shape))
        if c["weights"]:
            fresh = ((j >= n[:, None] - q_len) & (j < n[:, None]))[:, None, :]
            w = p.sum((2, 3))
            s["weights"].copy_(torch.where(fresh, w, s["weights"] + w))
            pos = (s["seen"].long() - n)[:, None, None] + j
            s["positions"].copy_(torch.where(fresh, pos.int(), s["positions"]))
    out = [s["out"], s["lse"]]
    return out + [s["weights"], s["positions"]] if c["weights"] else out


def _evict(s):
    c = s["case"]
    if own:
        from iquestrt_b200 import ops
        ops.kv_evict(s["k"], s["v"], s["table"], s["lengths"], s["weights"], s["positions"],
                     s["seen"], page_size=c["page"], budget=c["budget"], keep_first=c["first"],
                     keep_last=c["last"], lengths_out=s["lengths_out"],
                     weights_out=s["weights_out"], positions_out=s["positions_out"],
                     work=s["work"], scratch=s["scratch"])
    else:
        w, pos, n = s["weights"], s["positions"], s["lengths"].long()
        batch, hk, rows = w.shape
        budget, dev = c["budget"], w.device
        j = torch.arange(rows, device=dev)
        live = (j < n[:, None])[:, None, :].expand(batch, hk, rows)
        safe = (pos < c["first"]) | (pos >= s["seen"][:, None, None] - c["last"])
        key = torch.where(live, torch.where(safe, math.inf, w), -math.inf)
        rank = torch.empty_like(j).expand(batch, hk, rows).clone()
        order = key.argsort(dim=-1, descending=True, stable=True)
        rank.scatter_(2, order, j.expand(batch, hk, rows).contiguous())
        keep = live & (rank < budget)
        cut = (n > budget)[:, None, None]
        holes = cut & (j < budget) & ~keep
        moved = cut & (j >= budget) & keep
        # the i-th hole of a (sequence, head) takes its i-th moved row: both come out of
        # nonzero() in ascending order, and there are as many of one as of the other
        hole, move = holes.nonzero(), moved.nonzero()
        at = _cache_rows(s)
        to, frm = at[hole[:, 0], hole[:, 2]], at[move[:, 0], move[:, 2]]
        for cache in (s["k"], s["v"]):
            flat = cache.view(torch.uint8 if cache.dtype == E4M3 else torch.int16)
            flat[to, hole[:, 1]] = flat[frm, move[:, 1]]
        stay = j < torch.minimum(n, torch.tensor(budget, device=dev))[:, None]
        for src, dst in ((w, s["weights_out"]), (pos, s["positions_out"])):
            new = src.clone()
            new[hole[:, 0], hole[:, 1], hole[:, 2]] = src[move[:, 0], move[:, 1], move[:, 2]]
            dst.copy_(torch.where(stay[:, None, :], new, dst))
        s["lengths_out"].copy_(n.clamp_max(budget))
    return [s["k"], s["v"], s["weights_out"], s["positions_out"], s["lengths_out"]]


def _advance(s):
    c = s["case"]
    if own:
        from iquestrt_b200 import ops
        ops.kv_advance(s["table"], s["lengths"], s["seen"], s["slot"], s["pos"],
                       page_size=c["page"], capacity=s["capacity"], q_len=c["q_len"],
                       lengths_out=s["lengths_out"], seen_out=s["seen_out"],
                       scratch=s["scratch"])
    else:
        r = torch.arange(c["q_len"], device=s["table"].device)
        at = s["lengths"].long()[:, None] + r
        page = torch.gather(s["table"].long(), 1, at // c["page"])
        s["slot"].copy_((page * c["page"] + at % c["page"]).reshape(-1))
        s["pos"].copy_((s["seen"].long()[:, None] + r).reshape(-1))
        s["lengths_out"].copy_(s["lengths"] + c["q_len"])
        s["seen_out"].copy_(s["seen"] + c["q_len"])
    return [s["slot"], s["pos"], s["lengths_out"], s["seen_out"]]


def work(case):
    lengths = _lengths(case)
    if case["op"] == "advance":
        # a table entry and two words read, two 8-byte indices a row and two words written
        n = case["batch"] * case["q_len"]
        return {"bytes": 20 * n + 16 * case["batch"], "flops": 0}
    elt = 2 if case["kv"] == "bf16" else 1
    hk, dim = case["kv_heads"], case["dim"]
    if case["op"] == "evict":
        # weights and positions of the live rows read, those of the kept rows written; the
        # moved rows (with weights spread evenly, the kept share of the rows past the budget)
        # read and written
        budget, held = case["budget"], 0
        for n in lengths:
            if n <= budget:
                held += hk * 16 * n
                continue
            moved = budget * (n - budget) / n
            held += hk * (8 * n + 8 * budget + moved * 4 * dim * elt)
        return {"bytes": held + 16 * len(lengths), "flops": 0}
    q_len, window = case["q_len"], case["window"]
    rows = pairs = 0
    for n in lengths:
        low = n
        for r in range(q_len):
            at = n - q_len + r
            first = max(0, at - window + 1) if window else 0
            pairs += max(0, at + 1 - first)
            low = min(low, first)
        rows += n - low
    heads = case["batch"] * q_len * case["q_heads"]
    total = rows * hk * dim * elt * 2 + heads * (4 * dim + 4) + 4 * (rows // case["page"])
    if case["weights"]:
        total += 8 * rows * hk
    return {"bytes": total, "flops": 4 * dim * case["q_heads"] * pairs}


def exact(case, seed):
    s = prepare(case, seed)
    lengths, page = _lengths(case), case["page"]
    if case["op"] == "advance":
        return None                                # whole numbers: the two sides must be equal
    table = s["table"].tolist()

    def row_ids(b, n):
        return torch.tensor([table[b][i // page] * page + i % page for i in range(n)],
                            dtype=torch.int64, device="cuda")

    hk = case["kv_heads"]
    if case["op"] == "evict":
        # one (sequence, head) at a time, in plain lists
        seen = s["seen"].tolist()
        for b, n in enumerate(lengths):
            s["lengths_out"][b] = min(n, case["budget"])
            ids = row_ids(b, n).tolist()
            for h in range(hk):
                w, pos = s["weights"][b, h, :n].tolist(), s["positions"][b, h, :n].tolist()
                new_w, new_pos, src = w[:case["budget"]], pos[:case["budget"]], []
                if n > case["budget"]:
                    edge = seen[b] - case["last"]
                    safe = [p < case["first"] or p >= edge for p in pos]
                    best = sorted(range(n), key=lambda i: (not safe[i], 0.0 if safe[i] else -w[i], i))
                    kept = set(best[:case["budget"]])
                    src = sorted(i for i in kept if i >= case["budget"])
                    dst = sorted(i for i in range(case["budget"]) if i not in kept)
                    for d, i in zip(dst, src):
                        new_w[d], new_pos[d] = w[i], pos[i]
                    to = torch.tensor([ids[d] for d in dst], dtype=torch.int64, device="cuda")
                    frm = torch.tensor([ids[i] for i in src], dtype=torch.int64, device="cuda")
                    for cache in (s["k"], s["v"]):
                        flat = cache.view(torch.uint8)
                        flat[to, h] = flat[frm, h]
                m = len(new_w)
                s["weights_out"][b, h, :m] = torch.tensor(new_w, device="cuda")
                s["positions_out"][b, h, :m] = torch.tensor(new_pos, dtype=torch.int32,
                                                            device="cuda")
        return [s["k"].double(), s["v"].double(), s["weights_out"].double(), s["positions_out"],
                s["lengths_out"]]
    q_len, group = case["q_len"], case["q_heads"] // hk
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.full(s["q"].shape[:3], -math.inf, dtype=torch.float64, device="cuda")
    weights = s["weights"].double() if case["weights"] else None
    for b, n in enumerate(lengths):
        ids = row_ids(b, n)
        if case["weights"]:
            for i in range(max(0, n - q_len), n):
                weights[b, :, i] = 0.0
                s["positions"][b, :, i] = int(s["seen"][b]) - n + i
        for r in range(q_len):
            at = n - q_len + r
            low = max(0, at - case["window"] + 1) if case["window"] else 0
            if at < low:
                continue
            mine = ids[low:at + 1]
            for h in range(hk):
                heads = slice(h * group, (h + 1) * group)
                k, v = s["k"][mine, h].double(), s["v"][mine, h].double()
                sc = torch.einsum("gd,jd->gj", s["q"][b, r, heads].double(), k) * case["dim"] ** -0.5
                z = torch.logsumexp(sc, 1)
                p = (sc - z[:, None]).exp()
                out[b, r, heads], lse[b, r, heads] = p @ v, z
                if case["weights"]:
                    weights[b, h, low:at + 1] += p.sum(0)
    done = [out, lse]
    return done + [weights, s["positions"]] if case["weights"] else done
