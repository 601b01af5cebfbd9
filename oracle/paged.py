"""The paged-cache operators in plain 64-bit arithmetic, one row at a time: attention of a
few new tokens over a paged key/value cache, eviction by accumulated attention weight, and
the next tokens' cache rows."""

import torch


def rows_of(table, b, n, page):
    """The cache rows of sequence `b`'s first `n` rows."""
    return torch.tensor([int(table[b, j // page]) * page + j % page for j in range(n)],
                        dtype=torch.int64, device=table.device)


def attn_decode(q, k_cache, v_cache, table, lengths, page, *, scale=None, window=0, weights=None,
                positions=None, seen=None):
    """Returns a dict: `out` and `lse` in 64 bits, `mass` (sum of weight x |v|: what a relative
    error of the weights can move an output by), `reach` (largest sum |q_i k_i| scale of a row:
    what rounding in the scores can move), and the updated `weights` / `positions`."""
    batch, q_len, q_heads, d = q.shape
    kv_heads = k_cache.shape[1]
    group = q_heads // kv_heads
    scale = d ** -0.5 if scale is None else scale
    dev = q.device
    out = torch.zeros(q.shape, dtype=torch.float64, device=dev)
    mass = torch.zeros_like(out)
    lse = torch.full(q.shape[:3], -torch.inf, dtype=torch.float64, device=dev)
    reach = torch.zeros_like(lse)
    weights = None if weights is None else weights.double().clone()
    positions = None if positions is None else positions.clone()
    for b in range(batch):
        n = int(lengths[b])
        if weights is not None:
            for j in range(max(0, n - q_len), n):
                weights[b, :, j] = 0
                if positions is not None:
                    positions[b, :, j] = int(seen[b]) - n + j
        rows = rows_of(table, b, n, page)
        for r in range(q_len):
            at = n - q_len + r
            lo = max(0, at - window + 1) if window else 0
            if at < lo:
                continue
            for h in range(kv_heads):
                k, v = k_cache[rows[lo:at + 1], h].double(), v_cache[rows[lo:at + 1], h].double()
                hs = slice(h * group, (h + 1) * group)
                qq = q[b, r, hs].double()
                s = scale * (qq @ k.t())
                z = torch.logsumexp(s, -1)
                p = torch.exp(s - z[:, None])
                out[b, r, hs], lse[b, r, hs] = p @ v, z
                mass[b, r, hs] = p @ v.abs()
                reach[b, r, hs] = abs(scale) * (qq.abs() @ k.abs().t()).amax(-1)
                if weights is not None:
                    weights[b, h, lo:at + 1] += p.sum(0)
    return dict(out=out, lse=lse, mass=mass, reach=reach, weights=weights, positions=positions)


def kept_rows(weights, positions, n, seen, budget, first, last):
    """The rows of one (sequence, head) that stay: protected ones, then by weight, then by row."""
    w = [float("-inf") if x != x else x for x in weights[:n].tolist()]
    pos = positions[:n].tolist()
    safe = [p < first or p >= seen - last for p in pos]
    order = sorted(range(n), key=lambda i: (not safe[i], 0.0 if safe[i] else -w[i], i))
    return sorted(order[:budget])


def kv_evict(k_cache, v_cache, table, lengths, weights, positions, seen, page, *, budget, first=0,
             last=0):
    """Copies of the caches, weights, positions and lengths after eviction."""
    k, v, w, pos = k_cache.clone(), v_cache.clone(), weights.clone(), positions.clone()
    new = lengths.clone()
    for b in range(lengths.shape[0]):
        n = int(lengths[b])
        if n <= budget:
            continue
        new[b] = budget
        rows = rows_of(table, b, n, page)
        for h in range(k.shape[1]):
            kept = kept_rows(weights[b, h], positions[b, h], n, int(seen[b]), budget, first, last)
            stay = set(i for i in kept if i < budget)
            free = [i for i in range(budget) if i not in stay]
            moved = [i for i in kept if i >= budget]
            for to, frm in zip(free, moved):
                k[rows[to], h], v[rows[to], h] = k_cache[rows[frm], h], v_cache[rows[frm], h]
                w[b, h, to], pos[b, h, to] = weights[b, h, frm], positions[b, h, frm]
    return k, v, w, pos, new
