"""Attention over a paged KV cache, eviction from it by accumulated attention weight, and the
next tokens' cache rows, through the C ABI against 64-bit arithmetic (`oracle/paged.py`)."""

import pytest
import torch

from oracle import paged as P

pytestmark = pytest.mark.gpu

E4M3 = torch.float8_e4m3fn
BF16 = torch.bfloat16
DEV = "cuda"


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _table(lengths, page, g, spare=2, cover=None):
    """Pages in random order; -1 where a sequence does not reach; the cache's rows."""
    need = [-(-n // page) for n in lengths]
    width = max(1, *need) if cover is None else -(-cover // page)
    ids = torch.randperm(sum(need) + spare, generator=g, device=DEV).int()
    table = torch.full((len(lengths), width), -1, dtype=torch.int32, device=DEV)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = ids[at:at + n]
        at += n
    return table, (sum(need) + spare) * page


def _garbage(cache, table, lengths, page):
    """NaN in every row of the cache that no sequence holds."""
    held = torch.zeros(cache.shape[0], dtype=torch.bool, device=DEV)
    for b, n in enumerate(lengths):
        held[P.rows_of(table, b, n, page)] = True
    cache[~held] = torch.full((), float("nan"), device=DEV).to(cache.dtype)


def _case(lengths, q_len, q_heads, kv_heads, d, kv, page, seed=1, sharp=2.5, cover=None):
    g = _gen(seed)
    table, capacity = _table(lengths, page, g, cover=cover)
    k = torch.randn(capacity, kv_heads, d, generator=g, device=DEV).to(kv)
    v = torch.randn(capacity, kv_heads, d, generator=g, device=DEV).to(kv)
    _garbage(k, table, lengths, page)
    _garbage(v, table, lengths, page)
    q = (sharp * torch.randn(len(lengths), q_len, q_heads, d, generator=g, device=DEV)).to(BF16)
    return q, k, v, table, torch.tensor(lengths, dtype=torch.int32, device=DEV)


def _check(got, lse, want, kv, d, n):
    """Outputs are off by: half a step of bf16; a relative error of each softmax weight times
    the weighted |v| (`mass`).  A weight is off by its rounding for the product with v (bf16
    2^-8, half 2^-11, both times 1 + that), by what fp32 sums of d products leave in its score
    (at most d + 2 steps of 2^-23 of `reach`, which enter the weight and the normaliser), by
    ex2 (2^-22) and by the sums over n weights (n steps of 2^-24, as the terms are positive).
    Half precision keeps the weights relative to a reference the largest weight is 2^8 or
    more of; the steps of its smallest numbers are 2^-24, so a weight may be off by 2^-25
    absolutely, and all n of them by n 2^-33 of the sum: of the largest |v| (at most 6 here)."""
    out, mass, reach = want["out"], want["mass"], want["reach"][..., None]
    u = 2.0 ** -8 if kv == BF16 else 2.0 ** -11
    score = (d + 2) * 2.0 ** -23 * reach
    rel = u + 2 * score + 2.0 ** -21 + 2 * n * 2.0 ** -24
    room = 1.01 * (2.0 ** -8 * out.abs() + (1 + 2.0 ** -8) * rel * mass) + 6 * n * 2.0 ** -33
    off = (got.double() - out).abs()
    assert torch.isfinite(got.float()).all()
    assert (off <= room).all(), float((off / room).max())
    if lse is not None:
        empty = want["lse"] == -torch.inf
        assert torch.equal(lse == -torch.inf, empty)
        room = score[..., 0] + 2.0 ** -21 + n * 2.0 ** -24 + 2.0 ** -22 * want["lse"].abs()
        off = (lse.double() - want["lse"]).abs()[~empty]
        assert (off <= room[~empty]).all(), float((off / room[~empty]).max())


SHAPES = [
    # lengths, q_len, q_heads, kv_heads, d, page, window
    ([1], 1, 8, 1, 128, 64, 0),
    ([0, 1, 2, 17], 1, 8, 2, 128, 16, 0),
    ([127, 128, 129, 1000], 1, 4, 4, 64, 1, 0),
    ([4097], 1, 8, 1, 128, 64, 0),
    ([4097, 31], 1, 16, 2, 128, 64, 100),
    ([777, 3, 0, 64], 2, 10, 2, 128, 24, 0),
    ([1500, 5], 4, 16, 2, 128, 16, 0),
    ([1500, 5, 8], 8, 16, 2, 128, 16, 3),
    ([1500, 4, 9], 8, 8, 8, 64, 32, 700),
    ([513, 2], 3, 5, 1, 80, 8, 0),
    ([300, 40], 1, 16, 1, 48, 16, 33),
    ([2100], 1, 16, 1, 256, 128, 0),
    ([900, 77], 4, 16, 2, 256, 64, 500),
    ([700], 8, 64, 8, 192, 16, 0),
    ([600, 1], 8, 32, 2, 128, 64, 0),        # 128 query rows a head: two blocks
    ([333, 20], 6, 32, 2, 16, 16, 0),
    ([333, 64, 0, 1], 2, 4, 2, 64, 5, 77),
    ([333, 47], 1, 8, 2, 128, 1, 100),
    ([0, 0], 2, 4, 2, 64, 8, 0),
    ([2000, 700, 90], 2, 24, 6, 128, 64, 0),
    ([3000, 10], 8, 40, 1, 128, 32, 0),      # 320 query rows a head: five blocks
]


@pytest.mark.parametrize("kv", [E4M3, BF16], ids=["e4m3", "bf16"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: f"q{s[1]}h{s[2]}-{s[3]}d{s[4]}n{max(s[0])}w{s[6]}")
def test_attention_against_64_bits(scratch, shape, kv):
    from iquestrt_b200 import ops
    lengths, q_len, qh, kh, d, page, window = shape
    q, k, v, table, n = _case(lengths, q_len, qh, kh, d, kv, page)
    out = torch.full_like(q, float("nan"))
    lse = torch.full(q.shape[:3], float("nan"), device=DEV)
    ops.attn_decode(q, k, v, table, n, page_size=page, window=window, out=out, lse=lse,
                    scratch=scratch)
    assert scratch.status() == 0
    want = P.attn_decode(q, k, v, table, n, page, window=window)
    _check(out, lse, want, kv, d, max(lengths))
    empty = want["lse"] == -torch.inf
    assert float(out[empty].float().abs().sum()) == 0
    # a second call on the same buffers gives the same bits
    again = ops.attn_decode(q, k, v, table, n, page_size=page, window=window, scratch=scratch)
    assert torch.equal(again.view(torch.int16), out.view(torch.int16))


@pytest.mark.parametrize("kv", [E4M3, BF16], ids=["e4m3", "bf16"])
@pytest.mark.parametrize("q_len,window", [(4, 0), (3, 50), (8, 2)])
def test_a_row_is_not_touched_by_what_it_does_not_see(scratch, kv, q_len, window):
    """NaN in the newest key and value, and in keys and values that slid out of a window:
    every row that does not see them is as it is without them; those that do are NaN."""
    from iquestrt_b200 import ops
    q, k, v, table, n = _case([400, 390], q_len, 8, 2, 128, kv, 16, seed=3)
    call = dict(page_size=16, window=window, scratch=scratch)
    clean = ops.attn_decode(q, k, v, table, n, **call).clone()
    nan = torch.full((), float("nan"), device=DEV).to(kv)
    rows = P.rows_of(table, 0, 400, 16)
    k[rows[399]], v[rows[399]] = nan, nan
    if window:                               # row 0 of the step still sees this one, later rows not
        v[rows[400 - q_len - window + 1]] = nan
    got = ops.attn_decode(q, k, v, table, n, **call)
    assert torch.isnan(got[0, q_len - 1].float()).all()
    assert torch.equal(got[1], clean[1])
    sound = slice(1 if window else 0, q_len - 1)
    assert torch.equal(got[0, sound], clean[0, sound])
    if window:
        assert torch.isnan(got[0, 0].float()).all()
    if kv == BF16 and not window:
        # infinities in single channels of the newest value; a NaN that all see stays one
        k[rows[399]], v[rows[399]] = 0.5, 0.25
        v[rows[399], 0, 7], v[rows[399], 1, 9] = float("inf"), float("-inf")
        v[rows[10], 0, 7] = float("nan")
        got = ops.attn_decode(q, k, v, table, n, **call).float()
        assert torch.isnan(got[0, :, :4, 7]).all()
        assert (got[0, -1, 4:, 9] == float("-inf")).all()
        got[0, :, :4, 7] = got[0, -1, 4:, 9] = 0
        assert torch.isfinite(got).all()


def test_scores_of_any_size(scratch):
    """Very large and very small scores, a negative scale, a bf16 q near the ends of its
    range: softmax stays finite and right."""
    from iquestrt_b200 import ops
    for kv in (E4M3, BF16):
        q, k, v, table, n = _case([700, 50], 2, 8, 2, 128, kv, 16, seed=5)
        for factor, scale in ((2.0 ** 100, 2.0 ** -103), (2.0 ** -100, 2.0 ** 97), (1.0, -0.3),
                              (0.0, 1.0), (8.0, 0.5)):
            qq = (q.float() * factor).to(BF16)
            out = torch.full_like(qq, float("nan"))
            lse = torch.empty(q.shape[:3], device=DEV)
            ops.attn_decode(qq, k, v, table, n, page_size=16, scale=scale, out=out, lse=lse,
                            scratch=scratch)
            want = P.attn_decode(qq, k, v, table, n, 16, scale=scale)
            _check(out, lse, want, kv, 128, 700)
    assert scratch.status() == 0


def test_strided_operands(scratch):
    """q as a slice of a fused [.., q | k | v] row, K and V interleaved in one buffer, an
    output with gaps: the same bits as with contiguous operands."""
    from iquestrt_b200 import ops
    for kv in (E4M3, BF16):
        q, k, v, table, n = _case([260, 35], 2, 8, 2, 128, kv, 16, seed=7)
        want = ops.attn_decode(q, k, v, table, n, page_size=16, scratch=scratch)
        fused = torch.zeros(2, 2, 12, 128, dtype=BF16, device=DEV)
        fused[:, :, :8] = q
        both = torch.stack([k.view(torch.uint8), v.view(torch.uint8)], 1).view(kv)
        wide = torch.zeros(2, 2, 8, 256, dtype=BF16, device=DEV)
        tables = torch.full((2, table.shape[1] + 3), -1, dtype=torch.int32, device=DEV)
        tables[:, :table.shape[1]] = table
        got = ops.attn_decode(fused[:, :, :8], both[:, 0], both[:, 1], tables[:, :table.shape[1]], n,
                              page_size=16, out=wide[..., :128], scratch=scratch)
        # heads outermost
        hk, hv = (x.view(torch.uint8).transpose(0, 1).contiguous().transpose(0, 1).view(kv)
                  for x in (k, v))
        assert torch.equal(ops.attn_decode(q, hk, hv, table, n, page_size=16, scratch=scratch), want)
        assert torch.equal(got, want) and float(wide[..., 128:].float().abs().sum()) == 0


@pytest.mark.parametrize("kv", [E4M3, BF16], ids=["e4m3", "bf16"])
@pytest.mark.parametrize("q_len,qh,kh,window", [(1, 8, 2, 0), (4, 8, 2, 0), (3, 16, 1, 60),
                                                (8, 32, 2, 0)])
def test_accumulated_weights_and_positions(scratch, kv, q_len, qh, kh, window):
    """weights gain every row's softmax weights (the step's own rows are set), positions of the
    step's own rows are set, everything past a sequence's end stays as it was."""
    from iquestrt_b200 import ops
    lengths, page = [700, 0, q_len - 1, 33], 16
    q, k, v, table, n = _case(lengths, q_len, qh, kh, 128, kv, page, seed=11)
    rows = table.shape[1] * page
    g = _gen(12)
    w = torch.rand(4, kh, rows + 5, generator=g, device=DEV)
    pos = torch.randint(0, 99, w.shape, generator=g, device=DEV, dtype=torch.int32)
    seen = n + 1000
    want = P.attn_decode(q, k, v, table, n, page, window=window, weights=w, positions=pos, seen=seen)
    out = torch.empty_like(q)
    w0 = w.clone()
    ops.attn_decode(q, k, v, table, n, page_size=page, window=window, out=out, weights=w,
                    positions=pos, seen=seen, scratch=scratch)
    assert scratch.status() == 0
    _check(out, None, want, kv, 128, 700)
    assert torch.equal(pos, want["positions"])
    for b, m in enumerate(lengths):
        assert torch.equal(w[b, :, m:], w0[b, :, m:])
    # each weight: scores' rounding in the weight and in its normaliser, ex2, the sums
    score = (128 + 2) * 2.0 ** -23 * want["reach"].max()
    room = (2 * score + 2.0 ** -20 + 700 * 2.0 ** -24) * (want["weights"] + 1) + 2.0 ** -23
    assert ((w.double() - want["weights"]).abs() <= room).all()


def test_offsets_past_32_bits(scratch):
    """Pages at the far end of a cache of more than 2^32 bytes."""
    from iquestrt_b200 import ops
    kh, d, page = 8, 128, 64
    capacity = 2_200_000 // page * page          # x 2048 bytes: 4.5 GB
    for kv in (BF16,):
        k = torch.empty(capacity, kh, d, dtype=kv, device=DEV)
        v = torch.empty(capacity, kh, d, dtype=kv, device=DEV)
        pages = capacity // page
        lengths = [300, 129]
        ids = [pages - 1, 0, pages - 2, pages // 2, pages - 5, 7, pages - 9, 3]
        table = torch.tensor([ids[:5], ids[5:] + [-1, -1]], dtype=torch.int32, device=DEV)
        n = torch.tensor(lengths, dtype=torch.int32, device=DEV)
        g = _gen(21)
        for b, m in enumerate(lengths):
            rows = P.rows_of(table, b, m, page)
            k[rows] = torch.randn(m, kh, d, generator=g, device=DEV).to(kv)
            v[rows] = torch.randn(m, kh, d, generator=g, device=DEV).to(kv)
        q = torch.randn(2, 1, 64, d, generator=g, device=DEV).to(BF16)
        out = ops.attn_decode(q, k, v, table, n, page_size=page, scratch=scratch)
        _check(out, None, P.attn_decode(q, k, v, table, n, page), kv, d, 300)
        # and a row moved from one end to the other
        w = torch.rand(2, kh, 320, generator=g, device=DEV)
        pos = torch.arange(320, dtype=torch.int32, device=DEV).repeat(2, kh, 1)
        keep_k, keep_v = k[P.rows_of(table, 0, 300, page)], v[P.rows_of(table, 0, 300, page)]
        small = torch.arange(5, dtype=torch.int32, device=DEV)[None]
        seen = n.clone()
        want = P.kv_evict(keep_k, keep_v, small, n[:1], w[:1], pos[:1], seen, page, budget=150)
        out_n = torch.empty_like(n)
        ops.kv_evict(k, v, table, n, w, pos, seen, page_size=page, budget=150, lengths_out=out_n,
                     scratch=scratch)
        assert out_n.tolist() == [150, 129] and scratch.status() == 0
        rows = P.rows_of(table, 0, 150, page)
        assert torch.equal(k[rows], want[0][:150]) and torch.equal(v[rows], want[1][:150])


def _bits(t):
    return t.contiguous().view(torch.uint8)


EVICT = [
    # lengths, kv_heads, d, page, budget, first, last
    ([5], 1, 16, 4, 1, 0, 0),
    ([5], 1, 16, 4, 1, 1, 0),
    ([100, 0, 1, 64, 65], 2, 128, 16, 64, 0, 0),
    ([100, 200], 3, 48, 24, 50, 4, 46),
    ([129], 8, 128, 64, 128, 4, 16),
    ([5000, 4097, 4096], 2, 64, 64, 4096, 16, 1000),
    ([3000, 700], 2, 256, 1, 500, 3, 7),
    ([9000, 20000], 2, 128, 16, 6000, 16, 64),
    ([100_000], 1, 32, 64, 70_000, 16, 64),
    ([40_000, 33_000, 2], 3, 16, 128, 30_000, 0, 0),
]


@pytest.mark.parametrize("kv", [E4M3, BF16], ids=["e4m3", "bf16"])
@pytest.mark.parametrize("case", EVICT, ids=lambda c: f"n{max(c[0])}to{c[4]}d{c[2]}")
@pytest.mark.parametrize("in_place", [False, True], ids=["out", "inplace"])
def test_eviction_against_plain_lists(scratch, case, kv, in_place):
    from iquestrt_b200 import ops
    lengths, kh, d, page, budget, first, last = case
    g = _gen(31)
    table, capacity = _table(lengths, page, g)
    k = torch.randn(capacity, kh, d, generator=g, device=DEV).to(kv)
    v = torch.randn(capacity, kh, d, generator=g, device=DEV).to(kv)
    n = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    rows = table.shape[1] * page
    # many equal weights, zeros of both signs, a negative, infinities and a NaN
    w = torch.randint(0, 40, (len(lengths), kh, rows), generator=g, device=DEV).float() / 8
    w[:, :, 1::7] = -0.0
    w[:, :, 3::11] = 1e-30
    w[0, 0, 2] = float("nan")
    w[0, 0, min(4, rows - 1)] = -1.0
    w[-1, -1, lengths[-1] // 2] = float("inf")
    pos = torch.rand(w.shape, generator=g, device=DEV).argsort(dim=-1).int() * 2
    seen = torch.full_like(n, 2 * rows)
    want = P.kv_evict(k, v, table, n, w, pos, seen, page, budget=budget, first=first, last=last)
    w_out, pos_out = (None, None) if in_place else (torch.full_like(w, 77.0), torch.full_like(pos, 7))
    new_n = torch.full_like(n, -1)
    k0, v0, w0 = k.clone(), v.clone(), w.clone()
    ops.kv_evict(k, v, table, n, w, pos, seen, page_size=page, budget=budget, keep_first=first,
                 keep_last=last, lengths_out=new_n, weights_out=w_out, positions_out=pos_out,
                 scratch=scratch)
    assert scratch.status() == 0
    assert torch.equal(new_n, want[4])
    # the whole caches: moved rows in place, every other byte as it was
    assert torch.equal(_bits(k), _bits(want[0])) and torch.equal(_bits(v), _bits(want[1]))
    for b, m in enumerate(new_n.tolist()):
        got_w, got_p = (w, pos) if in_place else (w_out, pos_out)
        assert torch.equal(_bits(got_w[b, :, :m]), _bits(want[2][b, :, :m]))
        assert torch.equal(got_p[b, :, :m], want[3][b, :, :m])
        if in_place:
            assert torch.equal(_bits(w[b, :, m:]), _bits(w0[b, :, m:]))
        else:
            assert (w_out[b, :, m:] == 77.0).all() and (pos_out[b, :, m:] == 7).all()


@pytest.mark.parametrize("batch,q_len,page", [(1, 1, 64), (3, 4, 1), (300, 8, 24)])
def test_advance(scratch, batch, q_len, page):
    from iquestrt_b200 import ops
    g = _gen(41)
    lengths = torch.randint(0, 200, (batch,), generator=g, device=DEV).tolist()
    table, capacity = _table([n + q_len for n in lengths], page, g)
    n = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    seen = n + 50
    slot = torch.full((batch * q_len,), -5, dtype=torch.int64, device=DEV)
    pos = torch.full_like(slot, -5)
    ops.kv_advance(table, n, seen, slot, pos, page_size=page, capacity=capacity, q_len=q_len,
                   scratch=scratch)
    assert scratch.status() == 0
    assert n.tolist() == [m + q_len for m in lengths]
    assert seen.tolist() == [m + 50 + q_len for m in lengths]
    for b, m in enumerate(lengths):
        want = P.rows_of(table.cpu(), b, m + q_len, page)[m:].tolist()
        assert slot[b * q_len:(b + 1) * q_len].tolist() == want
        assert pos[b * q_len:(b + 1) * q_len].tolist() == list(range(m + 50, m + 50 + q_len))


def test_bad_pages_and_lengths_set_the_status(scratch):
    """Pages outside the cache and lengths outside the table: nothing is read or written out of
    place, the status word says so, and the sound sequences are as they should be."""
    from iquestrt_b200 import ops
    q, k, v, table, n = _case([100, 60, 40], 2, 8, 2, 128, E4M3, 16, seed=51)
    good = ops.attn_decode(q, k, v, table, n, page_size=16, scratch=scratch)
    assert scratch.status() == 0
    for bad in (-7, k.shape[0] // 16, 2 ** 30):
        broken = table.clone()
        broken[1, 1] = bad
        out = ops.attn_decode(q, k, v, broken, n, page_size=16, scratch=scratch)
        assert scratch.status() == 5
        assert torch.equal(out[0], good[0]) and torch.equal(out[2], good[2])
    for m in (-3, 10_000):
        broken = n.clone()
        broken[2] = m
        full = table.clamp_min(0)
        out = ops.attn_decode(q, k, v, full, broken, page_size=16, scratch=scratch)
        assert scratch.status() == 5
        assert torch.equal(out[:2], good[:2])
    slot = torch.zeros(3, dtype=torch.int64, device=DEV)
    pos, seen = torch.zeros_like(slot), n + 0
    full_rows = torch.tensor([112, 64, 40], dtype=torch.int32, device=DEV)
    before = full_rows.clone()
    ops.kv_advance(table, full_rows, seen, slot, pos, page_size=16, capacity=k.shape[0],
                   scratch=scratch)
    assert scratch.status() == 5
    assert slot.tolist()[:2] == [-1, -1] and full_rows.tolist() == before.tolist()[:2] + [41]
    assert pos.tolist() == [0, 0, 40]
    # positions at the end of a rotary table
    some = torch.tensor([3, 4, 5], dtype=torch.int32, device=DEV)
    seen = torch.tensor([9, 10, 11], dtype=torch.int32, device=DEV)
    ops.kv_advance(table, some, seen, slot, pos, page_size=16, capacity=k.shape[0],
                   max_positions=11, scratch=scratch)
    assert scratch.status() == 5
    assert pos.tolist() == [9, 10, 0] and seen.tolist() == [10, 11, 11] and some.tolist() == [4, 5, 5]
    assert slot.tolist()[2] == -1


def test_captured_step_advances_by_itself(scratch):
    """advance -> cache write -> attention with weights -> evict as one graph: each replay
    gives what the same calls give one by one, for lengths that grow past the budget."""
    from iquestrt_b200 import ops
    page, qh, kh, d, budget = 16, 8, 2, 128, 60
    g = _gen(61)
    table = torch.randperm(8, generator=g, device=DEV).int().view(2, 4)
    capacity = 8 * page

    def state():
        s = dict(n=torch.tensor([50, 3], dtype=torch.int32, device=DEV),
                 grown=torch.zeros(2, dtype=torch.int32, device=DEV),
                 seen=torch.tensor([50, 3], dtype=torch.int32, device=DEV),
                 k=torch.zeros(capacity, kh, d, dtype=E4M3, device=DEV),
                 v=torch.zeros(capacity, kh, d, dtype=E4M3, device=DEV),
                 w=torch.zeros(2, kh, 64, device=DEV),
                 pos=torch.arange(64, dtype=torch.int32, device=DEV).repeat(2, kh, 1),
                 slot=torch.zeros(2, dtype=torch.int64, device=DEV),
                 at=torch.zeros(2, dtype=torch.int64, device=DEV),
                 qkv=torch.zeros(2, (qh + 2 * kh) * d, device=DEV),
                 q=torch.zeros(2, qh, d, dtype=BF16, device=DEV),
                 out=torch.zeros(2, 1, qh, d, dtype=BF16, device=DEV),
                 cos=torch.ones(2, 32, dtype=BF16, device=DEV),
                 sin=torch.zeros(2, 32, dtype=BF16, device=DEV),
                 work=ops.AttnWork(batch=2, q_len=1, q_heads=qh, kv_heads=kh, head_dim=d, rows=64,
                                   weights=True),
                 ework=ops.EvictWork(batch=2, kv_heads=kh, rows=64))
        fill = torch.randn(64, kh, d, generator=_gen(62), device=DEV)
        for b, m in enumerate((50, 3)):
            rows = P.rows_of(table, b, m, page)
            s["k"][rows], s["v"][rows] = fill[:m].to(E4M3), fill[:m].flip(0).to(E4M3)
        return s

    ones = torch.ones(d, device=DEV)

    def step(s):
        ops.kv_advance(table, s["n"], s["seen"], s["slot"], s["at"], page_size=page,
                       capacity=capacity, lengths_out=s["grown"], scratch=scratch, pdl=True)
        ops.qkv_heads(s["qkv"], ones, ones, s["cos"], s["sin"], s["slot"], s["q"], s["k"], s["v"],
                      q_heads=qh, kv_heads=kh, rotary_dim=32, eps=1e-6, scratch=scratch, pdl=True)
        ops.attn_decode(s["q"].view(2, 1, qh, d), s["k"], s["v"], table, s["grown"], page_size=page,
                        out=s["out"], weights=s["w"], positions=s["pos"], seen=s["seen"],
                        work=s["work"], scratch=scratch, pdl=True)
        ops.kv_evict(s["k"], s["v"], table, s["grown"], s["w"], s["pos"], s["seen"], page_size=page,
                     budget=budget, keep_first=2, keep_last=20, lengths_out=s["n"],
                     work=s["ework"], scratch=scratch, pdl=True)

    eager, graphed = state(), state()
    warm = state()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step(warm)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            step(graphed)
    torch.cuda.synchronize()
    for i in range(25):
        x = torch.randn(2, (qh + 2 * kh) * d, generator=_gen(100 + i), device=DEV)
        eager["qkv"].copy_(x)
        graphed["qkv"].copy_(x)
        # this step's attention against 64 bits, on what the cache then holds
        step(eager)
        graph.replay()
        torch.cuda.synchronize()
        for key in ("n", "grown", "seen", "k", "v", "w", "pos", "slot", "at", "q", "out"):
            assert torch.equal(_bits(eager[key]), _bits(graphed[key])), (i, key)
        assert eager["n"].tolist() == [min(budget, 51 + i), min(budget, 4 + i)]
    assert scratch.status() == 0
    # the first and the latest tokens are protected, and each position is held once
    held = graphed["pos"][0, 0, :budget].tolist()
    assert len(set(held)) == budget and {0, 1} <= set(held)
    assert set(range(75 - 20, 75)) <= set(held)


def test_two_streams_at_once(scratch):
    """Calls with work areas of their own on two streams do not disturb one another."""
    from iquestrt_b200 import ops
    cases = [_case([3000 + 500 * i, 100], 1, 8, 2, 128, E4M3, 16, seed=70 + i) for i in range(2)]
    want = [ops.attn_decode(*c, page_size=16, scratch=scratch) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[], []]
    for _ in range(20):
        for i, (c, s) in enumerate(zip(cases, streams)):
            with torch.cuda.stream(s):
                got[i].append(ops.attn_decode(*c, page_size=16, scratch=scratch))
    torch.cuda.synchronize()
    for i in range(2):
        for x in got[i]:
            assert torch.equal(x, want[i])


def test_many_sequences(scratch):
    """As many sequences as a call takes, most of them empty or short, one long."""
    from iquestrt_b200 import ops
    lengths = [(7 * i) % 40 if i % 3 else 0 for i in range(1024)]
    lengths[500] = 5000
    q, k, v, table, n = _case(lengths, 1, 4, 2, 64, BF16, 8, seed=81)
    lse = torch.empty(q.shape[:3], device=DEV)
    out = ops.attn_decode(q, k, v, table, n, page_size=8, lse=lse, scratch=scratch)
    assert scratch.status() == 0
    _check(out, lse, P.attn_decode(q, k, v, table, n, 8), BF16, 64, 5000)


@pytest.mark.parametrize("kv", [E4M3, BF16], ids=["e4m3", "bf16"])
@pytest.mark.parametrize("page", [1, 2, 3, 8, 16, 24, 64, 256, 1000])
def test_pages_of_any_size(scratch, kv, page):
    """Whole boxes, pieces of boxes and single rows: whatever a page's size makes of the copies,
    the result differs by nothing but the order of no sum."""
    from iquestrt_b200 import ops
    for q_len, qh, kh, d in ((1, 8, 4, 128), (4, 16, 2, 64), (2, 4, 1, 256)):
        lengths = [1200, 333, 0, 65]
        g = _gen(91)
        rows = [torch.randn(m, 2, kh, d, generator=g, device=DEV).to(kv) for m in lengths]
        q = (2.5 * torch.randn(4, q_len, qh, d, generator=g, device=DEV)).to(BF16)
        n = torch.tensor(lengths, dtype=torch.int32, device=DEV)

        def run(page):
            table, capacity = _table(lengths, page, _gen(92))
            k = torch.full((capacity, kh, d), float("nan"), device=DEV).to(kv)
            v = k.clone()
            for b, m in enumerate(lengths):
                at = P.rows_of(table, b, m, page)
                k[at], v[at] = rows[b][:, 0], rows[b][:, 1]
            return ops.attn_decode(q, k, v, table, n, page_size=page, window=900, scratch=scratch)

        want = run(128)
        got = run(page)
        assert scratch.status() == 0
        assert torch.isfinite(got.float()).all()
        if d == 64 and kv == E4M3 and page % 2:      # these run at twice the width: another tiling
            assert (got.float() - want.float()).abs().max() <= 2.0 ** -7 * want.float().abs().max()
        else:
            assert torch.equal(got, want)


@pytest.mark.parametrize("budget", [None, 40])
def test_decode_slice_over_a_paged_cache(budget):
    """A slice whose attention reads the cache its prologue writes: each step's attention of
    every layer against 64 bits on what the cache held, the layers' outputs bit for bit those
    of a slice fed these attention outputs as stand-ins, and replays of the captured step bit
    for bit the eager steps."""
    from iquestrt_b200 import synth
    from iquestrt_b200.kernels import PagedKvCache
    from iquestrt_b200.layer import DecodeSlice
    shape = synth.LayerShape(hidden=1024, q_dim=1024, n_experts=16, top_k=2, inter=256)
    heads = synth.HeadShape(q_heads=8, kv_heads=2)
    layers = [(synth.make_layer(shape, device=DEV, seed=9, layer=i),
               synth.make_prologue(shape, heads, device=DEV, seed=9, layer=i)) for i in range(2)]

    def make():
        kv = PagedKvCache(2, 2, 2, 128, rows=64, page_size=16, budget=budget, keep_first=2,
                          keep_last=10)
        g = _gen(95)
        for x in kv.k + kv.v:
            x.copy_(torch.randn(x.shape, generator=g, device=DEV))
        kv.set_lengths([33, 5])
        return DecodeSlice(shape, layers, heads=heads, q_len=2, kv=kv, max_positions=200)

    g = _gen(96)
    inputs = [(torch.randn(2, 1024, generator=g, device=DEV).to(BF16),
               torch.randn(2, 1024, generator=g, device=DEV).to(BF16)) for _ in range(12)]
    sl, graphed = make(), make()
    stand_in = DecodeSlice(shape, layers, heads=heads, q_len=2)
    res, xn = (torch.empty_like(x) for x in inputs[0])
    stream = torch.cuda.Stream()
    warm = make()                           # every kernel's first launch, outside the capture
    warm.step(*inputs[0])
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            replayed = graphed.step(res, xn)
            replayed2 = graphed.step(res, xn)  # both all-reduce outputs' slots
    torch.cuda.synchronize()
    held = [33, 5]
    for i in range(0, 12, 2):
        eager = []
        for s in (i, i + 1):
            seen = []

            def visit(layer, q, out, norm):
                c = sl.kv
                seen.append((q.clone(), sl.attention.out.clone(), c.k[layer].clone(),
                             c.v[layer].clone(), c.lengths.clone(), out.clone(), norm.clone()))

            sl.step(*inputs[i], visit=visit)
            held = [n + 1 for n in held]
            for q, ao, k, v, n, _, _ in seen:
                assert n.tolist() == held
                want = P.attn_decode(q.view(2, 1, 8, 128), k, v, sl.kv.page_table, n, 16)
                _check(ao.view(2, 1, 8, 128), None, want, E4M3, 128, 64)
            got = stand_in.step(*inputs[i], [x[1] for x in seen])
            assert torch.equal(got[0], seen[-1][5]) and torch.equal(got[1], seen[-1][6])
            eager.append(got[0].clone())
            if budget is not None:
                held = [min(n, budget) for n in held]
            assert sl.kv.held.tolist() == held
        res.copy_(inputs[i][0])
        xn.copy_(inputs[i][1])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(replayed2[0], eager[1])
        for a, b in zip(sl.kv.k + sl.kv.v, graphed.kv.k + graphed.kv.v):
            assert torch.equal(_bits(a), _bits(b))
        assert graphed.kv.seen.tolist() == [33 + i + 2, 5 + i + 2]
    sl.check()
    graphed.check()
    assert sl.kv.scratch.status() == 0


def _slices(kv_heads=2, q_heads=8, layers=2, q_len=2, batch=2, **kv_args):
    """A maker of equal small slices over paged caches with the same prompts' rows in them."""
    from iquestrt_b200 import synth
    from iquestrt_b200.kernels import PagedKvCache
    from iquestrt_b200.layer import DecodeSlice
    shape = synth.LayerShape(hidden=1024, q_dim=128 * q_heads, n_experts=16, top_k=2, inter=256)
    heads = synth.HeadShape(q_heads=q_heads, kv_heads=kv_heads)
    weights = [(synth.make_layer(shape, device=DEV, seed=9, layer=i),
                synth.make_prologue(shape, heads, device=DEV, seed=9, layer=i))
               for i in range(layers)]

    def make(window=0, max_positions=200):
        kv = PagedKvCache(layers, batch, kv_heads, 128, q_len=q_len // batch,
                          **{**dict(rows=64, page_size=16), **kv_args})
        g = _gen(95)
        for x in kv.k + kv.v:
            x.copy_(torch.randn(x.shape, generator=g, device=DEV))
        return DecodeSlice(shape, weights, heads=heads, q_len=q_len, kv=kv, window=window,
                           max_positions=max_positions)

    def inputs(i):
        g = _gen(1000 + i)
        return tuple(torch.randn(q_len, 1024, generator=g, device=DEV).to(BF16) for _ in range(2))

    return make, inputs


def test_slice_check_sees_errors_over_the_cache():
    """A page outside the cache, below the rows that the step writes: attention reads zeros there
    and says so, and so does the slice."""
    from iquestrt_b200._lib import IqError
    make, inputs = _slices()
    sl = make()
    sl.kv.set_lengths([33, 5])
    sl.step(*inputs(0))
    sl.check()
    sl.kv.page_table[0, 0] = sl.kv.capacity // 16
    sl.step(*inputs(1))
    with pytest.raises(IqError, match="paged KV cache"):
        sl.check()
    sl.kv.page_table[0, 0] = 0
    sl.step(*inputs(2))
    sl.check()


def test_a_reused_cache_is_as_a_fresh_one():
    """Second prompts in a cache that has decoded and evicted before: every step past the budget
    as with a cache of their own, bit for bit."""
    make, inputs = _slices(budget=40, keep_first=2, keep_last=10)
    used, fresh = make(), make()
    used.kv.set_lengths([39, 12])
    for i in range(8):
        used.step(*inputs(50 + i))
    used.check()
    for a, b in zip(used.kv.k + used.kv.v, fresh.kv.k + fresh.kv.v):
        a.copy_(b)
    for sl in (used, fresh):
        sl.kv.set_lengths([36, 40])
    for i in range(8):
        got = [x.clone() for x in used.step(*inputs(i))]
        want = fresh.step(*inputs(i))
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        held = fresh.kv.held.tolist()
        assert used.kv.held.tolist() == held == [min(40, 37 + i), 40]
        for layer in range(2):
            for name in ("k", "v"):
                assert torch.equal(_bits(getattr(used.kv, name)[layer]), _bits(getattr(fresh.kv, name)[layer]))
            for name in ("weights", "positions"):
                for b, n in enumerate(held):
                    a, c = (getattr(sl.kv, name)[layer][b, :, :n] for sl in (used, fresh))
                    assert torch.equal(_bits(a), _bits(c))
    for sl in (used, fresh):
        sl.check()


def test_host_step_waits_for_the_callers_stream():
    """A prompt's rows that the caller's stream is still writing when the step is called: the
    step attends over them, as a step on that stream does."""
    from iquestrt_b200.layer import HostSliceStep
    make, inputs = _slices()
    on_stream, from_host = make(), make()
    host = HostSliceStep(from_host)
    g = _gen(97)
    prompt = [torch.randn(x.shape, generator=g, device=DEV).to(x.dtype) for x in on_stream.kv.k]

    def write(kv, rows):
        for k, v, x in zip(kv.k, kv.v, rows):
            k.copy_(x)
            v.copy_(x)

    on_stream.kv.set_lengths([33, 5])
    write(on_stream.kv, prompt)
    want = on_stream.step(*inputs(0))[0].cpu()
    res, xn = (x.cpu() for x in inputs(0))
    from_host.kv.set_lengths([33, 5])
    write(from_host.kv, [torch.zeros_like(x) for x in prompt])
    torch.cuda.synchronize()
    torch.cuda._sleep(100_000_000)               # some 50 ms
    write(from_host.kv, prompt)
    assert torch.equal(host(res, xn), want)
    from_host.check()


@pytest.mark.parametrize("kv_args", [
    dict(), dict(budget=40, keep_first=2, keep_last=10),
    dict(q_len=8, page_size=1, budget=2, keep_first=0),      # more new rows than the budget
    dict(q_len=6, page_size=4, rows=16)], ids=["plain", "budget", "small", "tight"])
def test_host_steps_over_a_cache(kv_args):
    """Building a host step leaves the cache as it was, a full budget's rows among it; its steps
    are those of a slice that is called step by step, bit for bit."""
    from iquestrt_b200.layer import HostSliceStep
    make, inputs = _slices(**kv_args)
    sl, other = make(), make()
    full = kv_args.get("budget") or 7
    g = _gen(98)
    w = None
    if sl.kv.budget is not None:
        w = [torch.rand(x.shape, generator=g, device=DEV) for x in sl.kv.weights]
    for s in (sl, other):
        s.kv.set_lengths([full, 1], weights=w)
    names = ("held", "lengths", "seen", "slot", "pos", "page_table", "k", "v", "weights", "positions")

    def state(kv):
        parts = [getattr(kv, n) for n in names]
        return [x.clone() for part in parts if part is not None
                for x in (part if isinstance(part, list) else [part])]

    before = state(sl.kv)
    host = HostSliceStep(sl)
    assert all(torch.equal(_bits(a), _bits(b)) for a, b in zip(before, state(sl.kv)))
    for i in range(3):
        res, xn = (x.cpu() for x in inputs(i))
        got = host(res, xn).clone()
        assert torch.equal(got, other.step(*inputs(i))[0].cpu())
        assert sl.kv.held.tolist() == other.kv.held.tolist()
        assert sl.kv.seen.tolist() == other.kv.seen.tolist()
        for a, b in zip(sl.kv.k + sl.kv.v, other.kv.k + other.kv.v):
            assert torch.equal(_bits(a), _bits(b))
        for b, n in enumerate(sl.kv.held.tolist()):
            for a, c in zip((sl.kv.weights or []) + (sl.kv.positions or []),
                            (other.kv.weights or []) + (other.kv.positions or [])):
                assert torch.equal(_bits(a[b, :, :n]), _bits(c[b, :, :n]))
    sl.check()
    other.check()


@pytest.mark.parametrize("kv", [E4M3, BF16], ids=["e4m3", "bf16"])
@pytest.mark.parametrize("page,cut", [(64, 1), (64, 40), (24, 5), (3, 1), (256, 200)])
def test_a_page_that_straddles_the_caches_end(scratch, kv, page, cut):
    """A cache whose rows are no whole number of pages: up to its last row all is well; a row
    behind it is read as zeros and the status says so, whether pages are copied in boxes or
    gathered row by row."""
    from iquestrt_b200 import ops
    g = _gen(71)
    table = torch.randperm(10, generator=g, device=DEV).int().view(2, 5)
    table = torch.where(table == table[0, 4], 10, table)     # sequence 0 ends in the last page
    capacity = 11 * page - cut
    k = torch.zeros(11 * page, 2, 128, device=DEV)
    v = torch.zeros_like(k)
    k[:capacity] = torch.randn(capacity, 2, 128, generator=g, device=DEV)
    v[:capacity] = torch.randn(capacity, 2, 128, generator=g, device=DEV)
    k, v = k.to(kv), v.to(kv)
    q = (2.5 * torch.randn(2, 2, 8, 128, generator=g, device=DEV)).to(BF16)
    for over in (0, 1, cut):
        lengths = [5 * page - cut + over, 4 * page]
        n = torch.tensor(lengths, dtype=torch.int32, device=DEV)
        out = ops.attn_decode(q, k[:capacity], v[:capacity], table, n, page_size=page, scratch=scratch)
        assert scratch.status() == (5 if over else 0), over
        _check(out, None, P.attn_decode(q, k, v, table, n, page), kv, 128, max(lengths))


@pytest.mark.parametrize("q_len", [1, 3])
def test_a_sequence_without_room_keeps_its_weights(scratch, q_len):
    """Slots of -1: the sequence's weights and positions stay, the others' are what they are
    without slots, bit for bit."""
    from iquestrt_b200 import ops
    page, kh = 16, 2
    q, k, v, table, n = _case([700, 1500, 40], q_len, 8, kh, 128, E4M3, page, seed=14)
    g = _gen(15)
    w = torch.rand(3, kh, table.shape[1] * page, generator=g, device=DEV)
    pos = torch.randint(0, 99, w.shape, generator=g, device=DEV, dtype=torch.int32)
    slot = torch.arange(3 * q_len, device=DEV)
    slot.view(3, q_len)[1] = -1
    got = []
    for more in (dict(), dict(slot=slot)):
        ww, pp = w.clone(), pos.clone()
        out = ops.attn_decode(q, k, v, table, n, page_size=page, weights=ww, positions=pp, seen=n + 9,
                              scratch=scratch, **more)
        got.append((out, ww, pp))
    assert scratch.status() == 0
    (out, ww, pp), (out2, ww2, pp2) = got
    assert torch.equal(out, out2)
    for b in (0, 2):
        assert torch.equal(ww[b], ww2[b]) and torch.equal(pp[b], pp2[b])
    assert torch.equal(ww2[1], w[1]) and torch.equal(pp2[1], pos[1])
    assert not torch.equal(ww[1], w[1]) and not torch.equal(pp[1], pos[1])


def test_a_slice_keeps_the_state_of_a_sequence_at_its_end():
    """A sequence that reaches `max_positions` while another goes on: from then on its rows,
    weights, positions and counts stay as they are, and the status says so at every step."""
    from iquestrt_b200._lib import IqError
    make, inputs = _slices(budget=40, keep_first=2, keep_last=10)
    sl = make(max_positions=60)
    sl.kv.set_lengths([39, 8])

    def state():
        kv = sl.kv
        return [kv.held[:1].clone(), kv.seen[:1].clone()] + \
            [x[0, :, :40].clone() for x in kv.weights + kv.positions] + \
            [x[P.rows_of(kv.page_table, 0, 40, 16)].clone() for x in kv.k + kv.v]

    for i in range(21):
        sl.step(*inputs(i))
        sl.check()
    assert sl.kv.seen.tolist() == [60, 29] and sl.kv.held.tolist() == [40, 29]
    before = state()
    for i in range(21, 25):
        sl.step(*inputs(i))
        with pytest.raises(IqError):
            sl.check()
        assert all(torch.equal(_bits(a), _bits(b)) for a, b in zip(before, state()))
    assert sl.kv.seen.tolist() == [60, 33] and sl.kv.held.tolist() == [40, 33]
    assert sl.kv.positions[1][1, 0, :33].tolist() == list(range(33))


@pytest.mark.parametrize("kv", [E4M3, BF16], ids=["e4m3", "bf16"])
@pytest.mark.parametrize("down,heard", [(14, False), (14, True), (17, False), (20, False)])
def test_elements_of_q_far_below_the_rows_largest(scratch, kv, heard, down):
    """One channel of q lies some 2^`down` above the others, and the keys have something there
    (`heard`) or zeros, so that the scores are the small elements' alone.  With e4m3 caches q is
    rounded to 2^-25 of the power of two at or below the row's largest, here 1: a score is off by
    that times scale sum |k| (beside what fp32 sums leave), a weight relative to the others by
    twice that in the exponent; with bf16 caches q is taken as it is."""
    from iquestrt_b200 import ops
    lengths, d = [700, 40], 128
    q, k, v, table, n = _case(lengths, 2, 8, 2, d, kv, 16, seed=23, sharp=2.0 ** -down)
    q = q.clamp(-4 * 2.0 ** -down, 4 * 2.0 ** -down)
    q[..., 5] = 1.0
    if not heard:
        k[..., 5] = 0.0
    scale = 2.0 ** down * d ** -0.5
    out = torch.full_like(q, float("nan"))
    lse = torch.empty(q.shape[:3], device=DEV)
    ops.attn_decode(q, k, v, table, n, page_size=16, scale=scale, out=out, lse=lse, scratch=scratch)
    assert scratch.status() == 0
    want = P.attn_decode(q, k, v, table, n, 16, scale=scale)
    rows = torch.cat([P.rows_of(table, b, m, 16) for b, m in enumerate(lengths)])
    step = scale * 2.0 ** -25 * float(k[rows].double().abs().sum(-1).max()) if kv == E4M3 else 0.0
    score = (d + 2) * 2.0 ** -23 * want["reach"][..., None] + step
    u = 2.0 ** -8 if kv == BF16 else 2.0 ** -11
    rel = torch.expm1(2 * score) + u * (1 + torch.expm1(2 * score)) + 2.0 ** -21 + 2 * 700 * 2.0 ** -24
    room = 1.01 * (2.0 ** -8 * want["out"].abs() + (1 + 2.0 ** -8) * rel * want["mass"]) + 6 * 700 * 2.0 ** -33
    off = (out.double() - want["out"]).abs()
    assert (off <= room).all(), float((off / room).max())
    room = score[..., 0] + 2.0 ** -21 + 700 * 2.0 ** -24 + 2.0 ** -22 * want["lse"].abs()
    off = (lse.double() - want["lse"]).abs()
    assert (off <= room).all(), float((off / room).max())


@pytest.mark.parametrize("window", [112, 10 ** 6, 1 << 31, 1 << 62])
def test_windows_past_the_page_table_are_none(scratch, window):
    from iquestrt_b200 import ops
    q, k, v, table, n = _case([100, 60], 2, 8, 2, 128, E4M3, 16, seed=52)
    assert table.shape[1] * 16 == 112
    want = ops.attn_decode(q, k, v, table, n, page_size=16, scratch=scratch)
    assert torch.equal(ops.attn_decode(q, k, v, table, n, page_size=16, window=window, scratch=scratch), want)


@pytest.mark.parametrize("kv", [E4M3, BF16], ids=["e4m3", "bf16"])
@pytest.mark.parametrize("d,page,q_len,qh", [(48, 16, 4, 8), (64, 3, 3, 8), (64, 64, 2, 4), (80, 64, 8, 16),
                                             (128, 1, 4, 32), (192, 24, 2, 10), (256, 64, 4, 16)])
@pytest.mark.parametrize("length", [90, 6000])
def test_values_that_are_not_finite_stay_in_their_channel(scratch, kv, d, page, q_len, qh, length):
    """Single NaNs and infinities among the values that only some rows of a step see (the newest
    token's, one that slides out of the window), in sequences of one CTA and of many: the
    channels of the rows and heads that see them get them, all else keeps its bits."""
    from iquestrt_b200 import ops
    window = 70 if length < 1000 else 5900
    q, k, v, table, n = _case([length, 33], q_len, qh, 2, d, kv, page, seed=24)
    call = dict(page_size=page, window=window, scratch=scratch)
    clean = ops.attn_decode(q, k, v, table, n, **call).clone()
    rows = P.rows_of(table, 0, length, page)
    first, group = length - q_len - window + 1, qh // 2
    bad = [(rows[-1], 0, 7, float("nan"), q_len - 1), (rows[-1], 1, d - 1, float("-inf"), q_len - 1),
           (rows[first], 1, d // 2 + 1, float("inf"), 0), (rows[first], 0, 0, float("nan"), 0)]
    want = clean.clone()
    for row, h, c, x, r in bad:
        if kv == E4M3:
            x = float("nan")                     # (the type has no infinities)
        v[row, h, c] = x
        want[0, r, h * group:(h + 1) * group, c] = x
    got = ops.attn_decode(q, k, v, table, n, **call)
    assert scratch.status() == 0
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(torch.nan_to_num(got, nan=0.0), torch.nan_to_num(want, nan=0.0))


@pytest.mark.parametrize("window", [0, 20])
def test_slice_of_several_tokens_a_sequence_over_pages_of_its_own(window):
    """Three sequences of two tokens a step, over a page table in any order with pages to spare:
    every layer's attention of every step against 64 bits on what the cache held."""
    g = _gen(99)
    table = torch.randperm(20, generator=g, device=DEV).int()[:15].view(3, 5)
    make, inputs = _slices(q_len=6, batch=3, rows=20, page_size=4, page_table=table, capacity=80)
    sl = make(window=window)
    sl.kv.set_lengths([10, 0, 3])
    checked = []

    def visit(layer, q, out, norm):
        c = sl.kv
        want = P.attn_decode(q.view(3, 2, 8, 128), c.k[layer], c.v[layer], table, c.lengths, 4,
                             window=window)
        _check(sl.attention.out.view(3, 2, 8, 128), None, want, E4M3, 128, 20)
        checked.append(layer)

    for i in range(5):
        sl.step(*inputs(i), visit=visit)
        sl.check()
        assert sl.kv.held.tolist() == [12 + 2 * i, 2 + 2 * i, 5 + 2 * i]
    assert checked == [0, 1] * 5


def test_a_scratch_of_another_device_is_refused():
    """Its status word would be written from this device."""
    from iquestrt_b200 import ops
    other = ops.Scratch("cpu")
    q, k, v, table, n = _case([40, 3], 1, 8, 2, 128, E4M3, 16, seed=53)
    w = torch.zeros(2, 2, table.shape[1] * 16, device=DEV)
    pos = torch.zeros_like(w, dtype=torch.int32)
    slot = torch.zeros(2, dtype=torch.int64, device=DEV)
    before = n.clone()
    calls = [lambda: ops.attn_decode(q, k, v, table, n, page_size=16, scratch=other),
             lambda: ops.kv_evict(k, v, table, n, w, pos, n, page_size=16, budget=8,
                                  lengths_out=n.clone(), scratch=other),
             lambda: ops.kv_advance(table, n, n.clone(), slot, slot.clone(), page_size=16,
                                    capacity=k.shape[0], scratch=other)]
    for call in calls:
        with pytest.raises(ValueError, match="scratch must be on cuda:0"):
            call()
    assert torch.equal(n, before)
