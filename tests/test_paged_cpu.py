"""Refusals of the paged-cache operators (no GPU needed: the checks come before any launch),
the sizes of their work areas, and the oracle's own arithmetic on cases small enough to work
out otherwise."""

import ctypes as C

import pytest
import torch

from oracle import paged as P


def _lib():
    from iquestrt_b200 import _lib as L
    return L, L.load()


def _attn_args():
    """Arguments that pass every check up to the device query (addresses are never read)."""
    L, lib = _lib()
    a = L.AttnArgs()
    a.q = a.k_cache = a.v_cache = a.page_table = a.lengths = a.out = a.work = 4096
    a.q_b, a.q_r, a.q_h, a.o_b, a.o_r, a.o_h = 1024, 1024, 128, 1024, 1024, 128
    a.k_row = a.v_row = 128
    a.k_head = a.v_head = 128
    a.kv_kind, a.capacity, a.table_stride, a.page_size, a.max_pages = 0, 640, 10, 64, 10
    a.batch, a.q_len, a.q_heads, a.kv_heads, a.head_dim = 1, 1, 8, 1, 128
    a.scale, a.work_bytes = 0.1, 1 << 40
    return L, lib, a


@pytest.mark.parametrize("field,value,code", [
    ("q", None, 1), ("k_cache", None, 1), ("v_cache", None, 1), ("page_table", None, 1),
    ("lengths", None, 1), ("out", None, 1), ("work", None, 1), ("page_size", 0, 1),
    ("max_pages", 0, 1), ("capacity", 0, 1), ("window", -1, 1), ("kv_kind", 2, 1),
    ("work_bytes", 100, 1), ("k_cache", 4096 + 8, 1), ("v_cache", 4096 + 8, 1), ("k_row", 120, 1),
    ("v_row", 120, 1), ("v_head", 8, 1), ("q", 4104, 1), ("q_h", 127, 1), ("q_r", 1028, 1), ("out", 4104, 1), ("o_h", 132, 1),
    ("k_row", -128, 1), ("v_head", 1 << 41, 1), ("work", 4104, 1),
    ("positions", 4096, 1), ("seen", 4096, 1),
    ("batch", 0, 6), ("batch", 1025, 6), ("q_len", 0, 6), ("q_len", 9, 6), ("q_heads", 0, 6),
    ("head_dim", 8, 6), ("head_dim", 100, 6), ("head_dim", 272, 6), ("q_heads", 513, 6),
    ("kv_heads", 3, 6), ("max_pages", 1 << 25, 6),
])
def test_attention_refuses(field, value, code):
    L, lib, a = _attn_args()
    setattr(a, field, value)
    assert lib.iq_attn_decode(C.byref(a), None) == code
    assert lib.iq_attn_decode(None, None) == L.IQ_ERR_ARG


def test_attention_weights_refusals():
    L, lib, a = _attn_args()
    a.weights, a.weights_rows = 4096, 639                # fewer than the table covers
    assert lib.iq_attn_decode(C.byref(a), None) == L.IQ_ERR_ARG
    a.weights_rows, a.positions = 640, 4096              # positions without seen
    assert lib.iq_attn_decode(C.byref(a), None) == L.IQ_ERR_ARG


def test_work_sizes():
    _, lib = _lib()
    plain = lib.iq_attn_work_bytes(4, 1, 64, 8, 128, 4096, 0)
    weighted = lib.iq_attn_work_bytes(4, 1, 64, 8, 128, 4096, 1)
    assert 0 < plain and weighted - plain >= 4 * 4096 * 64 * 4
    for bad in ((0, 1, 8, 1, 128, 64, 0), (1, 9, 8, 1, 128, 64, 0), (1, 1, 8, 3, 128, 64, 0),
                (1, 1, 8, 1, 100, 64, 0), (1, 1, 8, 1, 128, 0, 0), (1025, 1, 8, 1, 128, 64, 0)):
        assert lib.iq_attn_work_bytes(*bad) == 0
    assert lib.iq_evict_work_bytes(2, 8, 4096) >= 2 * 8 * 2048 * 8
    for bad in ((0, 8, 64), (1, 0, 64), (1, 8, 0), (1, 8, 262145), (70000, 1, 64)):
        assert lib.iq_evict_work_bytes(*bad) == 0


def _evict_args():
    L, lib = _lib()
    a = L.EvictArgs()
    for f in ("k_cache", "v_cache", "page_table", "lengths", "seen", "weights", "positions",
              "weights_out", "positions_out", "work"):
        setattr(a, f, 4096)
    a.lengths_out = 8192
    a.k_row = a.v_row = a.k_head = a.v_head = 128
    a.kv_kind, a.capacity, a.table_stride, a.page_size, a.max_pages = 0, 640, 10, 64, 10
    a.batch, a.kv_heads, a.head_dim, a.budget, a.work_bytes = 1, 1, 128, 32, 1 << 40
    return L, lib, a


@pytest.mark.parametrize("field,value,code", [
    ("k_cache", None, 1), ("v_cache", None, 1), ("page_table", None, 1), ("lengths", None, 1),
    ("seen", None, 1), ("weights", None, 1), ("positions", None, 1), ("weights_out", None, 1),
    ("positions_out", None, 1), ("lengths_out", None, 1), ("work", None, 1), ("budget", 0, 1),
    ("keep_first", -1, 1), ("keep_last", -1, 1), ("keep_first", 33, 1), ("keep_last", 33, 1),
    ("lengths_out", 4096, 1), ("page_size", 0, 1), ("kv_kind", 5, 1), ("k_row", 8, 1),
    ("v_head", 8, 1), ("work_bytes", 10, 1), ("batch", 0, 6), ("kv_heads", 0, 6),
    ("max_pages", 1 << 20, 6), ("head_dim", 8, 6),
])
def test_eviction_refuses(field, value, code):
    L, lib, a = _evict_args()
    setattr(a, field, value)
    assert lib.iq_kv_evict(C.byref(a), None) == code
    assert lib.iq_kv_evict(None, None) == L.IQ_ERR_ARG


@pytest.mark.parametrize("field,value", [
    ("page_table", None), ("lengths", None), ("seen", None), ("lengths_out", None),
    ("seen_out", None), ("slot", None), ("pos", None), ("page_size", 0), ("max_pages", 0),
    ("capacity", 0), ("batch", 0), ("q_len", 0), ("q_len", 9), ("max_positions", -1),
])
def test_advance_refuses(field, value):
    L, lib = _lib()
    a = L.AdvanceArgs()
    for f in ("page_table", "lengths", "seen", "lengths_out", "seen_out", "slot", "pos"):
        setattr(a, f, 4096)
    a.page_size, a.max_pages, a.capacity, a.batch, a.q_len = 16, 4, 64, 1, 1
    setattr(a, field, value)
    assert lib.iq_kv_advance(C.byref(a), None) == L.IQ_ERR_ARG


def test_outputs_that_overlap_what_others_read_are_refused():
    """Lengths and counts in place mean element on element; a shifted view is an error, for the
    eviction (every head reads them) any overlap is."""
    L, lib = _lib()
    a = L.AdvanceArgs()
    for i, f in enumerate(("page_table", "lengths", "seen", "lengths_out", "seen_out", "slot", "pos")):
        setattr(a, f, 4096 * (i + 1))
    a.page_size, a.max_pages, a.capacity, a.batch, a.q_len = 16, 4, 64, 8, 1
    for field, value in (("lengths_out", a.lengths + 4), ("lengths_out", a.seen - 28),
                         ("seen_out", a.lengths - 4), ("seen_out", a.seen + 28),
                         ("seen_out", a.lengths_out + 8), ("seen_out", a.lengths_out)):
        was = getattr(a, field)
        setattr(a, field, value)
        assert lib.iq_kv_advance(C.byref(a), None) == L.IQ_ERR_ARG, (field, value)
        setattr(a, field, was)

    _, _, e = _evict_args()
    e.batch = 8
    for i, f in enumerate(("lengths", "seen", "lengths_out", "weights", "weights_out", "positions",
                           "positions_out")):
        setattr(e, f, 65536 * (i + 1))
    for change in (dict(lengths_out=e.lengths + 4), dict(lengths_out=e.seen - 28),
                   dict(lengths_out=e.seen), dict(weights_out=e.weights, wo_b=640),
                   dict(positions_out=e.positions, po_h=640)):
        was = {f: getattr(e, f) for f in change}
        for f, value in change.items():
            setattr(e, f, value)
        assert lib.iq_kv_evict(C.byref(e), None) == L.IQ_ERR_ARG, change
        for f, value in was.items():
            setattr(e, f, value)


def _tensors():
    bf = torch.bfloat16
    return dict(q=torch.zeros(2, 1, 8, 128, dtype=bf), k_cache=torch.zeros(64, 2, 128, dtype=bf),
                v_cache=torch.zeros(64, 2, 128, dtype=bf),
                page_table=torch.zeros(2, 4, dtype=torch.int32),
                lengths=torch.zeros(2, dtype=torch.int32), page_size=8)


@pytest.mark.parametrize("change,message", [
    (dict(q=torch.zeros(2, 8, 128)), "q must be"),
    (dict(q=torch.zeros(2, 1, 8, 128)), "dtype"),
    (dict(q=torch.zeros(2, 1, 8, 64, dtype=torch.bfloat16)), "does not fit"),
    (dict(q=torch.zeros(2, 1, 7, 128, dtype=torch.bfloat16)), "does not fit"),
    (dict(k_cache=torch.zeros(64, 2, 128)), "bf16 or both e4m3"),
    (dict(v_cache=torch.zeros(64, 2, 128, dtype=torch.float8_e4m3fn)), "dtype"),
    (dict(v_cache=torch.zeros(32, 2, 128, dtype=torch.bfloat16)), "shape"),
    (dict(page_table=torch.zeros(2, 4, dtype=torch.int64)), "dtype"),
    (dict(page_table=torch.zeros(3, 4, dtype=torch.int32)), "page_table"),
    (dict(page_table=torch.zeros(2, 0, dtype=torch.int32)), "page_table"),
    (dict(page_size=0), "page_size"),
    (dict(lengths=torch.zeros(3, dtype=torch.int32)), "shape"),
    (dict(lengths=torch.zeros(2)), "dtype"),
    (dict(lengths=torch.zeros(4, dtype=torch.int32)[::2]), "contiguous"),
    (dict(window=-1), "window"),
    (dict(out=torch.zeros(2, 1, 8, 128)), "dtype"),
    (dict(out=torch.zeros(1, 1, 8, 128, dtype=torch.bfloat16).expand(2, 1, 8, 128)), "overlap"),
    (dict(lse=torch.zeros(2, 1, 7)), "shape"),
    (dict(weights=torch.zeros(2, 2, 31)), "weights"),
    (dict(weights=torch.zeros(2, 2, 32), positions=torch.zeros(2, 2, 32, dtype=torch.int32)), "seen"),
    (dict(positions=torch.zeros(2, 2, 32, dtype=torch.int32),
          seen=torch.zeros(2, dtype=torch.int32)), "weights"),
    (dict(), "CUDA"),
])
def test_attention_wrapper_refuses(change, message):
    from iquestrt_b200 import ops
    with pytest.raises(ValueError, match=message):
        ops.attn_decode(**{**_tensors(), **change})


@pytest.mark.parametrize("change,message", [
    (dict(weights=torch.zeros(2, 2)), "weights must be"),
    (dict(weights=torch.zeros(2, 3, 32)), "weights must be"),
    (dict(weights=torch.zeros(2, 2, 32, dtype=torch.float64)), "dtype"),
    (dict(positions=torch.zeros(2, 2, 31, dtype=torch.int32)), "shape"),
    (dict(budget=0), "budget"), (dict(budget=4, keep_first=3, keep_last=2), "budget"),
    (dict(lengths_out=torch.zeros(3, dtype=torch.int32)), "shape"),
    (dict(k_cache=torch.zeros(1, 2, 128, dtype=torch.bfloat16).expand(64, 2, 128)), "overlap"),
    (dict(), "CUDA"),
])
def test_eviction_wrapper_refuses(change, message):
    from iquestrt_b200 import ops
    t = _tensors()
    del t["q"]
    t.update(weights=torch.zeros(2, 2, 32), positions=torch.zeros(2, 2, 32, dtype=torch.int32),
             seen=torch.zeros(2, dtype=torch.int32), lengths_out=torch.zeros(2, dtype=torch.int32),
             budget=8)
    with pytest.raises(ValueError, match=message):
        ops.kv_evict(**{**t, **change})
    t["lengths_out"] = t["lengths"]
    with pytest.raises(ValueError, match="lengths_out"):
        ops.kv_evict(**t)


def test_advance_wrapper_refuses():
    from iquestrt_b200 import ops
    i32 = torch.zeros(2, dtype=torch.int32)
    t = dict(page_table=torch.zeros(2, 4, dtype=torch.int32), lengths=i32, seen=i32.clone(),
             slot=torch.zeros(2, dtype=torch.int64), pos=torch.zeros(2, dtype=torch.int64),
             page_size=8, capacity=64)
    for change, message in ((dict(q_len=9), "q_len"), (dict(slot=torch.zeros(3, dtype=torch.int64)), "shape"),
                            (dict(pos=i32), "dtype"), (dict(capacity=0), "capacity"), (dict(), "CUDA")):
        with pytest.raises(ValueError, match=message):
            ops.kv_advance(**{**t, **change})


def test_oracle_attention_by_hand():
    """Two keys of one channel pair: softmax weights 3/4 and 1/4; a window of one row; an
    empty sequence."""
    import math
    q = torch.zeros(2, 1, 1, 2)
    q[:, 0, 0, 0] = math.log(3.0)
    k = torch.tensor([[[0.0, 0.0]], [[1.0, 0.0]], [[9.0, 9.0]]])
    v = torch.tensor([[[4.0, 0.0]], [[8.0, 4.0]], [[9.0, 9.0]]])
    table = torch.tensor([[1, 0, 2], [0, 0, 0]])
    n = torch.tensor([2, 0])
    w = torch.full((2, 1, 3), 10.0)
    pos, seen = torch.zeros(2, 1, 3, dtype=torch.int32), torch.tensor([7, 7])
    r = P.attn_decode(q, k, v, table, n, 1, scale=1.0, weights=w, positions=pos, seen=seen)
    assert torch.allclose(r["out"][0, 0, 0], torch.tensor([7.0, 3.0], dtype=torch.float64))
    assert abs(float(r["lse"][0, 0, 0]) - math.log(4.0)) < 1e-6
    assert float(r["lse"][1, 0, 0]) == -math.inf and float(r["out"][1].abs().sum()) == 0
    assert torch.allclose(r["weights"][0, 0], torch.tensor([10.75, 0.25, 10.0], dtype=torch.float64))
    assert r["positions"][0, 0].tolist() == [0, 6, 0]
    r = P.attn_decode(q, k, v, table, n, 1, scale=1.0, window=1)
    assert torch.allclose(r["out"][0, 0, 0], torch.tensor([4.0, 0.0], dtype=torch.float64))


def test_oracle_eviction_by_hand():
    """Five rows to three: position 0 is protected, row 4 is the latest, ties go low."""
    k = torch.arange(5.0).view(5, 1, 1).repeat(1, 1, 2)
    w = torch.tensor([[[0.0, 2.0, 2.0, 1.0, 0.5]]])
    pos = torch.tensor([[[0, 3, 5, 6, 9]]], dtype=torch.int32)
    out = P.kv_evict(k, k + 10, torch.tensor([[0, 1, 2, 3, 4]]), torch.tensor([5]), w, pos,
                     torch.tensor([10]), 1, budget=3, first=1, last=1)
    assert out[0][:, 0, 0].tolist() == [0.0, 1.0, 4.0, 3.0, 4.0]
    assert out[1][:3, 0, 0].tolist() == [10.0, 11.0, 14.0]
    assert out[2][0, 0, :3].tolist() == [0.0, 2.0, 0.5] and out[3][0, 0, :3].tolist() == [0, 3, 9]
    assert out[4].tolist() == [3]


@pytest.mark.parametrize("change,message", [
    (dict(page_size=0), "at least 1"), (dict(batch=0), "at least 1"), (dict(layers=0), "at least 1"),
    (dict(budget=3), "protected"), (dict(budget=20, keep_last=17), "protected"),
    (dict(budget=20, keep_first=-1), "protected"),
    (dict(page_table=torch.zeros(2, 3, dtype=torch.int32)), "capacity"),
    (dict(page_table=torch.zeros(1, 4, dtype=torch.int32), capacity=64), "page_table"),
    (dict(page_table=torch.zeros(2, 3, dtype=torch.int32), capacity=64), "page_table"),
])
def test_cache_holder_refuses(change, message):
    from iquestrt_b200.kernels import PagedKvCache
    args = dict(layers=1, batch=2, kv_heads=1, head_dim=128, rows=64, page_size=16, device="cpu")
    with pytest.raises(ValueError, match=message):
        PagedKvCache(**{**args, **change})


def test_holders_refuse():
    from iquestrt_b200.kernels import PagedAttention, PagedKvCache
    from iquestrt_b200.workspace import Workspace
    ok = dict(rows=64, page_size=16, device="cpu")
    for change, message in ((dict(q_len=9), "q_len"), (dict(dtype=torch.float16), "bf16 or e4m3"),
                            (dict(budget=64), "budget"), (dict(budget=0), "budget"),
                            (dict(page_table=torch.zeros(2, 4)), "capacity")):
        with pytest.raises(ValueError, match=message):
            PagedKvCache(1, 2, 2, 128, **{**ok, **change})
    kv = PagedKvCache(1, 2, 2, 128, **ok)
    assert kv.capacity == 128 and kv.page_table.tolist() == [[0, 1, 2, 3], [4, 5, 6, 7]]
    for lengths in ([1], [1, 65], [-1, 0]):
        with pytest.raises(ValueError, match="lengths"):
            kv.set_lengths(lengths)
    kv.set_lengths([3, 64])
    assert kv.held.tolist() == kv.seen.tolist() == [3, 64]
    ws = Workspace(device="cpu")
    with pytest.raises(ValueError, match="share"):
        PagedAttention(3, kv, ws=ws)
    with pytest.raises(ValueError, match="window"):
        PagedAttention(4, kv, ws=ws, window=-1)


def test_a_window_over_a_cache_that_evicts_is_refused():
    """Eviction fills freed rows with later ones, so the last rows are not the last tokens: five
    rows cut to four (row 1 has the least weight) leave token 4 in row 1, and the next token's
    window of two rows would see rows 3 and 4, tokens 3 and 5, instead of tokens 4 and 5."""
    from iquestrt_b200.kernels import PagedAttention, PagedKvCache
    from iquestrt_b200.workspace import Workspace
    pos = torch.arange(6, dtype=torch.int32).view(1, 1, 6)
    w = torch.tensor([[[5.0, 0.0, 3.0, 2.0, 1.0, 0.0]]])
    kv = torch.zeros(6, 1, 2)
    moved = P.kv_evict(kv, kv, torch.arange(6)[None], torch.tensor([5]), w, pos, torch.tensor([5]),
                       1, budget=4)[3]
    assert moved[0, 0, :4].tolist() == [0, 4, 2, 3]
    cache = PagedKvCache(1, 1, 1, 128, rows=64, page_size=16, budget=24, device="cpu")
    ws = Workspace(device="cpu")
    for window in (1, 8, 1000):
        with pytest.raises(ValueError, match="without a budget"):
            PagedAttention(4, cache, ws=ws, window=window)
    PagedAttention(4, cache, ws=ws)
    PagedAttention(4, PagedKvCache(1, 1, 1, 128, rows=64, page_size=16, device="cpu"), ws=ws, window=8)


@pytest.mark.parametrize("layer_code,cache_code", [(0, 0), (0, 5), (5, 0), (5, 3)])
def test_slice_check_reads_the_caches_status_too(layer_code, cache_code):
    """The attention, eviction and bookkeeping of a slice report to the cache's scratch: an error
    there is the slice's, and is not reported a second time."""
    from types import SimpleNamespace

    from iquestrt_b200._lib import IqError
    from iquestrt_b200.layer import DecodeSlice

    class Status:
        def __init__(self, code):
            self.code = code

        def status(self):
            code, self.code = self.code, 0
            return code

        def raise_on_error(self):
            code = self.status()
            if code:
                raise IqError("fake", code)

    sl = object.__new__(DecodeSlice)
    sl.layer = SimpleNamespace(check=Status(layer_code).raise_on_error)
    sl.kv = SimpleNamespace(scratch=Status(cache_code))
    if layer_code or cache_code:
        with pytest.raises(IqError):
            sl.check()
    sl.check()
    sl.kv = None
    sl.check()


def _budget_cache():
    from iquestrt_b200.kernels import PagedKvCache
    return PagedKvCache(2, 2, 3, 128, rows=64, page_size=16, budget=40, device="cpu")


def test_set_lengths_starts_the_bookkeeping_anew():
    """Nothing of the sequences that a cache held before is left: weights, positions, counts."""
    fresh, used = _budget_cache(), _budget_cache()
    for x in used.weights:
        x.fill_(5.0)
    for x in used.positions:
        x.fill_(-9)
    used.held.fill_(17)
    used.seen.fill_(18)
    for kv in (fresh, used):
        kv.set_lengths([33, 5])
        assert kv.held.tolist() == kv.seen.tolist() == [33, 5]
    for name in ("weights", "positions"):
        for a, b in zip(getattr(fresh, name), getattr(used, name)):
            assert torch.equal(a, b)
    assert float(used.weights[0].abs().sum()) == 0
    assert torch.equal(used.positions[1][1, 2], torch.arange(64, dtype=torch.int32))


def test_set_lengths_takes_a_prompts_weights_and_positions():
    kv = _budget_cache()
    g = torch.Generator().manual_seed(3)
    w = [torch.rand(2, 3, 40, generator=g) for _ in range(2)]
    pos = [torch.randint(0, 90, (2, 3, 64), generator=g, dtype=torch.int32) for _ in range(2)]
    kv.set_lengths([33, 40], seen=[90, 100], positions=pos, weights=w)
    assert kv.held.tolist() == [33, 40] and kv.seen.tolist() == [90, 100]
    for i in range(2):
        assert torch.equal(kv.weights[i][..., :40], w[i]) and torch.equal(kv.positions[i], pos[i])
    # the cache's own: filled already, and left as they are
    kept = [x.clone() for x in kv.weights + kv.positions]
    kv.set_lengths(torch.tensor([30, 1]), torch.tensor([95, 1]), positions=kv.positions,
                   weights=kv.weights)
    assert all(torch.equal(a, b) for a, b in zip(kept, kv.weights + kv.positions))
    assert kv.held.tolist() == [30, 1] and kv.seen.tolist() == [95, 1]
    # seen as many as held: nothing was evicted
    kv.set_lengths([30, 1], [30, 1])
    assert kv.positions[0][1, 0].tolist() == list(range(64)) and float(kv.weights[1].sum()) == 0


@pytest.mark.parametrize("change,message", [
    (dict(seen=[90]), "seen"), (dict(seen=90), "seen"), (dict(seen=[90, -1]), "seen"),
    (dict(seen=[32, 5]), "seen"), (dict(seen=[90, 5]), "positions"),
    (dict(positions=[torch.zeros(2, 3, 64, dtype=torch.int32)]), "2 layers"),
    (dict(positions=[torch.zeros(2, 3, 32, dtype=torch.int32)] * 2), "33..64"),
    (dict(positions=[torch.zeros(2, 3, 65, dtype=torch.int32)] * 2), "33..64"),
    (dict(positions=[torch.zeros(2, 3, 64)] * 2), "int32"),
    (dict(weights=[torch.zeros(2, 2, 64)] * 2), "weights"),
    (dict(weights=torch.zeros(2, 64)), "weights"),
])
def test_set_lengths_refuses(change, message):
    """And changes nothing where it refuses."""
    kv = _budget_cache()
    kv.weights[0].fill_(2.0)
    with pytest.raises(ValueError, match=message):
        kv.set_lengths([33, 5], **change)
    assert kv.held.tolist() == kv.seen.tolist() == [0, 0] and float(kv.weights[0].min()) == 2.0


def test_set_lengths_without_a_budget():
    """Positions are the rotary embedding's alone: any count that is not negative will do."""
    from iquestrt_b200.kernels import PagedKvCache
    kv = PagedKvCache(1, 2, 1, 128, rows=64, page_size=16, device="cpu")
    kv.set_lengths([3, 64], seen=[0, 700])
    assert kv.held.tolist() == [3, 64] and kv.seen.tolist() == [0, 700]
    for change, message in ((dict(seen=[-1, 3]), "seen"), (dict(weights=[torch.zeros(2, 1, 64)]), "budget")):
        with pytest.raises(ValueError, match=message):
            kv.set_lengths([3, 64], **change)


@pytest.mark.parametrize("budget,page", [(None, 16), (40, 16), (1, 2)])
def test_rehearsal_puts_back_what_a_step_writes(budget, page):
    """A step's writes (rows, weights and positions of the first tokens, counts) are undone, also
    when the step fails; the page table is the cache's own again."""
    from iquestrt_b200.kernels import PagedKvCache
    kv = PagedKvCache(2, 2, 3, 16, rows=64, q_len=3, page_size=page, budget=budget, device="cpu",
                      keep_first=0, dtype=torch.bfloat16)
    kv.set_lengths([33, 5])
    g = torch.Generator().manual_seed(5)
    for x in kv.k + kv.v + (kv.weights or []):
        x.copy_(torch.rand(x.shape, generator=g))

    def state():
        return [x.clone() for x in [kv.held, kv.lengths, kv.seen, kv.slot, kv.pos, kv.page_table,
                                    *kv.k, *kv.v, *(kv.weights or []), *(kv.positions or [])]]

    before, table = state(), kv.page_table
    for fail in (False, True):
        try:
            with kv.rehearsal():
                assert kv.held.tolist() == kv.seen.tolist() == [0, 0]
                for b in range(2):
                    rows = P.rows_of(kv.page_table, b, 3, page)
                    for x in kv.k + kv.v:
                        x[rows] = 7.0
                for x in (kv.weights or []) + (kv.positions or []):
                    x[..., :3] = 9
                for x in (kv.held, kv.lengths, kv.seen, kv.slot, kv.pos):
                    x.fill_(3)
                if fail:
                    raise ArithmeticError
        except ArithmeticError:
            assert fail
        assert kv.page_table is table
        assert all(torch.equal(a, b) for a, b in zip(before, state()))


def test_attention_slots_are_refused_without_weights():
    from iquestrt_b200 import ops
    L, lib, a = _attn_args()
    a.slot = 4096
    assert lib.iq_attn_decode(C.byref(a), None) == L.IQ_ERR_ARG
    slot = torch.zeros(2, dtype=torch.int64)
    w = torch.zeros(2, 2, 32)
    for change, message in ((dict(slot=slot), "weights"), (dict(slot=slot[:1], weights=w), "shape"),
                            (dict(slot=slot.int(), weights=w), "dtype")):
        with pytest.raises(ValueError, match=message):
            ops.attn_decode(**{**_tensors(), **change})
