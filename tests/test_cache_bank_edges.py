"""CacheBank: calls after an eviction, buffers changed from outside, values at the ends of their types.  Against tests/cache_ref.py (numpy, 64 bits)."""
import copy

import numpy as np
import pytest
import torch

from tests import cache_ref as cr
from tests.test_cache_bank import DT, _bank, _check_out, _filled, _ica, _np, _rand, _rows_equal, _same, _set_weights

gpu = pytest.mark.gpu


class AgedBank(cr.RefBank):
    """The reference bank whose ``trim`` goes by age: of each head the rows with the largest positions leave (of equal ones, which only a
    state from elsewhere has, the highest slots); freed slots below the cut take the rows that stay from above, in order."""

    def trim(self, lengths):
        for b in range(self.batch):
            n, length = int(lengths[b] if np.ndim(lengths) else lengths), self.length(b)
            gone = length - n
            if gone <= 0:
                continue
            last = -1
            for h in range(self.heads):
                pos = self.position[b][h]
                stay = set(sorted(range(length), key=lambda i: (pos[i], i))[:n])
                above = iter(sorted(i for i in stay if i >= n))
                source = [i if i in stay else next(above) for i in range(n)]
                for part in (self.key, self.value, self.weight, self.position):
                    part[b][h] = part[b][h][source]
                last = max([last, *self.position[b][h]])
            self.seen[b] = max(self.seen[b] - gone, last + 1)


def _aged(rs, B, H, dim, k, fill):
    bank, ref = _filled(rs, B, H, dim, k, fill)
    ref.__class__ = AgedBank
    return bank, ref


def _push(bank, ref, rs, T, counts=None):
    kv = [_rand(rs, (ref.batch, ref.heads, T, ref.dim), "bf16") for _ in range(2)]
    bank.push("kv", kv[0].cuda(), kv[1].cuda(), counts=counts)
    ref.push(_np(kv[0]), _np(kv[1]), counts)


def _weights_equal(bank, ref):
    for b in range(ref.batch):
        for h in range(ref.heads):
            _same(_np(bank.weights("kv"))[b, h, :ref.length(b)], ref.weight[b][h])


# ------------------------------------------------------------------------------------------------------------- trim by age
def test_reference_trim_takes_back_the_rows_pushed_last():
    """Rows in slot order: the cut is the end of the list.  After an eviction: a list of rows in push order says what has to stay."""
    ref = AgedBank(1, 1, 8, 16)
    one = np.ones((1, 1, 8, 8))
    ref.push(one, one)
    ref.trim(5)
    assert list(ref.position[0][0]) == [0, 1, 2, 3, 4] and ref.seen == [5]
    ref.push(one, one)
    ref.weight[0][0] = np.array([1.0, 9, 1, 8, 1, 1, 1, 1, 1, 1, 1, 7, 7])
    ref.evict(6, 2)
    pushed = sorted(ref.position[0][0])
    assert pushed == [0, 1, 2, 3, 11, 12]
    ref.trim(4)
    assert sorted(ref.position[0][0]) == pushed[:4] and ref.seen == [11]


@gpu
def test_a_row_pushed_after_evict_and_trim_is_a_recent_one():
    """Push, evict, take back a row, push, evict: ``recent`` keeps the rows pushed last, and no two rows have one position."""
    rs = np.random.RandomState(0)
    bank, ref = _aged(rs, 1, 1, 8, 16, 8)

    def weigh(w):
        bank.weights("kv")[0, 0, :len(w)] = torch.tensor(w)
        ref.weight[0][0] = np.array(w)
    weigh([1.0, 9, 1, 8, 1, 1, 1, 1])
    bank.evict("kv", 4, recent=2)
    ref.evict(4, 2)
    assert sorted(bank.positions("kv")[0, 0, :4].tolist()) == [1, 3, 6, 7]
    bank.trim("kv", 3)
    ref.trim(3)
    _rows_equal(bank, ref)
    assert sorted(bank.positions("kv")[0, 0, :3].tolist()) == [1, 3, 6] and bank._buffers["kv_seen"].tolist() == [7]
    _push(bank, ref, rs, 3)
    weigh([0.0, 9, 0, 8, 8, 8])
    bank.evict("kv", 4, recent=4)
    ref.evict(4, 4)
    _rows_equal(bank, ref)
    assert sorted(bank.positions("kv")[0, 0, :4].tolist()) == [6, 7, 8, 9]


@gpu
@pytest.mark.parametrize("each", [False, True])
@pytest.mark.parametrize("dim,B,H,fill,keep,recent,more,cut", [(8, 1, 1, 12, 9, 4, 0, 6), (64, 2, 3, 40, 20, 5, 4, 22), (64, 2, 3, 40, 20, 5, 4, 18), (128, 3, 2, 300, 200, 0, 7, 150), (256, 2, 2, 300, 299, 20, 1, 1),
                                                              (72, 2, 1, 5000, 3000, 700, 30, 1200), (8, 1, 2, 9000, 8500, 8000, 0, 3100), (128, 1, 1, 2500, 2400, 30, 64, 2400)])
def test_trim_after_evict_takes_the_rows_pushed_last(dim, B, H, fill, keep, recent, more, cut, each):
    """Cuts into rows pushed since the eviction, into those that it kept as recent, and below them (each head loses its youngest)."""
    rs = np.random.RandomState(fill + cut)
    bank, ref = _aged(rs, B, H, dim, fill + more + 3, fill)
    _set_weights(bank, ref, rs, "spread")
    bank.evict("kv", keep, recent=recent)
    ref.evict(keep, recent)
    if more:
        _push(bank, ref, rs, more)
    lengths = [max(0, cut - 3 * b) for b in range(B)] if each else cut
    bank.trim("kv", torch.tensor(lengths, device="cuda") if each else cut)
    ref.trim(lengths)
    _rows_equal(bank, ref)
    _weights_equal(bank, ref)
    assert bank._buffers["kv_seen"].tolist() == ref.seen
    _push(bank, ref, rs, 3)                                                              # and it goes on from there
    bank.evict("kv", 3 + cut // 2, recent=3)
    ref.evict(3 + cut // 2, 3)
    _rows_equal(bank, ref)
    for b in range(B):
        for h in range(H):
            assert len(set(ref.position[b][h])) == ref.length(b)
    bank.trim("kv")
    assert bank.lengths("kv").tolist() == [0] * B


@gpu
def test_trim_of_a_state_whose_positions_repeat():
    """A state from elsewhere may hold a position twice: the cut has its length all the same, and of equal ones the highest slots leave."""
    rs = np.random.RandomState(1)
    bank, ref = _aged(rs, 1, 2, 64, 3000, 3000)
    pos = rs.randint(-5, 40, (1, 2, 3000))
    bank.positions("kv").copy_(torch.from_numpy(pos))
    bank._buffers["kv_seen"].fill_(3500)
    ref.seen = [3500]
    for h in range(2):
        ref.position[0][h] = pos[0, h]
    for n in (2999, 1300, 40, 1):
        bank.trim("kv", n)
        ref.trim(n)
        _rows_equal(bank, ref)
        assert bank._buffers["kv_seen"].tolist() == ref.seen


@gpu
def test_trim_in_a_graph_goes_by_age():
    rs = np.random.RandomState(2)
    bank, ref = _aged(rs, 2, 2, 64, 80, 60)
    kv = [torch.zeros(2, 2, 4, 64, device="cuda") for _ in range(2)]
    lengths = torch.zeros(2, dtype=torch.int32, device="cuda")
    start = {n: t.clone() for n, t in bank.state_dict().items()}
    bank.trim("kv", lengths + 100)                                                       # once outside the graph
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        bank.evict("kv", 40, recent=6)
        bank.push("kv", *kv)
        bank.trim("kv", lengths)
    bank.load_state_dict(start)
    for i in range(4):
        _set_weights(bank, ref, rs, "spread")
        rows = [torch.from_numpy(rs.randn(2, 2, 4, 64).astype(np.float32)) for _ in range(2)]
        for t, x in zip(kv, rows):
            t.copy_(x)
        cut = [41, 42 - 5 * i]
        lengths.copy_(torch.tensor(cut))
        g.replay()
        torch.cuda.synchronize()
        ref.evict(40, 6)
        ref.push(_np(rows[0]), _np(rows[1]))
        ref.trim(cut)
        _rows_equal(bank, ref)
        _weights_equal(bank, ref)
        _push(bank, ref, rs, 20)                                                         # eager work between the replays


# ----------------------------------------------------------------------------------------------- buffers changed from outside
def _full(bank, value, part="length"):
    return torch.full((bank.shapes["kv"][0],), value, dtype=torch.int32, device="cuda")


@gpu
@pytest.mark.parametrize("how", ["before the first call", "in place", "through a view", "other memory", "after a copy", "after a pickle", "inference"])
def test_push_notices_lengths_that_were_changed(how):
    """Whatever torch wrote to a bank's lengths, before its first call, between calls or in a copy of it: a push that does not fit is refused."""
    import pickle
    bank = _ica().CacheBank()
    if how == "inference":
        with torch.inference_mode():
            bank.register("kv", dim=64, k=64, batch=2)
    else:
        bank.register("kv", dim=64, k=64, batch=2)
    z = torch.zeros(2, 1, 5, 64, device="cuda")
    if how not in ("before the first call",):
        bank.push("kv", z, z)
    if how == "after a copy":
        bank = copy.deepcopy(bank)
    if how == "after a pickle":
        bank = pickle.loads(pickle.dumps(bank))
    if how in ("in place", "inference"):
        with torch.inference_mode(how == "inference"):
            bank.lengths("kv").fill_(60)
    elif how == "through a view":
        bank.state_dict()["kv_length"][1:].add_(55)
    elif how == "other memory":
        bank._buffers["kv_length"].data = _full(bank, 60)
    else:
        bank.kv_length = _full(bank, 60)
    before = bank.lengths("kv").tolist()
    with pytest.raises(RuntimeError, match="do not fit"):
        bank.push("kv", z, z)
    assert bank.lengths("kv").tolist() == before
    bank.push("kv", z[:, :, :4], z[:, :, :4])
    assert max(bank.lengths("kv").tolist()) == 64
    with pytest.raises(RuntimeError, match="do not fit"):
        bank.push("kv", z[:, :, :1], z[:, :, :1])


@gpu
def test_push_does_not_look_where_lengths_are_known():
    bank = _ica().CacheBank()
    bank.register("kv", dim=64, k=64, batch=2)
    z = torch.zeros(2, 1, 8, 64, device="cuda")
    L = _ica()._lib.lib()
    real, looks = L.mi_cache_longest, []
    L.mi_cache_longest = lambda *a: looks.append(1) or real(*a)
    try:
        for _ in range(8):
            bank.push("kv", z, z)
        bank.evict("kv", 40)
        bank.push("kv", z, z)
        bank.trim("kv", 10)
        bank.push("kv", z, z)
        assert not looks
        bank.lengths("kv").fill_(3)
        bank.push("kv", z, z)
        assert len(looks) == 1
        for _ in range(5):
            bank.push("kv", z, z)
        assert len(looks) == 1 and bank.lengths("kv").tolist() == [51, 51]
    finally:
        L.mi_cache_longest = real


# ------------------------------------------------------------------------------------------------------ attend after an eviction
def _query(rs, ref, T, group=2):
    return _rand(rs, (ref.batch, ref.heads * group, T, ref.dim), "bf16", 0.3)


@gpu
def test_causal_attention_refuses_rows_that_an_eviction_moved():
    """Push a draft, evict, attend: the draft's rows are not the last ones any more, so that slots say nothing of who sees whom."""
    rs = np.random.RandomState(3)
    bank, ref = _aged(rs, 1, 2, 64, 20, 12)
    _push(bank, ref, rs, 4)
    bank.weights("kv")[..., :16] = torch.arange(16.0)
    for h in range(2):
        ref.weight[0][h] = np.arange(16.0)
    bank.evict("kv", 12, recent=4)
    ref.evict(12, 4)
    _rows_equal(bank, ref)
    assert list(ref.position[0][0]) == [12, 13, 14, 15, *range(4, 12)]
    q = _query(rs, ref, 4)
    before = bank.weights("kv").clone()
    for call in (dict(), dict(accumulate=True), dict(counts=[3]), dict(counts=torch.tensor([4], device="cuda"))):
        with pytest.raises(RuntimeError, match="evict"):
            bank.attend("kv", q.cuda(), **call)
    assert torch.equal(bank.weights("kv"), before)
    on_device = q.cuda()
    with pytest.raises(RuntimeError, match="evict"), torch.cuda.graph(torch.cuda.CUDAGraph(), stream=torch.cuda.Stream()):
        bank.attend("kv", on_device)
    # what does not go by the order of the rows: one row, rows that all see everything, no order at all
    _check_out(bank.attend("kv", q[:, :, :1].cuda()), *ref.attend(_np(q[:, :, :1])), "bf16")
    _check_out(bank.attend("kv", q.cuda(), counts=[1]), *ref.attend(_np(q), [1]), "bf16")
    _check_out(bank.attend("kv", q.cuda(), causal=False), *ref.attend(_np(q), causal=False), "bf16")
    # rows pushed since are in order, and a copy of the bank, or its state in another one, is as mixed as the bank
    twin = _bank(1, 2, 64, 20)
    twin.load_state_dict(bank.state_dict())
    for other in (twin, copy.deepcopy(bank)):
        with pytest.raises(RuntimeError, match="evict"):
            other.attend("kv", q.cuda())
    _push(bank, ref, rs, 4)
    _check_out(bank.attend("kv", q.cuda()), *ref.attend(_np(q)), "bf16")
    bank.trim("kv", 13)
    ref.trim(13)
    with pytest.raises(RuntimeError, match="evict"):
        bank.attend("kv", q.cuda())
    bank.trim("kv")
    ref.trim(0)
    _push(bank, ref, rs, 6)
    _check_out(bank.attend("kv", q.cuda()), *ref.attend(_np(q)), "bf16")


@gpu
def test_causal_attention_after_an_eviction_that_left_the_last_rows_in_order():
    """The device says whether the last rows are in their order: an eviction that moved nothing, or older rows only, stands in no one's way."""
    rs = np.random.RandomState(4)
    bank, ref = _aged(rs, 2, 1, 64, 40, 30)
    q = _query(rs, ref, 3)
    bank.trim("kv", torch.tensor([20, 20], device="cuda"))                               # the host still counts 30 rows
    ref.trim([20, 20])
    bank.evict("kv", 20)
    _check_out(bank.attend("kv", q.cuda()), *ref.attend(_np(q)), "bf16")
    for b, n in enumerate((20, ref.length(1))):                                          # one old row leaves, the youngest takes its slot: one is enough
        ref.weight[b][0] = np.arange(n) + 1.0
        bank.weights("kv")[b, 0, :n] = torch.arange(n) + 1.0
    keep = 19
    bank.evict("kv", keep)
    ref.evict(keep)
    assert list(ref.position[0][0]) == [19, *range(1, 19)]
    with pytest.raises(RuntimeError, match="evict"):
        bank.attend("kv", q.cuda())
    bank.register("small", dim=64, k=20, batch=2)
    bank.evict("kv", keep, into="small")                                                 # as it is, the mixed order with it
    with pytest.raises(RuntimeError, match="evict"):
        bank.attend("small", q.cuda())
    _push(bank, ref, rs, 5, [5, 3])
    _check_out(bank.attend("kv", q.cuda()), *ref.attend(_np(q)), "bf16")
    _check_out(bank.attend("kv", q.cuda(), counts=[2, 3]), *ref.attend(_np(q), [2, 3]), "bf16")


@gpu
def test_the_look_at_the_order_is_needed_once():
    """A restored state is looked at before its first causal attention over several rows; pushes and attention go on without."""
    rs = np.random.RandomState(5)
    bank, ref = _aged(rs, 1, 1, 64, 64, 40)
    other = _bank(1, 1, 64, 64)
    other.load_state_dict(bank.state_dict())
    looks, look = [], other._in_order

    def counting(*args):
        looks.append(1)
        return look(*args)
    other._in_order = counting
    q = _query(rs, ref, 8)
    for counts in (None, [3], None):
        _check_out(other.attend("kv", q.cuda(), counts=counts), *ref.attend(_np(q), counts), "bf16")
    assert len(looks) == 1
    other.evict("kv", 30)
    kv = torch.zeros(1, 1, 8, 64, device="cuda")
    for _ in range(2):
        other.push("kv", kv, kv)
        other.attend("kv", q.cuda())
    assert len(looks) == 1


@gpu
def test_order_of_rows_and_graphs():
    """A graph's pushes stand before its own attention; what a replay may have evicted is looked at outside of it."""
    rs = np.random.RandomState(9)
    bank, ref = _aged(rs, 1, 1, 64, 64, 40)
    kv = [torch.zeros(1, 1, 3, 64, device="cuda") for _ in range(2)]
    q = _query(rs, ref, 3)
    on_device = q.cuda()

    def step():
        bank.push("kv", *kv)
        out = bank.attend("kv", on_device)
        bank.evict("kv", 30)
        return out
    step()
    graphs = []
    for _ in range(2):                                                                   # captured twice: an eviction stands before the second
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step()
        graphs.append((g, out))
    ref.push(_np(kv[0]), _np(kv[1]))
    ref.evict(30)
    for i in range(4):
        rows = [torch.from_numpy(rs.randn(1, 1, 3, 64).astype(np.float32)) for _ in range(2)]
        for t, x in zip(kv, rows):
            t.copy_(x)
        bank.weights("kv").copy_(torch.rand(64, generator=torch.Generator().manual_seed(i)))
        ref.weight[0][0] = _np(bank.weights("kv"))[0, 0, :30]
        ref.push(_np(rows[0]), _np(rows[1]))
        want = ref.attend(_np(q))
        g, out = graphs[i % 2]
        g.replay()
        torch.cuda.synchronize()
        _check_out(out, *want, "bf16")
        ref.evict(30)
        _rows_equal(bank, ref)
        if list(ref.position[0][0][-3:]) != list(range(ref.seen[0] - 3, ref.seen[0])):
            with pytest.raises(RuntimeError, match="evict"):
                bank.attend("kv", on_device)
    _push(bank, ref, rs, 4)
    _check_out(bank.attend("kv", on_device), *ref.attend(_np(q)), "bf16")
    state = bank.state_dict()
    twin = _bank(1, 1, 64, 64)
    twin.load_state_dict(state)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):                                                            # a loaded state is taken to be in order: a graph cannot look
        out = twin.attend("kv", on_device)
    for _ in range(3):
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        _check_out(out, *ref.attend(_np(q)), "bf16")


@gpu
def test_order_of_rows_through_the_c_abi():
    import ctypes
    ica = _ica()
    L = ica._lib.lib()
    rs = np.random.RandomState(6)
    bank, _ = _aged(rs, 3, 2, 64, 64, 50)
    bank.trim("kv", torch.tensor([50, 9, 0], device="cuda"))
    view, held = bank._cache("kv", "test")
    out = torch.full((1,), 7, dtype=torch.int32, device="cuda")

    def ask(T, counts=None):
        c = None if counts is None else torch.tensor(counts, dtype=torch.int32, device="cuda")
        assert L.mi_cache_in_order(view, None if c is None else c.data_ptr(), T, out.data_ptr(), torch.cuda.current_stream().cuda_stream) == 0
        return int(out)
    assert ask(1) == ask(5) == ask(64) == 1
    held[7][0] += 10                                                                     # rows left the first sequence
    held[5][0, :, :50] += 10
    assert ask(50) == 1
    held[5][0, 1, 45] = 3
    assert ask(4) == 1 and ask(5) == 0 and ask(64) == 0 and ask(8, [4, 8, 8]) == 1 and ask(8, [8, 0, 0]) == 0 and ask(8, [-1, 9, 1]) == 1
    held[5][0, 1, 45] = 55
    held[5][0, 1, 49] = 0
    assert ask(1) == 1 and ask(2) == 0                                                   # one row sees everything, whatever the order


def test_abi_refuses_a_bad_look_at_the_order():
    import ctypes
    ica = _ica()
    L, at = ica._lib.lib(), 1 << 20
    cache = ctypes.byref(ica._lib.Cache(at, at, at, at, at, at, at, at, 2, 2, 64, 64, 60))
    assert L.mi_cache_in_order(cache, None, 1, None, None) == -1 and L.mi_cache_in_order(cache, None, -1, at, None) == -1
    assert L.mi_cache_in_order(None, None, 1, at, None) == -1 and b"null cache" in L.mi_last_error()


@gpu
def test_longest_does_not_run_over():
    """The most rows a bank may hold and the most a push may bring: their sum is 2^31, which an int cannot say."""
    import ctypes
    ica = _ica()
    L = ica._lib.lib()
    length = torch.tensor([1 << 30, 5], dtype=torch.int32, device="cuda")
    out = torch.zeros(1, dtype=torch.int32, device="cuda")
    at = out.data_ptr()                                                                  # (only lengths and counts are read)
    base = -(-at // 16) * 16
    view = ica._lib.Cache(base, base, base, base, base, base, length.data_ptr(), base, 2, 1, 64, 1 << 30, 1 << 30)
    for T, want in ((1 << 30, 2 ** 31 - 1), ((1 << 30) - 1, 2 ** 31 - 1), (7, (1 << 30) + 7)):
        assert L.mi_cache_longest(ctypes.byref(view), None, T, out.data_ptr(), torch.cuda.current_stream().cuda_stream) == 0
        assert int(out) == want



# ------------------------------------------------------------------------------------------------------------ ends of the types
@gpu
def test_held_float16_rows_stay_finite():
    """Above 7 * 2^13 the nearest value that 4 bits hold is 2^16, past the largest float16: what is returned saturates, what is held does not."""
    f16 = np.float16
    tops = [f16(57344), np.nextafter(f16(57344), f16(60000)), f16(60000), f16(65504), f16(-65504), f16(49152)]
    x = np.zeros((1, 1, len(tops), 64), f16)
    x[0, 0, :, 5] = tops
    x[0, 0, :, 6] = f16(1000)
    x[0, 0, :, 40] = f16(3)
    bank, ref = _bank(1, 1, 64, 16), cr.RefBank(1, 1, 64, 16)
    held = bank.push("kv", torch.from_numpy(x).cuda(), torch.from_numpy(-x).cuda(), held=True)
    want = ref.push(x.astype(np.float64), -x.astype(np.float64))
    assert np.abs(want[0]).max() == 65536
    _rows_equal(bank, ref)
    for got, w in zip(held, want):
        _same(_np(got), np.clip(w, -65504, 65504))


@gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("dim,T,group,fill,k", [(64, 1, 1, 40, 64), (72, 1, 2, 3000, 3000), (64, 40, 1, 60, 64), (128, 100, 2, 3000, 3000), (256, 3, 2, 700, 700), (72, 9, 2, 200, 200)])
def test_scores_that_are_all_minus_infinity(dtype, dim, T, group, fill, k):
    """A row that sees something and whose scores are all -inf has no softmax: NaN, as exp(-inf - -inf) says, and NaN for the sums that it
    takes part in.  Scores of which only some are -inf are ordinary; a row that sees nothing is zeros all the same."""
    rs = np.random.RandomState(dim + T)
    kv = [_rand(rs, (1, 1, fill, dim), "bf16", 0.3) for _ in range(2)]
    kv[0][0, 0, :, 3] = 1.0                                                              # every key has a positive entry there ...
    kv[0][0, 0, :, :32] = kv[0][0, 0, :, :32].clamp(-2, 2)
    q = _rand(rs, (1, group, T, dim), dtype, 0.3)
    q[0, :, T // 2, 3] = -float("inf")                                                   # ... so that -inf makes -inf of all scores
    for causal in (True, False):
        for n in (None, [T // 2 + 1]):
            bank, ref = _bank(1, 1, dim, k), cr.RefBank(1, 1, dim, k)
            bank.push("kv", kv[0].cuda(), kv[1].cuda())
            ref.push(_np(kv[0]), _np(kv[1]))
            assert (ref.key[0][0][:, 3] > 0).all()
            out = bank.attend("kv", q.cuda(), counts=n, causal=causal, accumulate=True)
            real = T if n is None else n[0]
            clean = q.clone()
            clean[0, :, T // 2, 3] = 0.0
            want, bound, weigh = ref.attend(_np(clean), n, causal=causal, accumulate=True)
            want[:, :, T // 2] = np.nan
            _check_out(out, want, bound, dtype, T * group)
            w = _np(bank.weights("kv"))[0, 0, :fill]
            sees = fill - real + T // 2 + 1 if causal else fill
            assert np.isnan(w[:sees]).all() and not np.isnan(w[sees:]).any()
            d = np.abs(w - ref.weight[0][0])[sees:]
            assert (d <= weigh[0][0][sees:] + 1e-12).all()


@gpu
@pytest.mark.parametrize("T", [1, 40])
def test_float32_queries_up_to_the_largest(T):
    """The largest float32 rounds to an infinity in bf16; its pieces must not."""
    rs = np.random.RandomState(8)
    top = np.finfo(np.float32).max
    key = (rs.randn(1, 1, 50, 64) * 2.0 ** -120).astype(np.float32)
    value = rs.randn(1, 1, 50, 64).astype(np.float32)
    q = np.zeros((1, 1, T, 64), np.float32)
    q[..., 0] = top
    q[..., 1] = -top
    q[..., 2] = np.float32(3.3961775e38)                                                 # the least that rounds up, and its neighbour below
    q[..., 3] = np.nextafter(np.float32(3.3961775e38), np.float32(0))
    bank, ref = _bank(1, 1, 64, 64), cr.RefBank(1, 1, 64, 64)
    bank.push("kv", torch.from_numpy(key).cuda(), torch.from_numpy(value).cuda())
    ref.push(key.astype(np.float64), value.astype(np.float64))
    out = bank.attend("kv", torch.from_numpy(q).cuda(), scale=0.01, accumulate=True)
    want, bound, weigh = ref.attend(q.astype(np.float64), scale=0.01, accumulate=True)
    assert np.isfinite(want).all() and np.ptp(want[0, 0, -1]) > 0
    _check_out(out, want, bound, "fp32", T)
    assert (np.abs(_np(bank.weights("kv"))[0, 0, :50] - ref.weight[0][0]) <= weigh[0][0] + 1e-12).all()


@gpu
def test_attend_refuses_a_forward_mode_tangent():
    import torch.autograd.forward_ad as fwd
    rs = np.random.RandomState(7)
    bank, _ = _filled(rs, 1, 1, 64, 16, 16)
    q = torch.randn(1, 1, 2, 64, device="cuda")
    want = bank.attend("kv", q)
    with fwd.dual_level():
        assert torch.equal(bank.attend("kv", q), want)                                   # no tangent, no objection
        dual = fwd.make_dual(q, torch.ones_like(q))
        with pytest.raises(RuntimeError, match="no gradient"):
            bank.attend("kv", dual)
        assert torch.equal(bank.attend("kv", dual.detach()), want)
        assert torch.equal(bank.attend("kv", fwd.unpack_dual(dual).primal), want)


@gpu
def test_the_order_after_an_eviction_goes_by_the_fewest_rows_pushed():
    """A list of counts says how many rows each sequence got: where one got fewer than the query has, its older rows are looked at."""
    rs = np.random.RandomState(10)
    bank, ref = _aged(rs, 2, 1, 64, 40, 30)
    bank.trim("kv", 20)
    ref.trim(20)
    _push(bank, ref, rs, 8)
    for b in range(2):
        n = ref.length(b)
        bank.weights("kv")[b, 0, :n] = torch.arange(n) + 1.0
        ref.weight[b][0] = np.arange(n) + 1.0
    keep = min(ref.length(b) for b in range(2)) - 2
    bank.evict("kv", keep)
    ref.evict(keep)
    assert list(ref.position[1][0][-2:]) != [ref.seen[1] - 2, ref.seen[1] - 1]
    _push(bank, ref, rs, 4, [4, 1])
    q = _query(rs, ref, 4)
    with pytest.raises(RuntimeError, match="evict"):
        bank.attend("kv", q.cuda())
    _check_out(bank.attend("kv", q.cuda(), counts=[4, 1]), *ref.attend(_np(q), [4, 1]), "bf16")
    _push(bank, ref, rs, 4, np.array([4, 4]))
    _check_out(bank.attend("kv", q.cuda()), *ref.attend(_np(q)), "bf16")


def _by_age(ref, q, n):
    """Causal attention by positions: query row t, pushed as the (n - t)-th last of its sequence, sees the rows pushed up to then."""
    out = np.zeros(q.shape)
    group = q.shape[1] // ref.heads
    for b in range(ref.batch):
        for h in range(ref.heads):
            for t in range(n[b]):
                sees = ref.position[b][h] <= ref.seen[b] - n[b] + t
                K, V = ref.key[b][h][sees], ref.value[b][h][sees]
                for g in range(group if sees.any() else 0):
                    s = K @ q[b, h * group + g, t] * ref.dim ** -0.5
                    p = np.exp(s - s.max())
                    out[b, h * group + g, t] = p @ V / p.sum()
    return out


@gpu
@pytest.mark.parametrize("seed", range(8))
def test_programs_of_calls_in_any_order(seed):
    """Push, attend, evict and trim at random: what is held follows the lists of the reference, and causal attention either goes by the age
    of the rows or is refused, and then only where slots would have said something else."""
    rs = np.random.RandomState(seed)
    B, H, group, dim, k = 3, 2, 2, [64, 128, 72, 256][seed % 4], 96
    bank = _ica().CacheBank()
    bank.register("kv", dim=dim, k=k, heads=H, batch=B)
    ref = AgedBank(B, H, dim, k)
    refused = right = 0
    for step in range(60):
        op = rs.choice(["push", "push", "draft", "evict", "trim", "ask"])
        longest = max(ref.length(b) for b in range(B))
        if op in ("push", "draft"):
            T = int(rs.randint(1, 9))
            if longest + T > k:
                op = "evict"
            else:
                counts = None if rs.rand() < 0.5 else [int(n) for n in rs.randint(0, T + 1, B)]
                given = counts if counts is None or rs.rand() < 0.5 else torch.tensor(counts, device="cuda")
                kv = [_rand(rs, (B, H, T, dim), "bf16", 0.3) for _ in range(2)]
                bank.push("kv", kv[0].cuda(), kv[1].cuda(), counts=given)
                ref.push(_np(kv[0]), _np(kv[1]), counts)
                if op == "draft":
                    q = _query(rs, ref, T, group)
                    out = _np(bank.attend("kv", q.cuda(), counts=given, accumulate=True))
                    want, bound, weigh = ref.attend(_np(q), counts, accumulate=True)
                    age = _by_age(ref, _np(q), [T] * B if counts is None else counts)
                    assert np.allclose(want, age, rtol=1e-9, atol=1e-12)
                    assert (np.abs(out - want) <= 2.0 ** -8 * np.abs(want) + bound * 3).all()
                    for b in range(B):
                        for h in range(H):
                            got = _np(bank.weights("kv"))[b, h, :ref.length(b)]
                            assert (np.abs(got - ref.weight[b][h]) <= weigh[b][h] + 1e-12).all()
                            ref.weight[b][h] = got
        if op == "evict" and longest:
            keep = int(rs.randint(1, longest + 2))
            recent = int(rs.randint(0, keep + 1))
            bank.evict("kv", keep, recent=recent)
            ref.evict(keep, recent)
        if op == "trim":
            cut = [max(0, ref.length(b) - int(rs.randint(0, 6))) for b in range(B)]
            if rs.rand() < 0.2:
                cut = [int(rs.choice([0, 20]))] * B
            bank.trim("kv", cut[0] if len(set(cut)) == 1 else torch.tensor(cut, device="cuda"))
            ref.trim(cut)
        if op == "ask":
            T = int(rs.randint(1, 6))
            q = _query(rs, ref, T, group)
            age, by_slot = _by_age(ref, _np(q), [T] * B), ref.attend(_np(q))
            in_order = all(list(ref.position[b][h][-T:]) == list(range(ref.seen[b] - min(T, ref.length(b)), ref.seen[b]))
                           for b in range(B) for h in range(H) if ref.length(b)) or T == 1
            try:
                out = _np(bank.attend("kv", q.cuda()))
                assert in_order and np.allclose(by_slot[0], age, rtol=1e-9, atol=1e-12), step
                assert (np.abs(out - age) <= 2.0 ** -8 * np.abs(age) + by_slot[1] * 3).all()
                right += 1
            except RuntimeError as e:
                assert "evict" in str(e) and not in_order, step
                refused += 1
        _rows_equal(bank, ref)
        assert bank._buffers["kv_seen"].tolist() == ref.seen
    assert right > 0
