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
