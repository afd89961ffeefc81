"""CacheBank: keys and values in 4 bits, attention over them, eviction.  Kernels against tests/cache_ref.py (numpy, 64 bits).

What is held is compared bit for bit (values on a grid times a power of two), eviction too.  Attention outputs are off by half a step of
their type (finfo.eps / 2) and the float32 bound that cache_ref.RefBank.attend derives.  Probabilities enter the second product in bf16
pieces: three for float32 queries (2^-24 of each p is left out), two for float16 and for few rows of bfloat16 (2^-17), one for more than
32 bfloat16 rows of a head: that rounds each p by at most 2^-8 of itself, so the result by at most 2^-8 sum p|v|."""
import copy

import numpy as np
import pytest
import torch

from tests import cache_ref as cr

DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
gpu = pytest.mark.gpu


def _ica():
    import image_classification_amd as pkg
    return pkg


def _bank(batch, heads, dim, k, name="kv"):
    bank = _ica().CacheBank()
    bank.register(name, dim=dim, k=k, heads=heads, batch=batch, device="cpu")
    return bank.cuda()


def _rand(rs, shape, dtype, spread=1.0):
    x = rs.randn(*shape) * np.exp(spread * rs.randn(shape[0], shape[1], 1, shape[3]))
    return torch.from_numpy(x.astype(np.float32)).to(DT[dtype])


def _np(t):
    return t.detach().cpu().double().numpy()


def _same(got, ref):
    assert got.shape == ref.shape
    assert np.array_equal(np.isnan(got), np.isnan(ref))
    assert np.array_equal(got[~np.isnan(ref)], ref[~np.isnan(ref)])


def _rows_equal(bank, ref, name="kv"):
    keys, values = (_np(t) for t in bank[name])
    lengths = bank.lengths(name).tolist()
    for b in range(ref.batch):
        n = ref.length(b)
        assert lengths[b] == n
        for h in range(ref.heads):
            _same(keys[b, h, :n], ref.key[b][h])
            _same(values[b, h, :n], ref.value[b][h])
            assert bank.positions(name)[b, h, :n].tolist() == list(ref.position[b][h])
        assert not keys[b, :, n:].any() and not values[b, :, n:].any()


def _check_out(out, want, bound, dtype, rows=1):
    got = _np(out)
    tail = 2.0 ** -24 if dtype == "fp32" else 2.0 ** -8 if dtype == "bf16" and rows > 32 else 2.0 ** -17
    assert np.array_equal(np.isnan(got), np.isnan(want))
    ok = ~np.isnan(want)
    info = torch.finfo(DT[dtype])
    # bound is rel * sum p|v| with rel >= 64 * 2^-24: the pieces of p add `tail` of the same sum
    tol = info.eps / 2 * np.abs(want) + bound * (1 + tail / (64 * 2.0 ** -24)) + info.tiny * info.eps
    assert (np.abs(got - want)[ok] <= tol[ok]).all(), (np.abs(got - want) - tol)[ok].max()


# ---------------------------------------------------------------------------------------------------------------- on the CPU
def test_reference_quantiser_is_nearest_and_within_half_a_step():
    rs = np.random.RandomState(0)
    x = rs.randn(200, 64) * np.exp(4 * rs.randn(200, 1))
    v, e = cr.quantise(x)
    y = x.reshape(200, 2, 32) / 2.0 ** e[..., None]
    assert np.abs(y).max() <= 7.0 and (np.abs(y).max(-1) > 3.5).all()               # the smallest exponent that covers the block
    step = np.where(np.abs(y) < 2, 0.5, np.where(np.abs(y) < 4, 1.0, 2.0))
    assert (np.abs(v - y) <= step / 2).all()


def test_refusals_on_the_cpu():
    ica = _ica()
    bank = ica.CacheBank()
    for dim in (0, 4, 12, 260, 264):
        with pytest.raises(ValueError, match="dim"):
            bank.register("x", dim=dim, k=8)
    for bad in (dict(k=0), dict(k=8, heads=0), dict(k=8, batch=0)):
        with pytest.raises(ValueError, match="positive"):
            bank.register("x", dim=64, **bad)
    bank.register("kv", dim=64, k=100, heads=2, batch=3, device="cpu")
    assert bank.sizes["kv"] == 100 and set(bank.state_dict()) == {f"kv_{p}" for p in
                                                                  ("key", "key_scale", "value", "value_scale", "weight", "position", "length", "seen")}
    assert bank._buffers["kv_key"].shape == (3, 2, 128, 32)
    z = torch.zeros(3, 2, 1, 64)
    for call in (lambda: bank.push("kv", z, z), lambda: bank.attend("kv", z), lambda: bank.evict("kv", 5), lambda: bank.trim("kv"), lambda: bank["kv"]):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            call()
    with pytest.raises(KeyError, match="no bank"):
        bank.push("other", z, z)
    assert copy.deepcopy(bank).sizes == bank.sizes


def test_abi_refuses_bad_calls_before_touching_the_device():
    ica = _ica()
    L, lib = ica._lib.lib(), ica._lib
    import ctypes
    assert [L.mi_cache_width(d) for d in (0, 7, 8, 64, 72, 128, 136, 256, 264)] == [0, 0, 64, 64, 128, 128, 256, 256, 0]
    at = 1 << 20                                                                     # aligned, never read: every call below is refused first
    good = dict(key=at, key_scale=at, value=at, value_scale=at, weight=at, position=at, length=at, seen=at, batch=2, heads=2, dim=64, rows=64, limit=60)

    def cache(**changes):
        return ctypes.byref(lib.Cache(**{**good, **changes}))

    s = (ctypes.c_int64 * 3)(128, 64, 64)

    def push(c=None, key=at, strides=s, dtype=1, T=1, held=(None, None)):
        return L.mi_cache_push(c or cache(), key, strides, at, s, dtype, T, None, held[0], held[1], None)

    for c, rc, text in ((cache(key=None), -1, b"null pointer"), (cache(weight=at + 4), -1, b"aligned"), (cache(batch=0), -1, b"shape"),
                        (cache(dim=60), -4, b"dim"), (cache(dim=512), -4, b"dim"), (cache(rows=60), -1, b"capacity"), (cache(limit=65), -1, b"capacity"),
                        (cache(limit=0), -1, b"capacity"), (cache(batch=1 << 20, heads=1 << 20), -1, b"shape")):
        assert push(c) == rc and text in L.mi_last_error(), L.mi_last_error()
    assert push(dtype=7) == -1 and push(T=-1) == -1 and push(key=None) == -1 and push(key=at + 8) == -1
    assert push(strides=(ctypes.c_int64 * 3)(128, 60, 64)) == -1 and b"16 bytes" in L.mi_last_error()
    assert push(strides=(ctypes.c_int64 * 3)(-128, 64, 64)) == -1
    assert push(held=(at, None)) == -1 and push(held=(at, at + 2)) == -1
    assert L.mi_cache_push(None, at, s, at, s, 1, 1, None, None, None, None) == -1
    assert L.mi_cache_trim(cache(), None, -1, None) == -1
    assert L.mi_cache_longest(cache(), None, 1, None, None) == -1 and L.mi_cache_longest(cache(), None, -1, at, None) == -1
    assert L.mi_cache_read(cache(), None, at, None) == -1

    def attend(scale=1.0, ws=at, nbytes=1 << 30, group=1, T=1, dtype=1, out=at):
        return L.mi_cache_attend(cache(), at, s, out, s, dtype, T, group, None, scale, 1, 0, 10, ws, nbytes, None)

    for scale in (0.0, -1.0, float("nan"), float("inf"), 3e38, 1e-39):
        assert attend(scale=scale) == -1 and b"scale" in L.mi_last_error()
    assert attend(ws=None) == -1 and attend(nbytes=1) == -3 and attend(group=0) == -1 and attend(T=-1) == -1 and attend(dtype=3) == -1 and attend(out=None) == -1
    assert L.mi_cache_attend_workspace_bytes(cache(), 1, 0, 1, 10, 1, 0) == 0 and L.mi_cache_attend_workspace_bytes(cache(), 9, 1, 1, 10, 1, 0) == 0
    assert L.mi_cache_attend_workspace_bytes(cache(), 1, 1, 1, 10, 1, 0) > 0
    assert L.mi_cache_evict_workspace_bytes(cache(), 10) >= 4 * 10 * 8 and L.mi_cache_evict_workspace_bytes(cache(), 0) == 0

    def evict(into=None, keep=10, recent=0, ws=at, nbytes=1 << 30):
        return L.mi_cache_evict(cache(), into, keep, recent, 60, ws, nbytes, None)

    assert evict(keep=0) == -1 and evict(keep=61) == -1 and evict(recent=-1) == -1 and evict(recent=11) == -1 and evict(ws=None) == -1 and evict(nbytes=8) == -3
    assert evict(into=cache()) == -1 and b"share" in L.mi_last_error()
    assert evict(into=cache(key=2 * at, length=2 * at, dim=72)) == -1 and b"differ" in L.mi_last_error()


# ------------------------------------------------------------------------------------------------------------------- push
@gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("dim", [8, 64, 72, 128, 160, 256])
def test_push_holds_the_nearest_values(dtype, dim):
    rs = np.random.RandomState(dim)
    B, H, k = 3, 2, 70
    bank, ref = _bank(B, H, dim, k), cr.RefBank(B, H, dim, k)
    for T, counts in ((1, None), (37, [37, 0, 5]), (2, torch.tensor([1, 2, 2]))):
        key, value = _rand(rs, (B, H, T, dim), dtype, 2.0), _rand(rs, (B, H, T, dim), dtype, 2.0)
        dev = counts.cuda() if isinstance(counts, torch.Tensor) else counts
        held = bank.push("kv", key.cuda(), value.cuda(), counts=dev, held=True)
        want = ref.push(_np(key), _np(value), counts)
        for got, w in zip(held, want):
            assert got.dtype == DT[dtype]
            _same(_np(got), w)
        _rows_equal(bank, ref)
        for b in range(B):
            assert not bank.weights("kv")[b, :, :ref.length(b)].any()


@gpu
def test_push_edge_values():
    """Ties, midpoints one step to either side, zeros of both signs, subnormals, the largest numbers, and rows with NaN or infinities."""
    dim = 32
    f32 = np.float32
    mids = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0], f32)
    around = np.concatenate([mids, np.nextafter(mids, f32(0)), np.nextafter(mids[:-1], f32(8)), -mids])[:31]
    rows = []
    for e in (0, -3, 11, -120, 100):
        rows.append(np.concatenate([[f32(6.5)], around]).astype(f32) * f32(2.0) ** f32(e))
    rows.append(np.zeros(dim, f32))
    rows.append(-np.zeros(dim, f32))
    rows.append(np.full(dim, 1e-45, f32) * np.arange(dim).astype(f32))                # subnormals
    rows.append(np.full(dim, 2.0 ** -127, f32))
    rows.append(np.full(dim, np.finfo(f32).max, f32))
    rows.append(np.linspace(-3e38, 3e38, dim).astype(f32))
    rows.append((7.0 * 2.0 ** np.arange(-16, 16)).astype(f32))                         # block maxima on the border of a scale
    for bad in (np.nan, np.inf, -np.inf):
        r = np.ones(dim, f32)
        r[17] = bad
        rows.append(r)
    key = np.stack(rows)[None, None]
    value = np.ones_like(key)
    value[0, 0, 2, 3] = np.inf                                                         # a bad value makes its key NaN as well
    T = key.shape[2]
    bank, ref = _bank(1, 1, dim, 100), cr.RefBank(1, 1, dim, 100)
    held = bank.push("kv", torch.from_numpy(key).cuda(), torch.from_numpy(value).cuda(), held=True)
    want = ref.push(key.astype(np.float64), value.astype(np.float64))
    for got, w in zip(held, want):
        _same(_np(got), w)
    assert np.isnan(want[0][0, 0, [2, T - 3, T - 2, T - 1]]).all() and not np.isnan(want[0][0, 0, [0, 1, 3, 4]]).any()
    _rows_equal(bank, ref)


@gpu
def test_push_reads_any_layout_and_leaves_other_rows_alone():
    rs = np.random.RandomState(3)
    B, H, T, dim = 2, 3, 5, 72
    packed = torch.from_numpy(rs.randn(B, T, 3, H, dim).astype(np.float32)).cuda().bfloat16()   # as one projection leaves q, k, v
    key, value = packed[:, :, 1].transpose(1, 2), packed[:, :, 2].transpose(1, 2)
    bank, ref = _bank(B, H, dim, 64), cr.RefBank(B, H, dim, 64)
    before = {n: t.clone() for n, t in bank.state_dict().items()}
    bank.push("kv", key, value, counts=[2, 4])
    ref.push(_np(key), _np(value), [2, 4])
    _rows_equal(bank, ref)
    for b, n in ((0, 2), (1, 4)):                                                       # rows behind the last one
        for part in ("key", "value", "weight", "position"):
            assert torch.equal(bank.state_dict()["kv_" + part][b, :, n:], before["kv_" + part][b, :, n:])
        for part in ("key_scale", "value_scale"):
            assert torch.equal(bank.state_dict()["kv_" + part][b, :, :, n:], before["kv_" + part][b, :, :, n:])
    odd = torch.from_numpy(rs.randn(B * H * T * dim + 1).astype(np.float32)).cuda()[1:].view(B, H, T, dim)      # rows off 16 bytes
    flipped = torch.from_numpy(rs.randn(B, H, dim, T).astype(np.float32)).cuda().transpose(2, 3)                # dims not contiguous
    one = torch.from_numpy(rs.randn(1, H, 1, dim).astype(np.float32)).cuda().expand(B, H, T, dim)               # strides of zero
    for x in (odd, flipped, one):
        bank.push("kv", x, x)
        ref.push(_np(x), _np(x))
        _rows_equal(bank, ref)
    bank.push("kv", x[:, :, :0], x[:, :, :0])                                           # no rows at all
    _rows_equal(bank, ref)


@gpu
def test_push_refuses_what_does_not_fit():
    bank = _bank(2, 1, 64, 10)
    z = torch.zeros(2, 1, 6, 64, device="cuda")
    bank.push("kv", z, z, counts=[6, 1])
    with pytest.raises(RuntimeError, match="do not fit"):
        bank.push("kv", z, z)
    assert bank.lengths("kv").tolist() == [6, 1]
    bank.push("kv", z, z, counts=[4, 6])                                                # the bound says 12, the device 10: it fits
    assert bank.lengths("kv").tolist() == [10, 7]
    bank.trim("kv", torch.tensor([3, 9], device="cuda"))
    assert bank.lengths("kv").tolist() == [3, 7]
    bank.push("kv", z[:, :, :3], z[:, :, :3])
    assert bank.lengths("kv").tolist() == [6, 10]
    for bad, text in ((dict(counts=[1]), "counts"), (dict(counts=[7, 0]), "counts"), (dict(counts=[-1, 0]), "counts"),
                      (dict(counts=torch.tensor([1.0, 1.0], device="cuda")), "counts"), (dict(counts=torch.tensor([1, 1])), "counts")):
        with pytest.raises(ValueError, match=text):
            bank.push("kv", z, z, **bad)
    for key, value in ((z.double(), z.double()), (z, z.half()), (z, z[:, :, :2]), (z[..., :32], z[..., :32]), (z[:1], z[:1]), (z[0], z[0])):
        with pytest.raises(ValueError):
            bank.push("kv", key, value)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        bank.push("kv", z.cpu(), z.cpu())
    with pytest.raises(RuntimeError, match="dtype"):
        bank.half().push("kv", z, z)


# ----------------------------------------------------------------------------------------------------------------- attend
def _filled(rs, B, H, dim, k, fill, dtype="bf16", spread=0.7):
    """A bank and its reference with ragged lengths up to `fill`."""
    bank, ref = _bank(B, H, dim, k), cr.RefBank(B, H, dim, k)
    if fill:
        key, value = _rand(rs, (B, H, fill, dim), dtype, spread), _rand(rs, (B, H, fill, dim), dtype, spread)
        counts = [fill] + [int(n) for n in rs.randint(0, fill + 1, B - 1)]
        bank.push("kv", key.cuda(), value.cuda(), counts=counts)
        ref.push(_np(key), _np(value), counts)
    return bank, ref


@gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("dim,H,group,T,fill", [(64, 1, 1, 1, 1), (64, 2, 1, 1, 31), (128, 2, 4, 1, 33), (72, 1, 3, 1, 257), (256, 2, 2, 1, 700), (128, 1, 16, 1, 1500),
                                                (128, 1, 17, 1, 300), (64, 1, 2, 9, 65), (160, 2, 1, 5, 129), (128, 1, 4, 40, 40), (96, 1, 1, 70, 200), (128, 1, 4, 70, 330), (64, 1, 3, 100, 640), (256, 1, 3, 50, 128), (8, 1, 1, 200, 513)])
def test_attend_against_64_bits(dtype, dim, H, group, T, fill):
    rs = np.random.RandomState(dim + T + fill)
    B = 3
    bank, ref = _filled(rs, B, H, dim, fill + 3, fill)
    q = _rand(rs, (B, H * group, T, dim), dtype, 0.3)
    for causal, counts in ((True, None), (False, None), (True, [min(T, ref.length(b)) // (b + 1) for b in range(B)])):
        for accumulate in (False, True):
            out = bank.attend("kv", q.cuda(), counts=counts, causal=causal, accumulate=accumulate)
            want = ref.attend(_np(q), counts, causal=causal, accumulate=accumulate)
            assert out.dtype == DT[dtype] and out.shape == q.shape
            _check_out(out, want[0], want[1], dtype, T * group)
            if accumulate:
                for b in range(B):
                    for h in range(H):
                        n = ref.length(b)
                        d = np.abs(_np(bank.weights("kv"))[b, h, :n] - ref.weight[b][h])
                        assert (d <= want[2][b][h] + 1e-12).all(), d.max()
                        ref.weight[b][h] = _np(bank.weights("kv"))[b, h, :n]           # later sums start from what the bank has


@gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("dim,H,group,T,fill", [(64, 1, 1, 1100, 1150), (128, 1, 2, 1000, 1000), (256, 2, 1, 777, 1290), (128, 2, 1, 1025, 2000)])
def test_attend_causal_prompts_in_pieces(dtype, dim, H, group, T, fill):
    """Few heads and mostly their own rows: the bank is cut into pieces whose order changes with the tile; most rows see only some of
    them, and those of the shorter sequences (less than T rows) nothing at all at first."""
    rs = np.random.RandomState(T)
    bank, ref = _filled(rs, 2, H, dim, fill, fill)
    q = _rand(rs, (2, H * group, T, dim), dtype, 0.3)
    for counts in (None, [T - 1, T // 3]):
        out = bank.attend("kv", q.cuda(), counts=counts, accumulate=True)
        want = ref.attend(_np(q), counts, accumulate=True)
        _check_out(out, want[0], want[1], dtype, T * group)
        for b in range(2):
            for h in range(H):
                n = ref.length(b)
                d = np.abs(_np(bank.weights("kv"))[b, h, :n] - ref.weight[b][h])
                assert (d <= want[2][b][h] + 1e-12).all(), d.max()
                ref.weight[b][h] = _np(bank.weights("kv"))[b, h, :n]


@gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_attend_large_scores_and_other_scales(dtype):
    """Scores of several hundred: one row takes all, in a far corner of the bank, and the running maximum moves late."""
    rs = np.random.RandomState(0)
    bank, ref = _filled(rs, 2, 1, 128, 1000, 1000, spread=0.0)
    q = _rand(rs, (2, 2, 3, 128), dtype, 0.0) * 8
    for scale in (None, 1.0, 1e-3, 5.0):
        out = bank.attend("kv", q.cuda(), scale=scale)
        want = ref.attend(_np(q), scale=scale)
        _check_out(out, *want, dtype)


@gpu
def test_attend_rows_that_see_nothing_are_zeros():
    rs = np.random.RandomState(1)
    bank, ref = _filled(rs, 2, 2, 64, 40, 5)
    bank.trim("kv", torch.tensor([2, 0], device="cuda"))
    ref.trim([2, 0])
    q = _rand(rs, (2, 4, 6, 64), "bf16", 0.0).cuda()
    q[0, :, 1] = float("nan")                                                           # a row that sees nothing may hold anything
    before = bank.weights("kv").clone()
    out = bank.attend("kv", q, accumulate=True)                                         # 6 query rows, 2 and 0 rows in the bank
    want, bound, _ = ref.attend(_np(q), accumulate=True)
    _check_out(out, want, bound, "bf16")
    assert not out[0, :, :4].any() and not out[1].any() and out[0, :, 4:].any()
    assert torch.equal(bank.weights("kv")[1], before[1])
    out = bank.attend("kv", q, counts=[0, 0])
    assert not out.any()


@gpu
def test_attend_nan_rows_reach_only_who_sees_them():
    """A NaN row (a bad key or a bad value) makes NaN of the rows that see it and of nobody else, also inside one tile."""
    rs = np.random.RandomState(2)
    T = 40
    for side in (0, 1):
        kv = [_rand(rs, (1, 1, T, 64), "fp32", 0.0) for _ in range(2)]
        kv[side][0, 0, 20, 7] = float("inf") if side else float("nan")
        bank, ref = _bank(1, 1, 64, 64), cr.RefBank(1, 1, 64, 64)
        bank.push("kv", kv[0].cuda(), kv[1].cuda())
        ref.push(_np(kv[0]), _np(kv[1]))
        q = _rand(rs, (1, 2, T, 64), "fp32", 0.0)
        q[0, :, 25] = 0.0
        out = bank.attend("kv", q.cuda(), accumulate=True)
        got = _np(out)
        assert np.isnan(got[:, :, 20:]).all() and not np.isnan(got[:, :, :20]).any()
        w = _np(bank.weights("kv"))[0, 0]
        assert np.isnan(w[:T]).all()                                                    # row 39 sees every slot
        bank.trim("kv", 20)                                                             # the NaN row is behind the last one now
        ref.trim(20)
        q = q[:, :, :20]
        out = bank.attend("kv", q.cuda(), causal=False)
        _check_out(out, *ref.attend(_np(q), causal=False), "fp32")


@gpu
@pytest.mark.parametrize("T,fill", [(1, 1), (1, 600), (70, 70), (200, 900)])
def test_attend_rows_that_see_nothing_but_nan(T, fill):
    kv = torch.full((1, 1, fill, 64), float("nan"), device="cuda")
    bank = _bank(1, 1, 64, fill)
    bank.push("kv", kv, kv)
    q = torch.randn(1, 1, T, 64, device="cuda", generator=torch.Generator("cuda").manual_seed(0))
    for dtype in (torch.float32, torch.bfloat16):
        out = bank.attend("kv", q.to(dtype), accumulate=True)
        assert torch.isnan(out).all() and torch.isnan(bank.weights("kv")).all()


@gpu
def test_attend_keeps_the_layout_of_its_query():
    rs = np.random.RandomState(4)
    bank, ref = _filled(rs, 2, 2, 72, 50, 50)
    base = torch.from_numpy(rs.randn(2, 7, 4, 72).astype(np.float32)).cuda().half()     # [batch, rows, heads, dim]
    q = base.transpose(1, 2)
    out = bank.attend("kv", q)
    assert out.stride() == q.stride()
    _check_out(out, *ref.attend(_np(q)), "fp16")
    big = torch.zeros(2, 4, 7, 3, 72, device="cuda", dtype=torch.float16)
    for x in (base.permute(0, 2, 1, 3)[:, :, ::2], big.copy_(q.unsqueeze(3).expand_as(big))[:, :, :, 1], q[:, :, :1].expand(2, 4, 7, 72),
              q.transpose(2, 3).contiguous().transpose(2, 3)):
        out = bank.attend("kv", x)
        _check_out(out, *ref.attend(_np(x)), "fp16")
    assert bank.attend("kv", q[:, :, :0]).shape == (2, 4, 0, 72)


@gpu
def test_attend_refusals():
    bank = _bank(2, 2, 64, 10)
    z = torch.zeros(2, 4, 1, 64, device="cuda")
    for q in (z[:, :3], z[:, :0], z[..., :32], z[:1], z.double()):
        with pytest.raises(ValueError):
            bank.attend("kv", q)
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        with pytest.raises(ValueError, match="scale"):
            bank.attend("kv", z, scale=scale)
    with pytest.raises(RuntimeError, match="no gradient"):
        bank.attend("kv", z.clone().requires_grad_())
    with torch.no_grad():
        assert not bank.attend("kv", z.clone().requires_grad_()).any()
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        bank.attend("kv", z.cpu())


@gpu
def test_attend_offsets_beyond_32_bits():
    """The last sequences of a bank of 2.7 GB a side."""
    rs = np.random.RandomState(5)
    B, H, dim, k = 40, 16, 128, 65536
    bank = _bank(B, H, dim, k)
    T = 33
    key, value = (torch.from_numpy(rs.randn(B, H, T, dim).astype(np.float32)).cuda().bfloat16() for _ in range(2))
    bank.push("kv", key, value)
    q = torch.from_numpy(rs.randn(B, H, 2, dim).astype(np.float32)).cuda().bfloat16()
    out = bank.attend("kv", q, accumulate=True)
    ref = cr.RefBank(1, 2, dim, k)
    ref.push(_np(key[-1:, -2:]), _np(value[-1:, -2:]))
    want, bound, wb = ref.attend(_np(q[-1:, -2:]), accumulate=True)
    _check_out(out[-1:, -2:], want, bound, "bf16")
    for h in range(2):
        assert (np.abs(_np(bank.weights("kv")[-1, -2 + h, :T]) - ref.weight[0][h]) <= wb[0][h]).all()
    bank.evict("kv", 8)
    keys, _ = bank._buffers["kv_key"], None
    assert bank.lengths("kv").tolist() == [8] * B and keys.numel() > 2 ** 31


# ------------------------------------------------------------------------------------------------------------------ evict
def _set_weights(bank, ref, rs, style):
    w = bank.weights("kv")
    x = np.exp(2 * rs.randn(*w.shape)).astype(np.float32)
    if style == "ties":
        x = rs.randint(0, 3, w.shape).astype(np.float32) - 1.0
        x[x == 0] = np.where(rs.rand(*x[x == 0].shape) < 0.5, 0.0, -0.0)
    elif style == "equal":
        x = np.full(w.shape, 0.25, np.float32)
    elif style == "special":
        pick = rs.rand(*w.shape)
        x = np.where(pick < 0.2, np.float32(np.nan), np.where(pick < 0.3, np.float32(np.inf), np.where(pick < 0.4, np.float32(-np.inf), x)))
    w.copy_(torch.from_numpy(x))
    for b in range(ref.batch):
        for h in range(ref.heads):
            ref.weight[b][h] = x[b, h, :ref.length(b)].astype(np.float64)


@gpu
@pytest.mark.parametrize("style", ["spread", "ties", "equal", "special"])
@pytest.mark.parametrize("dim,fill,keep,recent", [(64, 1, 1, 0), (64, 70, 1, 1), (128, 300, 299, 10), (128, 300, 64, 64), (256, 1000, 37, 5), (72, 5000, 4500, 300), (64, 2500, 1200, 0), (32, 9000, 8500, 100), (64, 20000, 10000, 7), (8, 40000, 15000, 70), (8, 32768, 700, 3), (8, 32769, 31000, 1)])
def test_evict_in_place_and_into(style, dim, fill, keep, recent):
    rs = np.random.RandomState(fill + keep)
    B, H = 3, 2
    bank, ref = _filled(rs, B, H, dim, fill, fill)
    _set_weights(bank, ref, rs, style)
    bank.register("small", dim=dim, k=keep + 5, heads=H, batch=B, device="cuda")
    filler = torch.ones(B, H, keep + 5, dim, device="cuda")
    bank.push("small", filler, filler)
    before = {n: t.clone() for n, t in bank.state_dict().items() if n.startswith("kv_")}
    bank.evict("kv", keep, recent=recent, into="small")
    for n, t in bank.state_dict().items():
        if n.startswith("kv_"):
            assert torch.equal(t.view(torch.uint8) if t.dtype == torch.float32 else t, before[n].view(torch.uint8) if t.dtype == torch.float32 else before[n]), n
    ref.evict(keep, recent)
    bank.evict("kv", keep, recent=recent)
    for name in ("small", "kv"):
        _rows_equal(bank, ref, name)
        for b in range(B):
            for h in range(H):
                _same(_np(bank.weights(name))[b, h, :ref.length(b)], ref.weight[b][h])
    assert bank._buffers["small_seen"].tolist() == ref.seen == bank._buffers["kv_seen"].tolist()
    x = _rand(rs, (B, H, 3, dim), "bf16")                                               # both go on from there
    bank.push("small", x.cuda(), x.cuda())
    ref.push(_np(x), _np(x))
    _rows_equal(bank, ref, "small")


@gpu
def test_evict_refusals():
    bank = _bank(2, 2, 64, 20)
    bank.register("other", dim=64, k=5, heads=2, batch=2, device="cuda")
    bank.register("wrong", dim=64, k=5, heads=1, batch=2, device="cuda")
    for kw in (dict(keep=0), dict(keep=21), dict(keep=5, recent=6), dict(keep=5, recent=-1), dict(keep=6, into="other"), dict(keep=5, into="kv"), dict(keep=2, into="wrong")):
        with pytest.raises(ValueError):
            bank.evict("kv", **kw)
    with pytest.raises(KeyError):
        bank.evict("kv", 5, into="absent")
    with pytest.raises(ValueError):
        bank.trim("kv", -1)
    with pytest.raises(ValueError):
        bank.trim("kv", torch.zeros(3, dtype=torch.int32, device="cuda"))


# --------------------------------------------------------------------------------------------------------------- together
@gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_generation_under_a_budget(dtype):
    """A prompt, then single tokens and a rejected draft, with eviction whenever the bank is full: push, attend and evict as used together."""
    rs = np.random.RandomState(7)
    B, H, group, dim, k, keep = 2, 2, 3, 64, 48, 32
    bank, ref = _bank(B, H, dim, k), cr.RefBank(B, H, dim, k)

    def step(T, counts=None):
        kv = [_rand(rs, (B, H, T, dim), dtype, 0.5) for _ in range(2)]
        q = _rand(rs, (B, H * group, T, dim), dtype, 0.5)
        bank.push("kv", kv[0].cuda(), kv[1].cuda(), counts=counts)
        ref.push(_np(kv[0]), _np(kv[1]), counts)
        out = bank.attend("kv", q.cuda(), counts=counts, accumulate=True)
        want, bound, wb = ref.attend(_np(q), counts, accumulate=True)
        _check_out(out, want, bound, dtype, T * group)
        for b in range(B):
            for h in range(H):
                got = _np(bank.weights("kv"))[b, h, :ref.length(b)]
                assert (np.abs(got - ref.weight[b][h]) <= wb[b][h] + 1e-12).all()
                ref.weight[b][h] = got                                                  # eviction goes by the float32 sums
    step(30, [30, 17])
    for i in range(40):
        step(1)
        if i % 7 == 3:                                                                  # a draft of four, all of it rejected but the first
            lengths = bank.lengths("kv") + 1
            step(4)
            bank.trim("kv", lengths)
            ref.trim(lengths.cpu().numpy())
        if max(ref.length(b) for b in range(B)) > k - 6:
            bank.evict("kv", keep, recent=8)
            ref.evict(keep, 8)
        _rows_equal(bank, ref)


@gpu
def test_feature_bank_without_heads_matches_the_smoothing_it_stands_beside():
    """heads = batch = 1 over held features is the softmax-weighted read of smooth_prob (alpha = 0) on the same values."""
    import torch.nn.functional as F
    rs = np.random.RandomState(8)
    n, dim, classes = 500, 64, 10
    f = F.normalize(torch.from_numpy(rs.randn(n, dim).astype(np.float32)), dim=1)
    prob = torch.softmax(torch.from_numpy(rs.randn(n, classes).astype(np.float32)), 1)
    bank = _bank(1, 1, dim, n)
    bank.push("kv", f[None, None].cuda(), F.pad(prob, (0, dim - classes))[None, None].cuda())
    keys, values = (t[0, 0].float() for t in bank["kv"])
    q = F.normalize(torch.from_numpy(rs.randn(7, dim).astype(np.float32)), dim=1).cuda()
    got = bank.attend("kv", q[None, None], scale=1 / 0.2, causal=False)[0, 0, :, :classes]
    want = _ica().smooth_prob(q, keys, values[:, :classes].contiguous(), torch.zeros(7, classes, device="cuda"), 0.2, 0.0)
    assert np.allclose(_np(got), _np(want), rtol=1e-5, atol=1e-7)


@gpu
def test_graph_capture_replays_like_eager():
    rs = np.random.RandomState(9)
    B, H, group, dim, k, keep = 2, 2, 2, 128, 200, 100
    graphed, eager = _bank(B, H, dim, k), _bank(B, H, dim, k)
    fill = [torch.from_numpy(rs.randn(B, H, 90, dim).astype(np.float32)).cuda() for _ in range(2)]
    for bank in (graphed, eager):
        bank.push("kv", *fill)
    kv = [torch.zeros(B, H, 3, dim, device="cuda") for _ in range(2)]
    q = torch.zeros(B, H * group, 3, dim, device="cuda")

    def step(bank):
        bank.push("kv", *kv)
        out = bank.attend("kv", q, accumulate=True)
        bank.evict("kv", keep, recent=6)
        return out
    for bank in (graphed, eager):                                                       # once outside a graph, equally
        step(bank)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step(graphed)
    for i in range(6):
        for t in kv + [q]:
            t.copy_(torch.from_numpy(rs.randn(*t.shape).astype(np.float32)))
        g.replay()
        want = step(eager)
        torch.cuda.synchronize()
        assert torch.equal(out, want), i
        for a, b in zip(graphed.state_dict().values(), eager.state_dict().values()):
            n = int(eager.lengths("kv")[0])
            if a.dim() == 4 and a.shape[2] == dim // 32:
                a, b = a[..., :n], b[..., :n]
            elif a.dim() > 1:
                a, b = a[:, :, :n], b[:, :, :n]
            assert torch.equal(a, b)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side), pytest.raises(RuntimeError, match="cannot capture counts"):
        with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=side):
            graphed.push("kv", *kv, counts=[1, 1])
    # the host does not know the lengths any more: it looks, and refuses what does not fit
    big = torch.zeros(B, H, k - keep + 1, dim, device="cuda")
    with pytest.raises(RuntimeError, match="do not fit"):
        graphed.push("kv", big, big)
    graphed.push("kv", big[:, :, 1:], big[:, :, 1:])
    assert graphed.lengths("kv").tolist() == [k, k]


@gpu
def test_other_streams_state_dicts_and_copies():
    rs = np.random.RandomState(10)
    bank, ref = _filled(rs, 2, 1, 64, 64, 50)
    q = _rand(rs, (2, 1, 2, 64), "bf16", 0.3).cuda()
    want = bank.attend("kv", q)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = bank.attend("kv", q)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    twin = _bank(2, 1, 64, 64)
    twin.load_state_dict(bank.state_dict())
    assert torch.equal(twin.attend("kv", q), want)
    z = torch.zeros(2, 1, 20, 64, device="cuda")
    with pytest.raises(RuntimeError, match="do not fit"):                               # lengths came with the state
        twin.push("kv", z, z)
    bank.register("here", dim=64, k=4, batch=2)
    assert bank.lengths("here").is_cuda
    other = copy.deepcopy(bank)
    other.trim("kv")
    assert torch.equal(bank.attend("kv", q), want) and not other.attend("kv", q).any()
    _rows_equal(bank, ref)


@gpu
def test_buffers_that_were_replaced():
    rs = np.random.RandomState(11)
    bank, ref = _filled(rs, 2, 1, 64, 64, 50)
    q = _rand(rs, (2, 1, 2, 64), "bf16", 0.3).cuda()
    want = bank.attend("kv", q)
    for part in ("key", "value", "length"):                                             # the same tensors over other memory
        old = bank._buffers[f"kv_{part}"].data
        bank._buffers[f"kv_{part}"].data = old.clone()
        old.zero_()
    assert torch.equal(bank.attend("kv", q), want)
    _rows_equal(bank, ref)
    bank.trim("kv", 10)
    bank.kv_length = torch.full((2,), 60, dtype=torch.int32, device="cuda")
    z = torch.zeros(2, 1, 5, 64, device="cuda")
    with pytest.raises(RuntimeError, match="do not fit"):
        bank.push("kv", z, z)
    bank.kv_weight = bank.kv_weight[:1].clone()
    with pytest.raises(RuntimeError, match="kv_weight"):
        bank.attend("kv", q)
