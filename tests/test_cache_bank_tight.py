"""CacheBank.attend held to its own roundings, no more: a tolerance that a wrong sign, a missing mask or sums that were not rescaled cannot pass.

An output is off by half a step of its type, by the float32 bound that cache_ref.RefBank.attend derives (here for all rows at once), and by
what the pieces of the probabilities leave out, a share of sum p|v| of the same row and channel: 2^-24 for float32 (three bf16 pieces), 2^-17
for float16 and for up to 32 rows of bfloat16 (two), 2^-8 for more rows of bfloat16 (one piece: half a step of bf16 of each p).  What is
left of a result below the least normal number is a whole step of the type there."""
import numpy as np
import pytest
import torch

from tests import cache_ref as cr
from tests.test_cache_bank import DT, _bank, _filled, _ica, _np, _rand

gpu = pytest.mark.gpu


def _reference(ref, query, counts=None, causal=True):
    """out, bound, sum p|v| [batch, heads * group, T, dim], sums of p and their bound [batch][heads] -> [rows]: RefBank.attend, a head at a time."""
    group, T = query.shape[1] // ref.heads, query.shape[2]
    out, bound, spread = np.zeros(query.shape), np.zeros(query.shape), np.zeros(query.shape)
    got = [[np.zeros(len(w)) for w in row] for row in ref.weight]
    off = [[np.zeros(len(w)) for w in row] for row in ref.weight]
    for b in range(ref.batch):
        n = T if counts is None else int(counts[b])
        for h in range(ref.heads):
            K, V = ref.key[b][h], ref.value[b][h]
            see = np.clip(len(K) - n + np.arange(n) + 1, 0, None) if causal else np.full(n, len(K))
            mask, any_ = np.arange(len(K)) < see[:, None], see > 0
            for g in range(group):
                q = query[b, h * group + g, :n]
                s = np.where(mask, q @ K.T * ref.dim ** -0.5, -np.inf)
                p = np.exp(s - np.where(any_, s.max(1, initial=-np.inf), 0.0)[:, None])
                p = p / np.where(any_, p.sum(1), 1.0)[:, None]
                mag = np.where(mask, np.abs(q) @ np.abs(K).T, 0.0).max(1, initial=0.0) * ref.dim ** -0.5
                rel = 2.0 ** -24 * (4 * (ref.dim + 16) * mag + see / 16 + 64)
                out[b, h * group + g, :n], spread[b, h * group + g, :n] = p @ V, p @ np.abs(V)
                bound[b, h * group + g, :n] = rel[:, None] * (p @ np.abs(V)) + 4 * 2.0 ** -126 * (mask @ np.abs(V))
                got[b][h] += p.sum(0)
                off[b][h] += rel @ p
            off[b][h] += 2.0 ** -24 * 64 * got[b][h]
    return out, bound, spread, got, off


def _tolerance(want, bound, spread, dtype, rows):
    tail = 2.0 ** -24 if dtype == "fp32" else 2.0 ** -8 if dtype == "bf16" and rows > 32 else 2.0 ** -17
    info = torch.finfo(DT[dtype])
    return info.eps / 2 * (np.abs(want) + bound + tail * spread) + bound + tail * spread + info.tiny * info.eps


def _check(bank, ref, q, dtype, counts=None, causal=True, power=0.9):
    """One call with sums; `power`: how many of the elements a flipped sign has to fail at, so that the tolerance says something."""
    rows = q.shape[2] * (q.shape[1] // ref.heads)
    want, bound, spread, got, off = _reference(ref, _np(q), counts, causal)
    tol = _tolerance(want, bound, spread, dtype, rows)
    assert (2 * np.abs(want) > tol)[spread > 0].mean() > power
    bank.weights("kv").zero_()
    out = _np(bank.attend("kv", q.cuda(), counts=counts, causal=causal, accumulate=True))
    assert np.isfinite(out).all() and (np.abs(out - want) <= tol).all(), (np.abs(out - want) / tol).max()
    for b in range(ref.batch):
        for h in range(ref.heads):
            w = _np(bank.weights("kv"))[b, h, :ref.length(b)]
            assert (np.abs(w - got[b][h]) <= off[b][h] + 1e-12).all(), (np.abs(w - got[b][h]) - off[b][h]).max()


def test_reference_agrees_with_the_one_row_at_a_time():
    rs = np.random.RandomState(0)
    ref = cr.RefBank(2, 2, 16, 64)
    ref.push(rs.randn(2, 2, 40, 16), rs.randn(2, 2, 40, 16), [40, 3])
    q = rs.randn(2, 4, 6, 16)
    for causal in (True, False):
        for counts in (None, [5, 2]):
            out, bound, _, got, off = _reference(ref, q, counts, causal)
            ref.weight = [[np.zeros(len(w)) for w in row] for row in ref.weight]
            o, bd, wb = ref.attend(q, counts, causal=causal, accumulate=True)
            assert np.allclose(out, o, rtol=1e-12, atol=1e-14) and np.allclose(bound, bd, rtol=1e-12, atol=0)
            for b in range(2):
                for h in range(2):
                    assert np.allclose(got[b][h], ref.weight[b][h], rtol=1e-12) and np.allclose(off[b][h], wb[b][h], rtol=1e-9)


@gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("dim,H,group,T,fill", [(64, 1, 1, 5, 300), (64, 2, 9, 1, 700), (128, 1, 9, 1, 500), (128, 1, 3, 9, 401), (128, 2, 4, 8, 1300), (160, 1, 5, 4, 600), (256, 1, 4, 5, 333),
                                                (256, 2, 4, 8, 700), (256, 1, 17, 1, 1100), (256, 1, 1, 32, 64), (64, 1, 3, 100, 640), (64, 2, 1, 300, 900), (72, 1, 1, 200, 513),
                                                (128, 1, 4, 70, 330), (128, 2, 4, 300, 1200), (128, 1, 2, 1000, 1000), (256, 1, 3, 50, 128), (256, 2, 1, 500, 900)])
def test_attend_to_its_own_roundings(dtype, dim, H, group, T, fill):
    """Few and many rows; from 17 to 32 rows of 256 dims two tiles of the streaming form, whose sums take a product of their own."""
    rs = np.random.RandomState(dim + T + fill)
    bank, ref = _filled(rs, 2, H, dim, fill + 3, fill, spread=0.2)
    q = _rand(rs, (2, H * group, T, dim), dtype, 0.2)
    for causal, counts in ((True, None), (False, None), (True, [min(T, ref.length(b)) // (b + 1) for b in range(2)])):
        _check(bank, ref, q, dtype, counts, causal)


def _moves(ref, q, causal, waves):
    """How often the tiled form has to move the exponent's reference after a workgroup's first tile, in tiles that all of its rows see whole
    and in others: a score passes the reference by 2^16."""
    T, group, rows, tokens = q.shape[2], q.shape[1] // ref.heads, 32 * waves, 16 * waves
    found = {True: 0, False: 0}
    K = ref.key[0][0]
    see = np.repeat(np.clip(len(K) - T + np.arange(T) + 1, 0, None) if causal else np.full(T, len(K)), group)
    s = np.moveaxis(_np(q)[0, :group], 0, 1).reshape(T * group, -1) @ K.T * ref.dim ** -0.5 * np.log2(np.e)
    s = np.where(np.arange(len(K)) < see[:, None], s, -np.inf)
    for wave in range(0, T * group, 32):
        group0 = wave // rows * rows
        mark = np.full(len(s[wave:wave + 32]), -np.inf)
        for t in range(0, see[min(group0 + rows, T * group) - 1], tokens):
            top = s[wave:wave + 32, t:t + tokens].max(1)
            if (top - 16 > mark).any():
                found[bool(t + tokens <= see[group0])] += bool(t and np.isfinite(mark).any())
                mark = np.maximum(mark, top)
    return found


def _steps(rs, B, H, dim, fill, T, dtype, group):
    """Keys (the same for all sequences) whose scores go up by 20 powers of two five times along the bank, three of them among the query's own rows."""
    u = np.sign(rs.randn(dim))
    at = [fill * 0.15, fill * 0.4, fill - T * 0.95, fill - T * 0.6, fill - T * 0.2] if T < fill else [fill * f for f in (0.15, 0.35, 0.5, 0.7, 0.85)]
    level = -28.0 + 14.0 * (np.arange(fill)[:, None] >= np.array(at)).sum(1)
    key = level[:, None] / dim ** 0.5 * u + 0.3 * rs.randn(1, H, fill, dim)
    value = rs.randn(1, H, fill, dim)
    q = u + 0.05 * rs.randn(B, H * group, T, dim)
    return [torch.from_numpy(x.astype(np.float32)) for x in (key, value)] + [torch.from_numpy(q.astype(np.float32)).to(DT[dtype])]


@gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("B,H,dim,group,T,fill", [(1, 1, 64, 1, 512, 1500), (1, 2, 128, 2, 400, 2000), (1, 1, 128, 1, 40, 1700), (1, 1, 256, 2, 300, 1100), (16, 8, 128, 1, 500, 900), (16, 16, 64, 1, 500, 700),
                                                  (12, 8, 256, 1, 300, 600), (1, 2, 128, 1, 1024, 1024), (1, 1, 72, 3, 200, 1000)])
def test_sums_are_rescaled_where_scores_climb(dtype, B, H, dim, group, T, fill):
    """The maximum passes the slack of the exponent in later tiles, whole ones and bordering ones; in one piece and in several."""
    rs = np.random.RandomState(dim + T)
    key, value, q = _steps(rs, B, H, dim, fill, T, dtype, group)
    bank, ref, one = _bank(B, H, dim, fill), cr.RefBank(B, H, dim, fill), cr.RefBank(1, H, dim, fill)
    bank.push("kv", key.cuda().expand(B, -1, -1, -1), value.cuda().expand(B, -1, -1, -1))
    one.push(_np(key), _np(value))
    ref.key, ref.value, ref.weight = one.key * B, one.value * B, one.weight * B
    for waves in (4, 8):
        for causal in (True, False):
            m = _moves(ref, q, causal, waves)
            # (not causal: the last tile alone is not whole, where the bank's length is no multiple of it)
            assert m[True] > 0 and (m[False] > 0 or not causal), (m, waves, causal)
    if B == 1 and fill >= 1000:
        ica = _ica()
        view = bank._cache("kv", "test")[0]
        assert ica._lib.lib().mi_cache_attend_workspace_bytes(view, {"fp32": 0, "bf16": 1, "fp16": 2}[dtype], T, group, fill, 1, 0) > 256      # pieces
    for causal in (True, False):
        _check(bank, ref, q, dtype, None, causal, power=0.8)


@gpu
@pytest.mark.parametrize("dim,B,H,T,fill", [(64, 16, 16, 500, 700), (128, 16, 8, 500, 900), (256, 12, 8, 300, 600)])
def test_the_cases_above_in_one_piece_are_so(dim, B, H, T, fill):
    bank = _bank(B, H, dim, fill)
    view = bank._cache("kv", "test")[0]
    sizes = [_ica()._lib.lib().mi_cache_attend_workspace_bytes(view, dtype, T, 1, fill, 1, 0) for dtype in range(3)]
    assert sizes == [256] * 3
