"""Cases over the 4-bit cache bank: rows of keys and values held in 4 bits (``push``), softmax attention over them (``attend``), and
eviction by the attention that each row got (``evict``).

Held format: a row of ``dim`` values is padded with zeros to ``width`` (64, 128 or 256) and cut into blocks of 32.  A block has one scale
2**e, e the smallest integer with max|x| <= 7 * 2**e (kept within -126..125), stored as the byte e + 127; each value is x / 2**e rounded to
nearest, ties to even, on {0, .5, 1, 1.5, 2, 3, 4, 6} with a sign bit, two values a byte, the even one in the low four bits.  Codes are
[batch, heads, rows, width / 2], scales [batch, heads, width / 32, rows]; ``rows`` is the capacity rounded up to 64."""
import math

import torch

own = False

GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
NAME = "kv"


# ---------------------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # a decoding step's write: one new row for each of 64 sequences of unequal length
        dict(name="push one token", op="push", batch=64, heads=8, dim=128, k=4096, rows=1, dtype="bf16", fill=3900),
        # eight prompts of unequal length, padded to one tensor, enter an empty bank
        dict(name="push ragged prompts", op="push", batch=8, heads=8, dim=128, k=2048, rows=2000, dtype="fp16", fill=0),
        # the smallest call: one query, a few hundred rows, where only latency counts
        dict(name="attend one query, short", op="attend", batch=1, heads=4, group=1, dim=64, k=384, fill=333, rows=1, dtype="fp32", causal=True, weigh=False, ragged=False),
        # one user's long conversation: the whole card reads one sequence
        dict(name="attend one token, long", op="attend", batch=1, heads=8, group=4, dim=128, k=131072, fill=131071, rows=1, dtype="bf16", causal=True, weigh=False, ragged=False),
        # a serving batch's decoding step that keeps the sums which eviction needs
        dict(name="attend ragged batch, weigh", op="attend", batch=64, heads=8, group=4, dim=128, k=8192, fill=8100, rows=1, dtype="bf16", causal=True, weigh=True, ragged=True),
        # a draft of five tokens checked at once, in a padded batch, wide heads
        dict(name="attend draft of five", op="attend", batch=16, heads=4, group=4, dim=256, k=4096, fill=4001, rows=5, dtype="fp16", causal=True, weigh=False, ragged=True),
        # a prompt that attends to itself
        dict(name="attend prompt", op="attend", batch=1, heads=8, group=4, dim=128, k=4096, fill=4096, rows=4096, dtype="bf16", causal=True, weigh=False, ragged=False),
        # one chunk of a long prompt, with the sums for eviction after it
        dict(name="attend chunk, weigh", op="attend", batch=2, heads=4, group=4, dim=128, k=16384, fill=16000, rows=1000, dtype="bf16", causal=True, weigh=True, ragged=False),
        # features against a feature bank, as the soft-label smoothing does: no heads, no order
        dict(name="attend feature bank", op="attend", batch=1, heads=1, group=1, dim=64, k=14336, fill=14336, rows=448, dtype="fp32", causal=False, weigh=False, ragged=False),
        # generation under a fixed budget: 16 rows come in, 16 go, in place
        dict(name="evict streaming", op="stream", batch=32, heads=8, dim=128, k=2064, keep=2048, rows=16, recent=256, dtype="bf16"),
        # a read prompt is cut down to what mattered, into a bank of its own
        dict(name="evict long prompt", op="compress", batch=4, heads=8, dim=128, k=32768, keep=2048, recent=64, dtype="bf16"),
        # the same for one short sequence
        dict(name="evict short", op="compress", batch=1, heads=2, dim=64, k=700, keep=300, recent=32, dtype="bf16"),
    ]


def draw(rng):
    def span(lo, hi):
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    op = rng.choice(["push", "attend", "attend", "attend", "stream", "compress"])
    dim = rng.choice([64, 128, 128, 256, 32, 72, 80, 96, 104, 160])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    heads = rng.choice([1, 2, 3, 4, 5, 8, 16])
    if op == "push":
        rows = span(1, 2000)
        batch = span(1, max(1, min(128, 16_000_000 // (rows * heads * dim))))
        k = rows + span(1, 2000)
        return dict(op=op, batch=batch, heads=heads, dim=dim, k=k, rows=rows, dtype=dtype, fill=k - rows)
    if op == "attend":
        group = rng.choice([1, 2, 3, 4, 6, 7, 8, 16])
        fill = span(1, 131072)
        rows = 1 if rng.random() < 0.4 else span(1, min(4096, fill))
        batch = span(1, max(1, min(64, 200_000_000 // (fill * heads * dim), 400_000_000 // (fill * heads * group * rows))))
        while batch * heads * group * rows * fill > 400_000_000:
            rows = (rows + 1) // 2
        return dict(op=op, batch=batch, heads=heads, group=group, dim=dim, k=fill + rng.randrange(100), fill=fill, rows=rows, dtype=dtype,
                    causal=rng.random() < 0.75, weigh=rng.random() < 0.4, ragged=rng.random() < 0.5)
    k = span(64, 32768 if op == "compress" else 4096)
    keep = span(16, k - 16)
    batch = span(1, max(1, min(64, 100_000_000 // (k * heads * dim))))
    recent = rng.randrange(0, min(keep, 512))
    if op == "stream":
        rows = min(k - keep, span(1, 64))
        return dict(op=op, batch=batch, heads=heads, dim=dim, k=keep + rows, keep=keep, rows=rows, recent=recent, dtype=dtype)
    return dict(op=op, batch=batch, heads=heads, dim=dim, k=k, keep=keep, recent=recent, dtype=dtype)


def _width(dim):
    return 64 if dim <= 64 else 128 if dim <= 128 else 256


def _held_bytes(case):
    return case["dim"] // 2 + -(-case["dim"] // 32)      # one row of one side: codes and scales of its own values


def work(case):
    size = TYPES[case["dtype"]].itemsize
    lanes = case["batch"] * case["heads"]
    held = 2 * _held_bytes(case)
    if case["op"] == "push":
        part = 1.0 if case["rows"] == 1 else 0.75        # unequal counts: three quarters of the padded rows on average
        n = lanes * case["rows"]
        return {"bytes": n * (2 * case["dim"] * size * (part + 1) + part * (held + 8)), "flops": 0}
    if case["op"] == "attend":
        fill = case["fill"] * (0.75 if case["ragged"] else 1.0)
        rows, q = case["rows"], lanes * case["group"] * case["rows"]
        seen = fill - (rows - 1) / 2 if case["causal"] else fill
        moved = lanes * fill * (held + (8 if case["weigh"] else 0)) + 2 * q * case["dim"] * size
        return {"bytes": moved, "flops": q * max(seen, 1.0) * case["dim"] * (6 if case["weigh"] else 4)}
    if case["op"] == "stream":
        n, moves = lanes * (case["keep"] + case["rows"]), lanes * case["rows"]
        read_back = lanes * case["k"] * 2 * case["dim"] * 2 + lanes * case["keep"] * held
        return {"bytes": n * 8 + moves * (2 * case["dim"] * size + 3 * held) + read_back, "flops": 0}
    n = lanes * case["k"] * 0.75
    kept = lanes * case["keep"]
    return {"bytes": n * 8 + kept * (3 * held + 8) + kept * 2 * case["dim"] * 2, "flops": 0}


# --------------------------------------------------------------------------------------------------------------- inputs
def _scale_bytes(top):
    """The byte e + 127 for blocks whose largest magnitude is ``top`` (float32): 1.75 * 2**(e + 2) is the most that e takes."""
    bits = top.view(torch.int32)
    return ((bits >> 23) - 2 + ((bits & 0x7FFFFF) > 0x600000)).clamp_(1, 252)


def _pack(x):
    """float32 [..., rows, width] -> codes [..., rows, width / 2], scale bytes [..., rows, width / 32]."""
    blocks = x.unflatten(-1, (-1, 32))
    byte = _scale_bytes(blocks.abs().amax(-1))
    a = torch.ldexp(blocks.abs(), (127 - byte).unsqueeze(-1)).clamp_(max=6.0)
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    a = torch.round(a / step) * step
    code = torch.where(a < 2, a * 2, torch.where(a < 4, a + 2, a / 2 + 4)).to(torch.uint8)
    code = (code | (torch.signbit(blocks).to(torch.uint8) << 3)).flatten(-2)
    return code[..., 0::2] | (code[..., 1::2] << 4), byte.to(torch.uint8)


def _values(codes, scales):
    """Codes [..., rows, width / 2] and scales [..., width / 32, rows] -> float32 [..., rows, width]."""
    four = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).int()
    low = four & 7
    a = torch.where(low < 4, low * 0.5, torch.where(low < 6, low - 2.0, low * 2.0 - 8.0))
    a = torch.where(four > 7, -a, a).unflatten(-1, (-1, 32))
    byte = scales.transpose(-1, -2).int()
    scale = torch.where(byte == 255, math.nan, torch.ldexp(torch.ones_like(byte, dtype=torch.float32), byte - 127))
    return (a * scale.unsqueeze(-1)).flatten(-2)


def _rows_like(gen, shape, dtype):
    """Keys or values as projections give them: a few channels are much larger than the others."""
    dim = shape[-1]
    spread = torch.exp(0.8 * torch.randn(shape[1], 1, dim, generator=gen, device="cuda"))
    x = torch.randn(shape, generator=gen, device="cuda")
    return x.mul_(spread).to(dtype)


def _empty_bank(case):
    rows, width = -(-case["k"] // 64) * 64, _width(case["dim"])
    b, h = case["batch"], case["heads"]
    z = dict(device="cuda")
    return dict(key=torch.zeros(b, h, rows, width // 2, dtype=torch.uint8, **z), key_scale=torch.ones(b, h, width // 32, rows, dtype=torch.uint8, **z),
                value=torch.zeros(b, h, rows, width // 2, dtype=torch.uint8, **z), value_scale=torch.ones(b, h, width // 32, rows, dtype=torch.uint8, **z),
                weight=torch.zeros(b, h, rows, **z), position=torch.zeros(b, h, rows, dtype=torch.int32, **z),
                length=torch.zeros(b, dtype=torch.int32, **z), seen=torch.zeros(b, dtype=torch.int32, **z))


def _padded(x, width):
    return torch.nn.functional.pad(x.float(), (0, width - x.shape[-1]))


def _lengths(gen, case, top, low):
    if low >= top:
        return torch.full((case["batch"],), top, dtype=torch.int32, device="cuda")
    n = torch.randint(low, top + 1, (case["batch"],), generator=gen, device="cuda", dtype=torch.int32)
    n[0] = top
    return n


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dtype, width = TYPES[case["dtype"]], _width(case["dim"])
    b, h, dim, op = case["batch"], case["heads"], case["dim"], case["op"]
    bank = _empty_bank(case)
    state = dict(case=case, bank=bank, width=width)
    fill = {"push": case.get("fill"), "attend": case.get("fill"), "stream": case.get("keep"), "compress": case["k"]}[op]
    if op != "push":
        for side in ("key", "value"):
            for i in range(b):                           # one sequence at a time: float32 copies of all would be large
                x = _rows_like(gen, (1, h, fill, dim), dtype)
                codes, scales = _pack(_padded(x[0], width))
                bank[side][i, :, :fill] = codes
                bank[side + "_scale"][i, :, :, :fill] = scales.transpose(-1, -2)
    if op in ("push", "attend", "compress"):
        even = op == "attend" and not case["ragged"]
        low = case["keep"] // 2 if op == "compress" else 0 if op == "push" else fill // 2
        bank["length"] = _lengths(gen, case, fill, fill if even else low)
    else:
        bank["length"].fill_(fill)
    gone = torch.randint(0, 1000, (b,), generator=gen, device="cuda", dtype=torch.int32)         # rows that left before
    bank["seen"] = bank["length"] + (gone if op in ("stream", "compress") else 0)
    slots = torch.arange(bank["weight"].shape[2], device="cuda", dtype=torch.int32)
    bank["position"] += (bank["seen"] - bank["length"])[:, None, None] + slots
    if op in ("stream", "compress"):
        # attention sums: most rows little, a few much, some none at all
        w = torch.exp(2.0 * torch.randn(bank["weight"].shape, generator=gen, device="cuda"))
        bank["weight"] = w.masked_fill_(torch.rand(w.shape, generator=gen, device="cuda") < 0.05, 0.0)
    if op == "attend":
        q = torch.randn(b, case["rows"], h * case["group"], dim, generator=gen, device="cuda")   # as a projection leaves them
        state["query"] = (q * 1.2).to(dtype).transpose(1, 2)
        if case["ragged"] and case["rows"] > 1:
            state["counts"] = torch.randint(1, case["rows"] + 1, (b,), generator=gen, device="cuda", dtype=torch.int32)
            state["counts"] = torch.minimum(state["counts"], bank["length"])
    if op in ("push", "stream"):
        rows = case["rows"]
        state["key"] = _rows_like(gen, (b, h, rows, dim), dtype)
        state["new"] = _rows_like(gen, (b, h, rows, dim), dtype)
        if op == "push" and rows > 1:
            state["counts"] = torch.randint(rows // 2, rows + 1, (b,), generator=gen, device="cuda", dtype=torch.int32)
        state["start"] = bank["length"].clone()
    if op == "compress":
        state["small"] = _empty_bank(dict(case, k=case["keep"]))
    if own:
        import image_classification_amd as ica
        state["cache"] = cache = ica.CacheBank()
        cache.register(NAME, dim=dim, k=case["k"], heads=h, batch=b)
        if op == "compress":
            cache.register("small", dim=dim, k=case["keep"], heads=h, batch=b)
        cache.cuda()
        cache.load_state_dict({NAME + "_" + part: t for part, t in bank.items()}, strict=False)
    return state


# ---------------------------------------------------------------------------------------------------------- plain forms
def _push(state):
    """Quantises the new rows and writes those that count behind each sequence's last one; returns the values held."""
    bank, case = state["bank"], state["case"]
    key, new, rows = _padded(state["key"], state["width"]), _padded(state["new"], state["width"]), case["rows"]
    bad = ~(torch.isfinite(key).all(-1) & torch.isfinite(new).all(-1))
    t = torch.arange(rows, device="cuda", dtype=torch.int32)
    counts = state.get("counts", torch.full_like(bank["length"], rows))
    real = t < counts[:, None]
    seq, row = real.nonzero(as_tuple=True)
    at = bank["length"][seq].long() + row
    held = []
    for side, x in (("key", key), ("value", new)):
        codes, scales = _pack(x.masked_fill(bad.unsqueeze(-1), 0.0))
        scales = scales.masked_fill(bad.unsqueeze(-1), 255)
        bank[side][seq, :, at] = codes[seq, :, row]
        bank[side + "_scale"][seq, :, :, at] = scales[seq, :, row]
        v = _values(codes, scales.transpose(-1, -2)).masked_fill(~real[:, None, :, None], 0.0)
        held.append(v[..., :case["dim"]].to(state["key"].dtype))
    bank["weight"][seq, :, at] = 0.0
    bank["position"][seq, :, at] = (bank["seen"][seq] + row.int())[:, None]
    bank["length"] += counts
    bank["seen"] += counts
    return held


def _trim(state):
    bank = state["bank"]
    gone = (bank["length"] - state["start"]).clamp_(min=0)
    bank["length"] -= gone
    bank["seen"] -= gone


def _attend(state):
    bank, case, q = state["bank"], state["case"], state["query"]
    b, h, g, rows, fill = case["batch"], case["heads"], case["group"], case["rows"], case["fill"]
    key = _values(bank["key"][:, :, :fill], bank["key_scale"][..., :fill])
    x = _padded(q, state["width"]).reshape(b, h, g * rows, state["width"])
    s = torch.matmul(x, key.transpose(-1, -2)).view(b, h, g, rows, fill).mul_(case["dim"] ** -0.5)
    del key
    t = torch.arange(rows, device="cuda", dtype=torch.int32)
    counts = state.get("counts", torch.full_like(bank["length"], rows))
    sees = bank["length"][:, None] - (counts[:, None] - 1 - t).clamp(min=0) if case["causal"] else bank["length"][:, None].expand(b, rows)
    sees = sees.masked_fill(t >= counts[:, None], 0)
    mask = torch.arange(fill, device="cuda") >= sees[:, None, None, :, None]
    s = s.masked_fill_(mask, -math.inf)
    s -= s.amax(-1, keepdim=True).masked_fill_(sees[:, None, None, :, None] <= 0, 0.0)
    p = s.exp_()
    p /= p.sum(-1, keepdim=True).masked_fill_(sees[:, None, None, :, None] <= 0, 1.0)
    value = _values(bank["value"][:, :, :fill], bank["value_scale"][..., :fill])
    out = torch.matmul(p.view(b, h, g * rows, fill), value)[..., :case["dim"]].reshape(b, h * g, rows, case["dim"]).to(q.dtype)
    if not case["weigh"]:
        return out
    bank["weight"][:, :, :fill] += p.view(b, h, g * rows, fill).sum(2)
    return out, bank["weight"][:, :, :case["k"]]


def _evict(state, into):
    """Ranks rows by (recent, weight, lower slot); freed slots below ``keep`` take the kept rows from above, both in ascending order."""
    bank, case = state["bank"], state["case"]
    b, h, keep, rows = case["batch"], case["heads"], case["keep"], bank["weight"].shape[2]
    slot = torch.arange(rows, device="cuda")
    used = slot < bank["length"][:, None, None]
    recent = bank["position"] >= (bank["seen"] - case["recent"])[:, None, None]
    rank = bank["weight"].double().masked_fill(recent, math.inf).masked_fill(~used, -math.inf)
    order = rank.sort(dim=-1, descending=True, stable=True).indices
    kept = torch.zeros_like(used.expand(b, h, rows)).scatter_(-1, order[..., :keep], True) & used
    # source of each slot below keep: itself if it is kept, else the next kept row from above
    source = slot[:keep].expand(b, h, keep).clone()
    below, above = kept[..., :keep], kept.clone()
    above[..., :keep] = False
    lane, head, hole = (~below & used[..., :keep]).nonzero(as_tuple=True)
    source[lane, head, hole] = above.nonzero(as_tuple=True)[2]
    for side in ("key", "value"):
        into[side][:, :, :keep] = bank[side].gather(2, source[..., None].expand(-1, -1, -1, bank[side].shape[-1]))
        into[side + "_scale"][..., :keep] = bank[side + "_scale"].gather(3, source[:, :, None].expand(-1, -1, bank[side + "_scale"].shape[2], -1))
    into["weight"][..., :keep] = bank["weight"].gather(2, source)
    into["position"][..., :keep] = bank["position"].gather(2, source)
    into["seen"].copy_(bank["seen"])
    into["length"].copy_(bank["length"].clamp(max=keep))


def _read(bank, case, k):
    there = torch.arange(k, device="cuda") < bank["length"][:, None, None]
    return [_values(bank[side][:, :, :k], bank[side + "_scale"][..., :k])[..., :case["dim"]].masked_fill(~there.unsqueeze(-1), 0.0).bfloat16()
            for side in ("key", "value")]


def run(state):
    case = state["case"]
    op, keep = case["op"], case.get("keep")
    if own:
        cache = state["cache"]
        if op == "push":
            cache.trim(NAME, state["start"])
            held = cache.push(NAME, state["key"], state["new"], counts=state.get("counts"), held=True)
            return {"held": held, "lengths": cache.lengths(NAME)}
        if op == "attend":
            out = cache.attend(NAME, state["query"], counts=state.get("counts"), causal=case["causal"], accumulate=case["weigh"])
            return (out, cache.weights(NAME)) if case["weigh"] else out
        if op == "stream":
            cache.push(NAME, state["key"], state["new"])
            cache.evict(NAME, keep, recent=case["recent"])
            return {"rows": cache[NAME], "positions": cache.positions(NAME)[..., :keep], "weights": cache.weights(NAME)[..., :keep]}
        cache.evict(NAME, keep, recent=case["recent"], into="small")
        n = cache.lengths("small")
        return {"rows": cache["small"], "lengths": n}
    if op == "push":
        _trim(state)
        held = _push(state)
        return {"held": held, "lengths": state["bank"]["length"]}
    if op == "attend":
        return _attend(state)
    if op == "stream":
        _push(state)
        _evict(state, state["bank"])
        return {"rows": _read(state["bank"], case, case["k"]), "positions": state["bank"]["position"][..., :keep], "weights": state["bank"]["weight"][..., :keep]}
    _evict(state, state["small"])
    return {"rows": _read(state["small"], case, keep), "lengths": state["small"]["length"]}


# ------------------------------------------------------------------------------------------------------ in 64 bits, apart
def _exact_held(x):
    """float64 [..., dim] -> the values that 4 bits hold: the nearest grid point by looking at every midpoint."""
    dim = x.shape[-1]
    x = torch.nn.functional.pad(x.double(), (0, -dim % 32)).unflatten(-1, (-1, 32))
    top = x.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2((top / 7).clamp(min=2.0 ** -126))).clamp(-126, 125)
    e = torch.where(top > 7 * torch.exp2(e), e + 1, torch.where(top <= 7 * torch.exp2(e - 1), e - 1, e)).clamp(-126, 125)
    y = x / torch.exp2(e)
    grid = torch.tensor(GRID, dtype=torch.float64, device=x.device)
    middle = (grid[1:] + grid[:-1]) / 2
    a = y.abs()
    up = torch.bucketize(a, middle, right=True)           # a on a midpoint goes up
    down = torch.bucketize(a, middle, right=False)        # a on a midpoint stays down
    at = torch.where(up % 2 == 0, up, down)               # of the two, the one with the even code
    return (grid[at] * torch.sign(y) * torch.exp2(e)).flatten(-2)[..., :dim]


def _exact_rows(codes, scales, dim):
    """One sequence and head: codes [rows, width / 2], scales [width / 32, rows] -> float64 [rows, dim], by a table."""
    table = torch.tensor(GRID + tuple(-v for v in GRID), dtype=torch.float64, device=codes.device)
    pair = torch.stack((table[(codes % 16).long()], table[(codes // 16).long()]), -1).flatten(-2)
    return (pair * torch.exp2(scales.t().double() - 127).repeat_interleave(32, -1))[:, :dim]


def exact(case, seed):
    state = prepare(case, seed)
    bank, op, dim = state["bank"], case["op"], case["dim"]
    length, seen = bank["length"].tolist(), bank["seen"].tolist()
    if op == "push":
        counts = state["counts"].tolist() if "counts" in state else [case["rows"]] * case["batch"]
        held = [_exact_held(state[part]) for part in ("key", "new")]
        for x in held:
            for i, n in enumerate(counts):
                x[i, :, n:] = 0
        return {"held": held, "lengths": None}
    if op == "attend":
        g, rows = case["group"], case["rows"]
        counts = state["counts"].tolist() if "counts" in state else [rows] * case["batch"]
        out = torch.zeros(state["query"].shape, dtype=torch.float64, device="cuda")
        weight = bank["weight"].double()
        for i in range(case["batch"]):
            for j in range(case["heads"]):
                n = length[i]
                key, value = (_exact_rows(bank[side][i, j, :n], bank[side + "_scale"][i, j, :, :n], dim) for side in ("key", "value"))
                for m in range(g):
                    q = state["query"][i, j * g + m, :counts[i]].double()
                    s = q @ key.t() / math.sqrt(dim)
                    if case["causal"]:
                        limit = torch.arange(n - counts[i], n, device="cuda")
                        s = s.masked_fill(torch.arange(n, device="cuda") > limit[:, None], -math.inf)
                    p = torch.softmax(s, -1)
                    out[i, j * g + m, :counts[i]] = p @ value
                    weight[i, j, :n] += p.sum(0)
        return (out, weight[..., :case["k"]]) if case["weigh"] else out
    keep, k = case["keep"], case["k"] if op == "stream" else case["keep"]
    sides = {side: torch.zeros(case["batch"], case["heads"], k, dim, dtype=torch.float64, device="cuda") for side in ("key", "value")}
    new = {"key": _exact_held(state["key"]), "value": _exact_held(state["new"])} if op == "stream" else None
    weights = torch.zeros(case["batch"], case["heads"], keep, dtype=torch.float64, device="cuda")
    for i in range(case["batch"]):
        for j in range(case["heads"]):
            n, last = length[i], seen[i]
            rows = {side: _exact_rows(bank[side][i, j, :n], bank[side + "_scale"][i, j, :, :n], dim) for side in ("key", "value")}
            w, at = bank["weight"][i, j, :n].tolist(), bank["position"][i, j, :n].tolist()
            if op == "stream":
                rows = {side: torch.cat((rows[side], new[side][i, j])) for side in rows}
                w, at = w + [0.0] * case["rows"], at + list(range(last, last + case["rows"]))
                n, last = n + case["rows"], last + case["rows"]
            best = sorted(range(n), key=lambda r: (at[r] < last - case["recent"], 0.0 if at[r] >= last - case["recent"] else -w[r], r))[:keep]
            stay = set(best)
            moved = iter(sorted(r for r in best if r >= keep))
            source = [r if r in stay else next(moved) for r in range(min(n, keep))]
            for side in rows:
                sides[side][i, j, :len(source)] = rows[side][source]
            weights[i, j, :len(source)] = torch.tensor([w[r] for r in source], dtype=torch.float64)
    rows = [sides["key"], sides["value"]]
    return {"rows": rows, "positions": None, "weights": weights} if op == "stream" else {"rows": rows, "lengths": None}
