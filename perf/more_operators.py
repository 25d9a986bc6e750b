"""Work of the paged key-value cache held in 4 bits: rows that enter it (with the norm and the rotation of queries and keys on the way), decode
attention that reads it, and attention of prompt portions that reads it.

A case names an operator ("op") and its sizes.  `run` computes it in plain 32-bit torch operations, or, where `own` is set, through the
framework's entry points.  The format: 16 neighbouring numbers of a head's row of 128 are kept as codes c of 4 bits (sign, and a magnitude
of 0, 0.5, 1, 1.5, 2, 3, 4 or 6) and a scale s of 8 bits (5 of exponent, 3 of mantissa: the fp16 number with these bits on top), and stand for c * s.
s is the nearest to the block's largest magnitude / 6 (half way: to the even mantissa), c the nearest to number / s (half way: to the smaller magnitude)."""
import importlib
import math

import torch

own = False

DEV = "cuda:0"
BF16, F32, F64, E4M3, I32, U8 = torch.bfloat16, torch.float32, torch.float64, torch.float8_e4m3fn, torch.int32, torch.uint8
DIM, EPS = 128, 1e-6
MAGNITUDES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
BORDERS = (0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0)
MOST_SCALE = 10240.0                        # 6 of it still is an fp16 number

_made = {}


def _framework():
    if not _made:
        _made["ops"] = importlib.import_module("nano-vllm-candle_b200.ops")
        _made["ctx"] = _made["ops"].Context(0)
    return _made["ops"], _made["ctx"]


# ------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # a decode step's new rows: one sequence of a small model, where latency alone counts, and a batch of 64 with a few padded places
        {"name": "append 1", "op": "append", "tokens": 1, "heads": 16, "kv": 8, "block": 256, "decode": True, "padded": 0},
        {"name": "append 64", "op": "append", "tokens": 64, "heads": 32, "kv": 8, "block": 256, "decode": True, "padded": 5},
        # a long prompt batch on its way into the cache
        {"name": "append 16000", "op": "append", "tokens": 16000, "heads": 32, "kv": 8, "block": 256, "decode": False, "padded": 0},
        # rows that are ready as they are (rotated elsewhere), in small pages
        {"name": "rows 4097", "op": "rows", "tokens": 4097, "heads": 40, "kv": 8, "block": 16, "decode": False, "padded": 0},
        # decode steps: one short sequence; a batch of ragged chats; a full batch in small pages, from one token on; few long documents
        {"name": "decode 1", "op": "decode", "seqs": 1, "heads": 16, "kv": 8, "block": 256, "least": 700, "most": 700},
        {"name": "decode 64", "op": "decode", "seqs": 64, "heads": 32, "kv": 8, "block": 256, "least": 200, "most": 1500},
        {"name": "decode 256", "op": "decode", "seqs": 256, "heads": 32, "kv": 8, "block": 16, "least": 1, "most": 4000},
        {"name": "decode 4 long", "op": "decode", "seqs": 4, "heads": 64, "kv": 8, "block": 256, "least": 30000, "most": 131000},
        # a few new tokens of each sequence behind its context: drafted tokens to be checked, the ends of chunked prompts
        {"name": "portions 32", "op": "portion", "seqs": 32, "heads": 32, "kv": 8, "block": 256, "least": 1, "most": 8, "before_least": 500, "before_most": 3000},
        # a short prompt of odd length; one chunk of a long prompt; a whole prompt
        {"name": "portion 333", "op": "portion", "seqs": 1, "heads": 16, "kv": 8, "block": 16, "least": 333, "most": 333, "before_least": 0, "before_most": 0},
        {"name": "portion 2048 of 16000", "op": "portion", "seqs": 1, "heads": 32, "kv": 8, "block": 256, "least": 2048, "most": 2048, "before_least": 13952, "before_most": 13952},
        {"name": "portion 8191", "op": "portion", "seqs": 1, "heads": 32, "kv": 8, "block": 256, "least": 8191, "most": 8191, "before_least": 0, "before_most": 0},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    op = rng.choice(["append", "append", "rows", "decode", "decode", "decode", "portion", "portion", "portion"])
    heads, kv = rng.choice([(16, 8), (32, 8), (40, 8), (64, 8), (16, 4), (8, 1), (5, 1), (4, 4), (24, 2)])
    block = rng.choice([16, 32, 64, 128, 256])
    case = {"op": op, "heads": heads, "kv": kv, "block": block}
    if op in ("append", "rows"):
        decode = rng.random() < 0.4
        tokens = _log(rng, 1, 512 if decode else 16000 * 48 // (heads + 2 * kv))
        return {**case, "tokens": min(tokens, 16000), "decode": decode, "padded": rng.randrange(0, 1 + tokens // 4) if rng.random() < 0.4 else 0}
    if op == "decode":
        seqs = _log(rng, 1, 256)
        most = _log(rng, 1, min(131000, 4000 * 256 * 8 // (seqs * max(kv, heads // 4))))
        return {**case, "seqs": seqs, "least": rng.choice([0, 1, most, rng.randint(0, most)]), "most": most}
    if rng.random() < 0.5:
        seqs, least, most = _log(rng, 1, 64), 1, _log(rng, 1, 32)
        before = _log(rng, 1, min(16000, 8192 * 8192 // (seqs * most)) * 8 // max(8, kv * 2))
    else:
        seqs = _log(rng, 1, 8)
        most = _log(rng, 32, 4096 // seqs + 32)
        least = rng.randint(most // 2, most)
        before = rng.choice([0, _log(rng, 1, 14000)])
        before = min(before, max(0, 8192 * 8192 * 16 // (seqs * most * max(heads, 32)) - most))
    return {**case, "seqs": seqs, "least": least, "most": most, "before_least": rng.randint(0, before), "before_most": before}


def _spread(least, most, n):
    return [most - (most - least) * i // max(1, n - 1) for i in range(n)]


def _lengths(case):
    """(new tokens, all tokens) of each sequence: both spread evenly over their ranges, the longest contexts with the fewest new tokens."""
    if case["op"] == "decode":
        whole = _spread(case["least"], case["most"], case["seqs"])
        return [1] * case["seqs"], whole
    new = _spread(case["least"], case["most"], case["seqs"])
    return new, [n + b for n, b in zip(new, reversed(_spread(case["before_least"], case["before_most"], case["seqs"])))]


# ------------------------------------------------------------------------------------------ the 4-bit format
def _blocks(x):
    return x.unflatten(-1, (-1, 16))


def _to_scale(v):
    """The nearest numbers of 5 exponent bits and 3 mantissa bits, half way to the even mantissa; v is not negative."""
    _, e = torch.frexp(v)
    step = torch.ldexp(torch.ones_like(v), e.clamp_min(-13) - 4)
    return (torch.round(v / step) * step).clamp_max(MOST_SCALE)


def _to_4bit(x):
    """fp32 [..., 128] -> (codes of their magnitudes and signs, uint8 [..., 128]; scales, fp32 [..., 8])."""
    b = _blocks(x)
    s = _to_scale((b.abs().amax(-1).double() / 6).float())
    q = b.abs() / torch.where(s > 0, s, torch.ones((), device=DEV))[..., None]
    c = torch.bucketize(q, torch.tensor(BORDERS, device=DEV), out_int32=True).to(U8)        # borders below the quotient: half way is the smaller one
    c = torch.where((s > 0)[..., None], c, torch.zeros((), dtype=U8, device=DEV))
    return (c + 8 * torch.signbit(b).to(U8)).flatten(-2), s


def _pack(codes):
    return codes[..., 0::2] + 16 * codes[..., 1::2]


def _scale_bits(s):
    return (s.half().view(torch.int16) >> 7).to(U8)


def _numbers(codes):
    m = torch.tensor(MAGNITUDES + tuple(-m for m in MAGNITUDES), device=DEV)
    return m[codes.int()]


def _read(codes, scales):
    """Packed rows [..., 64] and scale bytes [..., 8] -> fp32 [..., 128]."""
    both = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)
    s = (scales.to(torch.int16) << 7).view(torch.float16).float()
    return (_blocks(_numbers(both)) * s[..., None]).flatten(-2)


# ------------------------------------------------------------------------------------------ inputs
class _Rand:
    def __init__(self, seed):
        self.g = torch.Generator(device=DEV).manual_seed(int(seed))

    def __call__(self, *shape, scale=1.0, mean=0.0, dtype=F32):
        return torch.randn(*shape, generator=self.g, device=DEV, dtype=F32).mul_(scale).add_(mean).to(dtype)

    def order(self, n):
        return torch.randperm(n, generator=self.g, device=DEV)


def _cache(rand, blocks, kv, block, heads_far):
    """One side of a cache full of rows: channels that stand far out in keys, rows of different size.  Made a part at a time."""
    codes, scales = torch.empty(blocks, kv, block, DIM // 2, dtype=U8, device=DEV), torch.empty(blocks, kv, block, DIM // 16, dtype=U8, device=DEV)
    far = torch.exp(rand(1, kv, 1, DIM, scale=heads_far))
    part = max(1, (1 << 25) // (kv * block * DIM))
    for at in range(0, blocks, part):
        n = min(part, blocks - at)
        c, s = _to_4bit(rand(n, kv, block, DIM) * far * torch.exp(rand(n, kv, block, 1, scale=0.2)))
        codes[at:at + n], scales[at:at + n] = _pack(c), _scale_bits(s)
    return codes, scales


def prepare(case, seed):
    rand, op = _Rand(seed), case["op"]
    heads, kv, block = case["heads"], case["kv"], case["block"]
    s = {"case": case}
    if op in ("append", "rows"):
        n = case["tokens"]
        if case["decode"]:                                             # each token in a page of its own
            blocks = n + 3
            pages = rand.order(blocks)
            slots = pages[:n] * block + torch.randint(0, block, (n,), generator=rand.g, device=DEV)
            positions = torch.randint(0, 40960, (n,), generator=rand.g, device=DEV)
        else:                                                          # one prompt behind another
            blocks = -(-n // block) + 3
            at, pages = torch.arange(n, device=DEV), rand.order(blocks)
            slots = pages[at // block] * block + at % block
            positions = at % 8192
        slots[n - case["padded"]:] = -1
        s.update(slots=slots.to(I32), positions=positions.to(I32), spare=pages[-1:].to(I32))
        s["qkv"] = (rand(n, (heads + 2 * kv) * DIM) * torch.exp(rand(1, (heads + 2 * kv) * DIM, scale=0.5))).to(BF16)
        # a cache in use: what is written is what these tokens change
        s["k"], s["ks"] = _cache(rand, blocks, kv, block, 0.5)
        s["v"], s["vs"] = _cache(rand, blocks, kv, block, 0.0)
        if op == "append":
            s.update(qw=rand(DIM, scale=0.2, mean=1.0, dtype=BF16), kw=rand(DIM, scale=0.2, mean=1.0, dtype=BF16))
            angle = torch.arange(40960, device=DEV, dtype=F64)[:, None] * 1e6 ** (-torch.arange(0, DIM, 2, device=DEV, dtype=F64) / DIM)
            s["rope"] = torch.cat((angle.cos(), angle.sin()), 1).float()
            s["q"] = torch.empty(n, heads * DIM, dtype=BF16, device=DEV)
        return s
    new, whole = _lengths(case)
    b = len(new)
    need = [-(-c // block) for c in whole]
    order = rand.order(sum(need) + 1).to(I32)
    tables = torch.full((b, max(max(need), 1)), -1, dtype=I32)
    place = order.cpu()
    at = 0
    for i, m in enumerate(need):
        tables[i, :m] = place[at:at + m]
        at += m
    s["k"], s["ks"] = _cache(rand, sum(need) + 1, kv, block, 0.5)
    s["v"], s["vs"] = _cache(rand, sum(need) + 1, kv, block, 0.0)
    s["tables"], s["lens"] = tables.to(DEV), torch.tensor(whole, dtype=I32, device=DEV)
    s["cu"] = torch.tensor([0] + new, dtype=I32).cumsum(0).to(I32).to(DEV)
    s["most_new"], s["most"] = max(new), max(whole)
    s["q"] = rand(sum(new), heads * DIM, dtype=BF16)
    return s


# ------------------------------------------------------------------------------------------ one pass
def _context(s):
    """Every sequence's cached rows, padded: k and v fp32 [B, kv, most, 128]."""
    case = s["case"]
    block, t = case["block"], torch.arange(s["most"], device=DEV)
    at = s["tables"].long().clamp_min(0)[:, t // block]                # [B, most]
    off = (t % block).expand_as(at)
    rows = lambda c: c[at, :, off].transpose(1, 2)                     # noqa: E731
    return _read(rows(s["k"]), rows(s["ks"])), _read(rows(s["v"]), rows(s["vs"]))


def _attend(q, k, v, seen):
    """q [B, kv, rows, 128], seen [B, 1, rows, most]: rows that see nothing are zeros."""
    x = (q @ k.transpose(-1, -2)) * DIM ** -0.5
    x = torch.where(seen, x, torch.full((), -math.inf, device=DEV))
    top = x.amax(-1, keepdim=True).clamp_min(torch.finfo(F32).min)
    p = torch.exp(x - top)
    total = p.sum(-1, keepdim=True)
    return (p @ v) / torch.where(total > 0, total, torch.ones((), device=DEV))


def run(s):
    case = s["case"]
    op, heads, kv = case["op"], case["heads"], case["kv"]
    if own:
        ops, ctx = _framework()
        cache = ops.Fp4Cache(s["k"], s["ks"], s["v"], s["vs"])
        if op == "append":
            q = ops.qk_norm_rope_store_fp4(ctx, s["qkv"], s["qw"], s["kw"], EPS, s["rope"], s["positions"], heads, cache, s["slots"], q_out=s["q"])
            k, ks, v, vs = ops.read_kvcache_fp4(ctx, cache, s["slots"])
            return {"q": q, "k": k, "k_scale": ks, "v": v, "v_scale": vs}
        if op == "rows":
            w = heads * DIM
            ops.store_kvcache_fp4(ctx, s["qkv"][:, w:w + kv * DIM], s["qkv"][:, w + kv * DIM:], cache, s["slots"])
            k, ks, v, vs = ops.read_kvcache_fp4(ctx, cache, s["slots"])
            return {"k": k, "k_scale": ks, "v": v, "v_scale": vs}
        if op == "decode":
            return ops.paged_decode_attn_fp4(ctx, s["q"], cache, s["tables"], s["lens"], heads, DIM ** -0.5)
        return ops.prefill_attn_paged_fp4(ctx, s["q"], cache, s["tables"], s["lens"], s["cu"], s["most_new"], heads, DIM ** -0.5)
    if op in ("append", "rows"):
        x = s["qkv"].float().unflatten(1, (-1, DIM))
        out = {}
        k = x[:, heads:heads + kv]
        if op == "append":
            cs = s["rope"][s["positions"].long()][:, None]
            cos, sin = cs[..., :DIM // 2], cs[..., DIM // 2:]
            w = torch.cat((s["qw"].float().expand(heads, DIM), s["kw"].float().expand(kv, DIM)))
            y = x[:, :heads + kv]
            y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + EPS) * w
            lo, hi = y[..., :DIM // 2], y[..., DIM // 2:]
            y = torch.cat((lo * cos - hi * sin, hi * cos + lo * sin), -1).to(BF16)
            out["q"], k = y[:, :heads].flatten(1), y[:, heads:].float()
        live = (s["slots"] >= 0)[:, None, None, None]
        codes, scale = _to_4bit(torch.stack((k, x[:, heads + kv:]), 1))                          # [tokens, 2, kv, ...]
        # into the cache; places without a slot write the page that no token has as it is
        page = torch.where(s["slots"] < 0, s["spare"], s["slots"] // case["block"])
        off = s["slots"].clamp_min(0) % case["block"]
        bits, scale_bits = _pack(codes), _scale_bits(scale)
        s["k"][page, :, off] = torch.where(live[:, 0], bits[:, 0], s["k"][page, :, off])
        s["v"][page, :, off] = torch.where(live[:, 0], bits[:, 1], s["v"][page, :, off])
        s["ks"][page, :, off] = torch.where(live[:, 0], scale_bits[:, 0], s["ks"][page, :, off])
        s["vs"][page, :, off] = torch.where(live[:, 0], scale_bits[:, 1], s["vs"][page, :, off])
        zero = torch.zeros((), device=DEV)
        numbers, scale = torch.where(live, _numbers(codes), zero).to(E4M3), torch.where(live, scale, zero).to(BF16)
        out.update(k=numbers[:, 0], k_scale=scale[:, 0], v=numbers[:, 1], v_scale=scale[:, 1])
        return out
    k, v = _context(s)
    b, t, most_new = s["lens"].numel(), torch.arange(s["most"], device=DEV), s["most_new"]
    count = s["cu"][1:] - s["cu"][:-1]
    i = torch.arange(most_new, device=DEV)
    row = (s["cu"][:-1, None] + torch.minimum(i, count[:, None] - 1)).long()                     # [B, most_new]
    q = s["q"].float().view(-1, kv, heads // kv, DIM)[row].transpose(1, 2)                        # [B, kv, most_new, group, 128]
    sees = (s["lens"] - count)[:, None] + i                                                     # the last token that a row sees
    seen = (t <= sees[..., None])[:, None, :, None].expand(b, 1, most_new, heads // kv, t.numel()).flatten(2, 3)
    o = _attend(q.flatten(2, 3), k, v, seen).unflatten(2, (most_new, heads // kv)).transpose(1, 2).flatten(2)     # [B, most_new, heads * 128]
    return o[i < count[:, None]].to(BF16)


# ------------------------------------------------------------------------------------------ what it cannot do without
def work(case):
    op, heads, kv = case["op"], case["heads"], case["kv"]
    row = kv * 2 * (DIM // 2 + DIM // 16)                              # a token's rows in the cache
    if op in ("append", "rows"):
        n, live = case["tokens"], case["tokens"] - case["padded"]
        back = n * kv * 2 * (DIM + DIM // 16 * 2)                      # as they come back: numbers in 8 bits, scales in 16
        if op == "rows":
            return {"bytes": live * (kv * 2 * DIM * 2 + 2 * row) + n * 4 + back, "flops": 4 * live * kv * 2 * DIM}
        angles = min(n, 8192) * DIM * 4
        return {"bytes": n * (heads * 2 * DIM * 2 + kv * 2 * DIM * 2 + 8) + 2 * live * row + angles + back, "flops": 10 * n * (heads + 2 * kv) * DIM}
    new, whole = _lengths(case)
    seen = sum(n * c - n * (n - 1) // 2 for n, c in zip(new, whole) if c)
    return {"bytes": sum(whole) * row + sum(new) * heads * DIM * 4 + len(new) * 8 + sum(-(-c // case["block"]) for c in whole) * 4, "flops": 4 * DIM * heads * seen}


# ------------------------------------------------------------------------------------------ the same from the definition, in 64 bits
def _rows64(x):
    """Rows of 128 -> (what their codes stand for, scales)."""
    x = x.unflatten(-1, (8, 16))
    want = x.abs().amax(-1) / 6
    all_scales = torch.tensor([m / 8 * 2.0 ** -14 for m in range(8)] + [(8 + m) / 8 * 2.0 ** (e - 15) for e in range(1, 31) for m in range(8)], dtype=F64, device=DEV)
    all_scales = all_scales[all_scales <= MOST_SCALE]
    above = torch.searchsorted(all_scales, want.contiguous()).clamp(1, all_scales.numel() - 1)
    lo, hi = all_scales[above - 1], all_scales[above]
    up = (want - lo > hi - want) | ((want - lo == hi - want) & (above % 2 == 0))
    scale = torch.where(up, hi, lo)
    q = x / torch.where(scale > 0, scale, torch.ones_like(scale))[..., None]
    size = sum((q.abs() > b) * (m - l) for b, l, m in zip(BORDERS, MAGNITUDES, MAGNITUDES[1:]))
    return (torch.sign(q) * size * (scale > 0)[..., None]).flatten(-2), scale


def exact(case, seed):
    s, op = prepare(case, seed), case["op"]
    heads, kv = case["heads"], case["kv"]
    if op in ("append", "rows"):
        x = s["qkv"].to(F64).view(case["tokens"], heads + 2 * kv, DIM)
        k, out = x[:, heads:heads + kv], {}
        if op == "append":
            turned = []
            for lo, hi, w in ((0, heads, s["qw"]), (heads, heads + kv, s["kw"])):
                y = x[:, lo:hi]
                y = y / torch.sqrt((y * y).sum(-1, keepdim=True) / DIM + EPS) * w.to(F64)
                turn = s["rope"][s["positions"].long()].to(F64)
                c, n = turn[:, None, :DIM // 2], turn[:, None, DIM // 2:]
                a, b = y.chunk(2, -1)
                turned.append(torch.cat((a * c - b * n, b * c + a * n), -1))
            out["q"], k = turned[0].flatten(1), turned[1].to(BF16).to(F64)       # the cache takes the rows in bf16
        live = (s["slots"] >= 0).to(F64)[:, None, None]
        for name, rows in (("k", k), ("v", x[:, heads + kv:])):
            numbers, scale = _rows64(rows)
            out[name], out[name + "_scale"] = numbers * live, scale * live
        return out
    new, whole = _lengths(case)
    if sum(n * c for n, c in zip(new, whole)) * heads > 3e9:
        return None
    scale_of = torch.arange(256, dtype=torch.int16, device=DEV).bitwise_left_shift(7).view(torch.float16).to(F64)
    number_of = torch.tensor(MAGNITUDES + tuple(-m for m in MAGNITUDES), dtype=F64, device=DEV)
    group, outs, at = heads // kv, [], 0
    for i, (n, c) in enumerate(zip(new, whole)):
        q = s["q"][at:at + n].to(F64).view(n, kv, group, DIM)
        at += n
        if not c:
            outs.append(torch.zeros(n, heads * DIM, dtype=F64, device=DEV))
            continue
        pages = s["tables"][i, :-(-c // case["block"])].long()
        o = torch.empty(n, kv, group, DIM, dtype=F64, device=DEV)
        late = torch.arange(c, device=DEV)[None] > torch.arange(c - n, c, device=DEV)[:, None]
        for h in range(kv):
            k, v = (torch.stack((number_of[(m[pages, h].flatten(0, 1)[:c] & 15).long()], number_of[(m[pages, h].flatten(0, 1)[:c] >> 4).long()]), -1).flatten(1)
                    * scale_of[e[pages, h].flatten(0, 1)[:c].long()].repeat_interleave(16, 1) for m, e in ((s["k"], s["ks"]), (s["v"], s["vs"])))
            for g in range(group):
                p = torch.softmax((q[:, h, g] @ k.T / math.sqrt(DIM)).masked_fill(late, -math.inf), -1)
                o[:, h, g] = p @ v
        outs.append(o.flatten(1))
    return torch.cat(outs)
