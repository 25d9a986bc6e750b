"""Work of the 8-bit path: rows and weights in e4m3 with a scale for each block of 128, the norm and the gated unit that write such rows, and the
products that read them, dense and grouped by expert.

A case names an operator ("op") and its sizes.  `run` computes it in plain 32-bit torch operations, or, where `own` is set, through the
framework's entry points.  The 8-bit format: a block of 128 numbers along a row (of 128 x 128 in a weight) is kept as e4m3 numbers q and one fp32
scale = max(largest magnitude / 448, 2^-126), and stands for q * scale.  A row's last block may be shorter."""
import importlib
import math

import torch

own = False

DEV = "cuda:0"
BF16, F32, F64, E4M3 = torch.bfloat16, torch.float32, torch.float64, torch.float8_e4m3fn
EPS = 1e-6
TOP, LEAST = 448.0, 2.0 ** -126

_made = {}


def _framework():
    if not _made:
        _made["ops"] = importlib.import_module("nano-vllm-candle_b200.ops")
        _made["ctx"] = _made["ops"].Context(0)
    return _made["ops"], _made["ctx"]


# ------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # the norm in front of a small model's layer for one sequence's next token: latency alone
        {"name": "norm decode 1", "op": "norm", "tokens": 1, "width": 1024, "wide": False, "residual": True, "plain": False},
        # the same in front of a routed layer over a long prompt batch, with the bf16 row for the router beside the 8-bit one
        {"name": "norm prefill 16000", "op": "norm", "tokens": 16000, "width": 4096, "wide": False, "residual": True, "plain": True},
        # rows of a decode step on their way to their experts: gathered, groups padded, in 8 bits
        {"name": "gather decode 64", "op": "rows", "tokens": 64, "width": 2048, "act": "none", "wide": False, "experts": 16, "top": 2},
        # the gated unit between the two products of a feed-forward over a prompt batch of odd length
        {"name": "gate prefill 8191", "op": "rows", "tokens": 8191, "width": 12288, "act": "silu", "wide": False, "experts": 0, "top": 0},
        # a layer's weights brought to 8 bits while a model is loaded: one projection, and experts of a height that no block divides
        {"name": "weights 6144 x 4096", "op": "weights", "groups": 1, "rows": 6144, "cols": 4096, "wide": False},
        {"name": "weights 24 x 1520 x 1008", "op": "weights", "groups": 24, "rows": 1520, "cols": 1008, "wide": True},
        # products of a decode step: one token through a small layer, 64 through a wide gate and up projection, where the weights' way counts
        {"name": "product decode 1", "op": "product", "tokens": 1, "cols": 1024, "depth": 2048, "wide": False},
        {"name": "product decode 64", "op": "product", "tokens": 64, "cols": 24576, "depth": 4096, "wide": False},
        # a short prompt of odd length with fp32 results, and a long prompt batch, where the tensor cores count
        {"name": "product prefill 333", "op": "product", "tokens": 333, "cols": 4096, "depth": 2560, "wide": True},
        {"name": "product prefill 8192", "op": "product", "tokens": 8192, "cols": 24576, "depth": 4096, "wide": False},
        # gate and up projection of routed experts, decode step and prompt batch: ragged groups, some of them empty
        {"name": "experts decode 64", "op": "experts", "tokens": 64, "experts": 24, "top": 2, "cols": 1536, "depth": 2048, "wide": False},
        {"name": "experts prefill 4000", "op": "experts", "tokens": 4000, "experts": 16, "top": 2, "cols": 4096, "depth": 2048, "wide": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """A multiple of 16, most of them no multiple of 128."""
    return 16 * _log(rng, lo // 16, hi // 16)


def draw(rng):
    op = rng.choice(["norm", "rows", "weights", "product", "product", "experts"])
    wide = rng.random() < 0.3
    if op == "norm":
        width = rng.choice([1024, 2048, 2560, 4096, _width(rng, 256, 8192)])
        return {"op": op, "tokens": _log(rng, 1, min(16000, 65536000 // width)), "width": width, "wide": wide, "residual": rng.random() < 0.8,
                "plain": rng.random() < 0.4}
    if op == "rows":
        routed = rng.random() < 0.4
        width = rng.choice([768, 1536, 2048, 6144, 12288, _width(rng, 256, 12288)])
        tokens = _log(rng, 1, min(8191, 50000000 // width) // (4 if routed else 1) // (2 if wide else 1))
        return {"op": op, "tokens": tokens, "width": width, "act": rng.choice(["none", "silu"]), "wide": wide, "experts": rng.choice([8, 16, 24]) if routed else 0,
                "top": rng.choice([1, 2, 3]) if routed else 0}
    if op == "weights":
        groups = rng.choice([1, 1, 8, 16])
        rows, cols = _width(rng, 256, 12288 if groups == 1 else 2048), _width(rng, 256, 4096 if groups == 1 else 2048)
        return {"op": op, "groups": groups, "rows": rows, "cols": cols, "wide": wide}
    if op == "product":
        cols, depth = rng.choice([(4096, 1024), (6144, 4096), (24576, 4096), (1024, 2048), (19456, 2560), (_width(rng, 128, 8192), _width(rng, 128, 8192))])
        most = max(1, int(8192 * 24576 * 4096 // (cols * depth)))
        return {"op": op, "tokens": _log(rng, 1, 200) if rng.random() < 0.5 else _log(rng, 200, min(8192, most)), "cols": cols, "depth": depth, "wide": wide}
    return {"op": op, "tokens": _log(rng, 1, 256) if rng.random() < 0.5 else _log(rng, 257, 4000), "experts": rng.choice([8, 16, 24]), "top": rng.choice([1, 2, 3]),
            "cols": rng.choice([1536, 2048, _width(rng, 256, 4096)]), "depth": rng.choice([768, 1024, 2048, _width(rng, 256, 2048)]), "wide": wide}


# ------------------------------------------------------------------------------------------ inputs
class _Rand:
    def __init__(self, seed):
        self.g = torch.Generator(device=DEV).manual_seed(int(seed))

    def __call__(self, *shape, scale=1.0, mean=0.0, dtype=F32):
        return torch.randn(*shape, generator=self.g, device=DEV, dtype=F32).mul_(scale).add_(mean).to(dtype)

    def rows(self, n, width, dtype=F32):
        """Activations: a few channels stand far out, and rows differ in size."""
        t = self(n, width)
        t *= torch.exp(self(1, width, scale=0.7))
        t *= torch.exp(self(n, 1, scale=0.5))
        return t.to(dtype)


def _blocks(x):
    """[..., K] -> [..., blocks of 128, 128], zeros behind the last number."""
    k = x.shape[-1]
    x = torch.nn.functional.pad(x, (0, -k % 128))
    return x.view(*x.shape[:-1], -1, 128)


def _rows_8bit(x):
    """fp32 rows -> (e4m3 rows, scales)."""
    b = _blocks(x)
    s = (b.abs().amax(-1) / TOP).clamp_min(LEAST)
    q = (b * (1.0 / s)[..., None]).to(E4M3).flatten(-2)[..., :x.shape[-1]]
    return q.contiguous(), s


def _weights_8bit(w):
    """[groups, N, K] fp32 -> (e4m3, scales [groups, ceil(N / 128), ceil(K / 128)])."""
    g, n, k = w.shape
    t = torch.nn.functional.pad(w, (0, -k % 128, 0, -n % 128)).view(g, -(-n // 128), 128, -(-k // 128), 128)
    s = (t.abs().amax((2, 4)) / TOP).clamp_min(LEAST)
    q = (t * (1.0 / s)[:, :, None, :, None]).to(E4M3).reshape(g, -n % 128 + n, -k % 128 + k)[:, :n, :k]
    return q.contiguous(), s


def _groups(rand, case):
    """Tokens' experts -> the layout whose groups start at multiples of 128 rows: each row's token (-1: padding), rows in use, the expert of each 128 rows (-1: none)."""
    n, e, top = case["tokens"], case["experts"], case["top"]
    score = rand(n, e) + rand(1, e, scale=1.5)                        # experts are not equally liked: some of few tokens' get none
    idx = score.topk(top, 1).indices
    tiles = (n * top + e * 127 + 127) // 128
    count = torch.bincount(idx.flatten(), minlength=e)
    padded = (count + 127) // 128 * 128
    end = padded.cumsum(0)
    order = torch.argsort(idx.flatten(), stable=True)
    of = idx.flatten()[order]
    place = (end - padded)[of] + torch.arange(n * top, device=DEV) - (count.cumsum(0) - count)[of]
    src = torch.full((tiles * 128,), -1, dtype=torch.int32, device=DEV)
    src[place] = (order // top).to(torch.int32)
    first = torch.arange(tiles, device=DEV) * 128
    group = torch.searchsorted(end, first, right=True)
    group = torch.where(first < end[-1], group, torch.full_like(group, -1)).to(torch.int32)
    return src, end[-1:].to(torch.int32), group


def prepare(case, seed):
    rand, op = _Rand(seed), case["op"]
    wide = F32 if case["wide"] else BF16
    s = {"case": case}
    if op == "norm":
        n, h = case["tokens"], case["width"]
        s.update(x=rand.rows(n, h, wide), w=rand(h, scale=0.2, mean=1.0, dtype=BF16))
        if case["residual"]:
            s.update(residual=rand.rows(n, h), residual_out=torch.empty(n, h, dtype=F32, device=DEV))
    elif op == "rows":
        n, h = case["tokens"], case["width"]
        s.update(x=rand.rows(n, 2 * h if case["act"] == "silu" else h, wide), rows=None, num_rows=None)
        m = n
        if case["experts"]:
            s["rows"], s["num_rows"], _ = _groups(rand, case)
            m = s["rows"].numel()
        # what is behind the rows in use stays as it is
        s.update(q=torch.zeros(m, h, dtype=torch.uint8, device=DEV).view(E4M3), scale=torch.zeros(m, -(-h // 128), dtype=F32, device=DEV))
    elif op == "weights":
        s.update(w=rand(case["groups"], case["rows"], case["cols"], scale=case["cols"] ** -0.5, dtype=wide))
    else:
        k, n, groups = case["depth"], case["cols"], case.get("experts", 1)
        s["wq"], s["ws"] = _weights_8bit(rand(groups, n, k, scale=k ** -0.5))
        x = rand.rows(case["tokens"], k)
        if op == "experts":
            src, _, s["group"] = _groups(rand, case)
            x = torch.where(src[:, None] < 0, torch.zeros((), device=DEV), x[src.clamp_min(0)])
        s["q"], s["scale"] = _rows_8bit(x)
        if op == "product":
            s["wq"], s["ws"] = s["wq"][0], s["ws"][0]
    return s


# ------------------------------------------------------------------------------------------ one pass
def run(s):
    case = s["case"]
    op = case["op"]
    wide = F32 if case["wide"] else BF16
    if own:
        ops, ctx = _framework()
        if op == "norm":
            q, scale, out = ops.add_rmsnorm_fp8(ctx, s["x"], s["w"], EPS, residual=s.get("residual"), residual_out=s.get("residual_out"), want_out=case["plain"])
            return {"q": q, "scale": scale, "out": out, "residual": s.get("residual_out")}
        if op == "rows":
            q, scale = ops.quant_fp8(ctx, s["x"], act=ops.ACT_SILU_MUL if case["act"] == "silu" else ops.ACT_NONE, rows=s["rows"], num_rows=s["num_rows"], q=s["q"], scale=s["scale"])
            return {"q": q, "scale": scale}
        if op == "weights":
            q, scale = ops.quant_fp8_weight(ctx, s["w"])
            return {"q": q, "scale": scale}
        if op == "product":
            return ops.gemm_fp8(ctx, s["q"], s["scale"], s["wq"], s["ws"], out_dtype=wide)
        return ops.gemm_fp8_grouped(ctx, s["q"], s["scale"], s["wq"], s["ws"], s["group"], out_dtype=wide)
    if op == "norm":
        v = s["x"].float()
        if "residual" in s:
            v = v + s["residual"]
        y = v * torch.rsqrt(v.square().mean(-1, keepdim=True) + EPS) * s["w"].float()
        q, scale = _rows_8bit(y)
        return {"q": q, "scale": scale, "out": y.to(BF16) if case["plain"] else None, "residual": v if "residual" in s else None}
    if op == "rows":
        x = s["x"].float()
        if case["act"] == "silu":
            h = case["width"]
            x = x[:, :h] * torch.sigmoid(x[:, :h]) * x[:, h:]
        if s["rows"] is None:
            q, scale = _rows_8bit(x)
            return {"q": q, "scale": scale}
        x = torch.where(s["rows"][:, None] < 0, torch.zeros((), device=DEV), x[s["rows"].clamp_min(0)])
        q, scale = _rows_8bit(x)
        used = (torch.arange(x.shape[0], device=DEV) < s["num_rows"])[:, None]
        return {"q": torch.where(used, q.view(torch.uint8), s["q"].view(torch.uint8)).view(E4M3), "scale": torch.where(used, scale, s["scale"])}
    if op == "weights":
        q, scale = _weights_8bit(s["w"].float())
        return {"q": q, "scale": scale}
    k, n = case["depth"], case["cols"]
    a = s["q"].float() * s["scale"].repeat_interleave(128, -1)[:, :k]
    w = s["wq"].float() * s["ws"].repeat_interleave(128, -2)[..., :n, :].repeat_interleave(128, -1)[..., :k]
    if op == "product":
        return (a @ w.t()).to(wide)
    # rows of tiles that no expert has are zeros
    c = torch.bmm(a.view(-1, 128, k), w[s["group"].clamp_min(0).long()].transpose(1, 2))
    return torch.where(s["group"][:, None, None] < 0, torch.zeros((), device=DEV), c).view(-1, n).to(wide)


# ------------------------------------------------------------------------------------------ what it cannot do without
def work(case):
    op = case["op"]
    if op in ("norm", "rows"):
        n, h, size = case["tokens"], case["width"], 4 if case["wide"] else 2
        if op == "norm":
            b = n * h * (size + 1 + (8 if case["residual"] else 0) + (2 if case["plain"] else 0)) + 2 * h
            return {"bytes": b + 4 * n * -(-h // 128), "flops": 6 * n * h}
        m = n * max(case["top"], 1)                                    # each row read once, written once for each of its experts
        return {"bytes": n * h * size * (2 if case["act"] == "silu" else 1) + m * (h + 4 * -(-h // 128)), "flops": (10 if case["act"] == "silu" else 4) * m * h}
    if op == "weights":
        g, n, k = case["groups"], case["rows"], case["cols"]
        return {"bytes": g * (n * k * ((4 if case["wide"] else 2) + 1) + 4 * -(-n // 128) * -(-k // 128)), "flops": 3 * g * n * k}
    n, k, size = case["cols"], case["depth"], 4 if case["wide"] else 2
    m, groups = case["tokens"] * case.get("top", 1), min(case.get("experts", 1), case["tokens"] * case.get("top", 1))
    return {"bytes": m * (k + 4 * -(-k // 128)) + groups * (n * k + 4 * -(-n // 128) * -(-k // 128)) + m * n * size, "flops": 2 * m * n * k}


# ------------------------------------------------------------------------------------------ the same from the definition, in 64 bits
def _scales64(v, across):
    return torch.clamp(v.abs().amax(dim=across, keepdim=True) / 448, min=2.0 ** -126)


def _quotients64(y):
    """What the 8-bit numbers of rows stand for before they are rounded, and the scales: a column block at a time."""
    q, s = torch.empty_like(y), []
    for at in range(0, y.shape[1], 128):
        part = y[:, at:at + 128]
        s.append(_scales64(part, 1))
        q[:, at:at + 128] = part / s[-1]
    return q, torch.cat(s, 1)


def exact(case, seed):
    """The 8-bit numbers have the quotients in front of their rounding as their values, and so do bf16 results."""
    s, op = prepare(case, seed), case["op"]
    if op == "norm":
        v = s["x"].to(F64)
        if case["residual"]:
            v += s["residual"].to(F64)
        y = v / torch.sqrt((v * v).sum(1, keepdim=True) / v.shape[1] + EPS) * s["w"].to(F64)
        q, scale = _quotients64(y)
        return {"q": q, "scale": scale, "out": y if case["plain"] else None, "residual": v if case["residual"] else None}
    if op == "rows":
        x = s["x"].to(F64)
        if case["act"] == "silu":
            gate, up = x.chunk(2, 1)
            x = gate / (1 + torch.exp(-gate)) * up
        q, scale = _quotients64(x)
        if s["rows"] is not None:
            # a row of padding is a row of zeros
            used, of = int(s["num_rows"]), s["rows"].long()
            all_q, all_s = torch.zeros(of.numel(), q.shape[1], dtype=F64, device=DEV), torch.zeros(of.numel(), scale.shape[1], dtype=F64, device=DEV)
            all_s[:used] = 2.0 ** -126
            there = of >= 0
            all_q[there], all_s[there] = q[of[there]], scale[of[there]]
            q, scale = all_q, all_s
        return {"q": q, "scale": scale}
    if op == "weights":
        w = s["w"].to(F64)
        g, n, k = w.shape
        q, scale = torch.empty_like(w), torch.empty(g, -(-n // 128), -(-k // 128), dtype=F64, device=DEV)
        for i in range(scale.shape[1]):
            for j in range(scale.shape[2]):
                part = w[:, 128 * i:128 * i + 128, 128 * j:128 * j + 128]
                t = _scales64(part, (1, 2))
                q[:, 128 * i:128 * i + 128, 128 * j:128 * j + 128] = part / t
                scale[:, i, j] = t[:, 0, 0]
        return {"q": q, "scale": scale}
    a, wq, ws = s["q"].to(F64), s["wq"], s["ws"]
    for j in range(s["scale"].shape[1]):
        a[:, 128 * j:128 * j + 128] *= s["scale"][:, j:j + 1].to(F64)

    def weights(q, t):
        w = q.to(F64)
        for i in range(t.shape[0]):
            for j in range(t.shape[1]):
                w[128 * i:128 * i + 128, 128 * j:128 * j + 128] *= t[i, j].to(F64)
        return w

    if op == "product":
        return a @ weights(wq, ws).T
    c = torch.zeros(a.shape[0], case["cols"], dtype=F64, device=DEV)
    for e in range(case["experts"]):
        tiles = torch.nonzero(s["group"] == e).flatten().tolist()
        if tiles:
            w = weights(wq[e], ws[e])
            c[128 * tiles[0]:128 * (tiles[-1] + 1)] = a[128 * tiles[0]:128 * (tiles[-1] + 1)] @ w.T
    return c
