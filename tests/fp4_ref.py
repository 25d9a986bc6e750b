"""The 4-bit cache from its definition, in 64 bits, for the tests: rows to codes and scales, a cache to its numbers, attention over it."""
import math

import torch

F64 = torch.float64
MAGNITUDES = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=F64)
SCALES = torch.tensor([m / 8 * 2.0 ** -14 for m in range(8)] + [(1 + m / 8) * 2.0 ** (e - 15) for e in range(1, 32) for m in range(8)], dtype=F64)[:227]     # 0 .. 10240


def nearest(x, values, even):
    """Index of the nearest of ascending values; half way: the even index, or the lower one."""
    hi = torch.searchsorted(values, x.contiguous()).clamp(1, len(values) - 1)
    up, down = values[hi] - x, x - values[hi - 1]
    return torch.where((up < down) | ((up == down) & (hi % 2 == 0) & torch.tensor(even)), hi, hi - 1)


def to_fp4(x):
    """[..., 128] -> (numbers of the codes [..., 128] in 64 bits, scale bytes [..., 8]); a block with an infinity or a NaN: zeros and 255."""
    b = x.cpu().to(F64).unflatten(-1, (8, 16))
    bad = ~torch.isfinite(b).all(-1)
    b = torch.where(bad[..., None], torch.zeros((), dtype=F64), b)
    byte = nearest(b.abs().amax(-1) / 6, SCALES, True)
    s = SCALES[byte]
    q = b.abs() / torch.where(s > 0, s, torch.ones((), dtype=F64))[..., None]
    c = MAGNITUDES[nearest(q, MAGNITUDES, False)]
    c = torch.where((s > 0)[..., None], c, torch.zeros((), dtype=F64)) * torch.sign(b)
    return c.flatten(-2), torch.where(bad, torch.full_like(byte, 255), byte)


def numbers(codes, scales):
    """uint8 [..., 64], [..., 8] -> what they stand for, [..., 128] in 64 bits."""
    codes, scales = codes.cpu(), scales.cpu()
    c = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).long()
    v = MAGNITUDES[c & 7] * torch.where(c >= 8, -1.0, 1.0)
    table = torch.full((256,), math.nan, dtype=F64)
    table[:227] = SCALES
    return (v.unflatten(-1, (8, 16)) * table[scales.long()][..., None]).flatten(-2)


def context(cache, table, n, kvh):
    """A sequence's n cached keys and values of one key head; pages outside the pool are zeros."""
    bs, out = cache.block_size, []
    for codes, scales in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        rows = []
        for i in range(-(-n // bs)):
            blk = int(table[i])
            rows.append(numbers(codes[blk, kvh], scales[blk, kvh]) if 0 <= blk < cache.num_blocks else torch.zeros(bs, 128, dtype=F64))
        out.append(torch.cat(rows)[:n] if rows else torch.zeros(0, 128, dtype=F64))
    return out


def attention(q, cache, tables, lens, new, scale, nh):
    """(outputs [rows, nh, 128], how far each may be off), all in 64 bits.  new: rows of each sequence, the last positions of its context.

    What the kernels round: a key's weight to fp16 (2^-11 of it; the sum takes it unrounded), the query to fp16 behind a power of two that brings its largest number to [1, 2) (2^-11 of a
    number at least 2^-14 of the largest has no effect on bf16's 8 bits; a smaller one is off by 2^-25 of the largest), scores and sums in fp32 (2^-24 per product of 128 and per addition),
    the exponential (2^-22), and the result to bf16 (2^-8).  Weights below 2^-31 of the largest may vanish: of n keys, n * 2^-31 of the weight."""
    q = q.cpu().to(F64).view(q.shape[0], nh, 128)
    out, far = torch.zeros_like(q), torch.zeros_like(q)
    group, at = nh // cache.kv, 0
    for b, (n, c) in enumerate(zip(new, lens)):
        c = min(max(c, 0), tables.shape[1] * cache.block_size)
        for h in range(cache.kv):
            k, v = context(cache, tables[b].tolist(), c, h)
            for i in range(n):
                m = max(0, c - n + i + 1)
                if not m:
                    continue
                r = q[at + i, h * group:(h + 1) * group]
                p = torch.softmax(r @ k[:m].T * scale, -1)
                size = (r.abs() @ k[:m].abs().T * abs(scale)).amax(-1, keepdim=True)
                tiny = r.abs().amax(-1, keepdim=True) * 2.0 ** -25 * k[:m].abs().sum(-1).amax() * abs(scale)
                o, a = p @ v[:m], p @ v[:m].abs()
                weight = 2.0 ** -11 + 2 * (size * 132 * 2.0 ** -24 + tiny + 2.0 ** -20) + m * 2.0 ** -31
                # (m + 64) roundings of the sums over the keys, most of them of partial sums: m / 16 tiles of 16
                weight = weight + (m / 16 + 64) * 2.0 ** -24
                out[at + i, h * group:(h + 1) * group] = o
                far[at + i, h * group:(h + 1) * group] = 2.0 ** -8 * o.abs() + weight * a + m * 2.0 ** -31 * v[:m].abs().amax()
        at += n
    return out, far
