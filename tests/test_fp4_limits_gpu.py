"""The largest scores that the 4-bit attention documents (2^22 in magnitude): a row is the value of its one key."""
import pytest
import torch

import test_fp4_lists_gpu as T

pytestmark = pytest.mark.gpu
F64, DEV = torch.float64, "cuda:0"


@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("lens,new,nh,kv,bs,room", [([300, 77, 2000], [1, 1, 1], 8, 2, 16, 8192), ([300, 77, 2000], [1, 1, 1], 16, 8, 256, 16), ([700, 90], [5, 3], 8, 2, 48, 8192),
                                                    ([700, 90], [100, 90], 8, 2, 16, 8192), ([330], [330], 4, 1, 16, 16), ([3000, 1500], [400, 37], 16, 2, 256, 8192)])
def test_rows_of_one_key(ctx, lens, new, nh, kv, bs, room, sign):
    """Where the largest score is further from the next than their roundings (132 of 2^-24 of the sum of magnitudes, each) and 40, all other weights are below 2^-40: the value, exact in bf16."""
    c = T._case(ctx, lens, new, nh, kv, bs, 11, room=room)
    scale = sign * 128 ** -0.5
    at = done = 0
    rows = T.ops.read_kvcache_fp4(ctx, c["cache"], c["slots"])
    k, v = ((a.to(F64).unflatten(-1, (8, 16)) * s.to(F64)[..., None]).flatten(-2) for a, s in (rows[:2], rows[2:]))
    tops, checks = [], []
    for m, n in zip(lens, new):
        q = c["q"][done:done + n].to(F64).view(n, kv, nh // kv, 128)
        s = torch.einsum("nhgd,mhd->nhgm", q, k[at:at + m]) * scale
        size = (torch.einsum("nhgd,mhd->nhgm", q.abs(), k[at:at + m].abs()) * abs(scale)).amax(-1)
        sees = torch.arange(m - n, m, device=DEV)[:, None] >= torch.arange(m, device=DEV)
        s = s.masked_fill(~sees[:, None, None], -float("inf"))
        tops.append(float(s[torch.isfinite(s)].abs().max()))
        checks.append((s, size, v[at:at + m], done))
        at, done = at + m, done + n
    times = 2.0 ** int(torch.log2(torch.tensor(2.0 ** 22 / max(tops))).floor())                    # exact in bf16
    c["q"] = (c["q"].float() * times).to(torch.bfloat16)
    if max(new) == 1:
        got = T.ops.paged_decode_attn_fp4(ctx, c["q"], c["cache"], c["tables"], c["lens"], nh, scale)
    else:
        got = T.ops.prefill_attn_paged_fp4(ctx, c["q"], c["cache"], c["tables"], c["lens"], c["cu"], max(new), nh, scale)
    assert bool(torch.isfinite(got).all())
    for s, size, values, first in checks:
        n, group = s.shape[0], nh // kv
        best = torch.topk(s, min(2, s.shape[-1]), -1)
        gap = (best.values[..., 0] - best.values[..., -1]) if s.shape[-1] > 1 else torch.full(s.shape[:-1], float("inf"), dtype=F64, device=DEV)
        clear = gap * times > 2 * 132 * 2.0 ** -24 * size * times + 40
        assert float(clear.double().mean()) > 0.9
        want = torch.stack([values[best.indices[:, h, :, 0].flatten(), h].view(n, group, 128) for h in range(kv)], 1)
        out = got[first:first + n].to(F64).view(n, kv, group, 128)
        assert torch.equal(out[clear], want[clear])
