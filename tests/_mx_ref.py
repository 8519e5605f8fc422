"""Block-scaled codes from their definition, in 64 bits on the CPU."""
from __future__ import annotations

import torch

GRID = {4: torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64),
        8: torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).to(torch.float64)}


def encode_ref(x: torch.Tensor, bits: int) -> tuple[torch.Tensor, torch.Tensor]:
    """(codes one a byte, scale bytes) of fp32 ``x [..., dim]``: the nearest code by comparison with all of them, on a middle the even
    one; the smallest scale in which the largest magnitude is at most half a step past the largest code."""
    grid = GRID[bits]
    blocks = x.double().unflatten(-1, (-1, 32))
    amax = blocks.abs().amax(-1, keepdim=True)
    fine = torch.isfinite(amax)
    most = grid[-1] + (grid[-1] - grid[-2]) / 2
    powers = torch.exp2(torch.arange(-126.0, 128.0, dtype=torch.float64))  # bytes 1 .. 254
    byte = 1 + torch.searchsorted(powers * most, torch.where(fine, amax, 0.0))
    y = torch.where(fine, blocks, 0.0) * torch.exp2(127.0 - byte.double())
    middle = (grid[1:] + grid[:-1]) / 2
    up, down = torch.searchsorted(middle, y.abs(), right=True), torch.searchsorted(middle, y.abs(), right=False)
    code = torch.where(up % 2 == 0, up, down) + (8 if bits == 4 else 128) * torch.signbit(y).long()
    return code.flatten(-2), torch.where(fine, byte, 255).squeeze(-1)


def decode_ref(codes: torch.Tensor, scales: torch.Tensor, bits: int) -> torch.Tensor:
    """fp64 values of packed codes ``[..., bytes]`` and scale bytes ``[..., blocks]``."""
    codes, scales = codes.cpu(), scales.cpu()
    one = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).long() if bits == 4 else codes.long()
    sign, index = (one >> (bits - 1)) & 1, one & ((1 << (bits - 1)) - 1)
    grid = torch.cat((GRID[bits], torch.tensor([float("nan")], dtype=torch.float64)))
    v = grid[index.clamp(max=grid.numel() - 1)] * (1 - 2 * sign)
    s = torch.where(scales == 255, float("nan"), torch.exp2(scales.double() - 127))
    return (v.unflatten(-1, (-1, 32)) * s.unsqueeze(-1)).flatten(-2)


def pack_ref(codes: torch.Tensor, bits: int) -> torch.Tensor:
    if bits == 8:
        return codes.to(torch.uint8)
    pair = codes.unflatten(-1, (-1, 2))
    return (pair[..., 0] + 16 * pair[..., 1]).to(torch.uint8)


def rotate_axes_ref(x, positions, table, sections, interleaved):
    """x [T, heads, dim] in fp64 with its first rot columns turned, pair by pair; positions [axes, T]; outside the table NaN."""
    x, table = x.cpu().double().clone(), table.cpu().double()
    half = table.shape[1] // 2
    axis = torch.repeat_interleave(torch.arange(len(sections)), torch.tensor(sections))
    for i in range(half):
        pos = positions[axis[i]].long()
        inside = (pos >= 0) & (pos < table.shape[0])
        at = pos.clamp(0, table.shape[0] - 1)
        c, s = (torch.where(inside, table[at, j], float("nan")).view(-1, 1) for j in (i, half + i))
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
        u, w = x[:, :, a].clone(), x[:, :, b].clone()
        x[:, :, a], x[:, :, b] = u * c - w * s, w * c + u * s
    return x


def capped_attention_ref(q, k, v, present, seq_lens, starts, scale, softcap, window):
    """(out, lse, sum of p |v|) in fp64 of ``q [T, heads, dim]`` over ``k``, ``v`` (fp64, a [key heads, n, dim] for each sequence) and
    ``present`` (which of the n tokens are there): a token sees the last ``window`` of its sequence's up to itself."""
    q = q.cpu().double()
    t, h, d = q.shape
    out, mag = torch.zeros(t, h, d, dtype=torch.float64), torch.zeros(t, h, d, dtype=torch.float64)
    lse = torch.full((t, h), -float("inf"), dtype=torch.float64)
    for b, n in enumerate(seq_lens):
        a, c = starts[b], starts[b + 1]
        if n == 0 or a == c:
            continue
        at = n - (c - a) + torch.arange(c - a).view(-1, 1)
        j = torch.arange(n)
        sees = (j <= at) & (j > at - window) if window else j <= at
        sees = sees & present[b]
        some = sees.any(1)
        group = h // k[b].shape[0]
        for head in range(h):
            kk, vv = (torch.where(present[b].view(-1, 1), x[b][head // group], 0.0) for x in (k, v))
            s = q[a:c, head] @ kk.t() * scale
            s = softcap * torch.tanh(s / softcap) if softcap else s
            s = s.masked_fill(~sees, -float("inf"))[some]
            z = torch.logsumexp(s, 1)
            p = torch.exp(s - z.view(-1, 1))
            rows = torch.nonzero(some).flatten() + a
            lse[rows, head], out[rows, head], mag[rows, head] = z, p @ vv, p @ vv.abs()
    return out, lse, mag
