"""Plain restatement of the 4-bit KV cache and the request maps (CPU, no product code).

A pool is uint8 [num_blocks][kv_heads][block_size / 64][4608]: 64 tokens x 128
dims in 4-bit codes, then 64 x 4 bf16 scales.  32 consecutive dims share the
scale s = bf16(max|x| / 7); n = clamp(rint(x / s), -7, 7); the code is n + 8.
A group with a non-finite member has a NaN scale and codes of 8.
"""
from __future__ import annotations

import numpy as np
import torch

TILE, D, RECORD = 64, 128, 4608


def quantise(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """bf16 [..., 128] -> (n int64 [..., 128], scale bf16 [..., 4]), decided in 64 bits."""
    g = x.double().reshape(*x.shape[:-1], 4, 32)
    finite = torch.isfinite(g).all(-1)
    g = torch.where(finite[..., None], g, 0.0)
    s = (g.abs().amax(-1) / 7).to(torch.bfloat16)
    sd = s.double()[..., None]
    n = torch.where(sd > 0, torch.round(g / torch.where(sd > 0, sd, 1.0)).clamp(-7, 7), 0.0)
    s = torch.where(finite, s, torch.tensor(float("nan"), dtype=torch.bfloat16))
    return n.long().reshape(x.shape), s


def nibble_places(value: bool) -> np.ndarray:
    """[64, 128] place (in nibbles) of every (token, dim) in a record, spelled out."""
    at = np.empty((TILE, D), dtype=np.int64)
    for t in range(TILE):
        for d in range(D):
            if value:
                r, j, g = t % 16, d // 16, (d % 16) // 2
                byte = 1024 * (t // 16) + 512 * (r // 8) + 16 * ((r % 8) // 2) + 8 * (r % 2) + 64 * g + j
                at[t, d] = 2 * byte + d % 2
            else:
                w, c, e = d // 32, (d % 32) // 8, d % 8
                at[t, d] = 2 * (64 * t + 16 * c + 4 * w) + e // 2 + 4 * (e % 2)
    return at


_PLACES = {v: torch.from_numpy(nibble_places(v)) for v in (False, True)}


def pack(x: torch.Tensor, value: bool) -> torch.Tensor:
    """bf16 [..., 64, 128] -> uint8 [..., 4608] records."""
    n, s = quantise(x)
    u = torch.zeros(*x.shape[:-2], 2 * 4096, dtype=torch.uint8)
    u[..., _PLACES[value].flatten()] = (n + 8).to(torch.uint8).flatten(-2)
    codes = u[..., 0::2] | (u[..., 1::2] << 4)
    return torch.cat([codes, s.contiguous().view(torch.uint8).flatten(-2)], -1)


def unpack(rec: torch.Tensor, value: bool) -> torch.Tensor:
    """uint8 [..., 4608] -> float64 [..., 64, 128]."""
    u = torch.stack([rec[..., :4096] & 15, rec[..., :4096] >> 4], -1).flatten(-2)
    n = u[..., _PLACES[value].flatten()].double() - 8
    s = rec[..., 4096:].contiguous().view(torch.bfloat16).double()  # 64 x 4
    return (n.reshape(*rec.shape[:-1], TILE, 4, 32) * s.reshape(*rec.shape[:-1], TILE, 4, 1)).flatten(-2)


def pool_rows(pool: torch.Tensor, value: bool) -> torch.Tensor:
    """A pool as float64 [num_slots, kv_heads, 128] in flat slot order."""
    x = unpack(pool, value)  # [nb, H, tiles, 64, 128]
    return x.permute(0, 2, 3, 1, 4).flatten(0, 2)


def pool_from_rows(x: torch.Tensor, block_size: int, value: bool) -> torch.Tensor:
    """bf16 [num_slots, kv_heads, 128] in flat slot order -> pool."""
    y = x.reshape(-1, block_size // TILE, TILE, x.shape[1], D).permute(0, 3, 1, 2, 4)
    return pack(y, value)


def attend(q, k, v, scale: float):
    """q [Hq, 128], k/v float64 [n, Hkv, 128] -> (out, sum p|v|, logit reach, sum p s) in float64.

    The third is scale * max_t sum_groups s_g * sum|q_g|, what a logit is summed from per unit of code; the
    fourth has the V scale s of each dim's group.  s is taken as max|x| / 7: a group's largest code is 7."""
    G = q.shape[0] // k.shape[1]
    kk, vv = k.repeat_interleave(G, 1), v.repeat_interleave(G, 1)
    x = torch.einsum("hd,nhd->hn", q.double(), kk) * scale
    p = torch.softmax(x, -1)

    def group_scale(y):
        return y.abs().reshape(y.shape[0], y.shape[1], 4, 32).amax(-1) / 7
    qa = q.double().abs().reshape(-1, 4, 32).sum(-1)
    reach = abs(scale) * (group_scale(kk) * qa).sum(-1).amax(0)
    ps = torch.einsum("hn,nhg->hg", p, group_scale(vv)).repeat_interleave(32, -1)
    return torch.einsum("hn,nhd->hd", p, vv), torch.einsum("hn,nhd->hd", p, vv.abs()), reach, ps


def block_tables(lengths, block_size, max_blocks, free):
    """([S][max_blocks] int32, blocks used) by walking the list."""
    out, it = np.full((len(lengths), max_blocks), -1, dtype=np.int32), 0
    for i, n in enumerate(lengths):
        need = min(max(0, -(-int(n) // block_size)), max_blocks)
        for j in range(need):
            out[i, j] = free[it] if it < len(free) else -1
            it += 1
    return out, it


def slot_maps(lengths, starts, rows, tables, block_size, num_tokens):
    """(cu, positions, slots) by walking the tokens."""
    cu, pos, slots = [0], [], []
    for i, n in enumerate(lengths):
        for p in range(int(starts[i]), int(starts[i]) + max(0, int(n))):
            pos.append(p)
            r = int(rows[i])
            slots.append(-1 if r < 0 else int(tables[r][p // block_size]) * block_size + p % block_size)
        cu.append(len(pos))
    pad = num_tokens - len(pos)
    return np.array(cu), np.array(pos + [0] * pad), np.array(slots + [-1] * pad)
