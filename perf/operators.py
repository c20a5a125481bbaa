"""Workloads of the 4-bit paged KV cache: storing into it, loading from it, decode attention over it, and the
block tables and slot maps that address it.

A pool holds K or V of one layer as uint8 [num_blocks][kv_heads][block_size / 64][4608]: per 64 tokens and kv
head 4096 bytes of 4-bit codes, then 64 x 4 bf16 scales (one per 32 dims).  A code u stands for (u - 8) * scale.
"""
import math

import torch

own = False

D = 128          # head dim
GROUP = 32       # dims that share a scale
TILE = 64        # tokens of one tile record
CODES = TILE * D // 2
RECORD = CODES + TILE * (D // GROUP) * 2
WORKSPACE = 32 << 20  # split partials of the decode attention (bytes, zero-filled)


# ---------------------------------------------------------------- cases
def listed():
    return [
        # block tables of a handful of new requests, in a pool of the default block size
        {"name": "tables 8 requests", "kind": "tables", "S": 8, "lo": 1, "hi": 2048, "MB": 9, "bs": 256},
        # ... and of many requests with tables as wide as the longest context (40960 tokens)
        {"name": "tables 2048 requests", "kind": "tables", "S": 2048, "lo": 0, "hi": 40960, "MB": 161, "bs": 256},
        # slot maps of two prompts that continue a cached context
        {"name": "slots 2 prompts", "kind": "slots", "S": 2, "lo": 100, "hi": 700, "start": 500, "bs": 256, "pad": 0},
        # slot maps of a full prefill chunk: 256 prompts of about 1024 tokens, the token count padded
        {"name": "slots 256 prompts", "kind": "slots", "S": 256, "lo": 1, "hi": 2047, "start": 0, "bs": 256, "pad": 129},
        # the new token of each of 32 decode rows goes into the cache (and is read back)
        {"name": "store 32 rows", "kind": "store", "T": 32, "hkv": 8, "bs": 256, "run": 1, "strided": False},
        # one prefill chunk goes into the cache (and is read back)
        {"name": "store chunk 32768", "kind": "store", "T": 32768, "hkv": 8, "bs": 256, "run": 1024, "strided": True},
        # the cached context of one request for a prefill that continues it
        {"name": "load one context", "kind": "load", "S": 1, "lo": 1000, "hi": 1000, "hkv": 8, "bs": 256},
        # the contexts of a whole prefill batch
        {"name": "load 64 contexts", "kind": "load", "S": 64, "lo": 1, "hi": 1500, "hkv": 8, "bs": 256},
        # decode attention, latency: one short conversation
        {"name": "attend 1 x 333", "kind": "attend", "B": 1, "lo": 333, "hi": 333, "hq": 16, "hkv": 8, "bs": 256, "pad": 0},
        # one request at the longest context
        {"name": "attend 1 x 40960", "kind": "attend", "B": 1, "lo": 40960, "hi": 40960, "hq": 32, "hkv": 8, "bs": 256,
         "pad": 0},
        # a bucketed batch with padding rows and 8 query heads per kv head
        {"name": "attend 40 ragged", "kind": "attend", "B": 40, "lo": 1, "hi": 3001, "hq": 64, "hkv": 8, "bs": 256,
         "pad": 3},
        # the framework's decode-attention benchmark: 256 rows, contexts 512 to 4096
        {"name": "attend 256 rows", "kind": "attend", "B": 256, "lo": 512, "hi": 4096, "hq": 16, "hkv": 8, "bs": 256,
         "pad": 0},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["tables", "slots", "store", "load", "attend", "attend", "attend"])
    bs = rng.choice([64, 128, 256])
    if kind == "tables":
        hi = _log(rng, 1, 40960)
        return {"kind": kind, "S": _log(rng, 1, 2048), "lo": rng.choice([0, 1, hi // 2]), "hi": hi,
                "MB": -(-hi // 256) + rng.randint(0, 3), "bs": 256}
    if kind == "slots":
        S = _log(rng, 1, 256)
        return {"kind": kind, "S": S, "lo": rng.choice([0, 1]), "hi": _log(rng, 2, max(2, 262144 // S // 2)),
                "start": _log(rng, 1, 4000), "bs": bs, "pad": rng.choice([0, rng.randint(1, 300)])}
    if kind == "store":
        return {"kind": kind, "T": _log(rng, 1, 32768), "hkv": rng.choice([1, 2, 3, 4, 8]), "bs": bs,
                "run": rng.choice([1, _log(rng, 2, 2000)]), "strided": rng.random() < 0.5}
    if kind == "load":
        S = _log(rng, 1, 64)
        hi = _log(rng, 1, 48000 // S)
        return {"kind": kind, "S": S, "lo": rng.choice([1, hi]), "hi": hi, "hkv": rng.choice([1, 2, 3, 4, 8]), "bs": bs}
    B = _log(rng, 1, 256)
    hi = _log(rng, 1, min(40960, 256 * 2304 // B))
    hkv, g = rng.choice([1, 2, 4, 5, 8]), rng.choice([1, 2, 4, 8])
    return {"kind": kind, "B": B, "lo": rng.choice([1, hi // 8 + 1, hi]), "hi": hi, "hq": hkv * g, "hkv": hkv, "bs": bs,
            "pad": rng.randint(0, B // 4)}


# ---------------------------------------------------------------- the stored form, in elementary operations
def _quantise(x):
    """bf16 [..., 128] -> (n int32 [..., 128] in -7..7, scale bf16 [..., 4])."""
    xg = x.float().unflatten(-1, (D // GROUP, GROUP))
    amax = xg.abs().amax(-1, keepdim=True)
    scale = (amax / 7).to(torch.bfloat16)
    s = scale.float()
    n = torch.where(s > 0, torch.round(xg / torch.where(s > 0, s, 1.0)).clamp(-7, 7), 0.0)
    return n.to(torch.int32).flatten(-2), scale.squeeze(-1)


def _k_nibble(t, d):
    """Place (in 4-bit units inside a tile record) of K's token t, dim d."""
    w, c, e = d // 32, d % 32 // 8, d % 8
    return 2 * (64 * t + 4 * (4 * c + w)) + e // 2 + 4 * (e % 2)


def _v_nibble(t, d):
    r, j, g = t % 16, d // 16, d % 16 // 2
    return 2 * (1024 * (t // 16) + 512 * (r // 8) + 8 * (r % 2) + 16 * (r % 8 // 2) + 64 * g + j) + d % 2


def _places(dev, of):
    """int64 [64, 128]: the nibble of every (token, dim) of a tile record."""
    return of(torch.arange(TILE, device=dev)[:, None], torch.arange(D, device=dev)[None, :])


def _pack(n, scale, place):
    """n [..., 64, 128], scale [..., 64, 4] -> uint8 [..., 4608] tile records."""
    u = torch.empty(n.shape[:-2] + (TILE * D,), dtype=torch.uint8, device=n.device)
    u[..., place.flatten()] = (n + 8).to(torch.uint8).flatten(-2)
    u = u.unflatten(-1, (CODES, 2))
    codes = u[..., 0] | (u[..., 1] << 4)
    return torch.cat([codes, scale.contiguous().view(torch.uint8).flatten(-2)], -1)


def _unpack(records, place):
    """uint8 [..., 4608] -> float32 [..., 64, 128], the values that the codes stand for."""
    codes = records[..., :CODES]
    u = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)
    n = u[..., place].float() - 8
    scale = records[..., CODES:].contiguous().view(torch.bfloat16).unflatten(-1, (TILE, D // GROUP)).float()
    return (n.unflatten(-1, (D // GROUP, GROUP)) * scale[..., None]).flatten(-2)


def _put(pool, slots, x, place):
    """Quantise rows x [T, hkv, 128] into a pool's flat slots (-1 skips)."""
    n, scale = _quantise(x)
    keep = slots >= 0
    n, scale, slots = n[keep], scale[keep], slots[keep]
    nb, hkv, tiles, _ = pool.shape
    blk, tile, t = slots // (tiles * TILE), slots % (tiles * TILE) // TILE, slots % TILE
    pl = place[t]  # [T, 128]
    lo = torch.argsort(pl, -1)  # dims in the order of their nibbles: two make a byte
    u = torch.gather((n + 8), -1, lo[:, None, :].expand_as(n)).unflatten(-1, (D // 2, 2))
    byte = torch.gather(pl, -1, lo)[:, 0::2] // 2
    head = torch.arange(hkv, device=x.device)[None, :, None]
    pool[blk[:, None, None], head, tile[:, None, None], byte[:, None, :]] = (u[..., 0] | (u[..., 1] << 4)).to(torch.uint8)
    at = CODES + 8 * t[:, None, None] + torch.arange(8, device=x.device)
    pool[blk[:, None, None], head, tile[:, None, None], at] = scale.contiguous().view(torch.uint8)


def _get(pool, slots, place):
    """float32 [T, hkv, 128] of a pool's flat slots (all >= 0)."""
    nb, hkv, tiles, _ = pool.shape
    blk, tile, t = slots // (tiles * TILE), slots % (tiles * TILE) // TILE, slots % TILE
    head = torch.arange(hkv, device=slots.device)[None, :, None]
    pl = place[t][:, None, :]
    byte = pool[blk[:, None, None], head, tile[:, None, None], pl // 2].int()
    n = ((byte >> (4 * (pl % 2)).int()) & 15).float() - 8
    at = CODES + 8 * t[:, None, None] + torch.arange(8, device=slots.device)
    s = pool[blk[:, None, None], head, tile[:, None, None], at].contiguous().view(torch.bfloat16).float()
    return (n.unflatten(-1, (D // GROUP, GROUP)) * s[..., None]).flatten(-2)


# ---------------------------------------------------------------- inputs
def _rows(gen, T, hkv, dev):
    """K rows with a few strong channels, V rows without: what a cache holds."""
    k = torch.randn((T, hkv, D), generator=gen, device=dev)
    k = k * torch.where(torch.rand((hkv, D), generator=gen, device=dev) < 0.05, 8.0, 1.0)
    v = torch.randn((T, hkv, D), generator=gen, device=dev) * 0.7
    return k.to(torch.bfloat16), v.to(torch.bfloat16)


def _lengths(gen, n, lo, hi):
    """n lengths in lo..hi in a random order, in pairs around the middle: their sum is the same for every seed."""
    x = torch.randint(lo, hi + 1, ((n + 1) // 2,), generator=gen)
    both = torch.stack([x, lo + hi - x], 1).flatten()
    if n % 2:
        both = torch.cat([both[2:], torch.tensor([(lo + hi) // 2])])
    return both[torch.randperm(n, generator=gen)]


def _tables(gen, need, MB, nb, dev):
    """Random distinct blocks of a pool of nb blocks for rows that need `need` blocks each."""
    perm = torch.randperm(nb, generator=gen).to(torch.int32)
    off = torch.cumsum(need, 0) - need
    j = torch.arange(MB)[None]
    idx = (off[:, None] + j).clamp(max=nb - 1)
    return torch.where(j < need[:, None], perm[idx], -1).to(torch.int32).to(dev)


def _flat(lens, starts, tables, bs):
    """Flat slots of tokens start .. start + len of every row, packed (host int64)."""
    seq = torch.repeat_interleave(torch.arange(len(lens)), lens)
    pos = torch.arange(int(lens.sum())) - (torch.cumsum(lens, 0) - lens)[seq] + starts[seq]
    return tables[seq, pos // bs].long() * bs + pos % bs


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator().manual_seed(seed)            # host: lengths and tables
    gpu = torch.Generator(device=dev).manual_seed(seed)  # device: rows
    kind, s = case["kind"], {"case": dict(case)}
    if kind == "tables":
        lens = _lengths(gen, case["S"], case["lo"], case["hi"])
        total = int(((lens + case["bs"] - 1) // case["bs"]).sum())
        s["lengths"] = lens.to(torch.int32).to(dev)
        s["free"] = torch.randperm(total + 17, generator=gen).to(torch.int32).to(dev)
        s["out"] = torch.empty((case["S"], case["MB"]), dtype=torch.int32, device=dev)
        s["used"] = torch.empty(1, dtype=torch.int32, device=dev)
        return s
    if kind == "slots":
        S, bs = case["S"], case["bs"]
        lens = _lengths(gen, S, case["lo"], case["hi"])
        starts = _lengths(gen, S, 0, case["start"])
        need = (lens + starts + bs - 1) // bs
        R = S + 5  # the cache has more rows than the call has requests
        rows = torch.randperm(R, generator=gen)[:S]
        full = torch.zeros(R, dtype=torch.int64)
        full[rows] = need
        MB, nb = int(need.max()) + 1, int(need.sum()) + 9
        T = int(lens.sum()) + case["pad"]
        s.update(lengths=lens.to(torch.int32).to(dev), starts=starts.to(torch.int32).to(dev), rows=rows.to(dev),
                 tables=_tables(gen, full, MB, nb, dev), nb=nb, T=T,
                 cu=torch.empty(S + 1, dtype=torch.int32, device=dev),
                 positions=torch.empty(T, dtype=torch.int64, device=dev),
                 slots=torch.empty(T, dtype=torch.int64, device=dev))
        return s
    if kind == "store":
        T, hkv, bs = case["T"], case["hkv"], case["bs"]
        run_ = case["run"]  # tokens of one sequence that follow one another
        n = -(-T // run_)
        lens = torch.full((n,), run_, dtype=torch.int64)
        lens[-1] = T - run_ * (n - 1)
        starts = _lengths(gen, n, 0, 2 * bs)
        need = (lens + starts + bs - 1) // bs
        nb = int(need.sum()) + 3
        tables = _tables(gen, need, int(need.max()), nb, "cpu")
        slots = _flat(lens, starts, tables, bs)
        slots[T // 2:][::97][:T // 50] = -1  # padding tokens of a bucketed batch
        k, v = _rows(gpu, T, hkv, dev)
        if case["strided"]:  # rows of a fused projection's output
            wide = torch.empty((T, 2 * hkv + 1, D), dtype=torch.bfloat16, device=dev)
            wide[:, :hkv], wide[:, hkv:2 * hkv] = k, v
            k, v = wide[:, :hkv], wide[:, hkv:2 * hkv]
        pool = lambda: torch.zeros((nb, hkv, bs // TILE, RECORD), dtype=torch.uint8, device=dev)  # noqa: E731
        s.update(k=k, v=v, slots=slots.to(dev), kc=pool(), vc=pool(),
                 ko=torch.zeros((T, hkv, D), dtype=torch.bfloat16, device=dev),
                 vo=torch.zeros((T, hkv, D), dtype=torch.bfloat16, device=dev))
    if kind in ("load", "attend"):
        rows_n = case["S"] if kind == "load" else case["B"]
        hkv, bs = case["hkv"], case["bs"]
        lens = _lengths(gen, rows_n, case["lo"], case["hi"])
        need = (lens + bs - 1) // bs
        nb, MB = int(need.sum()) + 3, int(need.max())
        tables = _tables(gen, need, MB, nb, "cpu")
        s.update(kc=torch.zeros((nb, hkv, bs // TILE, RECORD), dtype=torch.uint8, device=dev),
                 vc=torch.zeros((nb, hkv, bs // TILE, RECORD), dtype=torch.uint8, device=dev),
                 tables=tables.to(dev), lens=lens)
        for name, of in (("kc", _k_nibble), ("vc", _v_nibble)):  # a pool filled to the brim, block by block
            place = _places(dev, of)
            for b0 in range(0, nb, 512):
                x = _rows(gpu, min(512, nb - b0) * bs, hkv, dev)[name == "vc"]
                n, scale = _quantise(x.unflatten(0, (-1, bs)).transpose(1, 2).unflatten(2, (bs // TILE, TILE)))
                s[name][b0:b0 + 512] = _pack(n, scale, place)
    if kind == "load":
        MB = -(-case["hi"] // bs)
        src = _flat(lens, torch.zeros_like(lens), tables, bs)
        dst = _flat(lens, torch.zeros_like(lens), torch.arange(rows_n * MB).view(rows_n, MB), bs)
        out = lambda: torch.zeros((rows_n * MB, hkv, bs, D), dtype=torch.bfloat16, device=dev)  # noqa: E731
        s.update(src=src.to(dev), dst=dst.to(dev), ko=out(), vo=out())
    if kind == "attend":
        B = case["B"]
        rows = torch.randperm(B, generator=gen)
        rows[B - case["pad"]:] = -1
        s.update(rows=rows.to(dev), seqlens=(lens - 1).to(torch.int32).to(dev), max_context=MB * bs,
                 q=torch.randn((B, case["hq"], D), generator=gpu, device=dev).to(torch.bfloat16),
                 out=torch.empty((B, case["hq"], D), dtype=torch.bfloat16, device=dev),
                 workspace=torch.zeros(WORKSPACE, dtype=torch.uint8, device=dev), longest=int(lens.max()))
    return s


# ---------------------------------------------------------------- one pass
def run(s):
    if own:
        return _run_own(s)
    kind, bs = s["case"]["kind"], s["case"]["bs"]
    if kind == "tables":
        lens, free, MB = s["lengths"].long(), s["free"], s["case"]["MB"]
        need = (lens + bs - 1) // bs
        off = torch.cumsum(need, 0) - need
        j = torch.arange(MB, device=lens.device)[None]
        table = torch.where(j < need[:, None], free[(off[:, None] + j).clamp(max=free.numel() - 1)], -1)
        return table, need.sum(dtype=torch.int64).to(torch.int32).view(1)
    if kind == "slots":
        lens, starts, T = s["lengths"].long(), s["starts"].long(), s["T"]
        end = torch.cumsum(lens, 0)
        cu = torch.cat([torch.zeros_like(end[:1]), end])
        t = torch.arange(T, device=lens.device)
        seq = torch.searchsorted(end, t, right=True)
        some = seq < lens.numel()
        seq = seq.clamp(max=lens.numel() - 1)
        pos = torch.where(some, t - cu[seq] + starts[seq], 0)
        slot = s["tables"][s["rows"][seq], torch.where(some, pos // bs, 0)].long() * bs + pos % bs
        return cu.to(torch.int32), pos, torch.where(some, slot, -1)
    if kind == "store":
        dev, some = s["k"].device, s["slots"] >= 0
        at, slots = some.nonzero().flatten(), s["slots"][some]
        outs = ()
        for x, pool, out, of in ((s["k"], s["kc"], s["ko"], _k_nibble), (s["v"], s["vc"], s["vo"], _v_nibble)):
            place = _places(dev, of)
            _put(pool, s["slots"], x, place)
            out[at] = _get(pool, slots, place).to(torch.bfloat16)
            outs += (out,)
        return outs
    if kind == "load":
        outs = ()
        for pool, out, of in ((s["kc"], s["ko"], _k_nibble), (s["vc"], s["vo"], _v_nibble)):
            out[s["dst"] // bs, :, s["dst"] % bs] = _get(pool, s["src"], _places(out.device, of)).to(torch.bfloat16)
            outs += (out,)
        return outs
    q, rows = s["q"], s["rows"]
    B, hq, _ = q.shape
    nb, hkv, tiles, _ = s["kc"].shape
    row = rows.clamp(min=0)
    ctx = torch.where(rows >= 0, s["seqlens"][row].long() + 1, 0)
    blocks = s["tables"][row][:, :-(-s["longest"] // bs)].long().clamp(min=0)  # [B, blocks]
    L = blocks.shape[1] * bs
    k = _unpack(s["kc"][blocks].transpose(1, 2), _places(q.device, _k_nibble)).reshape(B, hkv, L, D)
    x = (q.float().view(B, hkv, hq // hkv, D) * D ** -0.5) @ k.transpose(2, 3)
    del k
    x = x.masked_fill((torch.arange(L, device=q.device) >= ctx[:, None])[:, None, None], -math.inf)
    m = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(m > -math.inf, m, 0.0))
    v = _unpack(s["vc"][blocks].transpose(1, 2), _places(q.device, _v_nibble)).reshape(B, hkv, L, D)
    l = p.sum(-1, keepdim=True)
    o = (p @ v) / torch.where(l > 0, l, 1.0)
    return o.view(B, hq, D).to(torch.bfloat16)


def _run_own(s):
    from awesome_acceleration_b200 import kernels as K
    c = s["case"]
    kind, bs = c["kind"], c["bs"]
    if kind == "tables":
        K.build_block_tables(s["lengths"], bs, free_blocks=s["free"], out=s["out"], used=s["used"])
        return s["out"], s["used"]
    if kind == "slots":
        return K.build_slot_maps(s["lengths"], s["tables"], block_size=bs, num_blocks=s["nb"], num_tokens=s["T"],
                                 starts=s["starts"], rows=s["rows"], cu=s["cu"], positions=s["positions"],
                                 slots=s["slots"])
    if kind == "store":
        K.kv4_store(s["k"], s["v"], s["slots"], s["kc"], s["vc"])
        K.kv4_load(s["kc"], s["vc"], s["slots"], s["ko"], s["vo"])
        return s["ko"], s["vo"]
    if kind == "load":
        K.kv4_load(s["kc"], s["vc"], s["src"], s["ko"], s["vo"], out_slots=s["dst"])
        return s["ko"], s["vo"]
    return K.kv4_decode_attention(s["q"], s["kc"], s["vc"], s["tables"], s["rows"], s["seqlens"], ctx_add=1,
                                  scale=D ** -0.5, max_context=s["max_context"], workspace=s["workspace"],
                                  out=s["out"])


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    kind, row = case["kind"], 2 * (D // 2 + 2 * D // GROUP)  # packed K + V bytes of a (token, kv head)
    if kind == "tables":
        return {"bytes": 4 * case["S"] * (2 + case["MB"]) + 4 * case["S"] * (case["lo"] + case["hi"]) // 2 // case["bs"],
                "flops": 0}
    mean = (case["lo"] + case["hi"]) / 2 if "lo" in case else 0
    if kind == "slots":
        T = case["S"] * mean
        return {"bytes": int(16 * (T + case["pad"]) + 20 * case["S"] + 4 * (T / case["bs"] + case["S"])), "flops": 0}
    if kind == "store":  # rows in, packed out; packed in, rows out
        return {"bytes": case["T"] * (case["hkv"] * 2 * (4 * D + row) + 16), "flops": 0}
    if kind == "load":
        return {"bytes": int(case["S"] * mean * (case["hkv"] * (4 * D + row) + 16)), "flops": 0}
    tokens = (case["B"] - case["pad"]) * mean
    return {"bytes": int(tokens * case["hkv"] * row + case["B"] * (4 * case["hq"] * D + 12) + 4 * tokens / case["bs"]),
            "flops": int(4 * D * case["hq"] * tokens)}


# ---------------------------------------------------------------- from the definitions, in 64 bits
def _values(pool, tables_row, n, value):
    """float64 [n, hkv, 128] of one row's first n tokens: every nibble looked up at its place."""
    recs = pool[tables_row.long()]  # [blocks, hkv, tiles, 4608]
    nb, hkv, tiles, _ = recs.shape
    recs = recs.permute(0, 2, 1, 3).reshape(nb * tiles, hkv, RECORD)
    t = torch.arange(TILE, device=pool.device).view(-1, 1)
    d = torch.arange(D, device=pool.device).view(1, -1)
    if value:
        byte = (t >> 4) * 1024 + (t >> 3 & 1) * 512 + (t & 1) * 8 + (t >> 1 & 3) * 16 + (d >> 1 & 7) * 64 + (d >> 4)
        shift = (d & 1) * 4 + t * 0
    else:
        byte = t * 64 + (d >> 3 & 3) * 16 + (d >> 5) * 4 + (d & 1) * 2 + (d >> 2 & 1)
        shift = (d >> 1 & 1) * 4 + t * 0
    u = recs[:, :, byte].to(torch.int64) >> shift & 15
    scale = recs[:, :, CODES:].contiguous().view(torch.bfloat16).double().view(nb * tiles, hkv, TILE, D // GROUP)
    x = (u - 8).double() * scale.repeat_interleave(GROUP, -1)
    return x.transpose(1, 2).reshape(nb * tiles * TILE, hkv, D)[:n]


def exact(case, seed):
    if case["kind"] in ("tables", "slots"):
        return None  # whole numbers
    s = prepare(case, seed)
    if case["kind"] == "store":
        outs = []
        for x in (s["k"], s["v"]):
            g = x.double().reshape(x.shape[0], -1, D // GROUP, GROUP)
            scale = (g.abs().max(-1, keepdim=True).values / 7.0).to(torch.bfloat16).double()
            code = torch.zeros_like(g)
            ok = (scale > 0).expand_as(g)
            code[ok] = torch.round((g / scale)[ok])
            y = (torch.minimum(torch.maximum(code, code.new_tensor(-7.0)), code.new_tensor(7.0)) * scale).reshape(x.shape)
            y[s["slots"] < 0] = 0
            outs.append(y)
        return tuple(outs)
    if case["kind"] == "load":
        bs, outs = case["bs"], []
        for pool, value, out in ((s["kc"], False, s["ko"]), (s["vc"], True, s["vo"])):
            y = torch.zeros(out.shape, dtype=torch.float64, device=out.device)
            for i, n in enumerate(s["lens"].tolist()):
                used, at = -(-n // bs), i * -(-case["hi"] // bs)
                rows = _values(pool, s["tables"][i, :used], n, value)
                rows = torch.cat([rows, rows.new_zeros((used * bs - n,) + rows.shape[1:])])
                y[at:at + used] = rows.view(used, bs, -1, D).transpose(1, 2)
            outs.append(y)
        return tuple(outs)
    q = s["q"].double()
    out = torch.zeros_like(q)
    G, bs = case["hq"] // case["hkv"], case["bs"]
    for b, r in enumerate(s["rows"].tolist()):
        if r < 0:
            continue
        n = int(s["seqlens"][r]) + 1
        table = s["tables"][r, :-(-n // bs)]
        k, v = _values(s["kc"], table, n, False), _values(s["vc"], table, n, True)
        for h in range(case["hkv"]):
            logits = q[b, h * G:(h + 1) * G] @ k[:, h].T / math.sqrt(D)
            out[b, h * G:(h + 1) * G] = torch.softmax(logits, -1) @ v[:, h]
    return out
