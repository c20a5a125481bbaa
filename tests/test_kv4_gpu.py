"""The 4-bit KV cache (store, load, decode attention) and the request maps against plain 64-bit
restatements (oracle/kv4.py), through awesome_acceleration_b200.kernels."""
import math

import numpy as np
import pytest
import torch

from oracle import kv4 as O

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
SCALE = 128 ** -0.5


def K():
    from awesome_acceleration_b200 import kernels
    return kernels


def dev_err():
    from awesome_acceleration_b200 import _lib
    e = _lib.device_error()
    _lib.clear_device_error()
    return e


@pytest.fixture(autouse=True)
def _clean_error_word(cuda):
    dev_err()


def same(a, b):
    """Bitwise equality of bf16 tensors up to the payload of NaN and the sign of zero."""
    a, b = a.float(), b.float()
    return torch.equal(torch.nan_to_num(a, nan=12345.0), torch.nan_to_num(b, nan=12345.0))


def tables_for(ctx, bs, gen, extra=3, max_blocks=None):
    need = [-(-c // bs) for c in ctx]
    nb = sum(need) + extra
    mb = max_blocks or max(max(need), 1)
    perm = torch.randperm(nb, generator=gen).to(torch.int32)
    bt = torch.full((len(ctx), mb), -1, dtype=torch.int32)
    it = 0
    for i, n in enumerate(need):
        bt[i, :n] = perm[it:it + n]
        it += n
    return bt, nb


# --------------------------------------------------------------------------- store / load
@pytest.mark.parametrize("T,hkv,bs,strided", [(1, 1, 64, False), (1, 8, 256, True), (17, 3, 64, True),
                                              (300, 4, 128, False), (257, 8, 256, True)])
def test_store_then_load(cuda, T, hkv, bs, strided):
    g = torch.Generator().manual_seed(T + hkv)
    nb = -(-T // bs) + 2
    x = torch.randn((2, T, hkv, 128), generator=g) * torch.exp(3 * torch.randn((2, T, hkv, 1), generator=g))
    k, v = x.to(BF)
    slots = torch.randperm(nb * bs, generator=g)[:T]
    if T > 4:
        slots[::5] = -1
    kc = torch.full(K().kv4_cache_shape(nb, hkv, bs), 0x5a, dtype=torch.uint8)
    vc = torch.full_like(kc, 0xa5)
    kd, vd, sd = kc.to(cuda), vc.to(cuda), slots.to(cuda)
    if strided:
        wide = torch.empty((T, 2 * hkv + 3, 128), dtype=BF, device=cuda)
        wide[:, 1:hkv + 1], wide[:, hkv + 2:2 * hkv + 2] = k.to(cuda), v.to(cuda)
        K().kv4_store(wide[:, 1:hkv + 1], wide[:, hkv + 2:2 * hkv + 2], sd, kd, vd)
    else:
        K().kv4_store(k.to(cuda), v.to(cuda).view(T, hkv * 128), sd, kd, vd)
    keep = slots >= 0
    for pool, before, rows, value in ((kd, kc, k, False), (vd, vc, v, True)):
        # the pool bit by bit: what was stored as the oracle packs it, everything else left as it was
        want = O.pool_rows(before, value)
        got = O.pool_rows(pool.cpu(), value)
        n, s = O.quantise(rows)
        want[slots[keep]] = (n.double() * s.double().repeat_interleave(32, -1))[keep]
        assert torch.equal(got, want)
    ko = torch.full((T, hkv, 128), 3.0, dtype=BF, device=cuda)
    vo = torch.full((T, hkv, 128), 5.0, dtype=BF, device=cuda)
    K().kv4_load(kd, vd, sd, ko, vo)
    for out, rows, left in ((ko, k, 3.0), (vo, v, 5.0)):
        n, s = O.quantise(rows)
        want = (n.double() * s.double().repeat_interleave(32, -1)).to(BF)  # exact product, rounded once
        assert same(out.cpu()[keep], want[keep])
        assert (out.cpu()[~keep] == left).all()
    assert dev_err() == 0


def test_store_special_values(cuda):
    """Zeros, subnormals, the largest values, exact ties, infinities and NaN."""
    rows = torch.zeros((9, 1, 128), dtype=BF)
    rows[1] = 2.0 ** -133                       # subnormal in bf16
    rows[2] = torch.finfo(BF).max
    rows[3, 0, ::2] = -torch.finfo(BF).max
    rows[4, 0, :32] = torch.tensor([7.0 * 2 ** -4] + [(i % 15 - 7 + 0.5) * 2 ** -4 for i in range(31)])  # ties
    rows[5, 0, 40] = math.inf
    rows[6, 0, 127] = math.nan
    rows[7] = torch.randn(128, generator=torch.Generator().manual_seed(0)) * 1e-38
    rows[8, 0, 3] = -math.inf
    slots = torch.arange(9)
    for swap in (False, True):
        kd = torch.zeros(K().kv4_cache_shape(1, 1, 64), dtype=torch.uint8, device=cuda)
        vd = torch.zeros_like(kd)
        K().kv4_store(rows.to(cuda), rows.flip(0).to(cuda) if swap else rows.to(cuda), slots.to(cuda), kd, vd)
        k, v = K().kv4_load(kd, vd, slots.to(cuda))
        n, s = O.quantise(rows)
        want = (n.double() * s.double().repeat_interleave(32, -1)).to(BF)
        assert same(k.cpu(), want)
        assert same(v.cpu(), want.flip(0) if swap else want)
        # a non-finite member spoils its own group of 32 dims and no other
        assert torch.isnan(k.cpu()[5, 0, 32:64]).all() and torch.isfinite(k.cpu()[5, 0, :32]).all()
    assert dev_err() == 0


def test_store_quantisation_matches_the_oracle_on_every_bf16_magnitude(cuda):
    """x / s over all pairs of significands: the rounding decisions are those of exact arithmetic."""
    sig = torch.arange(128, 256).double()
    rows = torch.zeros((128, 4, 32), dtype=torch.float64)
    g = torch.Generator().manual_seed(5)
    rows[:, :, 0] = sig[:, None] * 2.0 ** torch.tensor([-7.0, 0.0, 30.0, -100.0])
    e = torch.randint(-6, 1, (128, 4, 31), generator=g)
    m = torch.randint(128, 256, (128, 4, 31), generator=g)
    rows[:, :, 1:] = torch.minimum(m * 2.0 ** e.double() * (rows[:, :, :1] / sig[:, None, None]), rows[:, :, :1])
    rows = rows.reshape(128, 1, 128).to(BF)
    kd = torch.zeros(K().kv4_cache_shape(2, 1, 64), dtype=torch.uint8, device=cuda)
    vd = torch.zeros_like(kd)
    K().kv4_store(rows.to(cuda), (-rows).to(cuda), torch.arange(128, device=cuda), kd, vd)
    assert torch.equal(kd.cpu(), O.pool_from_rows(rows, 64, False))
    assert torch.equal(vd.cpu(), O.pool_from_rows(-rows, 64, True))


def test_load_into_a_paged_cache_of_another_block_size(cuda):
    g = torch.Generator().manual_seed(3)
    hkv, T = 2, 200
    pool_k = O.pool_from_rows(torch.randn((512, hkv, 128), generator=g).to(BF), 128, False)
    pool_v = O.pool_from_rows(torch.randn((512, hkv, 128), generator=g).to(BF), 128, True)
    src = torch.randint(0, 512, (T,), generator=g)      # a slot may be loaded twice
    dst = torch.randperm(3 * 96, generator=g)[:T]
    src[7], dst[11] = -1, -1
    ko = torch.full((3, hkv, 96, 128), 7.0, dtype=BF, device=cuda)
    vo = torch.full_like(ko, -7.0)
    K().kv4_load(pool_k.to(cuda), pool_v.to(cuda), src.to(cuda), ko, vo, out_slots=dst.to(cuda))
    keep = (src >= 0) & (dst >= 0)
    for out, pool, value, left in ((ko, pool_k, False, 7.0), (vo, pool_v, True, -7.0)):
        want = torch.full((3 * 96, hkv, 128), left, dtype=BF)
        want[dst[keep]] = O.pool_rows(pool, value)[src[keep]].to(BF)
        assert same(out.cpu().permute(0, 2, 1, 3).reshape(-1, hkv, 128), want)
    assert dev_err() == 0


def test_store_and_load_skip_slots_outside_the_pool(cuda):
    kd = torch.zeros(K().kv4_cache_shape(2, 1, 64), dtype=torch.uint8, device=cuda)
    vd = torch.zeros_like(kd)
    ones = torch.ones((2, 1, 128), dtype=BF, device=cuda)
    K().kv4_store(ones, ones, torch.tensor([5, 128], device=cuda), kd, vd)
    assert dev_err() & 2
    # s = bf16(1 / 7) = 73/512, so a one is held as 7 s = 511/512, which rounds to 1 in bf16 (tie to even)
    assert float(O.pool_rows(kd.cpu(), False).sum()) == 128 * 511 / 512
    ko, vo = K().kv4_load(kd, vd, torch.tensor([5, 128], device=cuda))
    assert dev_err() & 2
    assert float(ko.float().sum()) == 128.0 and float(vo.float().sum()) == 128.0
    out = torch.zeros((1, 1, 128), dtype=BF, device=cuda)
    K().kv4_load(kd, vd, torch.tensor([5, 5], device=cuda), out, out.clone(), out_slots=torch.tensor([1, -1], device=cuda))
    assert dev_err() & 2 and not out.any()


def test_wrappers_refuse_other_types_shapes_and_layouts(cuda):
    pool = torch.zeros(K().kv4_cache_shape(2, 2, 64), dtype=torch.uint8, device=cuda)
    rows = torch.zeros((3, 2, 128), dtype=BF, device=cuda)
    i64, i32 = torch.zeros(3, dtype=torch.int64, device=cuda), torch.zeros(3, dtype=torch.int32, device=cuda)
    bt = torch.zeros((3, 2), dtype=torch.int32, device=cuda)
    ws = torch.zeros(K().kv4_decode_workspace_bytes(4, 2), dtype=torch.uint8, device=cuda)
    q = torch.zeros((3, 4, 128), dtype=BF, device=cuda)

    def store(k=rows, v=rows, s=i64, kc=pool, vc=pool):
        K().kv4_store(k, v, s, kc, vc)

    def load(kc=pool, vc=pool, s=i64, ko=rows, vo=rows.clone(), os=None):
        K().kv4_load(kc, vc, s, ko, vo, out_slots=os)

    def attend(q=q, kc=pool, vc=pool, bt=bt, r=i64, sl=i32, ws=ws, out=None):
        K().kv4_decode_attention(q, kc, vc, bt, r, sl, ctx_add=0, scale=1.0, max_context=64, workspace=ws, out=out)

    def maps(n=i32, bt=bt, st=None, r=None, cu=None, pos=None, sl=None):
        K().build_slot_maps(n, bt, block_size=64, num_blocks=2, num_tokens=5, starts=st, rows=r, cu=cu, positions=pos,
                            slots=sl)

    def tables(n=i32, out=None, fr=None, used=None, mb=2):
        K().build_block_tables(n, 64, max_blocks=mb, out=out, free_blocks=fr, used=used)
    half = torch.zeros((2, 2, 1, 4600), dtype=torch.uint8, device=cuda)
    wide = torch.zeros((3, 2, 256), dtype=BF, device=cuda)
    for f, kw in [
        (store, dict(kc=pool.to(torch.int8))), (store, dict(kc=half, vc=half)), (store, dict(vc=pool[:1])),
        (store, dict(kc=pool.transpose(0, 1))), (store, dict(k=rows.float())), (store, dict(v=rows[:2])),
        (store, dict(k=wide[..., ::2])), (store, dict(k=rows[:, :1])), (store, dict(s=i32)), (store, dict(s=i64[:2])),
        (store, dict(k=rows.cpu())), (store, dict(s=i64.cpu())),
        (load, dict(kc=half, vc=half)), (load, dict(s=i32)), (load, dict(os=i64[:2])), (load, dict(ko=None)),
        (load, dict(ko=rows.half())), (load, dict(ko=rows[:2])), (load, dict(ko=wide[..., :128], vo=wide[..., 128:])),
        (load, dict(ko=rows[:, :1].contiguous(), vo=rows[:, :1].contiguous())), (load, dict(ko=None, vo=None, os=i64)),
        (attend, dict(q=q.half())), (attend, dict(q=wide)), (attend, dict(r=i64[:2])), (attend, dict(r=i32)),
        (attend, dict(sl=i64)), (attend, dict(bt=bt[:2])), (attend, dict(bt=bt.long())), (attend, dict(ws=None)),
        (attend, dict(ws=ws[:-16])), (attend, dict(ws=ws.view(torch.int8))), (attend, dict(out=q[:2])),
        (attend, dict(out=q.float())), (attend, dict(kc=pool[:1], vc=pool)),
        (maps, dict(n=i64)), (maps, dict(n=i32.view(1, 3))), (maps, dict(bt=bt.long())), (maps, dict(st=i32[:2])),
        (maps, dict(r=i64[:2])), (maps, dict(r=i32)), (maps, dict(cu=i32)), (maps, dict(pos=i64)),
        (maps, dict(sl=i32)), (maps, dict(bt=bt.t())),
        (tables, dict(n=i64)), (tables, dict(mb=None)), (tables, dict(out=bt[:2])), (tables, dict(out=bt, mb=3)),
        (tables, dict(fr=i64)), (tables, dict(used=i32)),
    ]:
        with pytest.raises((ValueError, RuntimeError)):
            f(**kw)
    for f in (store, load, attend, maps, tables):
        f()
    with pytest.raises(RuntimeError, match="head ratio"):
        attend(q=torch.zeros((3, 6, 128), dtype=BF, device=cuda))
    with pytest.raises(RuntimeError, match="aligned"):
        buf = torch.zeros(3 * 256 + 4, dtype=BF, device=cuda)
        store(k=buf[4:].view(3, 2, 128))
    assert dev_err() == 0


def test_empty_calls(cuda):
    kd = torch.zeros(K().kv4_cache_shape(2, 2, 64), dtype=torch.uint8, device=cuda)
    none = torch.empty(0, dtype=torch.int64, device=cuda)
    rows = torch.empty((0, 2, 128), dtype=BF, device=cuda)
    K().kv4_store(rows, rows, none, kd, kd)
    k, v = K().kv4_load(kd, kd, none)
    assert k.shape == (0, 2, 128)
    q = torch.empty((0, 4, 128), dtype=BF, device=cuda)
    ws = torch.zeros(K().kv4_decode_workspace_bytes(4, 2), dtype=torch.uint8, device=cuda)
    out = K().kv4_decode_attention(q, kd, kd, torch.zeros((1, 1), dtype=torch.int32, device=cuda), none,
                                   torch.zeros(1, dtype=torch.int32, device=cuda), ctx_add=0, scale=1.0, max_context=64,
                                   workspace=ws)
    assert out.shape == (0, 4, 128)
    i32 = torch.empty(0, dtype=torch.int32, device=cuda)
    assert K().build_block_tables(i32, 64, max_blocks=3).shape == (0, 3)
    cu, pos, slots = K().build_slot_maps(i32, torch.zeros((1, 1), dtype=torch.int32, device=cuda), block_size=64,
                                         num_blocks=1, num_tokens=5)
    assert cu.tolist() == [0] and pos.tolist() == [0] * 5 and slots.tolist() == [-1] * 5
    assert not kd.any() and dev_err() == 0


# --------------------------------------------------------------------------- decode attention
def make_case(ctx, G, hkv, bs, seed, *, max_blocks=None, extra=3, outliers=True):
    g = torch.Generator().manual_seed(seed)
    bt, nb = tables_for(ctx, bs, g, extra, max_blocks)
    k = torch.randn((nb * bs, hkv, 128), generator=g)
    if outliers:
        k = k * torch.where(torch.rand((hkv, 128), generator=g) < 0.05, 8.0, 1.0)
    v = torch.randn((nb * bs, hkv, 128), generator=g) * 0.7
    q = torch.randn((len(ctx), G * hkv, 128), generator=g).to(BF)
    return dict(q=q, kp=O.pool_from_rows(k.to(BF), bs, False), vp=O.pool_from_rows(v.to(BF), bs, True), bt=bt, nb=nb,
                ctx=ctx, bs=bs, hkv=hkv, G=G)


def workspace(c, cuda):
    return torch.zeros(K().kv4_decode_workspace_bytes(c["G"] * c["hkv"], c["hkv"]), dtype=torch.uint8, device=cuda)


def call(c, cuda, *, rows=None, seqlens=None, ctx_add=1, scale=SCALE, max_context=None, ws=None, q=None, kp=None,
         vp=None, bt=None, out=None):
    B = c["q"].shape[0]
    rows = torch.arange(B) if rows is None else rows
    seqlens = torch.tensor(c["ctx"], dtype=torch.int32) - ctx_add if seqlens is None else seqlens
    return K().kv4_decode_attention(
        (c["q"] if q is None else q).to(cuda), (c["kp"] if kp is None else kp).to(cuda),
        (c["vp"] if vp is None else vp).to(cuda), (c["bt"] if bt is None else bt).to(cuda), rows.to(cuda),
        seqlens.to(cuda), ctx_add=ctx_add, scale=scale, max_context=max_context or c["bt"].shape[1] * c["bs"],
        workspace=workspace(c, cuda) if ws is None else ws, out=out)


def check(out, c, scale=SCALE, ctx=None):
    """Every output within its derived bound of the 64-bit result.

    Rounding: the output once to bf16 (2^-8 relative); each probability once and its product with the V scale
    once to fp16 (2^-11 relative each, so 2^-10 sum p|v|).
    Scores: fp32 sums of q (u - 8), from terms of at most (15 + 8)|q| a code, in at most 2^5 steps that round
    (or cut) to 2^-23 of the terms: |error| <= 23 * 2^-18 * scale * sum s|q|; exp makes it a relative error
    of p, above and below the fraction line.  2^-17 covers exp2 and the fp32 sums of a lane's weights.
    P V: fp32 sums of p s (u - 8) from terms of at most 23 p s a code.  Each of the two products for 16 tokens
    rounds (or cuts) to 2^-22 of its terms and of what it adds to, which is sum p |v| and 8 p s of those
    tokens: in all 2^-22 * 2 * 23 * sum p s, and 2^-22 * 2 * (tokens / 16 in one warp's run, below 2^8 here) *
    sum p|v|."""
    k_all, v_all = O.pool_rows(c["kp"], False), O.pool_rows(c["vp"], True)
    out = out.cpu().double()
    for b, n in enumerate(c["ctx"] if ctx is None else ctx):
        if n <= 0:
            assert not out[b].any(), f"row {b}: empty context"
            continue
        pos = torch.arange(n)
        slot = c["bt"][b].long()[pos // c["bs"]] * c["bs"] + pos % c["bs"]
        ref, mag, reach, ps = O.attend(c["q"][b], k_all[slot], v_all[slot], scale)
        rel = torch.expm1(2 * 23 * 2.0 ** -18 * reach)[:, None] + 2.0 ** -17
        tol = (2.0 ** -8 * ref.abs() + 2.0 ** -10 * mag) * (1 + 2.0 ** -7) + rel * (mag + ref.abs())
        tol += 2.0 ** -22 * 46 * ps + 2.0 ** -13 * mag
        bad = (out[b] - ref).abs() > tol
        assert not bad.any(), f"row {b} ctx {n}: {((out[b] - ref).abs() / tol).max().item():.2f} of the bound"


CTX = [1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 255, 256, 257, 511, 1000, 2049]


@pytest.mark.parametrize("G,hkv,bs", [(1, 2, 64), (2, 8, 256), (4, 3, 128), (8, 1, 256), (8, 5, 64)])
def test_decode_attention(cuda, G, hkv, bs):
    c = make_case(CTX, G, hkv, bs, 10 + G)
    check(call(c, cuda), c)
    assert dev_err() == 0


@pytest.mark.parametrize("G,hkv,ctx", [(2, 8, [333]), (4, 8, [40960]), (8, 8, [9000, 1, 3]), (1, 1, [5000]),
                                       (1, 1, [64] * 300), (8, 2, [70] * 200 + [3000])])
def test_decode_attention_few_and_many_rows(cuda, G, hkv, ctx):
    c = make_case(ctx, G, hkv, 256, sum(ctx) % 97)
    check(call(c, cuda), c)
    assert dev_err() == 0


@pytest.mark.parametrize("B", [513, 1300])
def test_decode_attention_batches_past_the_row_table(cuda, B):
    """More rows than the kernel keeps in shared memory, padding and empty rows among them."""
    g = torch.Generator().manual_seed(B)
    lens = torch.randint(1, 150, (B,), generator=g)
    lens[::7] = 0
    lens[1] = 1000
    c = make_case([max(int(n), 1) for n in lens], 2, 1, 64, B)
    rows = torch.arange(B)
    rows[5::11] = -1
    out = call(c, cuda, rows=rows, seqlens=lens.to(torch.int32), ctx_add=0)
    check(out, c, ctx=[int(n) if r >= 0 else 0 for n, r in zip(lens, rows)])
    assert dev_err() == 0


def test_decode_attention_rows_padding_and_empty_contexts(cuda):
    c = make_case([5, 100, 64, 300, 1], 2, 2, 64, 4)
    order = torch.tensor([3, -1, 0, 2, -7, 1])          # rows permuted, two padding rows
    seqlens = torch.tensor([5, 100, -1, 300, 1], dtype=torch.int32)  # row 2 is empty: nothing to attend to
    q = torch.randn((6, 4, 128), generator=torch.Generator().manual_seed(1)).to(BF)
    out = call(c, cuda, rows=order, seqlens=seqlens, ctx_add=0, q=q)
    ctx = [c["ctx"][r] if r >= 0 and r != 2 else 0 for r in order.tolist()]
    full = dict(c, q=q, ctx=ctx, bt=c["bt"][order.clamp(min=0)])
    check(out, full)
    assert dev_err() == 0
    # the same row twice is two reads
    both = call(c, cuda, rows=torch.tensor([3, 3, 1, 3, 1]), q=c["q"][:1].expand(5, -1, -1).contiguous())
    assert torch.equal(both[0], both[1]) or (both[0].float() - both[1].float()).abs().max() < 0.05


def test_decode_attention_ignores_what_lies_behind_the_context(cuda):
    """NaN scales and arbitrary codes behind the last token, in the last tile and in unused blocks."""
    ctx = [1, 17, 63, 65, 130]
    for G in (1, 8):
        c = make_case(ctx, G, 2, 64, 20 + G)
        clean = call(c, cuda)
        kp, vp = c["kp"].clone(), c["vp"].clone()
        used = torch.zeros(c["nb"] * 64, dtype=torch.bool)
        for b, n in enumerate(ctx):
            pos = torch.arange(n)
            used[c["bt"][b].long()[pos // 64] * 64 + pos % 64] = True
        for p in (kp, vp):
            rec = p.view(c["nb"], 2, 4608)
            s = rec[..., 4096:].contiguous().view(BF).view(c["nb"], 2, 64, 4)
            s[(~used).view(c["nb"], 1, 64).expand(-1, 2, -1)] = math.nan
            rec[..., 4096:] = s.view(c["nb"], 2, 256).contiguous().view(torch.uint8)
        dirty = call(c, cuda, kp=kp, vp=vp)
        assert torch.equal(clean, dirty)
    assert dev_err() == 0


def test_decode_attention_nan_in_the_context_spreads_to_its_heads_only(cuda):
    c = make_case([100, 50], 2, 2, 64, 8)
    x = torch.randn((64, 2, 128), generator=torch.Generator().manual_seed(2)).to(BF)
    x[3, 1, 5] = math.nan
    kd, vd = c["kp"].to(cuda), c["vp"].to(cuda)
    slots = c["bt"][0, 0].long() * 64 + torch.arange(64)
    K().kv4_store(x.to(cuda), x.nan_to_num().to(cuda), slots.to(cuda), kd, vd)
    out = call(c, cuda, kp=kd, vp=vd).cpu()
    assert torch.isnan(out[0, 2:]).all() and torch.isfinite(out[0, :2]).all() and torch.isfinite(out[1]).all()


def test_decode_attention_extreme_logits_and_scales(cuda):
    """One token far above the rest, logits of thousands, values near the ends of bf16's range."""
    c = make_case([70, 200, 1000], 4, 2, 64, 31)
    check(call(c, cuda, scale=40.0), c, scale=40.0)
    check(call(c, cuda, scale=0.0), c, scale=0.0)
    check(call(c, cuda, scale=-SCALE), c, scale=-SCALE)
    for mul in (1e-30, 1e30):
        g = torch.Generator().manual_seed(6)
        v = (torch.randn((c["nb"] * 64, 2, 128), generator=g) * mul).to(BF)
        big = dict(c, vp=O.pool_from_rows(v, 64, True))
        check(call(big, cuda), big)
    assert dev_err() == 0


def test_decode_attention_bad_blocks_rows_and_contexts_are_reported(cuda):
    c = make_case([100, 40, 64], 2, 2, 64, 12)
    good = call(c, cuda)
    assert dev_err() == 0
    for bad in (-1, c["nb"], 2 ** 31 - 1):
        bt = c["bt"].clone()
        bt[0, 1] = bad
        out = call(c, cuda, bt=bt)
        assert dev_err() == 1
        assert torch.equal(out[1:], good[1:])
    out = call(c, cuda, rows=torch.tensor([0, 3, 2]))   # there are 3 rows
    assert dev_err() == 2
    assert not out[1].any() and torch.equal(out[0], good[0]) and torch.equal(out[2], good[2])
    out = call(c, cuda, max_context=64)                 # row 0 has 100 tokens: cut at 64
    assert dev_err() == 32
    check(out, c, ctx=[64, 40, 64])
    out = call(c, cuda, seqlens=torch.tensor([2 ** 31 - 1, 39, 63], dtype=torch.int32))
    assert dev_err() & 32
    assert torch.equal(out[1:], good[1:])


def test_decode_attention_in_a_pool_past_32_bit_offsets(cuda):
    """Blocks at both ends of pools of more than 2^32 bytes each."""
    hkv, bs, nb = 8, 256, 30000
    shape = K().kv4_cache_shape(nb, hkv, bs)
    assert math.prod(shape) > 2 ** 32
    kd = torch.zeros(shape, dtype=torch.uint8, device=cuda)
    vd = torch.zeros_like(kd)
    g = torch.Generator().manual_seed(40)
    ctx = [300, 257, 64]
    bt = torch.tensor([[nb - 1, 0], [1, nb - 2], [nb - 3, -1]], dtype=torch.int32)
    T = sum(ctx)
    k, v = torch.randn((2, T, hkv, 128), generator=g).to(BF)
    cu, pos, slots = K().build_slot_maps(torch.tensor(ctx, dtype=torch.int32, device=cuda), bt.to(cuda), block_size=bs,
                                         num_blocks=nb, num_tokens=T)
    K().kv4_store(k.to(cuda), v.to(cuda), slots, kd, vd)
    ko, vo = K().kv4_load(kd, vd, slots)
    q = torch.randn((3, 16, 128), generator=g).to(BF)
    c = dict(q=q, ctx=ctx, bs=bs, hkv=hkv, G=2, bt=torch.tensor([[0, 1], [2, 3], [4, -1]], dtype=torch.int32), nb=6)
    kr, vr = torch.zeros((2, 6 * bs, hkv, 128), dtype=BF)
    at = 0
    for b, n in enumerate(ctx):
        p = torch.arange(n)
        s = c["bt"][b].long()[p // bs] * bs + p % bs
        kr[s], vr[s] = k[at:at + n], v[at:at + n]
        at += n
    c.update(kp=O.pool_from_rows(kr, bs, False), vp=O.pool_from_rows(vr, bs, True))
    out = call(c, cuda, kp=kd, vp=vd, bt=bt)
    check(out, c)
    n, s = O.quantise(k)
    assert same(ko.cpu(), (n.double() * s.double().repeat_interleave(32, -1)).to(BF))
    assert dev_err() == 0


def test_decode_attention_repeats_bit_for_bit_and_shares_a_workspace_between_shapes(cuda):
    """One workspace, calls of different batches, head counts and contexts in turn: each gives what it gives alone."""
    cases = [make_case([3000, 5, 900], 4, 2, 256, 1), make_case([64] * 40, 4, 2, 64, 2),
             make_case([9000], 4, 2, 256, 3), make_case([1], 4, 2, 64, 4)]
    alone = [call(c, cuda) for c in cases]
    ws = workspace(cases[0], cuda)
    for order in ([0, 1, 2, 3], [2, 0, 3, 1], [0, 0, 2, 2]):
        for i in order:
            assert torch.equal(call(cases[i], cuda, ws=ws), alone[i])
    assert dev_err() == 0


def test_decode_attention_in_a_graph_and_on_another_stream(cuda):
    """Captured once, replayed with contexts that grow in place; then an eager call on a side stream."""
    c = make_case([200, 64, 700], 2, 8, 64, 50)
    q, kp, vp, bt = (c[x].to(cuda) for x in ("q", "kp", "vp", "bt"))
    rows = torch.arange(3, device=cuda)
    seqlens = torch.tensor([100, 1, 3], dtype=torch.int32, device=cuda)
    ws, out = workspace(c, cuda), torch.empty_like(q)

    def go():
        K().kv4_decode_attention(q, kp, vp, bt, rows, seqlens, ctx_add=1, scale=SCALE, max_context=bt.shape[1] * 64,
                                 workspace=ws, out=out)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        go()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        go()
        K().advance_seqlens(rows, seqlens)
    seqlens.copy_(torch.tensor([198, 61, 640], dtype=torch.int32))
    for step in range(3):
        graph.replay()
        ctx = [199 + step, 62 + step, 641 + step]
        if step < 2:
            check(out, dict(c, ctx=ctx))
    with torch.cuda.stream(s):
        s.wait_stream(torch.cuda.current_stream())
        seqlens.copy_(torch.tensor([199, 63, 699], dtype=torch.int32))
        go()
    torch.cuda.current_stream().wait_stream(s)
    check(out, c)
    assert dev_err() == 0


def test_decode_attention_on_two_streams_at_once(cuda):
    """Calls in flight together, each with its own workspace, and one pool stored to by neither."""
    cases = [make_case([4000, 3, 700] * 5, 2, 8, 64, 60), make_case([9000, 130], 8, 8, 64, 61)]
    dev = [{x: c[x].to(cuda) for x in ("q", "kp", "vp", "bt")} for c in cases]
    lens = [torch.tensor(c["ctx"], dtype=torch.int32, device=cuda) for c in cases]
    rows = [torch.arange(len(c["ctx"]), device=cuda) for c in cases]
    ws, outs = [workspace(c, cuda) for c in cases], [torch.empty_like(d["q"]) for d in dev]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for _ in range(20):
        for i, (c, s) in enumerate(zip(cases, streams)):
            with torch.cuda.stream(s):
                K().kv4_decode_attention(dev[i]["q"], dev[i]["kp"], dev[i]["vp"], dev[i]["bt"], rows[i], lens[i],
                                         ctx_add=0, scale=SCALE, max_context=c["bt"].shape[1] * 64, workspace=ws[i],
                                         out=outs[i])
    torch.cuda.synchronize()
    for c, out in zip(cases, outs):
        check(out, c)
    assert dev_err() == 0


# --------------------------------------------------------------------------- request maps
def test_block_tables_of_no_request_take_no_block(cuda):
    used = torch.full((1,), 9, dtype=torch.int32, device=cuda)
    K().build_block_tables(torch.empty(0, dtype=torch.int32, device=cuda), 64, max_blocks=3, used=used)
    assert used.item() == 0 and dev_err() == 0


@pytest.mark.parametrize("lens,bs", [([0], 64), ([1], 64), ([64, 65, 0, 1, 128, 700], 64), ([256] * 300, 256),
                                     (list(range(0, 2600, 2)), 128)])
def test_block_tables(cuda, lens, bs):
    mb = max(1, max(-(-n // bs) for n in lens)) + 1
    total = sum(-(-n // bs) for n in lens)
    free = torch.randperm(total + 5, generator=torch.Generator().manual_seed(len(lens))).to(torch.int32)
    used = torch.full((1,), -5, dtype=torch.int32, device=cuda)
    for fr in (free, None):
        out = K().build_block_tables(torch.tensor(lens, dtype=torch.int32, device=cuda), bs, max_blocks=mb,
                                     free_blocks=None if fr is None else fr.to(cuda), used=used)
        want, n = O.block_tables(lens, bs, mb, range(total) if fr is None else fr.tolist())
        assert np.array_equal(out.cpu().numpy(), want) and int(used) == n == total
    assert dev_err() == 0


def test_block_tables_cut_and_exhausted(cuda):
    lens = torch.tensor([300, -4, 64, 2 ** 31 - 1, 65], dtype=torch.int32, device=cuda)
    out = K().build_block_tables(lens, 64, max_blocks=4)
    assert dev_err() == 32
    want, _ = O.block_tables([256, 0, 64, 256, 65], 64, 4, range(99))
    assert np.array_equal(out.cpu().numpy(), want)
    used = torch.zeros(1, dtype=torch.int32, device=cuda)
    free = torch.tensor([9, 8, 7], dtype=torch.int32, device=cuda)
    out = K().build_block_tables(torch.tensor([64, 65, 64], dtype=torch.int32, device=cuda), 64, max_blocks=2,
                                 free_blocks=free, used=used)
    assert dev_err() == 1
    assert out.tolist() == [[9, -1], [8, 7], [-1, -1]] and int(used) == 4


@pytest.mark.parametrize("lens,bs,pad", [([0], 64, 3), ([1], 64, 0), ([700, 0, 0, 1, 64, 513, 0], 64, 100),
                                         ([3] * 1500, 256, 1), ([5000], 128, 0), (list(range(60)), 256, 700),
                                         ([0] * 1100 + [600] + [0] * 1000 + [1], 64, 0)])
def test_slot_maps(cuda, lens, bs, pad):
    S = len(lens)
    g = torch.Generator().manual_seed(S)
    starts = torch.randint(0, 300, (S,), generator=g)
    rows = torch.randperm(S + 4, generator=g)[:S]
    if S > 3:
        rows[2] = -1
    mb = -(-(max(lens) + 300) // bs) + 1
    nb = (S + 4) * mb
    bt = torch.randperm(nb, generator=g).to(torch.int32).view(S + 4, mb)
    T = sum(lens) + pad
    i32 = dict(dtype=torch.int32, device=cuda)
    for st in (starts, torch.zeros_like(starts)):
        cu, pos, slots = K().build_slot_maps(torch.tensor(lens, **i32), bt.to(cuda), block_size=bs, num_blocks=nb,
                                             num_tokens=T, rows=rows.to(cuda), starts=st.to(**i32) if st.any() else None)
        wcu, wpos, wslots = O.slot_maps(lens, st.tolist(), rows.tolist(), bt.tolist(), bs, T)
        assert np.array_equal(cu.cpu().numpy(), wcu)
        assert np.array_equal(pos.cpu().numpy(), wpos) and np.array_equal(slots.cpu().numpy(), wslots)
    assert dev_err() == 0


def test_slot_maps_report_what_has_no_slot(cuda):
    i32 = dict(dtype=torch.int32, device=cuda)
    bt = torch.tensor([[0, 1], [2, -1], [3, 99]], **i32)

    def maps(lens, T, **kw):
        kw = {k: torch.tensor(v, device=cuda, dtype=torch.int64 if k == "rows" else torch.int32) for k, v in kw.items()}
        return [x.tolist() for x in K().build_slot_maps(torch.tensor(lens, **i32), bt, block_size=64, num_blocks=4,
                                                        num_tokens=T, **kw)]
    cu, pos, slots = maps([2, 2], 4, starts=[127, 63])
    assert dev_err() == 32 | 1 and pos == [127, 128, 63, 64] and slots == [127, -1, 191, -1]
    cu, pos, slots = maps([1, 1], 2, rows=[2, 3], starts=[64, 0])
    assert dev_err() == 1 | 2 and slots == [-1, -1]
    cu, pos, slots = maps([3, 4], 5)                    # two tokens do not fit
    assert dev_err() == 32 and cu == [0, 3, 7] and slots == [0, 1, 2, 128, 129]
    cu, pos, slots = maps([-3, 1], 2, starts=[0, -1])
    assert dev_err() == 32 and cu == [0, 0, 1] and slots == [-1, -1]


# --------------------------------------------------------------------------- together
def test_maps_store_load_and_attention_together(cuda):
    """A prefill of ragged requests through device-built tables and maps, then three decode steps that append
    one token each: every step attends to what the steps before stored."""
    g = torch.Generator().manual_seed(77)
    hkv, G, bs, lens = 2, 4, 64, [5, 64, 200, 1]
    S, steps = len(lens), 3
    cap = torch.tensor([n + steps for n in lens], dtype=torch.int32, device=cuda)
    used = torch.zeros(1, dtype=torch.int32, device=cuda)
    nb = sum(-(-(n + steps) // bs) for n in lens)
    free = torch.randperm(nb, generator=g).to(torch.int32).to(cuda)
    bt = K().build_block_tables(cap, bs, max_blocks=5, free_blocks=free, used=used)
    assert int(used) == nb
    kd = torch.zeros(K().kv4_cache_shape(nb, hkv, bs), dtype=torch.uint8, device=cuda)
    vd = torch.zeros_like(kd)
    rows = torch.arange(S, device=cuda)
    T = sum(lens)
    k, v = torch.randn((2, T + 7, hkv, 128), generator=g).to(BF)
    seqlens = torch.tensor(lens, dtype=torch.int32, device=cuda)
    cu, pos, slots = K().build_slot_maps(seqlens, bt, block_size=bs, num_blocks=nb, num_tokens=T + 7)
    K().kv4_store(k.to(cuda), v.to(cuda), slots, kd, vd)  # 7 padding rows are skipped
    hist_k = [k[int(cu[i]):int(cu[i + 1])] for i in range(S)]
    hist_v = [v[int(cu[i]):int(cu[i + 1])] for i in range(S)]
    ws = torch.zeros(K().kv4_decode_workspace_bytes(G * hkv, hkv), dtype=torch.uint8, device=cuda)
    one = torch.empty(S, dtype=torch.int64, device=cuda)
    for _ in range(steps):
        kn, vn = torch.randn((2, S, hkv, 128), generator=g).to(BF)
        q = torch.randn((S, G * hkv, 128), generator=g).to(BF)
        K().decode_slot_mapping(rows, seqlens, bt, bs, nb, one)
        K().kv4_store(kn.to(cuda), vn.to(cuda), one, kd, vd)
        out = K().kv4_decode_attention(q.to(cuda), kd, vd, bt, rows, seqlens, ctx_add=1, scale=SCALE,
                                       max_context=5 * bs, workspace=ws)
        K().advance_seqlens(rows, seqlens)
        for i in range(S):
            hist_k[i], hist_v[i] = torch.cat([hist_k[i], kn[i:i + 1]]), torch.cat([hist_v[i], vn[i:i + 1]])
        ctx = [h.shape[0] for h in hist_k]
        c = dict(q=q, kp=kd.cpu(), vp=vd.cpu(), bt=bt.cpu(), nb=nb, ctx=ctx, bs=bs, hkv=hkv, G=G)
        check(out, c)
        # and the pool holds the oracle's quantisation of every token
        ko, vo = K().kv4_load(kd, vd, K().build_slot_maps(seqlens, bt, block_size=bs, num_blocks=nb,
                                                           num_tokens=sum(ctx))[2])
        for got, hist in ((ko, hist_k), (vo, hist_v)):
            n, s = O.quantise(torch.cat(hist))
            assert same(got.cpu(), (n.double() * s.double().repeat_interleave(32, -1)).to(BF))
    assert dev_err() == 0
