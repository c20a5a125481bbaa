"""Decode attention over the 4-bit cache at the ends of its range: V groups that are not finite, V scales and
queries of very different magnitude in one context, each against the 64-bit restatement (oracle/kv4.py)."""
import math

import pytest
import torch

from oracle import kv4 as O
from test_kv4_gpu import SCALE, call, check, dev_err, make_case

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


@pytest.fixture(autouse=True)
def _clean_error_word(cuda):
    dev_err()
    yield
    assert dev_err() == 0


def slots_of(c, b):
    pos = torch.arange(c["ctx"][b])
    return c["bt"][b].long()[pos // c["bs"]] * c["bs"] + pos % c["bs"]


def rows(c, seed, hkv):
    """bf16 K or V rows for every slot of the case's pools."""
    return torch.randn((c["nb"] * c["bs"], hkv, 128), generator=torch.Generator().manual_seed(seed)).to(BF)


# --------------------------------------------------------------------------- V groups that are not finite
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("G", [1, 2, 4, 8])
def test_a_v_group_that_is_not_finite_spoils_its_own_dims_only(cuda, G, bad):
    """In the first, a middle and the last tile, and in all three; every head that attends to the token reads NaN
    in the group's 32 dims, and the 64-bit result in the other 96 and in the other kv head."""
    n, hkv = 300, 2
    for where in ([5], [130], [299], [5, 130, 299]):
        c = make_case([n, 70], G, hkv, 64, 90 + G)
        v = rows(c, 91, hkv)
        groups = set()
        for i, t in enumerate(where):
            w = (2 * i + 1) % 4
            v[slots_of(c, 0)[t], 1, 32 * w + 7 * i] = bad
            groups.add(w)
        c["vp"] = O.pool_from_rows(v, 64, True)
        out = call(c, cuda).cpu()
        check(out, c)
        nan = torch.zeros((2, hkv, G, 4, 32), dtype=torch.bool)
        for w in groups:
            nan[0, 1, :, w] = True
        assert torch.equal(torch.isnan(out), nan.view(2, hkv * G, 128))


def test_a_v_group_that_is_not_finite_in_a_split_context(cuda):
    """Contexts whose tiles are shared by many warps and CTAs: the partial that holds the group spoils no other dims."""
    for G, hkv in ((2, 8), (8, 1)):
        c = make_case([6000, 1], G, hkv, 256, 95)
        v = rows(c, 96, hkv)
        v[slots_of(c, 0)[3333], 0, 64] = math.nan
        c["vp"] = O.pool_from_rows(v, 256, True)
        out = call(c, cuda).cpu()
        check(out, c)
        bad = torch.isnan(out)
        assert bad[0, :G, 64:96].all() and bad.sum() == 32 * G


# --------------------------------------------------------------------------- V scales of very different magnitude
def check_v(out, c, **kw):
    """`check` holds every element to 2^-10 sum p|v| (and the roundings of the output and of fp32): a value may lie
    any way below the largest of its context, its tile or its token."""
    assert torch.isfinite(out).all()
    check(out, c, **kw)


def with_v(c, v):
    return dict(c, vp=O.pool_from_rows(v, c["bs"], True))


@pytest.mark.parametrize("e", [-10, -16, -24, -30, -45, -60])
@pytest.mark.parametrize("G", [1, 2, 4, 8])
def test_v_scales_across_groups(cuda, G, e):
    """Groups of 32 dims at 1, 2^e, 2^(e/2) and 2^(e/3) of one another."""
    c = make_case([200, 64, 1, 130], G, 2, 64, 100 + G)
    v = rows(c, 101, 2).float().view(-1, 2, 4, 32)
    v = v * 2.0 ** torch.tensor([0, e, e // 2, e // 3]).view(4, 1)
    c = with_v(c, v.view(-1, 2, 128).to(BF))
    check_v(call(c, cuda), c)


@pytest.mark.parametrize("e", [-10, -16, -24, -30, -45, -60])
@pytest.mark.parametrize("G", [1, 2, 4, 8])
def test_v_scales_across_tokens(cuda, G, e):
    """Every third token, whole tiles, or all but one token at 2^e of the rest."""
    for k, pick in enumerate((lambda t: t % 3 == 0, lambda t: t // 64 == 1, lambda t: t != 77)):
        c = make_case([200, 130], G, 2, 64, 110 + G)
        v = rows(c, 111 + k, 2).float()
        for b in (0, 1):
            at = slots_of(c, b)
            small = pick(torch.arange(c["ctx"][b]))
            v[at[small]] *= 2.0 ** e
        c = with_v(c, v.to(BF))
        check_v(call(c, cuda), c)


def logits_case(logit, G, hkv, ctx, seed, bs=64):
    """A case whose logits are near logit(t) (natural log) for token t of every row: q is one direction u for all
    heads, up to 1 part in 8, and k_t = logit(t) u."""
    c = make_case(ctx, G, hkv, bs, seed)
    g = torch.Generator().manual_seed(seed)
    u = torch.where(torch.rand(128, generator=g) < 0.5, -1.0, 1.0)
    c["q"] = (u * (1 + 0.125 * torch.rand(c["q"].shape, generator=g))).to(BF)
    k = torch.zeros((c["nb"] * bs, hkv, 128))
    for b, n in enumerate(ctx):
        x = logit(torch.arange(n)).float() / (128 * SCALE)
        k[slots_of(c, b)] = x.view(-1, 1, 1) * u
    c["kp"] = O.pool_from_rows(k.to(BF), bs, False)
    return c


@pytest.mark.parametrize("e", [10, 20, 30, 45, 60])
@pytest.mark.parametrize("G", [1, 2, 4, 8])
def test_a_huge_v_of_negligible_or_of_small_probability(cuda, G, e):
    """Token t0's V is 2^e times the others', its probability 2^-(e + 20) (it adds nothing), 2^-e (it adds as much
    as another) or 2^-(e - 6) (it is most of the output)."""
    for t0 in (3, 90, 199):
        for less in (e + 20, e, e - 6):
            c = logits_case(lambda t: torch.where(t == t0, -less * math.log(2.0), 0.25 * torch.cos(t.float())), G, 2,
                            [200], 120 + G)
            v = rows(c, 121, 2).float()
            v[slots_of(c, 0)[t0]] *= 2.0 ** e
            c = with_v(c, v.to(BF))
            check_v(call(c, cuda), c)


@pytest.mark.parametrize("e", [0, 8, 20, 26, 40, 60])
@pytest.mark.parametrize("G", [1, 2, 4, 8])
def test_a_token_of_all_the_probability_and_no_value(cuda, G, e):
    """An attention sink: one token's V is zero, in all groups or in one, and the others, at 2^-e of its
    probability, are the whole output."""
    for groups in ([0, 1, 2, 3], [2]):
        c = logits_case(lambda t: torch.where(t == 0, 0.0, -e * math.log(2.0) + torch.sin(t.float())), G, 2,
                        [150, 2], 130 + G)
        v = rows(c, 131, 2).view(-1, 2, 4, 32)
        for b in (0, 1):
            v[slots_of(c, b)[0], :, groups] = 0
        c = with_v(c, v.view(-1, 2, 128))
        check_v(call(c, cuda), c)


@pytest.mark.parametrize("G", [1, 2, 4, 8])
def test_small_values_over_a_long_context(cuda, G):
    """Thousands of tokens in one warp's run (1300 queries over the same 4000): a first tile of small V and most of
    the probability, then large V of little."""
    B, look = 1300, [0, 650, 1299]
    for e in (6, 9, 12, 20):
        c = logits_case(lambda t: torch.where(t < 64, 0.0, -(e + 14) * math.log(2.0)), G, 1, [4000], 140 + G, 256)
        q = c["q"] * (1 + torch.randint(0, 32, (B, 1, 1), generator=torch.Generator().manual_seed(e)) / 256)
        v = rows(c, 141, 1).float()
        v[slots_of(c, 0)[:64]] *= 2.0 ** -e
        c = with_v(c, v.to(BF))
        out = call(c, cuda, q=q.to(BF), rows=torch.zeros(B, dtype=torch.int64))
        check_v(out[look], dict(c, q=q.to(BF)[look], ctx=[4000] * 3, bt=c["bt"].expand(3, -1)))


@pytest.mark.parametrize("G", [2, 8])
def test_v_scales_down_to_2_100_of_the_largest_and_subnormal_ones(cuda, G):
    for top, low in ((2.0 ** 60, 2.0 ** -40), (2.0 ** -10, 2.0 ** -110), (2.0 ** -100, 2.0 ** -128)):
        c = make_case([100, 65], G, 2, 64, 150 + G)
        v = rows(c, 151, 2).float()
        v[::2] *= low
        v[1::2] *= top
        v.view(-1, 2, 4, 32)[1::4, :, 1] *= low / top
        c = with_v(c, v.to(BF))
        check_v(call(c, cuda), c)


@pytest.mark.parametrize("G", [1, 2, 4, 8])
def test_v_groups_that_are_not_finite_among_scales_of_every_size(cuda, G):
    """NaN, zero and far-apart scales in the same tiles."""
    c = make_case([200], G, 2, 64, 160 + G)
    v = rows(c, 161, 2).float()
    at = slots_of(c, 0)
    v[at[::3]] *= 2.0 ** -40
    v[at[5::7]] = 0
    v[at[100], 1, 40] = math.inf
    c = with_v(c, v.to(BF))
    out = call(c, cuda).cpu()
    check(out, c)
    bad = torch.isnan(out)
    assert bad[0, G:, 32:64].all() and bad.sum() == 32 * G


# --------------------------------------------------------------------------- queries of very different magnitude
@pytest.mark.parametrize("e", [-20, -28, -40, -60, -90])
@pytest.mark.parametrize("G", [1, 2, 4, 8])
def test_small_query_elements_that_meet_large_keys(cuda, G, e):
    """One group of q at 2^e of the others, where K is 2^-e times the others': all groups count alike in a logit."""
    c = make_case([200, 65, 2], G, 2, 64, 170 + G)
    up = torch.ones(4, 32)
    up[G % 4] = 2.0 ** -e
    k = rows(c, 171, 2).float().view(-1, 2, 4, 32) * up
    c["kp"] = O.pool_from_rows(k.view(-1, 2, 128).to(BF), 64, False)
    c["q"] = (c["q"].float().view(3, -1, 4, 32) / up).view(3, -1, 128).to(BF)
    for scale in (SCALE, -SCALE, 2.0):
        check_v(call(c, cuda, scale=scale), c, scale=scale)


@pytest.mark.parametrize("top", [110, 125, -100, -124])
@pytest.mark.parametrize("G", [1, 2, 4, 8])
def test_queries_at_the_ends_of_bf16(cuda, G, top):
    """q near 2^top and K near 2^-top: ordinary logits.  Other heads of the same kv head have q of zero or tiny q."""
    c = make_case([130, 1], G, 2, 64, 180 + G)
    low = max(-top, -120)
    k = rows(c, 181, 2).float() * 2.0 ** low
    c["kp"] = O.pool_from_rows(k.to(BF), 64, False)
    q = c["q"].float().clamp(-3, 3) * 2.0 ** (min(-low, 125))
    if G > 1:
        q[:, 1] = 0
        q[:, 2 * G - 1] *= 2.0 ** -60
    c["q"] = q.to(BF)
    check_v(call(c, cuda), c)


@pytest.mark.parametrize("scale", [1e-30, 1e-38, 1e30, 0.0])
def test_softmax_scales_of_every_size(cuda, scale):
    """A scale that q or K makes up for."""
    for G in (2, 8):
        c = make_case([130, 3], G, 2, 64, 190 + G)
        f = 1.0 if scale == 0 else 0.1 / scale
        a = 2.0 ** round(math.log2(f) / 2)
        k = rows(c, 191, 2).float() * a
        c["kp"] = O.pool_from_rows(k.to(BF), 64, False)
        c["q"] = (c["q"].float() * a).to(BF)
        check_v(call(c, cuda, scale=scale), c, scale=scale)


@pytest.mark.parametrize("G", [1, 2, 4, 8])
def test_a_query_that_is_not_finite_spoils_its_own_head_only(cuda, G):
    c = make_case([150, 20], G, 2, 64, 200 + G)
    clean = c["q"].clone()
    for bad in (math.nan, math.inf, -math.inf):
        c["q"] = clean.clone()
        c["q"][0, G, 17] = bad
        out = call(c, cuda).cpu()
        nan = torch.isnan(out)
        assert nan[0, G].all() and nan.sum() == 128
        check(out, c)


@pytest.mark.parametrize("G", [1, 2, 4, 8])
def test_tiles_of_zeros(cuda, G):
    """A pool never written reads as zeros; tiles and tokens of zero V before, between and after others, with most of
    the probability or little of it."""
    for e in (0, 30):
        for pick in (lambda t: t < 64, lambda t: (t >= 64) & (t < 128), lambda t: t >= 190, lambda t: t % 5 == 0,
                     lambda t: t < 130, lambda t: t >= 0):
            c = logits_case(lambda t: torch.where(pick(t), 0.0, -e * math.log(2.0)) + torch.sin(t.float()), G, 2,
                            [200, 70], 220 + G)
            v = rows(c, 221, 2)
            for b in (0, 1):
                v[slots_of(c, b)[pick(torch.arange(c["ctx"][b]))]] = 0
            c = with_v(c, v)
            check_v(call(c, cuda), c)


@pytest.mark.parametrize("level", [-90, -40, 60])
@pytest.mark.parametrize("scale", [2.0 ** -80, SCALE, 2.0 ** 45])
def test_small_query_elements_at_every_scale(cuda, scale, level):
    """Query elements near 2^level and 2^-70 of that, K to make up for both, so that logits are ordinary whatever the
    softmax scale."""
    low = round(-level - math.log2(scale / SCALE))
    if low + 70 > 120:
        level, low = level + (low - 50), 50
    for G in (1, 8):
        c = make_case([130, 3], G, 2, 64, 230 + G)
        k = rows(c, 231, 2).float().view(-1, 2, 4, 32) * 2.0 ** max(low, -120)
        k[:, :, 1] *= 2.0 ** 70
        q = c["q"].float().view(2, -1, 4, 32) * 2.0 ** level
        q[:, :, 1] *= 2.0 ** -70
        c["kp"] = O.pool_from_rows(k.view(-1, 2, 128).to(BF), 64, False)
        c["q"] = q.view(2, -1, 128).to(BF)
        assert c["q"].isfinite().all() and k.isfinite().all()
        check_v(call(c, cuda, scale=scale), c, scale=scale)
