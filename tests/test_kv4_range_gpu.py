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
