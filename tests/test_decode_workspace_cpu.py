"""The bf16 decode attention's workspace holds every call of fewer rows and shorter contexts, and the counters of one
never lie where another has partials."""
import pytest

from awesome_acceleration_b200 import _lib

ROW = (128 + 2) * 4  # fp32 partial O, max and sum of a query head and split


def splits(batch, hkv, ctx, split_tokens):
    """The splits of a call, as documented: a CTA's share of eight CTAs per SM, whole tiles, at most 2048 tokens."""
    if split_tokens <= 0:
        want = -(-148 * 8 // (batch * hkv))
        split_tokens = min(max(-(-(-(-ctx // want)) // 64) * 64, 64), 2048)
    return -(-ctx // split_tokens)


@pytest.mark.parametrize("hq,hkv", [(1, 1), (8, 1), (16, 8), (5, 5)])
@pytest.mark.parametrize("split_tokens", [0, 64, 1024])
def test_workspace_holds_smaller_calls(hq, hkv, split_tokens):
    size = _lib.load().aacc_paged_decode_workspace_bytes
    for batch in (1, 2, 7, 8, 33, 256, 1500):
        for ctx in (1, 64, 700, 9536, 40960):
            ws = size(batch, hq, ctx, split_tokens)
            counters = batch * hkv * 4  # at the end, of the largest call
            for b in {1, 2, 3, 7, batch // 2, batch - 1, batch} - {0}:
                for c in {1, 64, ctx // 2, ctx - 64, ctx}:
                    if b <= batch and 0 < c <= ctx:
                        n = splits(b, hkv, c, split_tokens)
                        assert n == 1 or b * hq * n * ROW + counters <= ws, (batch, ctx, b, c)
