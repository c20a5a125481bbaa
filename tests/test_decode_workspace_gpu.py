"""One workspace of the bf16 decode attention, shared in turn by calls of different batches, heads' splits and contexts
(as the decode step's batch buckets share it)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def K():
    from awesome_acceleration_b200 import kernels
    return kernels


def make(ctx, hq, hkv, bs, seed, dev):
    g = torch.Generator().manual_seed(seed)
    need = [-(-c // bs) for c in ctx]
    nb, mb = sum(need) + 1, max(need)
    perm, at = torch.randperm(nb, generator=g).to(torch.int32), 0
    bt = torch.full((len(ctx), mb), -1, dtype=torch.int32)
    for i, n in enumerate(need):
        bt[i, :n] = perm[at:at + n]
        at += n
    kv = torch.randn((2, nb, hkv, bs, 128), generator=g).to(BF).to(dev)
    return dict(q=torch.randn((len(ctx), hq, 128), generator=g).to(BF).to(dev), k=kv[0], v=kv[1], bt=bt.to(dev),
                rows=torch.arange(len(ctx), device=dev), lens=torch.tensor(ctx, dtype=torch.int32, device=dev))


def call(c, ws, max_context, split):
    out = torch.full_like(c["q"], math.nan)  # an output that nothing writes shows
    return K().paged_decode_attention(c["q"], c["k"], c["v"], c["bt"], c["rows"], c["lens"], ctx_add=0,
                                      scale=128 ** -0.5, max_context=max_context, workspace=ws, out=out,
                                      split_tokens=split)


@pytest.mark.parametrize("split", [0, 64, 512])
def test_calls_of_different_batches_share_a_workspace(cuda, split):
    from awesome_acceleration_b200 import _lib
    _lib.clear_device_error()
    hq, hkv, bs, max_context = 16, 8, 64, 6144
    ctxs = [[6144] * 64, [6000, 3, 2500], [5000], [700] * 7 + [4097], [1, 64, 6144, 65] * 8]
    cases = [make(c, hq, hkv, bs, i, cuda) for i, c in enumerate(ctxs)]
    size = K().decode_workspace_bytes(64, hq, max_context, split)
    alone = [call(c, torch.zeros(size, dtype=torch.uint8, device=cuda), max_context, split) for c in cases]
    assert all(torch.isfinite(a).all() for a in alone)
    ws = torch.zeros(size, dtype=torch.uint8, device=cuda)
    for order in ([0, 1, 2, 3, 4], [4, 3, 0, 2, 1], [1, 1, 0, 0, 3, 2, 4]):
        for i in order:
            assert torch.equal(call(cases[i], ws, max_context, split), alone[i])
    assert _lib.device_error() == 0
