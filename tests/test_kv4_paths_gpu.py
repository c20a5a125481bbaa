"""The 4-bit cache on the paths around one model on one GPU: a prefill's scratch memory, the tensor-parallel model and
engine, the hand-off over CUDA IPC, one row named twice in a decode batch."""
import weakref

import pytest
import torch

from oracle.weights import TINY, TINY_G4, init_weights, random_prompts
from test_kv4_gpu import SCALE, call, check, make_case
from test_kv4_model_gpu import TOL, CacheOracle, dequantised, make

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


@pytest.fixture(autouse=True)
def _clean_error_word(cuda):
    from awesome_acceleration_b200 import _lib
    _lib.clear_device_error()
    yield
    assert _lib.device_error() == 0


def test_prefill_holds_one_chunks_scratch_at_a_time(cuda):
    """What sizing counts: a chunk's bf16 context and staging rows are gone before the next chunk's are made."""
    m = make(TINY, init_weights(TINY, 84, norm_jitter=0.1), 4, 512, prefill_chunk_tokens=96)
    rt = m._rt()
    inner, alive, seen = rt._prefill_chunk, [], 0

    def chunk(*args):
        nonlocal seen
        assert not [r for r in alive if r() is not None], "the chunk before still holds its scratch"
        slots, attend = inner(*args)
        alive.append(weakref.ref(attend))
        seen += 1
        return slots, attend
    rt._prefill_chunk = chunk
    prompts = [p[:n] for p, n in zip(random_prompts(4, 200, TINY.vocab_size, 85), [200, 1, 150, 60])]
    rt.prefill(prompts, [0, 1, 2, 3])
    assert seen == 5
