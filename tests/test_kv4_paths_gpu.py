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


@pytest.mark.parametrize("src_bits,dst_bits", [(4, 4), (16, 4), (4, 16)])
def test_ipc_hand_off_into_a_cache_of_either_width(cuda, monkeypatch, src_bits, dst_bits):
    """export_request_kv_ipc and import_request_kv_ipc themselves, the exporter's buffer opened in this process: the
    importer holds the exported values, quantised where its cache has 4 bits, in its own slots and block size."""
    from awesome_acceleration_b200 import kernels as K
    sd = init_weights(TINY, 86, norm_jitter=0.1)
    src = make(TINY, sd, 2, 256, kv_bits=src_bits)
    dst = make(TINY, sd, 4, 256, kv_bits=dst_bits, block_size=64)
    n = 130
    src._rt().prefill(random_prompts(1, n, TINY.vocab_size, 87), [1])
    dst._rt().prefill(random_prompts(2, 100, TINY.vocab_size, 88), [0, 3])
    kept = [dst.kv.gather(i, 3, 100) for i in range(TINY.num_hidden_layers)]
    ticket, owner = src.export_request_kv_ipc(1, n)
    opened = []
    monkeypatch.setattr(K, "peer_buffer_open", lambda handle: opened.append(handle) or owner.ptr)
    monkeypatch.setattr(K, "peer_buffer_close", lambda ptr: opened.append(ptr))
    dst.import_request_kv_ipc(2, ticket)
    assert opened == [ticket.handle, owner.ptr] and dst.kv.lengths[2] == n
    owner.release()
    for i in range(TINY.num_hidden_layers):
        for x, y in zip(src.kv.gather(i, 1, n), dst.kv.gather(i, 2, n)):
            want = dequantised(x.cpu()) if dst_bits == 4 else x.cpu()
            assert torch.equal(y.cpu(), want)
        assert all(torch.equal(x, y) for x, y in zip(kept[i], dst.kv.gather(i, 3, 100)))


def test_the_same_row_named_twice_and_more(cuda):
    """Every mention of a row is a query of its own, each held to the derived bound."""
    for G, hkv, ctx in ((2, 2, [5, 100, 64, 300, 1]), (8, 1, [3000, 7])):
        c = make_case(ctx, G, hkv, 64, 210 + G)
        rows = torch.tensor([0, len(ctx) - 1] * 3 + [1, 1, -1, 0])
        q = torch.randn((len(rows), G * hkv, 128), generator=torch.Generator().manual_seed(211)).to(BF)
        q[2] = q[0]
        out = call(c, cuda, rows=rows, q=q)
        at = rows.clamp(min=0)
        check(out, dict(c, q=q, bt=c["bt"][at], ctx=[ctx[r] if r >= 0 else 0 for r in rows.tolist()]), scale=SCALE)


# --------------------------------------------------------------------------- the tensor-parallel model and engine
def test_tensor_parallel_model_of_one_rank(cuda):
    """Qwen3ForCausalLMTP over a 4-bit cache: prefill in chunks and decode steps against the oracle over the cache's
    own values."""
    from awesome_acceleration_b200.model.model import Qwen3Config
    from awesome_acceleration_b200.model.model_tp import Qwen3ForCausalLMTP
    arch = TINY_G4
    sd = init_weights(arch, 89, norm_jitter=0.1)
    cfg = Qwen3Config(**{k: v for k, v in arch.as_dict().items() if k in Qwen3Config.__annotations__})
    m = Qwen3ForCausalLMTP.from_state_dict(sd, cfg, torch.device("cuda", 0))
    m.fuse_qkv()
    m.use_cuda_graphs, m.prefill_chunk_tokens = False, 100
    m.init_kv_cache(4, 256, torch.device("cuda", 0), BF, block_size=64, kv_bits=4)
    assert m.kv.bits == 4 and type(m._rt()).__name__ == "Qwen3RuntimeKV4"
    rt = m._rt()
    lens, rows = [130, 1, 64], [2, 0, 3]
    prompts = [p[:n] for p, n in zip(random_prompts(3, 130, arch.vocab_size, 90), lens)]
    feed, lg = rt.prefill(prompts, rows, last_logits=True)
    orc = CacheOracle(arch, sd, m, rows, lens)
    for b, (r, p) in enumerate(zip(rows, prompts)):
        assert (lg[b].float().cpu() - orc.logits(r, p, 0)[-1]).abs().max().item() <= TOL
    feed, pos = feed.tolist(), list(lens)
    rt.load_decode_inputs(feed, pos, rows)
    for _ in range(3):
        lg = torch.empty((3, arch.vocab_size), dtype=BF, device=cuda)
        got = rt.decode_step(rows, logits=lg).tolist()
        orc = CacheOracle(arch, sd, m, rows, [p + 1 for p in pos])
        for b, r in enumerate(rows):
            assert (lg[b].float().cpu() - orc.logits(r, feed[b:b + 1], pos[b])[0]).abs().max().item() <= TOL
        feed, pos = got, [p + 1 for p in pos]


def test_tensor_parallel_engine_of_one_rank(cuda):
    """LLMTP(kv_bits=4) gives what LLM(kv_bits=4) gives for the same weights and prompts."""
    from awesome_acceleration_b200.llm import LLM
    from awesome_acceleration_b200.llm_tp import LLMTP
    from awesome_acceleration_b200.model.model import Qwen3Config
    sd = init_weights(TINY, 91, norm_jitter=0.1)
    cfg = Qwen3Config(**{k: v for k, v in TINY.as_dict().items() if k in Qwen3Config.__annotations__})
    prompts = [p[:n] for p, n in zip(random_prompts(5, 70, TINY.vocab_size, 92), [70, 1, 13, 64, 40])]
    outs = []
    for engine in (LLMTP(None, max_num_seqs=3, max_seq_len=200, enable_tp=False, config=cfg, state_dict=sd, kv_bits=4),
                   LLM(model=make(TINY, sd, 1, 64), max_num_seqs=3, max_seq_len=200, kv_bits=4)):
        assert engine.model.kv.bits == 4
        out = engine.generate_ids(prompts, max_tokens=8, ignore_eos=True).result(timeout=120)
        engine.stop()
        assert [o.generated_tokens for o in out] == [8] * 5
        outs.append([o.token_ids for o in out])
    assert outs[0] == outs[1]
    with pytest.raises(ValueError, match="kv_bits"):
        LLMTP(None, max_num_seqs=1, max_seq_len=64, enable_tp=False, config=cfg, state_dict=sd, kv_bits=8)
