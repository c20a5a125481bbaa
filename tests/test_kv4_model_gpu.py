"""The model and the engine over the 4-bit KV cache (init_kv_cache(kv_bits=4), LLM(kv_bits=4)): what is stored,
prefill against decode, decode against the CPU oracle over the cache's own values, hand-offs."""
import pytest
import torch

from oracle import kv4 as O
from oracle.qwen3_oracle import Qwen3Oracle
from oracle.weights import TINY, TINY_G4, init_weights, random_prompts

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
TOL = 2e-2  # logits max-abs between two bf16 computations of the same values (as for the bf16 cache)


@pytest.fixture(autouse=True)
def _clean_error_word(cuda):
    from awesome_acceleration_b200 import _lib
    _lib.clear_device_error()
    yield
    assert _lib.device_error() == 0


def make(arch, sd, slots, max_seq_len, kv_bits=4, block_size=256, **kw):
    from awesome_acceleration_b200.model.model import Qwen3Config, Qwen3ForCausalLM
    cfg = Qwen3Config(**{k: v for k, v in arch.as_dict().items() if k in Qwen3Config.__annotations__})
    with torch.device("meta"):
        m = Qwen3ForCausalLM(cfg)
    m = m.to_empty(device="cuda").to(BF)
    m.load_state_dict({k: v.to(BF) for k, v in sd.items()}, strict=False)
    for k, v in kw.items():
        setattr(m, k, v)
    m.fuse_qkv()
    m.init_kv_cache(slots, max_seq_len, "cuda", BF, block_size=block_size, kv_bits=kv_bits)
    return m


def dequantised(x):
    """bf16 rows as the 4-bit cache reads them back."""
    n, s = O.quantise(x)
    return (n.double() * s.double().repeat_interleave(32, -1)).to(BF)


@pytest.mark.parametrize("arch,block_size", [(TINY, 64), (TINY_G4, 256)])
def test_prefill_stores_the_quantised_rows(cuda, arch, block_size):
    """Layer 0's K and V do not depend on attention: the 4-bit cache holds the quantisation of the bf16 cache's."""
    sd = init_weights(arch, 70, norm_jitter=0.1)
    prompts = [p[:n] for p, n in zip(random_prompts(3, 300, arch.vocab_size, 71), [300, 1, 130])]
    a = make(arch, sd, 3, 512, kv_bits=16, block_size=block_size)
    b = make(arch, sd, 3, 512, block_size=block_size, prefill_chunk_tokens=128)
    for m in (a, b):
        m._rt().prefill(prompts, [2, 0, 1])
    for row, p in zip([2, 0, 1], prompts):
        for x, y in zip(a.kv.gather(0, row, len(p)), b.kv.gather(0, row, len(p))):
            assert torch.equal(dequantised(x.cpu()), y.cpu())


def test_chunked_prefill_equals_whole(cuda):
    """What a chunk attends to is what the cache holds, so cutting the prompts differently changes only the order
    of sums."""
    sd = init_weights(TINY, 72, norm_jitter=0.1)
    prompts = [p[:n] for p, n in zip(random_prompts(3, 600, TINY.vocab_size, 73), [600, 257, 90])]
    res = []
    for chunk in (1 << 20, 256, 100):
        m = make(TINY, sd, 3, 1024, prefill_chunk_tokens=chunk)
        tok, lg = m._rt().prefill(prompts, [0, 1, 2], last_logits=True)
        res.append((tok.cpu(), lg.float().cpu()))
    for tok, lg in res[1:]:
        assert (lg - res[0][1]).abs().max().item() <= TOL


class CacheOracle(Qwen3Oracle):
    """The CPU oracle with its K and V taken from a model's cache, the new tokens' among them: the values that
    the model attends to.  (Its own K/V, a bf16 step off here and there, would now and then quantise to the
    neighbouring code, a whole step of 1/7 of the group's maximum.)"""

    def __init__(self, arch, sd, model, rows, lens):
        super().__init__(arch, sd, BF, num_slots=1, max_seq_len=1)
        self.k_cache = [{r: model.kv.gather(i, r, n)[0].cpu() for r, n in zip(rows, lens)}
                        for i in range(arch.num_hidden_layers)]
        self.v_cache = [{r: model.kv.gather(i, r, n)[1].cpu() for r, n in zip(rows, lens)}
                        for i in range(arch.num_hidden_layers)]

    def logits(self, row, tokens, first):
        """Logits of `tokens` at positions first, first + 1, ... of cache row `row`, causal."""
        from oracle import qwen3_oracle as Q
        eps, lin = self.arch.rms_norm_eps, torch.nn.functional.linear
        cos, sin = self.rope_rows(list(range(first, first + len(tokens))))
        hidden = self.w["model.embed_tokens.weight"][torch.tensor(tokens)]
        for i in range(self.arch.num_hidden_layers):
            q, k, _ = self._qkv(i, Q.rms_norm(hidden, self._lw(i, "input_layernorm.weight"), eps))
            q, _ = Q.apply_rope(q, k, cos, sin)
            o = torch.cat([Q.fa.attend(q[t:t + 1], self.k_cache[i][row][:first + t + 1],
                                       self.v_cache[i][row][:first + t + 1], self.scaling, False)
                           for t in range(len(tokens))])
            hidden = hidden + lin(o.reshape(len(tokens), -1), self._lw(i, "self_attn.o_proj.weight"))
            hidden = hidden + self._mlp(i, Q.rms_norm(hidden, self._lw(i, "post_attention_layernorm.weight"), eps))
        return self.head(hidden).float()


def test_last_token_by_prefill_and_by_decode(cuda):
    """The last prompt token's logits through kv4_load + prefill attention and through kv4_decode_attention, each
    against the oracle over the values in its cache."""
    for arch, lens in ((TINY, [65, 2, 200]), (TINY_G4, [64, 129, 3])):
        sd = init_weights(arch, 74, norm_jitter=0.1)
        prompts = [p[:n] for p, n in zip(random_prompts(3, 200, arch.vocab_size, 75), lens)]
        m = make(arch, sd, 6, 256, block_size=64)
        rt = m._rt()
        _, whole = rt.prefill(prompts, [0, 1, 2], last_logits=True)
        rt.prefill([p[:-1] for p in prompts], [3, 4, 5])
        rt.load_decode_inputs([p[-1] for p in prompts], [n - 1 for n in lens], [3, 4, 5])
        lg = torch.empty((3, arch.vocab_size), dtype=BF, device=cuda)
        rt.decode_step([3, 4, 5], logits=lg)
        orc = CacheOracle(arch, sd, m, range(6), lens + lens)
        for b, p in enumerate(prompts):
            assert (whole[b].float().cpu() - orc.logits(b, p, 0)[-1]).abs().max().item() <= TOL
            # the hidden states of the tokens before are in the cache only, so the last token alone is enough
            assert (lg[b].float().cpu() - orc.logits(3 + b, p[-1:], len(p) - 1)[0]).abs().max().item() <= TOL


@pytest.mark.parametrize("graphs", [False, True])
def test_decode_steps_against_the_oracle_over_the_cached_values(cuda, graphs):
    arch = TINY_G4
    sd = init_weights(arch, 76, norm_jitter=0.1)
    lens, rows = [63, 1, 140, 64, 7], [3, 1, 0, 4, 2]
    prompts = [p[:n] for p, n in zip(random_prompts(5, 140, arch.vocab_size, 77), lens)]
    m = make(arch, sd, 5, 256, block_size=64, use_cuda_graphs=graphs)
    rt = m._rt()
    feed = rt.prefill(prompts, rows).tolist()
    pos = list(lens)
    rt.load_decode_inputs(feed, pos, rows)
    for step in range(4):
        if graphs:
            rt.decode_step(rows)
            got = rt.read_tokens(5)
        else:
            lg = torch.empty((5, arch.vocab_size), dtype=BF, device=cuda)
            got = rt.decode_step(rows, logits=lg).tolist()
        orc = CacheOracle(arch, sd, m, rows, [p + 1 for p in pos])
        for b, row in enumerate(rows):
            want = orc.logits(row, feed[b:b + 1], pos[b])[0]
            if not graphs:
                assert (lg[b].float().cpu() - want).abs().max().item() <= TOL
            # the token is a maximum of the oracle's logits within the tolerance
            assert want.max().item() - want[got[b]].item() <= 2 * TOL
        feed, pos = got, [p + 1 for p in pos]


def test_decode_graph_equals_eager(cuda):
    sd = init_weights(TINY, 78, norm_jitter=0.1)
    prompts = [p[:n] for p, n in zip(random_prompts(5, 70, TINY.vocab_size, 79), [70, 3, 33, 64, 65])]
    outs = []
    for graphs in (False, True):
        # eager steps run 5 rows, graphs the 8-row bucket with three padding rows
        m = make(TINY, sd, 5, 256, use_cuda_graphs=graphs, block_size=64)
        rt = m._rt()
        rows = [4, 2, 0, 1, 3]
        first = rt.prefill(prompts, rows).tolist()
        rt.load_decode_inputs(first, [len(p) for p in prompts], rows)
        seq = [first]
        for _ in range(8):
            rt.decode_step(rows)
            seq.append(rt.read_tokens(5))
        outs.append(seq)
    assert outs[0] == outs[1]


def test_llm_generates_over_a_4_bit_cache(cuda):
    """Continuous batching with more prompts than slots: every future resolves, and the same requests give the
    same tokens again."""
    from awesome_acceleration_b200.llm import LLM
    sd = init_weights(TINY, 80, norm_jitter=0.1)
    prompts = [p[:n] for p, n in zip(random_prompts(7, 60, TINY.vocab_size, 81), [60, 1, 13, 33, 2, 59, 20])]
    runs = []
    for _ in range(2):
        m = make(TINY, sd, 1, 64)
        llm = LLM(model=m, max_num_seqs=3, max_seq_len=200, kv_bits=4)
        assert m.kv.bits == 4 and llm.max_num_seqs == 3
        out = llm.generate_ids(prompts, max_tokens=10, ignore_eos=True).result(timeout=120)
        llm.stop()
        assert [o.generated_tokens for o in out] == [10] * 7
        runs.append([o.token_ids for o in out])
    assert runs[0] == runs[1]
    with pytest.raises(ValueError, match="kv_bits"):
        LLM(model=make(TINY, sd, 1, 64), max_num_seqs=1, max_seq_len=64, kv_bits=8)


def test_export_and_import_between_caches(cuda):
    """A 4-bit cache exports the values it holds; importing quantises again, at most another half step off."""
    sd = init_weights(TINY, 82, norm_jitter=0.1)
    m = make(TINY, sd, 4, 256)
    wide = make(TINY, sd, 4, 256, kv_bits=16)
    n = 200
    prompt = random_prompts(1, n, TINY.vocab_size, 83)[0]
    m._rt().prefill([prompt], [0])
    payload = m.export_request_kv(0, n)
    m.import_request_kv(3, payload, n)
    wide.import_request_kv(1, payload, n)
    for i in range(TINY.num_hidden_layers):
        for x, y, z in zip(m.kv.gather(i, 0, n), m.kv.gather(i, 3, n), wide.kv.gather(i, 1, n)):
            assert torch.equal(x, z)
            assert torch.equal(dequantised(x.cpu()), y.cpu())
            # half a step of s <= (max|x| / 7)(1 + 2^-8), and the rounding of what is read back to bf16
            step = x.float().reshape(n, -1, 4, 32).abs().amax(-1, keepdim=True) / 7 * (1 + 2.0 ** -8)
            off = (x.float() - y.float()).reshape(n, -1, 4, 32).abs()
            assert (off <= 0.5 * step * (1 + 2.0 ** -7) + 2.0 ** -8 * 7 * step).all()
    assert m.kv.lengths[3] == n


def test_kv_ipc_ticket_into_a_4_bit_cache(cuda):
    """import_request_kv_ipc's storing call, with the exporter's buffer in this process."""
    from awesome_acceleration_b200 import _lib
    from awesome_acceleration_b200 import kernels as K
    hkv, n = 2, 70
    x = torch.randn((2, n, hkv, 128), generator=torch.Generator().manual_seed(1)).to(BF).to(cuda)
    kd = torch.zeros(K.kv4_cache_shape(2, hkv, 64), dtype=torch.uint8, device=cuda)
    vd = torch.zeros_like(kd)
    slots = torch.arange(n, device=cuda)
    rs = hkv * 128
    assert _lib.load().aacc_kv4_store(x[0].data_ptr(), x[1].data_ptr(), n, rs, 128, rs, 128, slots.data_ptr(),
                                      kd.data_ptr(), vd.data_ptr(), 2, hkv, 64,
                                      torch.cuda.current_stream().cuda_stream) == 0
    k, v = K.kv4_load(kd, vd, slots)
    assert torch.equal(k.cpu(), dequantised(x[0].cpu())) and torch.equal(v.cpu(), dequantised(x[1].cpu()))
