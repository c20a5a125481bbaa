"""The 4-bit KV cache and request maps without a GPU: the oracle's storage format, and what the entry points
refuse before any CUDA call."""
import pytest
import torch

from awesome_acceleration_b200 import _lib
from awesome_acceleration_b200 import kernels as K
from oracle import kv4 as O

BF = torch.bfloat16


def test_every_nibble_has_one_place_and_packing_round_trips():
    for value in (False, True):
        assert sorted(O.nibble_places(value).flatten().tolist()) == list(range(2 * 4096))
        x = torch.randn((3, 64, 128), generator=torch.Generator().manual_seed(int(value))).to(BF)
        n, s = O.quantise(x)
        rec = O.pack(x, value)
        assert rec.shape == (3, 4608)
        assert torch.equal(O.unpack(rec, value), n.double() * s.double().repeat_interleave(32, -1))
        # a value is at most half a step of its group's scale off (7 s rounds within 2^-8 of max|x|)
        step = s.double().repeat_interleave(32, -1)
        assert ((O.unpack(rec, value) - x.double()).abs() <= step * (0.5 + 7 * 2.0 ** -8)).all()


def test_cache_shape():
    assert K.kv4_cache_shape(10, 8, 256) == (10, 8, 4, 4608)
    for bs in (0, -64, 63, 100):
        with pytest.raises(ValueError):
            K.kv4_cache_shape(1, 1, bs)


def test_wrappers_refuse_tensors_off_the_gpu():
    pool = torch.zeros(K.kv4_cache_shape(2, 2, 64), dtype=torch.uint8)
    rows, slots = torch.zeros((3, 2, 128), dtype=BF), torch.zeros(3, dtype=torch.int64)
    i32 = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(ValueError, match="current CUDA device"):
        K.kv4_store(rows, rows, slots, pool, pool)
    with pytest.raises(ValueError, match="current CUDA device"):
        K.kv4_load(pool, pool, slots)
    with pytest.raises(ValueError, match="current CUDA device"):
        K.kv4_decode_attention(rows, pool, pool, i32.view(1, 3), slots, i32, ctx_add=0, scale=1.0, max_context=64,
                               workspace=None)
    with pytest.raises(ValueError, match="current CUDA device"):
        K.build_block_tables(i32, 64, max_blocks=2)
    with pytest.raises(ValueError, match="current CUDA device"):
        K.build_slot_maps(i32, i32.view(1, 3), block_size=64, num_blocks=1, num_tokens=3)


def test_c_abi_checks_arguments_before_any_cuda_call():
    lib = _lib.load()
    st = lib.aacc_kv4_store

    def store(T=3, ks=256, kh=128, nb=2, hkv=2, bs=64, k=16, slots=16):
        return st(k, 16, T, ks, kh, 256, 128, slots, 16, 16, nb, hkv, bs, None)
    for kw in (dict(T=-1), dict(nb=0), dict(hkv=0), dict(bs=0), dict(bs=96), dict(ks=100), dict(kh=127), dict(k=8),
               dict(k=None), dict(slots=None)):
        assert store(**kw) == 1, kw
        assert b"kv4_store" in lib.aacc_last_error()
    assert store(T=2 ** 30, hkv=2) == 3 and store(nb=2 ** 25) == 3
    assert store(T=0) == 0

    def load(T=3, nb=2, hkv=2, bs=64, ob=3, obs=1, k=16):
        return lib.aacc_kv4_load(k, 16, nb, hkv, bs, 16, None, T, 16, 16, ob, obs, None)
    for kw in (dict(T=-1), dict(nb=0), dict(hkv=0), dict(bs=100), dict(ob=-1), dict(obs=0), dict(k=8),
               dict(k=None)):
        assert load(**kw) == 1, kw
        assert b"kv4_load" in lib.aacc_last_error()
    assert load(T=2 ** 30, hkv=2) == 3 and load(nb=2 ** 25) == 3 and load(ob=2 ** 31) == 3
    assert load(T=0) == 0

    def attend(B=2, hq=4, hkv=2, bs=64, nb=2, mb=2, rows=2, ctx=128, q=16):
        return lib.aacc_kv4_decode_attention(q, 16, 16, 16, nb, 16, rows, mb, 16, 16, 1, B, hq, hkv, bs, 0.1, ctx, None,
                                             0, None)
    for kw in (dict(B=-1), dict(hkv=0), dict(hq=0), dict(hq=5), dict(bs=96), dict(bs=0), dict(nb=0), dict(mb=0),
               dict(rows=-1), dict(ctx=0), dict(q=8), dict(q=None)):
        assert attend(**kw) == 1, kw
        assert b"kv4_decode_attention" in lib.aacc_last_error()
    for hq in (6, 32):
        assert attend(hq=hq) == 3, hq  # 3 and 16 query heads per kv head
    # units of work are counted in 32 bits
    assert attend(B=2 ** 31) == 3 and attend(B=2 ** 26, mb=2 ** 10, ctx=2 ** 16) == 3
    assert attend(B=0) == 0

    def tables(S=2, bs=64, nf=4, mb=2, lens=16):
        return lib.aacc_build_block_tables(lens, S, bs, None, nf, 16, mb, None, None)
    for kw in (dict(lens=None), dict(S=-1), dict(S=2 ** 31), dict(bs=0), dict(nf=-1), dict(mb=0)):
        assert tables(**kw) == 1, kw
    assert tables(S=0) == 0

    def maps(S=2, nr=2, mb=2, bs=64, nb=2, T=4, cu=16, slots=16):
        return lib.aacc_build_slot_maps(16, None, None, S, 16, nr, mb, bs, nb, cu, None, slots, T, None)
    for kw in (dict(cu=None), dict(slots=None), dict(S=-1), dict(nr=-1), dict(mb=0), dict(bs=0), dict(nb=0), dict(T=-1), dict(T=2 ** 31)):
        assert maps(**kw) == 1, kw


def test_cache_of_either_width():
    from awesome_acceleration_b200.kv_cache import PagedKV4Cache, PagedKVCache, kv_cache_class
    assert kv_cache_class(16) is PagedKVCache and kv_cache_class(4) is PagedKV4Cache
    for bits in (8, 0, 32):
        with pytest.raises(ValueError, match="kv_bits"):
            kv_cache_class(bits)
    kv = PagedKV4Cache(3, 2, 4, 1000, block_size=128, device="cpu")
    assert kv.k.shape == (3, kv.num_blocks, 2, 2, 4608) and kv.k.dtype == torch.uint8 and kv.bits == 4
    assert PagedKVCache.bytes_per_token_head() == 512 and PagedKV4Cache.bytes_per_token_head() == 144
    kv.reserve(1, 300)
    kv.sync()
    assert kv.block_tables[1, :4].tolist() == [0, 1, 2, -1]
    assert kv.slot_mapping(1, 127, 130).tolist() == [127, 128, 129]
    with pytest.raises(ValueError, match="bf16"):
        PagedKV4Cache(1, 1, 1, 64, device="cpu", dtype=torch.float16)


def test_runtime_of_either_width(monkeypatch):
    """The 4-bit runtime projects into its staging rows and stores them, then attends to the 4-bit pools."""
    import types

    from awesome_acceleration_b200 import runtime as R
    calls = []

    class Rec:
        CLUSTER_MAX_ROWS, SKINNY_MAX_ROWS = K.CLUSTER_MAX_ROWS, K.SKINNY_MAX_ROWS

        def __getattr__(self, name):
            return lambda *a, **kw: calls.append((name, a, kw))
    monkeypatch.setattr(R, "K", Rec())
    assert R.runtime_class(types.SimpleNamespace(bits=4)) is R.Qwen3RuntimeKV4
    assert R.runtime_class(types.SimpleNamespace(bits=16)) is R.Qwen3Runtime
    rt = R.Qwen3RuntimeKV4.__new__(R.Qwen3RuntimeKV4)
    rt.eps, rt.rope, rt.Hq, rt.Hkv, rt.skinny_rows, rt.cluster_gemm = 1e-6, None, 4, 2, 0, False
    rt.device, rt.scale, rt.max_context, rt.kv4_ws = torch.device("cpu"), 1.0, 256, None
    rt.kv = types.SimpleNamespace(k=["k0"], v=["v0"], block_tables="bt", seqlens="sl")
    rt._stage = rt._stage_decode = rt._staging(8)
    lw = types.SimpleNamespace(wqkv=torch.empty((1024, 256)), q_norm=None, k_norm=None)
    slot_map = torch.tensor([5, -1, 9])
    rt._qkv(0, lw, torch.empty((3, 256)), None, slot_map, None, None)
    assert [c[0] for c in calls] == ["qkv_norm_rope_store", "kv4_store"]
    a = calls[0][1]
    assert a[7].tolist() == [0, 1, 2] and a[8].shape == (8, 2, 1, 128)  # staging slots and pool
    k, v, slots, kc, vc = calls[1][1]
    assert k.shape == v.shape == (3, 2, 128) and slots is slot_map and (kc, vc) == ("k0", "v0")
    assert k.data_ptr() == rt._stage[0].data_ptr() and k.stride() == (256, 128, 1)
    rt._decode_attend(0, "q", "out", "rows")
    assert calls[2][0] == "kv4_decode_attention" and calls[2][1][:3] == ("q", "k0", "v0")


def test_sizing_leaves_room_for_a_chunk_of_many_short_prompts(monkeypatch):
    """A prefill chunk's scratch pool has a whole block for each sequence, however short."""
    from awesome_acceleration_b200.llm import kv_sized_max_seqs
    from awesome_acceleration_b200.model.model import Qwen3Config
    from awesome_acceleration_b200.runtime import Qwen3RuntimeKV4
    cfg = Qwen3Config(hidden_size=512, num_hidden_layers=1, num_attention_heads=4, num_key_value_heads=4, head_dim=128,
                      intermediate_size=1024, vocab_size=256)
    free = 4 << 30
    monkeypatch.setattr(torch.cuda, "synchronize", lambda *a: None)
    monkeypatch.setattr(torch.cuda, "empty_cache", lambda: None)
    monkeypatch.setattr(torch.cuda, "mem_get_info", lambda *a: (free, 180 << 30))
    chunk, seq, want = 4096, 1024, 4000
    n = kv_sized_max_seqs(cfg, want, seq, 1.0, "cuda", 1, chunk, 4)
    pool = n * seq * 4 * 144
    scratch = n * Qwen3RuntimeKV4.SCRATCH_BLOCK * 4 * 128 * 2 * 2  # n prompts of one token in one chunk
    rows = chunk * 4 * 128 * 2 * 2
    assert 1 < n < want and pool + scratch + rows <= free - (1 << 30)


def test_tensor_parallel_cache_has_its_ranks_heads():
    """A rank's 4-bit cache holds its share of the kv heads, and its runtime is the 4-bit one."""
    from awesome_acceleration_b200 import runtime as R
    from awesome_acceleration_b200.kv_cache import PagedKV4Cache
    from awesome_acceleration_b200.model import model_tp
    from awesome_acceleration_b200.model.model import Qwen3Config
    cfg = Qwen3Config(hidden_size=512, num_hidden_layers=2, num_attention_heads=8, num_key_value_heads=4, head_dim=128,
                      intermediate_size=1024, vocab_size=256)
    with torch.device("meta"):
        m = model_tp.Qwen3ForCausalLMTP(cfg)
    m.tp_size = 2
    m.init_kv_cache(3, 500, "cpu", torch.bfloat16, block_size=128, kv_bits=4)
    assert isinstance(m.kv, PagedKV4Cache) and m.kv.num_kv_heads == 2
    assert m.kv.k.shape == (2, m.kv.num_blocks, 2, 2, 4608) and m.max_batch == 3
    assert m.model.layers[1].self_attn._kv_cache.data_ptr() == m.kv.k[1].data_ptr()
    assert R.runtime_class(m.kv) is R.Qwen3RuntimeKV4
    m.init_kv_cache(3, 500, "cpu", torch.bfloat16, block_size=128)
    assert m.kv.bits == 16 and R.runtime_class(m.kv) is R.Qwen3Runtime
    with pytest.raises(ValueError, match="kv_bits"):
        m.init_kv_cache(3, 500, "cpu", torch.bfloat16, kv_bits=8)
