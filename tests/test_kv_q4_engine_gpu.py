"""QwenEngine with the 4-bit KV cache: decode, dense prefill and the next turn behind a cached context."""
import dataclasses

import numpy as np
import pytest
import torch

from oracle import mirror as M
from tests import _kv_q4 as R

pytestmark = pytest.mark.gpu


class QuantisedCache:
    """The oracle's KV cache with each row replaced by what the 4-bit cache holds of it."""

    def __init__(self, inner):
        self.inner = inner

    def append(self, layer, pos, k, v):
        def held(x):
            codes, scales = R.quantise(np.asarray(x, np.float16).reshape(-1, 128))
            return R.values(codes, scales).astype(np.float16).reshape(np.shape(x))
        self.inner.append(layer, pos, held(k), held(v))

    def rows(self, layer):
        return self.inner.rows(layer)


@pytest.fixture(scope="module")
def model():
    from llamamps_b200.config import QWEN2_5_1_5B
    from llamamps_b200.weights import model_host_arrays, synth_model
    cfg = dataclasses.replace(QWEN2_5_1_5B, n_layers=2, vocab=8192)
    mw = synth_model(cfg, seed=41, device="cuda")
    return cfg, mw, model_host_arrays(mw)


def _engine(mw, **kw):
    from llamamps_b200.engine import QwenEngine
    return QwenEngine(weights=mw, kv_bits=4, **kw)


def test_logits_follow_the_quantised_oracle(cuda, model):
    """Logits at 40 positions, fed the same tokens: nearer to the oracle with quantised K and V than half of
    what the quantisation itself moves them.  (K rows that differ by an fp16 step may land on another code: at
    most a few in a thousand elements, each off by one step where quantising leaves all of them off by a
    twelfth of its square; so a tenth or so is expected.)"""
    cfg, mw, host = model
    eng = _engine(mw, max_seq_len=64)
    q4, fp = (M.OracleModel(host, M.OracleConfig(n_layers=2, vocab=cfg.vocab)) for _ in range(2))
    q4.cache = QuantisedCache(q4.cache)
    ids = np.random.default_rng(3).integers(0, cfg.vocab, 40)
    off = moved = 0.0
    for t in ids:
        vec = host["embed"][t]
        got, want, plain = eng.run_inference(vec).astype(np.float64), q4.step_vector(vec), fp.step_vector(vec)
        off += np.square(got - want.astype(np.float64)).sum()
        moved += np.square(plain.astype(np.float64) - want.astype(np.float64)).sum()
    assert moved > 0 and off <= 0.25 * moved, f"rms off the quantised oracle {off ** 0.5:.3g}, moved {moved ** 0.5:.3g}"


@pytest.mark.parametrize("batch,page_size", [(3, 64), (6, 16)])
def test_graph_eager_and_batch_agree(cuda, model, batch, page_size):
    """Graph replay, eager launches and permuted pages give the same ids; sequences do not depend on their batch."""
    cfg, mw, _ = model
    prompts = np.random.default_rng(5).integers(0, cfg.vocab, (batch, 9))
    kw = dict(max_batch=batch, max_seq_len=96, page_size=page_size, gemv_max_batch=8)
    eng = _engine(mw, **kw)
    ids = eng.generate_batch(prompts, 12)
    assert np.array_equal(_engine(mw, use_graphs=False, **kw).generate_batch(prompts, 12), ids)
    n = eng.cache.n_pages
    order = list(np.random.default_rng(6).permutation(n))
    assert np.array_equal(_engine(mw, page_order=order, **kw).generate_batch(prompts, 12), ids)
    for b in range(batch):
        assert np.array_equal(eng.generate_batch(prompts[b:b + 1], 12)[0], ids[b])


def test_dense_prefill_and_next_turn_fill_the_same_cache(cuda, model):
    """The cached values after a dense prefill, after two dense chunks (the second behind the first) and after
    the prompt token by token: layer 0's rows (same inputs) within fp16 roundings of the projection and one code
    step; decoding goes on from there."""
    from llamamps_b200 import kernels as K
    cfg, mw, _ = model
    B, P, cut = 2, 200, 70
    prompts = torch.from_numpy(np.random.default_rng(7).integers(0, cfg.vocab, (B, P)).astype(np.int32)).cuda()
    engines = [_engine(mw, max_batch=B, max_seq_len=256) for _ in range(3)]
    for e in engines:
        e.reset(B)
        e._ensure_history(4)
    engines[0].prefill(prompts, dense=True)
    engines[1].prefill(prompts[:, :cut], dense=True)
    engines[1].prefill(prompts[:, cut:], dense=True)
    engines[2].prefill(prompts, dense=False)
    for e in engines:
        assert e.host_pos == P and e.pos[:B].tolist() == [P] * B and e.seq_lens[:B].tolist() == [P + 1] * B
        e.check_kv_error()
    for b in range(B):
        k0, v0 = engines[0].cache.read_positions(b, 0, P)
        scale = k0.float().unflatten(1, (-1, 32)).abs().amax(-1).repeat_interleave(32, 1) / 7
        vscale = v0.float().unflatten(1, (-1, 32)).abs().amax(-1).repeat_interleave(32, 1) / 7
        for e in engines[1:]:
            k, v = e.cache.read_positions(b, 0, P)
            assert ((k - k0).float().abs() <= 1.02 * scale + 1e-6).all()
            assert ((v - v0).float().abs() <= 1.02 * vscale + 1e-6).all()
            assert ((k != k0).float().mean() < 0.05) and ((v != v0).float().mean() < 0.05)
    for e in engines:
        e.decode_steps(3)
        e.check_kv_error()
        assert e.pos[:B].tolist() == [P + 3] * B
    assert K.Q4_ROW_BYTES * 2 * cfg.n_kv_heads * cfg.n_layers == cfg.kv_bytes_per_position(4)


def test_sampled_generation_is_reproducible(cuda, model):
    cfg, mw, _ = model
    eng = _engine(mw, max_seq_len=64)
    a = eng.generate([5, 900, 77], 10, temperature=0.9, top_k=20, seed=4)
    assert eng.generate([5, 900, 77], 10, temperature=0.9, top_k=20, seed=4) == a


def test_reported_errors_raise(cuda, model):
    """A block table entry outside the pool is not followed: the engine raises, and works again after a repair."""
    cfg, mw, _ = model
    eng = _engine(mw, max_seq_len=64, use_graphs=False)
    ids = eng.generate([1, 2, 3], 4)
    eng.reset(1)
    eng.cache.block_table[0, 0] = eng.cache.n_pages + 3
    with pytest.raises(RuntimeError, match="outside the pool"):
        eng.step_tokens([1])
    eng.cache.block_table[0, 0] = eng.cache.pages(0)[0]
    assert eng.generate([1, 2, 3], 4) == ids


def test_refusals_and_launches(cuda, model):
    from llamamps_b200.engine import QwenEngine
    cfg, mw, _ = model
    for decoder in ("persistent", "batched"):
        with pytest.raises(ValueError, match="fp16 cache"):
            QwenEngine(weights=mw, kv_bits=4, decoder=decoder)
    with pytest.raises(ValueError, match="kv_bits"):
        QwenEngine(weights=mw, kv_bits=8)
    with pytest.raises(ValueError, match="page_size"):
        QwenEngine(weights=mw, kv_bits=4, page_size=24)
    # embedding, 2 x 7 in the layers, final norm, head and its argmax, advance
    assert _engine(mw, max_seq_len=64).launches_per_step() == 1 + 2 * 7 + 1 + 2 + 1
    eng = _engine(mw, max_seq_len=64)
    with pytest.raises(ValueError, match="longer"):
        eng.prefill(torch.zeros(1, 64, dtype=torch.int32))
