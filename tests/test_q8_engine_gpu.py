"""QwenEngine with 8-bit projections (w8a8): dense prefill, decode steps of larger batches, tensor-parallel ranks."""
import dataclasses
import threading

import numpy as np
import pytest
import torch

from tests import _q8 as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def model():
    from llamamps_b200.config import QWEN2_5_1_5B
    from llamamps_b200.weights import synth_model
    cfg = dataclasses.replace(QWEN2_5_1_5B, n_layers=2, vocab=8192)
    return cfg, synth_model(cfg, seed=43, device="cuda")


def _engine(mw, **kw):
    from llamamps_b200.engine import QwenEngine
    return QwenEngine(weights=mw, **{"w8a8": True, **kw})


def _prompts(cfg, B, P, seed=7):
    return torch.from_numpy(np.random.default_rng(seed).integers(0, cfg.vocab, (B, P)).astype(np.int32)).cuda()


def test_weights_in_8_bits(cuda, model):
    """The 8-bit copies against the values of the Q4 matrices, gate rows before up rows."""
    from llamamps_b200.quant import unpack_q4
    from llamamps_b200.weights import add_q8
    cfg, mw = model
    add_q8(mw)
    lw = mw.layers[1]
    kept = lw.q8
    add_q8(mw)
    assert lw.q8 is kept
    gate = unpack_q4(lw.gate_packed, lw.gate_scales, cfg.intermediate, cfg.hidden)
    up = unpack_q4(lw.up_packed, lw.up_scales, cfg.intermediate, cfg.hidden)
    p, s = lw.gate_packed[:16].cpu().numpy(), float(lw.gate_scales[0])
    first = np.stack([p & 15, p >> 4], axis=1).reshape(-1).astype(np.float64) - 8  # the first 32 elements of row 0
    assert np.array_equal(gate[0, :32].cpu().numpy(), (first * s).astype(np.float16))
    for (codes, scales), x in ((lw.q8.gate_up, torch.cat([gate, up])),
                               (lw.q8.down, unpack_q4(lw.down_packed, lw.down_scales, cfg.hidden, cfg.intermediate)),
                               (lw.q8.qkv, unpack_q4(lw.qkv_packed, lw.qkv_scales, cfg.qkv_rows, cfg.hidden)),
                               (lw.q8.o, unpack_q4(lw.o_packed, lw.o_scales, cfg.hidden, cfg.q_dim))):
        R.check_rows(x.double(), codes, scales)


@pytest.mark.parametrize("B,P", [(2, 200), (1, 300)])
def test_dense_prefill(cuda, model, B, P):
    """Layer 0's cached V rows are the formula's; the hidden rows behind both layers are off the fp16 activations'
    by what 8 bits take: a row's largest of 1536 elements is some 3.5 rms, so codes and weights are each off by
    3.5 / 127 / sqrt(12) = 0.8 % of a product, the long-tailed input of the down projection by two to three times
    as much; a few per cent together on the branches, less on the residual stream they join."""
    from llamamps_b200 import kernels as K
    cfg, mw = model
    prompts = _prompts(cfg, B, P)
    rows = []
    for w8a8 in (True, False):
        eng = _engine(mw, max_batch=B, max_seq_len=P + 8, w8a8=w8a8)
        eng.reset(B)
        eng._ensure_history(4)
        eng.prefill(prompts, dense=True)
        eng.check_gemm_error()
        rows.append(eng.buf_residual[:B].double())
        if w8a8:
            x = mw.embed[prompts.reshape(-1).long()].contiguous()
            lw = mw.layers[0]
            c, s = K.rms_norm_q8(x, lw.in_norm, cfg.eps)
            at = cfg.q_dim + cfg.kv_dim
            v = torch.cat([eng.cache.read_positions(b, 0, P)[1] for b in range(B)]).cuda()
            R.check_linear(v, c, s, lw.q8.qkv[0][at:], lw.q8.qkv[1][at:], lw.qkv_bias[at:])
            eng.decode_steps(3)
            assert eng.pos[:B].tolist() == [P + 3] * B
    off = float((rows[0] - rows[1]).norm() / rows[1].norm())
    assert 0.002 < off < 0.08, off


@pytest.mark.parametrize("kv_bits,batch", [(16, 6), (4, 6), (16, 40)])
def test_graph_eager_and_batch_agree(cuda, model, kv_bits, batch):
    """Graph replay and eager launches give the same ids, and a sequence the same ids in another batch."""
    cfg, mw = model
    prompts = _prompts(cfg, batch, 9, seed=5).cpu().numpy()
    kw = dict(max_batch=batch, max_seq_len=96, kv_bits=kv_bits, decoder="kernels")
    eng = _engine(mw, **kw)
    ids = eng.generate_batch(prompts, 10)
    assert np.array_equal(_engine(mw, use_graphs=False, **kw).generate_batch(prompts, 10), ids)
    assert np.array_equal(eng.generate_batch(prompts[:5], 10), ids[:5])


def test_launches(cuda, model):
    cfg, mw = model
    eng = _engine(mw, max_batch=8, max_seq_len=64, kv_bits=4)
    eng.reset(8)
    # embedding, 2 x (norm, q|k|v, attention, quantiser, o, norm, gate|up, quantiser, down), norm, head, argmax, advance
    assert eng.launches_per_step() == 1 + 2 * 9 + 1 + 2 + 1
    eng.reset(2)  # up to gemv_max_batch sequences the Q4 weights serve
    assert eng.launches_per_step() == 1 + 2 * 7 + 1 + 2 + 1


def test_small_batches_are_those_of_the_q4_engine(cuda, model):
    cfg, mw = model
    prompts = _prompts(cfg, 2, 9).cpu().numpy()
    kw = dict(max_batch=2, max_seq_len=64)
    assert np.array_equal(_engine(mw, **kw).generate_batch(prompts, 8), _engine(mw, w8a8=False, **kw).generate_batch(prompts, 8))


def test_the_batched_decoder_keeps_the_q4_weights(cuda, model):
    """decoder="batched": a dense prompt is in 8 bits as with the per-stage kernels, steps are those without w8a8."""
    cfg, mw = model
    B, P = 8, 40
    kw = dict(max_batch=B, max_seq_len=96, decoder="batched")
    short = _prompts(cfg, B, 5).cpu().numpy()
    eng = _engine(mw, **kw)
    assert np.array_equal(eng.generate_batch(short, 8), _engine(mw, w8a8=False, **kw).generate_batch(short, 8))
    stages = _engine(mw, max_batch=B, max_seq_len=96)
    assert stages.decoder == "kernels"
    for e in (eng, stages):
        e.reset(B)
        e._ensure_history(4)
        e.prefill(_prompts(cfg, B, P), dense=True)
        e.check_gemm_error()
    for b in range(B):
        for layer in range(2):
            for x, y in zip(eng.cache.read_positions(b, layer, P), stages.cache.read_positions(b, layer, P)):
                assert torch.equal(x, y)
    assert torch.equal(eng.tokens, stages.tokens)


def test_a_reported_timeout_raises(cuda, model):
    cfg, mw = model
    eng = _engine(mw, max_batch=8, max_seq_len=64)
    prompts = _prompts(cfg, 8, 5).cpu().numpy()
    ids = eng.generate_batch(prompts, 3)
    eng.gemm_err.fill_(1)
    with pytest.raises(RuntimeError, match="timed out"):
        eng.generate_batch(prompts, 3)
    assert np.array_equal(eng.generate_batch(prompts, 3), ids)


@pytest.mark.parametrize("kw", [dict(), dict(use_graphs=False), dict(decoder="kernels"), dict(kv_bits=4)])
def test_run_inference_raises_a_reported_timeout(cuda, model, kw):
    """Logits behind a prompt whose products gave up are not handed out, eager (the first token) and replayed (later
    ones), with a reset in between too; the error is raised once."""
    cfg, mw = model
    eng = _engine(mw, max_batch=1, max_seq_len=320, **kw)
    prompt, vec = _prompts(cfg, 1, 300), mw.embed[17].cpu().numpy()
    eng._ensure_history(4)

    def logits(report=False, reset=False):
        eng.reset(1)
        eng.prefill(prompt, dense=True)
        if report:
            eng.gemm_err.fill_(1)
        if reset:
            eng.reset(1)
        return eng.run_inference(vec)
    want = None
    for _ in range(3):
        with pytest.raises(RuntimeError, match="timed out"):
            logits(report=True)
        got = logits()
        assert np.isfinite(got).all() and (want is None or np.array_equal(got, want))
        want = got
    with pytest.raises(RuntimeError, match="timed out"):
        logits(report=True, reset=True)
    assert int(eng.gemm_err.item()) == 0


def test_tensor_parallel_ranks(cuda, model):
    """Both ranks on one GPU, a thread a rank, the all-reduce a host rendezvous between steps: layer 0's cached rows
    of rank r are KV head r's of the whole engine, bit for bit, and both ranks name the same tokens."""
    from llamamps_b200 import kernels as K
    from llamamps_b200.tp import TPEngine
    cfg, mw = model
    B, P = 2, 150
    prompts = _prompts(cfg, B, P)
    parts, meet, out = [None, None], threading.Barrier(2, timeout=60), [None, None]

    class Rank(TPEngine):
        def _reduce_add(self, part, x, site=-1):
            torch.cuda.current_stream().synchronize()
            parts[self.rank] = part
            meet.wait()
            total = parts[0] + parts[1]
            torch.cuda.current_stream().synchronize()
            meet.wait()
            K.residual_add(x, total, out=x)

    kw = dict(max_batch=B, max_seq_len=P + 8)
    engines = [Rank(mw, r, 2, comm="nccl", w8a8=True, **kw) for r in range(2)]
    whole = _engine(mw, **kw)
    for e in engines + [whole]:
        e.reset(B)
        e._ensure_history(4)
    whole.prefill(prompts, dense=True)
    torch.cuda.synchronize()

    def work(r):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                engines[r].prefill(prompts, dense=True)
                torch.cuda.current_stream().synchronize()
        except BaseException as e:  # noqa: BLE001  (raised in the test's thread)
            out[r] = e
            meet.abort()
    threads = [threading.Thread(target=work, args=(r,)) for r in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(120)
    for o in out:
        if o is not None:
            raise o
    for b in range(B):
        kw_, vw = whole.cache.read_positions(b, 0, P)
        for r in range(2):
            k, v = engines[r].cache.read_positions(b, 0, P)
            assert torch.equal(k, kw_[:, 128 * r:128 * (r + 1)]) and torch.equal(v, vw[:, 128 * r:128 * (r + 1)])
    assert torch.equal(engines[0].tokens, engines[1].tokens)
    off = (engines[0].buf_residual.double() - whole.buf_residual.double()).norm() / whole.buf_residual.double().norm()
    assert float(off) < 0.08


@pytest.mark.parametrize("B", [6, 40])
def test_decode_steps_of_tensor_parallel_ranks(cuda, model, B):
    """Steps of a batch on both ranks (one GPU, a thread a rank, host rendezvous): layer 0's cached rows of rank r are
    KV head r's of the whole engine, bit for bit, both ranks name the same tokens, and the hidden rows are off the
    whole engine's by what partial sums quantised apart take."""
    from tests.test_kv_q4_tp_gpu import _both, _rank_engines
    cfg, mw = model
    P = 7
    prompts = _prompts(cfg, B, P, seed=B)
    kw = dict(max_batch=B, max_seq_len=64, kv_bits=4, w8a8=True)
    whole = _engine(mw, **kw)
    kw.pop("kv_bits")
    ranks = _rank_engines(mw, **kw)

    def feed(e):
        e.reset(B)
        for t in range(P):
            e.tokens[:B].copy_(prompts[:, t])
            e.decode_step(record=False)
        torch.cuda.current_stream().synchronize()
        e.check_gemm_error()
        e.check_kv_error()
    feed(whole)
    _both(ranks, feed)
    for e in ranks:
        assert e.q8_rows is not None and e.pos[:B].tolist() == [P] * B
        off = (e.buf_residual.double() - whole.buf_residual.double()).norm() / whole.buf_residual.double().norm()
        assert float(off) < 0.08
    for b in range(B):
        full = whole.cache.read_positions(b, 0, P)
        for r, e in enumerate(ranks):
            for x, y in zip(full, e.cache.read_positions(b, 0, P)):
                assert torch.equal(x[:, 128 * r:128 * (r + 1)], y)
    assert torch.equal(ranks[0].tokens, ranks[1].tokens) and torch.equal(ranks[0].buf_residual, ranks[1].buf_residual)


def test_demo_runs_with_8_bit_projections(cuda, capsys):
    from llamamps_b200 import demo
    from llamamps_b200.config import QWEN2_5_1_5B
    cfg = dataclasses.replace(QWEN2_5_1_5B, n_layers=1, vocab=4096)
    out = demo.main(["--synthetic", "--w8a8", "--ids", ",".join(str(i) for i in range(300)), "--new", "3"], config=cfg)
    assert len(out) == 3 and "Generated token IDs" in capsys.readouterr().out
