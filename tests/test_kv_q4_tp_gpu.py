"""The two-way tensor-parallel engine on the 4-bit KV cache, both ranks on one GPU: a thread a rank, the
all-reduce a host rendezvous between steps (no kernel waits for another)."""
import dataclasses
import threading

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def _rank_engines(mw, **kw):
    from llamamps_b200 import kernels as K
    from llamamps_b200.tp import TPEngine
    parts, meet = [None, None], threading.Barrier(2, timeout=60)

    class Rank(TPEngine):
        def _reduce_add(self, part, x, site=-1):
            torch.cuda.current_stream().synchronize()
            parts[self.rank] = part
            meet.wait()
            total = parts[0] + parts[1]
            torch.cuda.current_stream().synchronize()
            meet.wait()
            K.residual_add(x, total, out=x)

    return [Rank(mw, r, 2, comm="nccl", kv_bits=4, **kw) for r in range(2)]


def _both(engines, call):
    out = [None, None]

    def work(r):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                out[r] = call(engines[r])
                torch.cuda.current_stream().synchronize()
        except BaseException as e:  # noqa: BLE001  (raised in the test's thread)
            out[r] = e
    torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=(r,)) for r in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(120)
    for o in out:
        if isinstance(o, BaseException):
            raise o
    return out


@pytest.mark.parametrize("P", [9, 150])
def test_ranks_hold_their_heads_of_the_same_cache(cuda, P):
    """Token by token and by dense prefill: layer 0's cached rows of rank r are KV head r's of the whole engine,
    byte for byte; layer 1's (behind partial sums in another order) within a code step, nearly all equal; both
    ranks name the same tokens, and the next turn goes on from there."""
    from llamamps_b200.config import QWEN2_5_1_5B
    from llamamps_b200.engine import QwenEngine
    from llamamps_b200.weights import synth_model
    cfg = dataclasses.replace(QWEN2_5_1_5B, n_layers=2, vocab=8192)
    mw = synth_model(cfg, seed=41, device="cuda")
    B, n = 2, 5
    prompts = np.random.default_rng(P).integers(0, cfg.vocab, (B, P))
    kw = dict(max_batch=B, max_seq_len=256)
    whole = QwenEngine(weights=mw, kv_bits=4, **kw)
    ranks = _rank_engines(mw, **kw)
    whole.generate_batch(prompts, 1)
    ids = _both(ranks, lambda e: e.generate_batch(prompts, n))
    assert np.array_equal(*ids)
    for b in range(B):
        for layer in range(2):
            full = whole.cache.read_positions(b, layer, P)
            for r, e in enumerate(ranks):
                for x, y in zip(full, e.cache.read_positions(b, layer, P)):
                    x = x[:, 128 * r:128 * r + 128].float()
                    step = x.unflatten(1, (-1, 32)).abs().amax(-1).repeat_interleave(32, 1) / 7
                    off = (x - y.float()).abs()
                    if layer == 0:
                        assert (off == 0).all()
                    else:
                        assert (off <= 1.02 * step + 1e-6).all() and (off > 0).float().mean() < 0.1
    more = torch.from_numpy(np.random.default_rng(1).integers(0, cfg.vocab, (B, 40)).astype(np.int32)).cuda()
    for e in ranks:
        assert e.host_pos == P + n - 1
    for dense in (True, False):
        _both(ranks, lambda e: e.prefill(more, dense=dense))
        assert torch.equal(ranks[0].tokens, ranks[1].tokens)
    for e in ranks:
        e.check_kv_error()
