"""What the 4-bit cache's calls report, and to whom."""
import numpy as np
import pytest
import torch

from tests import _kv_q4 as R
from tests.test_kv_q4_gpu import _cu

pytestmark = pytest.mark.gpu

D = 128


def test_prefill_without_an_error_word_raises(cuda):
    """A call that brings no error word raises what the kernel reports; a captured call needs a word."""
    from llamamps_b200 import kernels as K
    rng = np.random.default_rng(2)
    hq, hkv, page, seq = 6, 1, 16, 20
    c = R.Cache(rng, [seq, seq], hkv, page)
    q = _cu(rng.normal(0, 1, (2 * seq, hq * D)).astype(np.float16))
    out = torch.zeros(2 * seq, hq * D, dtype=torch.float16, device="cuda")
    starts = torch.zeros(2, dtype=torch.int32, device="cuda")

    def call(**kw):
        return K.prefill_attention_q4(q, c.k, c.v, c.bt, out, 2, seq, page, hq, hkv, D, c.max_seq_len, starts=starts, **kw)

    want = torch.empty_like(out)
    e = torch.zeros(1, dtype=torch.int32, device="cuda")
    want.copy_(call(error=e))
    assert call() is out and torch.equal(out, want) and e.item() == 0
    good = c.bt[1, 0].item()
    c.bt[1, 0] = c.k.shape[0]
    with pytest.raises(RuntimeError, match="outside the pool"):
        call()
    c.bt[1, 0] = good
    starts.fill_(c.max_seq_len)
    with pytest.raises(RuntimeError, match="position outside"):
        call()
    starts.zero_()
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.stream(stream):
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            call(error=e)
            with pytest.raises(ValueError, match="error"):
                call()
    out.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want) and e.item() == 0
