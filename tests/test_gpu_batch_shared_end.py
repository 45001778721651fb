"""A shared batch whose streams end at different times: a stream that has finished keeps its K/V while the others go on, as
the rings of a plain batch do."""
import numpy as np
import pytest

from tests.conftest import gpu_available
from tests.test_gpu_batch_shared import B, ctx, mini, rel_err, tokens  # noqa: F401 (fixtures)

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not gpu_available(), reason="needs a CUDA GPU")]


@pytest.mark.parametrize("mode", ["greedy", "ngram"])
def test_finished_stream_keeps_its_positions(ctx, mode):
    """Stream 0 ends at once (its first token is the end of text) with its last position alone in a page, the others take
    new pages; then stream 0 goes on from where it was."""
    from anetransformers_b200.engine import BatchContext
    rng = np.random.default_rng(31)
    eos, n, more = 2, 65, 80
    prefix, hist = tokens(rng, ctx.vocab, 40), tokens(rng, ctx.vocab, B, n)
    first = tokens(rng, ctx.vocab, B)
    first[0] = eos
    nxt = tokens(rng, ctx.vocab, B, 3)
    full = np.concatenate([hist, first[:, None]], 1)
    kw = dict(mode=mode, max_tokens=more, temp=0.0, rep_penalty=1.0, ignore_eos=False, spec_k=4, ngram_n=3)
    sh = BatchContext(ctx, B, max_seq=256, width=5, prefix=prefix)
    try:
        sh.prefill(hist)
        pos = np.full(B, n, np.int32)
        before = sh.forward(nxt, pos)
        sh.prefill(hist)
        outs, _ = sh.decode(full, first, **kw)
        assert len(outs[0]) == 0 and max(len(o) for o in outs[1:]) > 64
        after = sh.forward(nxt, np.array([n] + [n + more // 2] * (B - 1), np.int32))
    finally:
        sh.close()
    assert rel_err(after[0], before[0].astype(np.float64)) == 0.0
