"""A batch that is used again with other sizes gives what a fresh one gives."""
import numpy as np
import pytest

from tests.conftest import gpu_available
from tests.test_gpu_batch_shared import B, ctx, mini, tokens  # noqa: F401 (fixtures)

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not gpu_available(), reason="needs a CUDA GPU")]


def calls(bc, prompts, n, more, mode):
    """Tokens of generate and of decode (after a prefill) on the first n prompt tokens, sampled: greedy ones of this model
    depend little on the prompt."""
    kw = dict(mode=mode, max_tokens=more, temp=1.0, top_k=40, top_p=1.0, seed=n, rep_penalty=1.0, ignore_eos=True, spec_k=4, ngram_n=3)
    got, _ = bc.generate(prompts[:, :n], **kw)
    bc.prefill(prompts[:, :n - 1])
    dec, _ = bc.decode(prompts[:, :n], prompts[:, n - 1], **kw)
    return got, dec


@pytest.mark.parametrize("mode", ["greedy", "ngram"])
@pytest.mark.parametrize("shared", [False, True])
def test_shorter_after_longer(ctx, mode, shared):
    from anetransformers_b200.engine import BatchContext
    rng = np.random.default_rng(41)
    prompts = tokens(rng, ctx.vocab, B, 60)
    kw = dict(max_seq=256, width=5, **(dict(prefix=tokens(rng, ctx.vocab, 30)) if shared else {}))
    fresh, used = BatchContext(ctx, B, **kw), BatchContext(ctx, B, **kw)
    try:
        want = calls(fresh, prompts, 20, 12, mode)
        long = calls(used, prompts, 60, 80, mode)
        assert all(0 <= t < ctx.vocab for call in long for out in call for t in out)
        assert calls(used, prompts, 20, 12, mode) == want
    finally:
        fresh.close()
        used.close()
