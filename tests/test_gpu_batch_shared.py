"""Batched serving behind a shared prompt prefix (sd_batch_create_shared) on a small Mistral-geometry model.

Bars: logits within 1e-2 relative of the CPU oracle's single-stream forward over prefix + tokens, and within 5e-3 of a
plain batch's (both round Q and P to fp16 once); a stream's logits do not depend on the other streams, bit for bit;
generated tokens those of a plain batch over prefix + prompt, up to a near-tie.
"""
import numpy as np
import pytest

from tests.conftest import gpu_available

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not gpu_available(), reason="needs a CUDA GPU")]

B = 3


@pytest.fixture(scope="module")
def mini(tmp_path_factory):
    from anetransformers_b200 import gguf as G
    path = str(tmp_path_factory.mktemp("bs") / "mini.gguf")
    G.write_synthetic_gguf(path, G.MINI, seed=3)
    return path


@pytest.fixture(scope="module")
def ctx(mini):
    from anetransformers_b200.engine import Context
    c = Context(mini, max_seq=512)
    yield c
    c.close()


def rel_err(a, b):
    return float(np.max(np.abs(a.astype(np.float64) - b)) / max(np.max(np.abs(b)), 1e-30))


def tokens(rng, vocab, *shape):
    return rng.integers(3, vocab, shape).astype(np.int32)


@pytest.mark.parametrize("n_prefix", [1, 64, 75])
def test_forward_matches_oracle(mini, ctx, oracle, n_prefix):
    """Prefill behind the prefix, then a forward at another position per stream (rolled back, as after rejected drafts)."""
    from anetransformers_b200 import gguf as G
    from anetransformers_b200.engine import BatchContext
    rng = np.random.default_rng(n_prefix)
    prefix, prom, nxt = tokens(rng, ctx.vocab, n_prefix), tokens(rng, ctx.vocab, B, 20), tokens(rng, ctx.vocab, B, 5)
    pos = np.array([20, 17, 0], np.int32)
    bc = BatchContext(ctx, B, max_seq=128, width=8, prefix=prefix)
    try:
        bc.prefill(prom)
        lg = bc.forward(nxt, pos)
    finally:
        bc.close()
    om = oracle.OracleModel(G.GGUFFile(mini), max_seq=256)
    for s in range(B):
        kv = om.new_kv()
        seq = list(prefix) + list(prom[s, :pos[s]])
        for i, t in enumerate(seq):
            om.forward(kv, int(t), i)
        for j in range(5):
            ref = om.forward(kv, int(nxt[s, j]), len(seq) + j)
            assert rel_err(lg[s, j], ref) < 1e-2, (s, j)
        om.free_kv(kv)


def test_close_to_a_plain_batch(ctx):
    from anetransformers_b200.engine import BatchContext
    rng = np.random.default_rng(8)
    prefix, prom, nxt = tokens(rng, ctx.vocab, 150), tokens(rng, ctx.vocab, B, 40), tokens(rng, ctx.vocab, B, 5)
    sh = BatchContext(ctx, B, max_seq=128, width=5, prefix=prefix)
    pl = BatchContext(ctx, B, max_seq=256, width=5)
    try:
        sh.prefill(prom)
        a = sh.forward(nxt, np.full(B, 40, np.int32))
        pl.prefill(np.concatenate([np.tile(prefix, (B, 1)), prom], 1))
        b = pl.forward(nxt, np.full(B, 190, np.int32))
    finally:
        sh.close()
        pl.close()
    for s in range(B):
        assert rel_err(a[s], b[s].astype(np.float64)) < 5e-3, s


def test_streams_are_independent(ctx):
    """Other streams' tokens and lengths change: stream 1's logits must not; the same call again gives the same bits."""
    from anetransformers_b200.engine import BatchContext
    rng = np.random.default_rng(9)
    prefix, prom, nxt = tokens(rng, ctx.vocab, 33), tokens(rng, ctx.vocab, B, 70), tokens(rng, ctx.vocab, B, 4)
    bc = BatchContext(ctx, B, max_seq=128, width=8, prefix=prefix)
    try:
        bc.prefill(prom)
        a = bc.forward(nxt, np.array([70, 66, 70], np.int32))
        prom2, nxt2 = tokens(rng, ctx.vocab, B, 70), tokens(rng, ctx.vocab, B, 4)
        prom2[1], nxt2[1] = prom[1], nxt[1]
        bc.prefill(prom2)
        b = bc.forward(nxt2, np.array([3, 66, 64], np.int32))
        bc.prefill(prom)
        c = bc.forward(nxt, np.array([70, 66, 70], np.int32))
    finally:
        bc.close()
    np.testing.assert_array_equal(a[1].view(np.uint32), b[1].view(np.uint32))
    np.testing.assert_array_equal(a.view(np.uint32), c.view(np.uint32))


def near_tie(ctx, prompt, one, other, rel=1e-2):
    n = min(len(one), len(other))
    if one[:n] == other[:n]:
        return True
    i = next(j for j in range(n) if one[j] != other[j])
    seq = list(prompt) + one[:i]
    ctx.prefill(seq[:-1], 0)
    lg, _ = ctx.forward([seq[-1]], len(seq) - 1)
    s = np.sort(lg[0])
    return (s[-1] - s[-2]) <= rel * np.max(np.abs(lg[0]))


@pytest.mark.parametrize("mode", ["greedy", "ngram"])
def test_generate_matches_plain_batch(ctx, mode):
    """Greedy and n-gram speculative output behind the prefix: at temp 0 without a repetition penalty both are the greedy
    continuation of prefix + prompt."""
    from anetransformers_b200.engine import BatchContext
    rng = np.random.default_rng(12)
    prefix = tokens(rng, ctx.vocab, 90)
    pool = tokens(rng, ctx.vocab, 3, 12)
    prompts = np.stack([np.concatenate([pool[(s + i) % 3] for i in range(4)]) for s in range(B)]).astype(np.int32)
    kw = dict(max_tokens=24, temp=0.0, rep_penalty=1.0, ignore_eos=True)
    sh = BatchContext(ctx, B, max_seq=128, width=5, prefix=prefix)
    pl = BatchContext(ctx, B, max_seq=256, width=5)
    try:
        want, _ = pl.generate(np.concatenate([np.tile(prefix, (B, 1)), prompts], 1), mode="greedy", **kw)
        got, st = sh.generate(prompts, mode=mode, **(dict(kw, spec_k=4, ngram_n=3) if mode == "ngram" else kw))
        again, _ = sh.generate(prompts, mode=mode, **(dict(kw, spec_k=4, ngram_n=3) if mode == "ngram" else kw))
    finally:
        sh.close()
        pl.close()
    assert got == again
    for s in range(B):
        assert len(got[s]) >= 23
        assert near_tie(ctx, list(prefix) + prompts[s].tolist(), want[s], got[s]), s


def test_decode_after_prefill(ctx):
    from anetransformers_b200.engine import BatchContext
    rng = np.random.default_rng(13)
    prefix, hist = tokens(rng, ctx.vocab, 64), tokens(rng, ctx.vocab, B, 30)
    first = tokens(rng, ctx.vocab, B)
    full = np.concatenate([hist, first[:, None]], 1)
    kw = dict(mode="ngram", max_tokens=16, temp=0.0, rep_penalty=1.0, ignore_eos=True, spec_k=4, ngram_n=3)
    sh = BatchContext(ctx, B, max_seq=128, width=5, prefix=prefix)
    try:
        sh.prefill(hist)
        outs, _ = sh.decode(full, first, **kw)
    finally:
        sh.close()
    for s in range(B):
        seq = list(prefix) + full[s].tolist()
        ctx.prefill(seq[:-1], 0)
        one, _ = ctx.decode(seq, int(first[s]), **kw)
        assert near_tie(ctx, seq, one, outs[s]), s


def test_bad_arguments(ctx):
    from anetransformers_b200 import _lib
    from anetransformers_b200.engine import BatchContext
    ok = np.arange(3, 10, dtype=np.int32)
    for kw in (dict(prefix=np.array([ctx.vocab], np.int32)), dict(prefix=np.zeros(0, np.int32)), dict(width=9), dict(max_seq=8),
               dict(n_streams=0), dict(n_streams=5000)):
        a = dict(n_streams=B, max_seq=64, width=5, prefix=ok)
        a.update(kw)
        with pytest.raises(_lib.SpecDecError):
            BatchContext(ctx, **a).close()
    bc = BatchContext(ctx, B, max_seq=64, width=5, prefix=ok)
    try:
        with pytest.raises(_lib.SpecDecError):
            bc.forward(np.ones((B, 5), np.int32), np.full(B, 60, np.int32))  # past the stream's positions
    finally:
        bc.close()
