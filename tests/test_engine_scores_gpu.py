"""The engine with a 4-bit cache, and the scores it reports: generated tokens with their alternatives, and given tokens.
A 4-bit engine's prompts run as a BF16 one's (their cached rows are the BF16 rows quantised, bit for bit), and its decode
steps attend over those; scores are held to log softmax in 64 bits of the rows the LM head saw."""

from __future__ import annotations

import math

import numpy as np
import pytest

from tests import _q4

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    yield
    from tempo_compiler_b200 import ops
    torch.cuda.synchronize()
    assert ops.watchdog() == 0


@pytest.fixture(scope="module")
def model():
    from tempo_compiler_b200.weights import GPT2Shape, random_gpt2
    return random_gpt2(5, GPT2Shape(layers=2))


def _ids(batch: int, tokens: int, seed: int = 0) -> np.ndarray:
    return np.random.default_rng(seed).integers(0, 50257, (batch, tokens)).astype(np.int32)


def _engine(model, batch: int, prompt: int, capacity: int, **kwargs):
    from tempo_compiler_b200.engine import Engine
    return Engine(*model, batch=batch, prompt=prompt, capacity=capacity, **kwargs)


def _cached(engine, layer: int, positions: int) -> np.ndarray:
    """Rows [batch, positions, 2 * heads * 64] of a 4-bit engine's cache."""
    from tempo_compiler_b200 import ops
    seq = torch.arange(engine.batch, dtype=torch.int32, device="cuda").repeat_interleave(positions)
    pos = torch.arange(positions, dtype=torch.int32, device="cuda").repeat(engine.batch)
    rows = ops.kv_load_q4(engine.kv_cache[layer], seq, pos)
    return rows.float().cpu().numpy().reshape(engine.batch, positions, -1)


def _quantised(engine, layer: int, positions: int) -> np.ndarray:
    """The same rows a BF16 engine cached, quantised."""
    parts = []
    for cache in (engine.k_cache[layer], engine.v_cache[layer]):
        x = cache[:, :, :positions].transpose(1, 2).float().cpu().numpy()
        parts.append(_q4.dequantise(x).reshape(engine.batch, positions, -1))
    return torch.from_numpy(np.concatenate(parts, 2)).float().to(torch.bfloat16).float().numpy()


@pytest.mark.parametrize("batch,options", [(2, {}), (2, dict(fuse_small_norms=False)), (11, {}),
                                           (11, dict(fold_layernorms=False)), (11, dict(decode_groups=3))])
def test_four_bit_engine(model, batch: int, options: dict) -> None:
    prompt, steps = 37, 9
    ids = _ids(batch, prompt)
    wide = _engine(model, batch, prompt, prompt + steps, **options)
    want = wide.generate(ids, 0)
    narrow = _engine(model, batch, prompt, prompt + steps, kv_bits=4, **options)
    # (one decode group's graph is captured anew for each number of steps)
    np.testing.assert_array_equal(narrow.generate(ids, 0), want)
    for layer in range(2):
        np.testing.assert_array_equal(_cached(narrow, layer, prompt), _quantised(wide, layer, prompt))
    tokens = narrow.generate(ids, steps)
    assert tokens.shape == (batch, steps + 1)
    np.testing.assert_array_equal(tokens[:, 0], want[:, 0])
    np.testing.assert_array_equal(narrow.generate(ids, steps, graph=False), tokens)
    # the first layer's rows of the generated tokens depend on the tokens alone: a prompt of them caches the same
    again = _engine(model, batch, prompt + steps, prompt + steps, kv_bits=4)
    again.generate(np.concatenate([ids, tokens[:, :steps]], 1), 0)
    a, b = _cached(narrow, 0, prompt + steps), _cached(again, 0, prompt + steps)
    np.testing.assert_array_equal(a[:, :prompt], b[:, :prompt])
    # (a decode projection may round a BF16 value the other way, which may move a code: one step, an eighth of the
    # range, plus what the row's ends moved by)
    reach = np.abs(b[:, prompt:]).max()
    assert np.abs(a[:, prompt:] - b[:, prompt:]).max() <= reach * (2 / 15 + 2.0 ** -6)


def test_four_bit_decode_step_is_the_average_over_the_cache(model) -> None:
    """One decode step's attention output against 64 bits, from the engine's own projection and cache."""
    engine = _engine(model, 3, 50, 64, kv_bits=4)
    engine.generate(_ids(3, 50), 3)
    # the last step's state: layer 1's projection rows are still in dqkv, its queries first, and 53 positions are cached
    q = engine.dqkv[:, :768].double().cpu().numpy().reshape(3, 12, 64)
    want, bound = _q4.attend(q, engine.kv_cache[1].cpu().numpy(), [53] * 3, 12)
    got = engine.dattn.double().cpu().numpy().reshape(want.shape)
    assert (np.abs(got - want) <= bound).all()


@pytest.mark.parametrize("batch,kv_bits", [(1, 16), (5, 4), (12, 16), (12, 4)])
def test_alternatives_of_generated_tokens(model, batch: int, kv_bits: int) -> None:
    prompt, steps, k = 24, 7, 4
    ids = _ids(batch, prompt, seed=batch)
    plain = _engine(model, batch, prompt, prompt + steps, kv_bits=kv_bits).generate(ids, steps)
    engine = _engine(model, batch, prompt, prompt + steps, kv_bits=kv_bits, alternatives=k)
    with pytest.raises(RuntimeError, match="scores"):
        engine.scores()
    tokens = engine.generate(ids, steps)
    np.testing.assert_array_equal(tokens, plain)
    scores = engine.scores()
    assert scores.logprob.shape == (batch, steps + 1) and scores.top_ids.shape == (batch, steps + 1, k)
    np.testing.assert_array_equal(scores.top_ids[..., 0], tokens)
    np.testing.assert_array_equal(scores.top_logprob[..., 0], scores.logprob)
    assert (np.diff(scores.top_logprob, axis=2) <= 0).all()
    assert (scores.entropy > 0).all() and (scores.entropy <= math.log(50257)).all()
    # the last step's rows are still there
    _check_scores(engine.dln, engine.wte, tokens[:, -1], k, [x[:, -1] for x in scores])
    np.testing.assert_array_equal(engine.generate(ids, steps, graph=False), tokens)
    for a, b in zip(engine.scores(), scores):
        np.testing.assert_array_equal(a, b)
    # scoring in between leaves the captured step alone
    engine.score(ids)
    np.testing.assert_array_equal(engine.generate(ids, steps), tokens)
    for a, b in zip(engine.scores(), scores):
        np.testing.assert_array_equal(a, b)


def _check_scores(rows, table, ids, k: int, got) -> None:
    """Scores against 64 bits of the normalised rows: a logit's FP32 accumulation of 768 products is off by at most
    768 2^-23 sum |a| |w|, which moves a log probability by at most twice that; the rest as in test_logprobs_gpu."""
    a, w = rows.double(), table.double()
    logits = a @ w.T
    slack = 2 * 768 * 2.0 ** -23 * (a.abs() @ w.abs().T).amax(1, keepdim=True).cpu().numpy()
    logs = torch.log_softmax(logits, 1)
    entropy = -(logs.exp() * logs).sum(1).cpu().numpy()
    logs = logs.cpu().numpy()
    own = 2.0 ** -21 + (50257 / 128 + 64) * 2.0 ** -24
    n = np.arange(len(ids))
    want = logs[n, ids]
    assert (np.abs(got[0] - want) <= slack[:, 0] + own + 2.0 ** -22 * np.abs(want)).all()
    weight = 2 + math.log(50257)
    assert (np.abs(got[1] - entropy) <= weight * (slack[:, 0] + own) + 2.0 ** -22 * entropy).all()
    if k:
        want = logs[n[:, None], got[3]]
        assert (np.abs(got[2] - want) <= slack + own + 2.0 ** -22 * np.abs(want)).all()
        best = -np.sort(-logs, 1)[:, :k]
        assert (np.abs(want - best) <= 2 * slack + 2.0 ** -22 * np.abs(best)).all()


@pytest.mark.parametrize("batch,prompt,kv_bits", [(1, 2, 16), (3, 65, 16), (9, 300, 4)])
def test_scores_of_given_tokens(model, batch: int, prompt: int, kv_bits: int) -> None:
    engine = _engine(model, batch, prompt, prompt, kv_bits=kv_bits)
    ids = _ids(batch, prompt, seed=3)
    scores = engine.score(ids, alternatives=3)
    assert scores.logprob.shape == (batch, prompt - 1) and scores.top_ids.shape == (batch, prompt - 1, 3)
    rows = engine.ln.view(batch, prompt, -1)[:, :-1].reshape(batch * (prompt - 1), -1)
    _check_scores(rows, engine.wte, ids[:, 1:].reshape(-1), 3, [x.reshape(-1, *x.shape[2:]) for x in scores])
    bare = engine.score(ids)
    np.testing.assert_array_equal(bare.logprob, scores.logprob)
    assert bare.top_ids.shape == (batch, prompt - 1, 0)


def test_padding_scores_zero(model) -> None:
    engine = _engine(model, 2, 10, 10)
    ids = _ids(2, 10)
    full = engine.score(ids)
    ids[1, 6:] = -1
    padded = engine.score(ids)
    assert (padded.logprob[1, 5:] == 0).all()
    np.testing.assert_array_equal(padded.logprob[1, :5], full.logprob[1, :5])
    np.testing.assert_array_equal(padded.logprob[0], full.logprob[0])


def test_ids_that_32_bits_do_not_hold_are_padding(model) -> None:
    engine = _engine(model, 2, 10, 10)
    ids = _ids(2, 10).astype(np.int64)
    ids[1, 6:] = -1
    want = engine.score(ids)
    for far in (2 ** 32 + 5, -2 ** 32 + 5, 2 ** 62):
        ids[1, 6:] = far
        for a, b in zip(engine.score(ids), want):
            np.testing.assert_array_equal(a, b)


def test_refusals(model) -> None:
    for kwargs, word in ((dict(kv_bits=8), "kv_bits"), (dict(alternatives=33), "alternatives"),
                         (dict(alternatives=-1), "alternatives"), (dict(kv_bits=4, persistent_decode=True), "persistent"),
                         (dict(alternatives=0, persistent_decode=True), "persistent"),
                         (dict(alternatives=0, decode_groups=2), "decode group")):
        with pytest.raises(ValueError, match=word):
            _engine(model, 4, 8, 16, **kwargs)
    engine = _engine(model, 2, 8, 16)
    with pytest.raises(ValueError, match="prompts of shape"):
        engine.score(_ids(2, 9))
    with pytest.raises(ValueError, match="alternatives"):
        engine.score(_ids(2, 8), alternatives=40)
    with pytest.raises(RuntimeError, match="scores"):
        engine.scores()
    with pytest.raises(ValueError, match="integers"):
        engine.score(_ids(2, 8).astype(np.float32))
