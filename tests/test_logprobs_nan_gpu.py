"""Rows of logits that hold a NaN, whatever else they hold: their scores are NaN."""

from __future__ import annotations

import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module", autouse=True)
def _device():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    from tempo_compiler_b200 import lib
    lib.load()
    yield
    from tempo_compiler_b200 import ops
    torch.cuda.synchronize()
    assert ops.watchdog() == 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [1, 7, 900, 50257])
@pytest.mark.parametrize("copies", [1, 30])
@pytest.mark.parametrize("rest", ["nan", "-inf", "lowest", "-1e10", "logits", "large"])
def test_a_row_with_a_nan_scores_nan(dtype, vocab: int, copies: int, rest: str) -> None:
    """One NaN, in the first, the last or a middle place, among nothing but NaN, masks, ordinary and large logits; a row of
    a cluster and of one CTA; rows beside it without a NaN keep their scores."""
    from tempo_compiler_b200 import ops
    rng = np.random.default_rng(vocab)
    clean = torch.from_numpy(rng.standard_normal((6, vocab)).astype(np.float32)).cuda().to(dtype)
    fill = {"nan": math.nan, "-inf": -math.inf, "lowest": torch.finfo(dtype).min, "-1e10": -1e10, "large": 1e30}
    rows = clean.clone()
    places = [0, vocab - 1, vocab // 2]
    for r, place in enumerate(places):
        if rest != "logits":
            rows[r] = fill[rest]
        rows[r, place] = math.nan
    rows, clean = rows.repeat(copies, 1), clean.repeat(copies, 1)
    ids = torch.from_numpy(rng.integers(0, vocab, len(rows)).astype(np.int32)).cuda()
    for top in sorted({0, min(5, vocab)}):
        got, want = ops.token_logprobs(rows, ids, top=top), ops.token_logprobs(clean, ids, top=top)
        for i in range(2 if top == 0 else 3):
            a, b = got[i].view(copies, 6, -1), want[i].view(copies, 6, -1)
            assert a[:, :3].isnan().all(), ("logprob", "entropy", "top_logprob")[i]
            assert torch.equal(a[:, 3:], b[:, 3:])
        if top:
            order = got.top_ids.view(copies, 6, top)
            assert torch.equal(order[:, 3:], want.top_ids.view(copies, 6, top)[:, 3:])
            for r, place in enumerate(places):
                first = list(range(top)) if rest == "nan" else [place]
                assert (order[:, r, :len(first)] == torch.tensor(first, device="cuda")).all()
    # a row without a token scores 0 all the same, and its entropy is NaN
    none = ops.token_logprobs(rows, torch.full_like(ids, -1))
    assert (none.logprob == 0).all() and none.entropy.view(copies, 6)[:, :3].isnan().all()
