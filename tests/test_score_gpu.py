"""Scoring of texts through the engine, the LLM and the command line against the plain implementation's logits."""
import json

import numpy as np
import pytest
import torch

from conftest import TINY
from plain_cache8 import logprobs
from test_replay_gpu import TOL

pytestmark = pytest.mark.gpu


def _text(name, n, seed):
    return np.random.default_rng(seed).integers(0, TINY[name]["vocab_size"], size=n).tolist()


def _close(score, ids, logits, tol, top):
    """Log-probabilities and entropies are differences of logits and sums of them: off by twice what the logits are, and an entropy by
    that times the logits' spread (below 4 here)."""
    want, entropy, order, top_lp = logprobs(torch.from_numpy(logits.astype(np.float64)), ids[1:] + [-1], top)
    off = 2 * (tol["atol"] + tol["rtol"] * np.abs(logits).max()) + 2e-5
    assert score.logprobs.shape == (len(ids) - 1,) and score.entropies.shape == (len(ids),) and score.top_ids.shape == (len(ids), top)
    assert (np.abs(score.logprobs - want[:-1]) <= off).all() and (np.abs(score.entropies - entropy) <= 4 * off).all()
    assert (np.abs(score.top_logprobs - top_lp) <= off).all()
    same = score.top_ids == order
    near = np.abs(top_lp[:, :, None] - top_lp[:, None, :]) <= 2 * off             # neighbours that rounding may have exchanged
    assert (same | (near.sum(axis=2) > 1) | (np.arange(top) == top - 1)).all()


@pytest.mark.parametrize("name,dtype,store", [("A", "float32", "f32"), ("B", "bfloat16", "bf16"), ("C", "float32", "f32")])
@pytest.mark.parametrize("portion", [256, 7])
def test_score_is_the_plain_model_s(model_dirs, plain_models, name, dtype, store, portion):
    from sandyrt_b200.engine.step import Engine
    from sandyrt_b200.models.model import load_model

    engine = Engine(load_model(model_dirs[name], device="cuda:0", dtype=getattr(torch, dtype)), max_tokens=256, max_requests=2)
    free = engine.cache.alloc.free_pages(0)
    ids = _text(name, 61, 4)
    for _ in range(2):                                            # the second time in the pages of the first
        _close(engine.score(ids, top=5, portion=portion), ids, plain_models(name, store).logits(ids), TOL[dtype], 5)
    one = engine.score(ids[:1])
    assert one.logprobs.shape == (0,) and one.entropies.shape == (1,) and one.top_ids.shape == (1, 0)
    assert engine.cache.alloc.free_pages(0) == free and not engine.cache.alloc.live()


def test_score_leaves_other_requests_alone_and_refuses(model_dirs):
    from sandyrt_b200.engine.llm import LLM
    from sandyrt_b200.errors import OutOfPages, StepError

    llm = LLM(model_dirs["A"], dtype="float32", cache_tokens=96, max_live=2)
    prompt = _text("A", 11, 6)
    want = llm.generate(prompt, max_tokens=6)[0].output_ids
    scores = llm.score([prompt + want, prompt])
    assert np.array_equal(scores[1].logprobs, llm.score(prompt)[0].logprobs)
    # greedy tokens are the likeliest ones
    full = llm.score(prompt + want, top=1)[0]
    assert full.top_ids[len(prompt) - 1:-1, 0].tolist() == want
    assert llm.generate(prompt, max_tokens=6)[0].output_ids == want
    for call, error in ((lambda: llm.score([[]]), StepError), (lambda: llm.score(prompt, top=33), StepError), (lambda: llm.engine.score(prompt, portion=0), StepError),
                        (lambda: llm.score(_text("A", 100, 1)), OutOfPages), (lambda: llm.score(_text("A", 129, 1)), (StepError, OutOfPages))):
        with pytest.raises(error):
            call()
    with pytest.raises(Exception, match="token id"):
        llm.score([3, TINY["A"]["vocab_size"], 5])
    llm.add_request(prompt, max_tokens=4)
    with pytest.raises(StepError, match="waiting or running"):
        llm.score(prompt)
    while llm.has_work():
        llm.step()
    assert np.array_equal(scores[1].logprobs, llm.score(prompt)[0].logprobs)


@pytest.mark.parametrize("at", [0, 1, 4, 5, 7, 8])
@pytest.mark.parametrize("bad", [-1, "vocab", 1 << 31, -(1 << 40)])
def test_score_names_a_token_outside_the_vocabulary(model_dirs, at, bad):
    """Wherever in a portion of 4 it stands: the first token of a portion is asked for with the portion before it."""
    from sandyrt_b200.engine.step import Engine
    from sandyrt_b200.errors import StepError
    from sandyrt_b200.models.model import load_model

    engine = Engine(load_model(model_dirs["A"], device="cuda:0", dtype=torch.float32), max_tokens=64, max_requests=2)
    free, ids = engine.cache.alloc.free_pages(0), _text("A", 9, 2)
    want = engine.score(ids, portion=4)
    wrong = list(ids)
    wrong[at] = TINY["A"]["vocab_size"] if bad == "vocab" else bad
    with pytest.raises(StepError, match="token id is outside the vocabulary"):
        engine.score(wrong, portion=4)
    assert engine.cache.alloc.free_pages(0) == free and not engine.cache.alloc.live()
    assert np.array_equal(engine.score(ids, portion=4).logprobs, want.logprobs)


def test_score_without_a_free_slot_leaves_nothing_behind(model_dirs):
    from sandyrt_b200.engine.step import Engine
    from sandyrt_b200.errors import NoFreeSlot
    from sandyrt_b200.models.model import load_model

    engine = Engine(load_model(model_dirs["A"], device="cuda:0", dtype=torch.float32), max_tokens=64, max_requests=1)
    engine.admit("mine")
    known = dict(engine.ids._to_int)
    for _ in range(3):
        with pytest.raises(NoFreeSlot):
            engine.score([1, 2, 3])
    assert engine.ids._to_int == known
    engine.release("mine")
    assert engine.score([1, 2, 3]).logprobs.shape == (2,)


def test_score_on_the_command_line(model_dirs, capsys):
    from sandyrt_b200.cli import main

    assert main(["score", "--model", model_dirs["A"], "--dtype", "float32", "--ids", "5,9,300", "--ids", "7", "--top", "2"]) == 0
    lines = [json.loads(l) for l in capsys.readouterr().out.strip().splitlines()]
    assert [len(l["logprobs"]) for l in lines] == [2, 0] and [len(l["top_ids"]) for l in lines] == [3, 1]
    assert lines[0]["logprob"] == pytest.approx(sum(lines[0]["logprobs"])) and all(len(r) == 2 for r in lines[0]["top_ids"])
