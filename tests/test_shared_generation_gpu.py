"""Generation behind a shared prompt, far beyond it: every step's logits are those of a sequence that shares nothing and has run
the same tokens in one prompt step."""
import numpy as np
import pytest

from helpers import BF16_REL_TO_MAX, F32_REL_TO_MAX, make_model
from test_shared_sequences_gpu import SHARED, tokens

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def share_whatever_can_be(monkeypatch):
    """The models here are small: sharing would not pay."""
    from nnis_b200.engine import sharing
    monkeypatch.setattr(sharing, "LEAST_BYTES", 1)


@pytest.fixture(scope="module")
def folder(tmp_path_factory):
    return make_model(str(tmp_path_factory.mktemp("shared")), SHARED, 3)


def logits_alone(llm, prompt, emitted):
    """The logits that each emitted token was picked from, by a sequence that shares nothing and takes all tokens in one step."""
    from nnis_b200.engine import SequenceStep
    engine = llm.engine
    slot = engine.acquire_slot()
    fed = prompt + emitted[:-1]
    logits = engine.step([SequenceStep(slot, fed, list(range(len(prompt) - 1, len(fed))))]).cpu().numpy()
    engine.release_slot(slot)
    return logits


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("last", [1, 9])
def test_greedy_steps_far_behind_a_shared_prompt(folder, dtype, last, monkeypatch):
    """Prompts that differ in their last token (or nine) and 700 tokens after them, eleven pages: every step's logits, and the
    tokens picked from them."""
    from nnis_b200 import LLM
    from nnis_b200.csrc import ops
    from nnis_b200.engine.api import EngineBackend
    from nnis_b200.engine.decode import GraphDecoder
    llm = LLM(folder, dtype=dtype, max_tokens=1 << 14, max_batch=8)
    document = tokens(2, 1100)
    prompts = [document + [7 + i] * last for i in range(5)]
    steps, used, real, made, launch = [], [], ops.attention_shared, EngineBackend._decoder, GraphDecoder.launch

    def launch_and_keep(dec):
        launch(dec)
        steps.append(dec.logits[:5].cpu().numpy())

    # (of the classes, so that no model outlives the test in a cycle)
    monkeypatch.setattr(EngineBackend, "_decoder", lambda self, rows, context, want=False, rooms=None: made(self, rows, context, True, rooms))
    monkeypatch.setattr(GraphDecoder, "launch", launch_and_keep)
    monkeypatch.setattr(ops, "attention_shared", lambda *a: (used.append(1), real(*a))[1])
    results = llm.generate(prompts, max_new_tokens=700, share_prefix=True, stop_token_ids=[])
    assert used and all(r.ok and len(r.token_ids) == 700 for r in results)
    assert len(steps) == 699 + (last == 1)  # (one token of a prompt's own runs as such a step, too)
    limit = F32_REL_TO_MAX if dtype == "float32" else BF16_REL_TO_MAX
    for row, (prompt, r) in enumerate(zip(prompts, results)):
        want, got = logits_alone(llm, prompt, r.token_ids)[1:], np.stack([s[row] for s in steps[-699:]])
        off = np.abs(got - want).max(axis=1) / np.maximum(1.0, np.abs(want).max(axis=1))
        assert off.max() <= limit, (row, int(off.argmax()), float(off.max()))
        assert (got.argmax(axis=1) == r.token_ids[1:]).all()
    llm.engine.check_status()
    assert llm.engine.cache.usage()["pages_held"] == [0]


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("name", ["A", "B", "C"])
def test_other_head_sizes_read_shared_pages_once(tmp_path, name, dtype, monkeypatch):
    """Forked sequences of other head layouts, where the rule of what pays would have them read row by row: captured steps' logits
    are those of sequences of their own."""
    from helpers import CONFIGS
    from nnis_b200 import LLM
    from nnis_b200.csrc import ops
    from nnis_b200.engine import SequenceStep, sharing
    monkeypatch.setattr(sharing, "PAGE_COST", {})
    used, real = [], ops.attention_shared
    monkeypatch.setattr(ops, "attention_shared", lambda *a: (used.append(1), real(*a))[1])
    vocab = CONFIGS[name]["vocab_size"]
    llm = LLM(make_model(str(tmp_path), {**CONFIGS[name], "max_position_embeddings": 2048}, 11), dtype=dtype, max_tokens=1 << 14, max_batch=8)
    engine, limit = llm.engine, F32_REL_TO_MAX if dtype == "float32" else BF16_REL_TO_MAX
    document = tokens(3, 1000, vocab)
    first = engine.acquire_slot()
    engine.step([SequenceStep(first, document, [])])
    slots = [first] + [engine.fork(first) for _ in range(4)]
    history = {s: list(document) for s in slots}
    for turn in range(70):
        new = tokens(200 + turn, 5, vocab)
        logits = llm.backend.step([SequenceStep(s, [t], [0]) for s, t in zip(slots, new)])
        for s, t in zip(slots, new):
            history[s].append(t)
        if turn in (0, 24, 25, 69):
            got, other = logits.float().cpu().numpy(), engine.acquire_slot()
            for r, s in enumerate(slots):
                engine.release_slot(other)
                other = engine.acquire_slot()
                want = engine.step([SequenceStep(other, history[s], [len(history[s]) - 1])])[0].cpu().numpy()
                assert np.abs(got[r] - want).max() <= limit * max(1.0, float(np.abs(want).max())), (turn, r)
            engine.release_slot(other)
    assert used
    engine.check_status()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_a_step_of_many_drafted_sequences(folder, dtype):
    """Forked sequences and one of its own with two to six tokens each in one step, wanted places in any order: the logits of steps
    that do not share, and what follows them."""
    from nnis_b200 import LLM
    from nnis_b200.engine import SequenceStep
    llm = LLM(folder, dtype=dtype, max_tokens=1 << 14, max_batch=16)
    engine, limit = llm.engine, F32_REL_TO_MAX if dtype == "float32" else BF16_REL_TO_MAX
    first, lone = engine.acquire_slot(), engine.acquire_slot()
    history = {first: tokens(80, 830), lone: tokens(81, 100)}
    for s, h in history.items():
        engine.step([SequenceStep(s, h, [])])
    for _ in range(3):
        new = engine.fork(first)
        history[new] = list(history[first])
    for turn in range(4):
        batch, want = [], []
        for i, s in enumerate(history):
            fresh = tokens(900 + 10 * turn + i, 2 + (i + turn) % 5)
            places = list(range(len(fresh)))[::-1 if i % 2 else 1]
            batch.append(SequenceStep(s, fresh, places))
            other = engine.acquire_slot()
            want.append(engine.step([SequenceStep(other, history[s] + fresh, [len(history[s]) + p for p in places])]).cpu().numpy())
            engine.release_slot(other)
        got = engine.step(batch, drafted=True).cpu().numpy()
        want = np.concatenate(want)
        assert got.shape == want.shape
        assert (np.abs(got - want).max(axis=1) <= limit * np.maximum(1.0, np.abs(want).max(axis=1))).all()
        for i, s in enumerate(batch):
            keep = len(s.tokens) - i % 2
            history[s.slot] += s.tokens[:keep]
            engine.truncate(s.slot, len(history[s.slot]))
        engine.cache.check()
    engine.check_status()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_sampled_tokens_behind_a_shared_prompt(folder, dtype):
    """Each prompt's tokens are drawn from its own logits: every drawn token is one that its policy can draw (of the 50 likeliest, by
    logits that are off by the type's tolerance on either side), lengths are whole, and a second run draws the same."""
    from nnis_b200 import LLM, SamplingConfig
    llm = LLM(folder, dtype=dtype, max_tokens=1 << 14, max_batch=8)
    document = tokens(4, 1100)
    prompts = [document + [7 + i] * (1 + 3 * i) for i in range(6)]
    sampling = [SamplingConfig(seed=i, temperature=0.9, top_k=50) for i in range(6)]
    drawn = [llm.generate(prompts, max_new_tokens=90, share_prefix=True, sampling=sampling, stop_token_ids=[]) for _ in range(2)]
    assert all(r.ok and len(r.token_ids) == 90 for run in drawn for r in run)
    assert [r.token_ids for r in drawn[0]] == [r.token_ids for r in drawn[1]]
    limit = 2 * (F32_REL_TO_MAX if dtype == "float32" else BF16_REL_TO_MAX)
    for prompt, r in zip(prompts, drawn[0]):
        logits = logits_alone(llm, prompt, r.token_ids)
        line = np.sort(logits, axis=1)[:, -50]
        assert (logits[np.arange(90), r.token_ids] >= line - limit * np.maximum(1.0, np.abs(logits).max(axis=1))).all()
