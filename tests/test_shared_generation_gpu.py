"""Generation behind a shared prompt, far beyond it: every token emitted is the likeliest by a sequence that shares nothing and
has run the same tokens in one prompt step."""
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


def short_of_the_likeliest(llm, prompt, emitted):
    """How far each emitted token's logit lies under the largest, of the logits' scale."""
    from nnis_b200.engine import SequenceStep
    engine = llm.engine
    slot = engine.acquire_slot()
    fed = prompt + emitted[:-1]
    logits = engine.step([SequenceStep(slot, fed, list(range(len(prompt) - 1, len(fed))))]).cpu().numpy()
    engine.release_slot(slot)
    scale = np.maximum(1.0, np.abs(logits).max(axis=1))
    return (logits.max(axis=1) - logits[np.arange(len(emitted)), emitted]) / scale


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("last", [1, 9])
def test_greedy_tokens_far_behind_a_shared_prompt(folder, dtype, last):
    """Prompts that differ in their last token (or nine) and 700 tokens after them, eleven pages.  Two forms' logits are each
    within the tolerance of the type, so the pick of one is short of the other's largest by twice that at most."""
    from nnis_b200 import LLM
    from nnis_b200.csrc import ops
    llm = LLM(folder, dtype=dtype, max_tokens=1 << 14, max_batch=8)
    document = tokens(2, 1100)
    prompts = [document + [7 + i] * last for i in range(5)]
    used, real = [], ops.attention_shared
    ops.attention_shared = lambda *a: (used.append(1), real(*a))[1]
    try:
        results = llm.generate(prompts, max_new_tokens=700, share_prefix=True, stop_token_ids=[])
    finally:
        ops.attention_shared = real
    assert used and all(r.ok and len(r.token_ids) == 700 for r in results)
    limit = 2 * (F32_REL_TO_MAX if dtype == "float32" else BF16_REL_TO_MAX)
    for prompt, r in zip(prompts, results):
        short = short_of_the_likeliest(llm, prompt, r.token_ids)
        assert short.max() <= limit, (int(short.argmax()), float(short.max()))
    llm.engine.check_status()
    assert llm.engine.cache.usage()["pages_held"] == [0]
