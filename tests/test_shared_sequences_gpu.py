"""Forked sequences and drafted tokens through the engine: the same tokens and logits as without sharing."""
import numpy as np
import pytest
import torch

from helpers import CONFIGS, F32_REL_TO_MAX, BF16_REL_TO_MAX, make_model

pytestmark = pytest.mark.gpu

SHARED = dict(architectures=["LlamaForCausalLM"], model_type="llama", vocab_size=311, hidden_size=192, intermediate_size=320,
              num_hidden_layers=2, num_attention_heads=6, num_key_value_heads=2, head_dim=64, max_position_embeddings=4096,
              rms_norm_eps=1e-5, rope_theta=10000.0, hidden_act="silu", tie_word_embeddings=True, attention_bias=False,
              torch_dtype="bfloat16")


@pytest.fixture(autouse=True)
def share_whatever_can_be(monkeypatch):
    """The models here are small: sharing would not pay."""
    from nnis_b200.engine import sharing
    monkeypatch.setattr(sharing, "LEAST_BYTES", 1)


@pytest.fixture(scope="module")
def folder(tmp_path_factory):
    return make_model(str(tmp_path_factory.mktemp("shared")), SHARED, 3)


@pytest.fixture(scope="module")
def small_folder(tmp_path_factory):
    return make_model(str(tmp_path_factory.mktemp("tiny")), {**CONFIGS["B"], "vocab_size": 311, "eos_token_id": None}, 5)


def tokens(seed, n, vocab=311):
    return np.random.default_rng(seed).integers(0, vocab, n).tolist()


def close(got, want, dtype):
    scale = max(1.0, float(np.abs(want).max()))
    return float(np.abs(got - want).max()) <= (F32_REL_TO_MAX if dtype == "float32" else BF16_REL_TO_MAX) * scale


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("graph", [False, True])
def test_forked_sequences_decode_as_sequences_of_their_own(folder, dtype, graph):
    """Steps of forked sequences beside one that shares nothing, captured and not, over page ends, while some fork again, end
    and go back; every step's logits against sequences that have run the same tokens alone."""
    from nnis_b200 import LLM
    from nnis_b200.engine import SequenceStep
    from nnis_b200.csrc import ops
    llm = LLM(folder, dtype=dtype, max_tokens=1 << 14, max_batch=32)
    engine = llm.engine
    step = llm.backend.step if graph else engine.step
    prompt = tokens(1, 1150)
    first = engine.acquire_slot()
    engine.step([SequenceStep(first, prompt, [])])
    lone = engine.acquire_slot()
    engine.step([SequenceStep(lone, tokens(9, 200), [])])
    history = {first: list(prompt), lone: tokens(9, 200)}
    for _ in range(5):
        new = engine.fork(first)
        history[new] = list(prompt)
    used = []
    real = ops.attention_shared
    ops.attention_shared = lambda *a: (used.append(1), real(*a))[1]
    try:
        for turn in range(70):
            slots = list(history)
            if turn == 20:
                new = engine.fork(slots[2])
                history[new] = list(history[slots[2]])
                slots.append(new)
            if turn == 30:
                engine.release_slot(slots[3])
                del history[slots[3]]
                slots = list(history)
            if turn == 40:
                engine.truncate(slots[2], 1140)
                del history[slots[2]][1140:]
            if turn == 45:
                engine.compact()
            t = tokens(100 + turn, len(slots))
            logits = step([SequenceStep(s, [x], [0]) for s, x in zip(slots, t)])
            for s, x in zip(slots, t):
                history[s].append(x)
            if turn in (0, 1, 21, 33, 41, 46, 69):
                got = logits.float().cpu().numpy()
                for r, s in enumerate(slots):
                    other = engine.acquire_slot()
                    want = engine.step([SequenceStep(other, history[s], [len(history[s]) - 1])])[0].cpu().numpy()
                    engine.release_slot(other)
                    assert close(got[r], want, dtype), (turn, s)
            engine.cache.check()
    finally:
        ops.attention_shared = real
    assert used
    engine.check_status()


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_generation_behind_a_shared_prompt(folder, dtype):
    """``share_prefix`` gives the tokens of generation without it (float32: the logits' differences of 1e-4 of their scale
    decide no pick of these; sampled, each with its seed), and gives all pages back."""
    from nnis_b200 import LLM, SamplingConfig
    llm = LLM(folder, dtype=dtype, max_tokens=1 << 14, max_batch=16)
    document = tokens(2, 1100)
    prompts = [document + tokens(20 + i, 1 + 3 * i) for i in range(7)] + [tokens(40, 50)] + [document + tokens(23, 4)]
    shared = llm.generate(prompts, max_new_tokens=40, share_prefix=True, stop_token_ids=[5])
    assert all(r.ok for r in shared)
    assert llm.engine.cache.usage()["pages_held"] == [0] and not llm.engine.cache.shares_pages()
    sampling = [SamplingConfig(seed=i, temperature=0.9, top_k=50) for i in range(9)]
    drawn = llm.generate(prompts, max_new_tokens=20, share_prefix=True, sampling=sampling)
    if dtype == "float32":
        alone = llm.generate(prompts, max_new_tokens=40, stop_token_ids=[5])
        assert [r.token_ids for r in shared] == [r.token_ids for r in alone]
        alone = llm.generate(prompts, max_new_tokens=20, sampling=sampling)
        assert [r.token_ids for r in drawn] == [r.token_ids for r in alone]
    else:  # (roundings differ between the kernels: the first tokens, before they add up, and the lengths)
        assert all(len(r.token_ids) in (40, r.token_ids.index(5) + 1 if 5 in r.token_ids else 40) for r in shared)


@pytest.mark.parametrize("name", ["A", "B", "C"])
def test_other_head_sizes_share_too(tmp_path, name):
    from nnis_b200 import LLM
    folder = make_model(str(tmp_path), {**CONFIGS[name], "max_position_embeddings": 2048}, 11)
    vocab = CONFIGS[name]["vocab_size"]
    llm = LLM(folder, dtype="float32", max_tokens=1 << 14, max_batch=8)
    document = tokens(3, 1000, vocab)
    prompts = [document + tokens(30 + i, 5, vocab) for i in range(4)]
    shared = llm.generate(prompts, max_new_tokens=12, share_prefix=True, stop_token_ids=[])
    alone = llm.generate(prompts, max_new_tokens=12, stop_token_ids=[])
    assert [r.token_ids for r in shared] == [r.token_ids for r in alone]


def test_sessions_fork(folder):
    from nnis_b200 import LLM
    llm = LLM(folder, dtype="float32", max_tokens=1 << 13, max_batch=8)
    a = llm.new_session()
    a.prefill(tokens(4, 100))
    b = a.fork()
    la = [a.decode_one(t) for t in (7, 8, 9)]
    lb = [b.decode_one(t) for t in (7, 8, 10)]
    assert b.position() == a.position() == 103
    assert close(lb[1], la[1], "float32")
    c = llm.new_session()
    c.prefill(tokens(4, 100) + [7, 8])
    assert close(c.decode_one(10), lb[2], "float32")
    for s in (a, b, c):
        s.close()
    assert llm.engine.cache.usage()["pages_held"] == [0]


def test_drafted_greedy_generation_is_greedy_generation(folder, small_folder):
    """Whatever is drafted, float32 greedy tokens are those of generation token by token; the session goes on from there."""
    from nnis_b200 import LLM, GenerationConfig, LookupDrafter, SessionDrafter, StreamControl

    class Wrong:
        def begin(self):
            self.n = 0

        def propose(self, told, count, temperature):
            self.n += 1
            return [(told[-1] * 31 + self.n + i) % 311 for i in range(count)], None

    llm = LLM(folder, dtype="float32", max_tokens=1 << 13, max_batch=8)
    draft = LLM(small_folder, dtype="float32", max_tokens=1 << 13, max_batch=2)
    prompt = tokens(6, 40) * 5
    want = llm.new_session().generate(prompt, GenerationConfig(30))
    itself = SessionDrafter(llm)
    for drafter, count in ((LookupDrafter(), 4), (Wrong(), 3), (SessionDrafter(draft), 5), (itself, 4), (itself, 1)):
        s = llm.new_session()
        assert s.generate_drafted(prompt, GenerationConfig(30), drafter, drafts=count) == want
        assert s.position() == len(prompt) + 30
        again = s.decode_one(3)
        s.close()
        ref = llm.new_session()
        ref.prefill(prompt + want)
        assert close(again, ref.decode_one(3), "float32")
        ref.close()
    # a stop token among drafts that are kept, and a callback that stops
    for stop_at in (0, 4, 11):
        cut = want.index(want[stop_at]) + 1
        s = llm.new_session()
        got = s.generate_drafted(prompt, GenerationConfig(30, (want[stop_at],)), itself, drafts=6)
        assert got == want[:cut] and s.position() == len(prompt) + cut
        s.reset()
        seen = []
        got = s.generate_drafted(prompt, GenerationConfig(30), itself, drafts=6,
                                 on_token=lambda t: (seen.append(t), StreamControl.STOP if len(seen) == stop_at + 1 else None)[1])
        assert got == seen == want[:stop_at + 1] and s.position() == len(prompt) + stop_at + 1
        s.close()
    itself.close()
    llm.engine.cache.check()
    llm.engine.check_status()


@pytest.mark.parametrize("at", [0, 1, 3, 6])
def test_a_callback_that_raises_leaves_no_draft_behind(folder, at):
    """The session holds the prompt and emitted tokens alone, and goes on from there."""
    from nnis_b200 import LLM, GenerationConfig, SessionDrafter
    llm = LLM(folder, dtype="float32", max_tokens=1 << 13, max_batch=8)
    prompt, shown = tokens(6, 40) * 5, []

    def on_token(token):
        if len(shown) == at:
            raise KeyError("enough")
        shown.append(token)

    s = llm.new_session()
    with pytest.raises(KeyError):
        s.generate_drafted(prompt, GenerationConfig(30), SessionDrafter(llm), drafts=4, on_token=on_token)
    held = s.position()
    assert len(prompt) <= held <= len(prompt) + len(shown)
    assert shown == llm.new_session().generate(prompt, GenerationConfig(30))[:at]
    ref = llm.new_session()
    ref.prefill(prompt + shown[:held - len(prompt)])
    assert close(s.decode_one(3), ref.decode_one(3), "float32")


def test_drafted_sampling_draws_from_the_target(folder, small_folder):
    """The first two tokens over 600 seeds, by a drafter of another distribution: as often as the target's probabilities say.
    A count of 600 draws is within 4.5 standard deviations of its mean, sqrt(600 p (1 - p)) each, for all of some 20
    likely tokens but once in 7,000 such tests (normal tails)."""
    from nnis_b200 import LLM, GenerationConfig, SamplingConfig, SessionDrafter
    from nnis_b200.engine import SequenceStep
    llm = LLM(folder, dtype="float32", max_tokens=1 << 13, max_batch=8)
    draft = LLM(small_folder, dtype="float32", max_tokens=1 << 13, max_batch=2)
    drafter = SessionDrafter(draft, seed=12345)
    prompt, n, t = tokens(7, 12), 600, 0.6
    s = llm.new_session()
    seconds, firsts = {}, {}
    for seed in range(n):
        a, b, _ = s.generate_drafted(prompt, GenerationConfig(3), drafter, drafts=2, sampling=SamplingConfig(seed=seed, temperature=t))
        firsts[a] = firsts.get(a, 0) + 1
        seconds[(a, b)] = seconds.get((a, b), 0) + 1
    slot = llm.engine.acquire_slot()
    p1 = torch.softmax(llm.engine.step([SequenceStep(slot, prompt, [11])])[0].double() / t, 0).cpu().numpy()
    for a in np.argsort(-p1)[:12]:
        assert abs(firsts.get(int(a), 0) - n * p1[a]) <= 4.5 * np.sqrt(n * p1[a] * (1 - p1[a])) + 1
    a = int(np.argmax(p1))
    p2 = torch.softmax(llm.engine.step([SequenceStep(slot, [a], [0])])[0].double() / t, 0).cpu().numpy()
    m = firsts[a]
    for b in np.argsort(-p2)[:8]:
        assert abs(seconds.get((a, int(b)), 0) - m * p2[b]) <= 4.5 * np.sqrt(m * p2[b] * (1 - p2[b])) + 1


def test_what_is_refused(folder, small_folder, tmp_path):
    from nnis_b200 import LLM, GenerationConfig, LookupDrafter, SamplingConfig, SessionDrafter
    llm = LLM(folder, dtype="float32", max_tokens=1 << 13, max_batch=4)
    s = llm.new_session()
    for kw in (dict(drafts=0), dict(sampling=SamplingConfig(seed=1, top_k=3)), dict(sampling=SamplingConfig(seed=1, temperature=-1.0))):
        with pytest.raises(ValueError):
            s.generate_drafted([1, 2], GenerationConfig(4), LookupDrafter(), **kw)
    with pytest.raises(ValueError):
        s.generate_drafted([], GenerationConfig(4), LookupDrafter())
    with pytest.raises(ValueError):
        s.generate_drafted([1] * 4095, GenerationConfig(4), LookupDrafter())
    other = LLM(make_model(str(tmp_path), CONFIGS["A"], 1), dtype="float32", max_tokens=1 << 12, max_batch=2)
    with pytest.raises(ValueError):
        s.generate_drafted([1, 2], GenerationConfig(4), SessionDrafter(other))


def test_designs_with_states_and_windows_fork_and_refuse_drafts(tmp_path):
    """States are copied where a sequence forks, whatever the mixers: a prompt shared by sequences of Nafezen, Sedopel and Selovik
    gives the tokens of each alone; drafts, which would have to be taken back, are refused."""
    import nafezen_models
    import sedopel_models
    import selovik_models
    from nnis_b200 import LLM, GenerationConfig, LookupDrafter
    for i, module in enumerate((nafezen_models, sedopel_models, selovik_models)):
        name, cfg = next((n, c) for n, c in module.CONFIGS.items())
        folder = module.make_model(str(tmp_path / f"m{i}"), cfg, 5)
        llm = LLM(folder, dtype="float32", max_tokens=1 << 13, max_batch=8)
        vocab = llm.spec.vocab_size
        document = tokens(50 + i, 70, vocab)
        prompts = [document + tokens(60 + j, 1 + j, vocab) for j in range(3)]
        shared = llm.generate(prompts, max_new_tokens=8, share_prefix=True, stop_token_ids=[])
        alone = [llm.generate([p], max_new_tokens=8, stop_token_ids=[])[0] for p in prompts]
        assert [r.error for r in shared] == [None] * 3, name
        assert [r.token_ids for r in shared] == [r.token_ids for r in alone], name
        assert set(llm.engine.cache.usage()["pages_held"]) <= {0}
        if llm.engine.cache.fixed_history():
            with pytest.raises(ValueError):
                llm.new_session().generate_drafted([1, 2], GenerationConfig(4), LookupDrafter())


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_captured_steps_of_drafts(folder, dtype):
    """Several tokens of a sequence as rows of a captured step, over page ends, with tokens taken back between them, two
    sessions and two numbers of tokens in turn, one of them forked: logits as token by token."""
    from nnis_b200 import LLM
    from nnis_b200.engine import SequenceStep
    llm = LLM(folder, dtype=dtype, max_tokens=1 << 14, max_batch=16)
    engine, backend = llm.engine, llm.backend
    a, b = engine.acquire_slot(), engine.acquire_slot()
    history = {a: tokens(70, 1270), b: tokens(71, 60)}
    for s, h in history.items():
        engine.step([SequenceStep(s, h, [])])
    for turn in range(24):
        if turn == 12:
            c = engine.fork(a)
            history[c] = list(history[a])
        for s, n in ((a, 5), (b, 3 if turn % 2 else 5)):
            new = tokens(1000 + 10 * turn + s, n)
            got = backend.drafted_logits(s, new, True).cpu().numpy()
            keep = 1 + turn % n
            if turn % 6 == 0:
                other = engine.acquire_slot()
                engine.step([SequenceStep(other, history[s], [])])
                want = np.concatenate([engine.step([SequenceStep(other, [t], [0])]).cpu().numpy() for t in new])
                engine.release_slot(other)
                assert close(got, want, dtype), (turn, s)
            history[s] += new[:keep]
            engine.truncate(s, len(history[s]))
            engine.cache.check()
    for s in (a, c):  # what was forked is as it was
        t = tokens(5, 1)
        got = engine.step([SequenceStep(s, t, [0])])[0].cpu().numpy()
        other = engine.acquire_slot()
        want = engine.step([SequenceStep(other, history[s] + t, [len(history[s])])])[0].cpu().numpy()
        engine.release_slot(other)
        assert close(got, want, dtype)
    engine.check_status()
