"""Models whose cache, matrices or both are held in 8 bits: logits against the plain decoder with the same roundings, generation."""
import random

import numpy as np
import pytest
import torch

import int8_plain
import plain_llama
from helpers import CONFIGS, load_plain_weights, make_model, read_config_json, read_step, three_cuts
from test_shared_sequences_gpu import SHARED, tokens

pytestmark = pytest.mark.gpu
KINDS = {"cache": dict(cache_dtype="int8"), "weights": dict(weight_dtype="int8"), "both": dict(cache_dtype="int8", weight_dtype="int8")}
# Of the largest logit.  A value that another order of sums moves by an ulp may fall to the neighbouring code, a step of top / 127:
# with top three times the rows' mean square root, 0.024 of that root.  Whatever that row meets afterwards is moved by it, so that in
# float32 too, once one code of a sequence has fallen otherwise, some of the codes of its later products, keys and values do: with one in
# ten, three layers of six such roundings carry sqrt(18 * 0.1) * 0.024 = 0.032 of a logit's mean square root, and the largest of the
# ten thousand logits compared at once is four times that, 0.13 of it, while the largest logit is three to four times it: 0.04.
# Half as much again for the weights' own spread.  (The operators alone are held to their last bits elsewhere.)
LIMIT = {"float32": 0.06, "bfloat16": 0.06}
MODELS = {**CONFIGS, "D": SHARED, "E": {**SHARED, "head_dim": 128, "num_attention_heads": 4}}


@pytest.fixture(scope="module", params=sorted(MODELS))
def folder(request, tmp_path_factory):
    return make_model(str(tmp_path_factory.mktemp("int8" + request.param)), MODELS[request.param], 11)


def near(got, want, dtype):
    scale = max(1.0, float(np.abs(want).max()))
    assert float(np.abs(got - want).max()) <= LIMIT[dtype] * scale


def plain_in_int8(monkeypatch, weights, cache, kind):
    """The plain decoder with 8-bit matrices (each row of activations in codes too) and 8-bit keys and values."""
    linear, attention = plain_llama.linear, plain_llama.causal_attention
    blocks = {id(t) for name, t in weights.items() if ".layers." in name}

    def values(x):
        codes, scales = int8_plain.codes_of(x)
        return codes.double() * scales.double()[..., None]

    if kind != "cache":
        monkeypatch.setattr(plain_llama, "linear", lambda x, w, b=None: linear(values(x), values(w), b) if id(w) in blocks else linear(x, w, b))
    if kind != "weights":
        monkeypatch.setattr(plain_llama, "causal_attention", lambda q, k, v, window=0: attention(q, values(k), values(v), window))


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("kind", sorted(KINDS))
def test_logits_are_the_plain_decoders(folder, dtype, kind, tmp_path, monkeypatch):
    """Whole prompts, tokens one by one after a prompt, ragged batches in chunks."""
    from nnis_b200.engine import Engine
    from nnis_b200.engine.replay import replay
    engine = Engine.from_dir(folder, dtype=dtype, max_tokens=1 << 13, **KINDS[kind])
    cfg = read_config_json(folder)
    trace, sequences = three_cuts(random.Random(5), cfg["vocab_size"])
    replay(engine, trace.lines, str(tmp_path))
    assert engine.cache.usage()["slots_held"] == 0 and engine.cache.usage()["pages_held"] == [0]
    engine.cache.check()
    weights, bf16 = load_plain_weights(folder, as_bf16=dtype == "bfloat16"), dtype == "bfloat16"
    plain_in_int8(monkeypatch, weights, True, kind)
    plain = {}
    for step, rows in trace.rows.items():
        got = read_step(str(tmp_path), step, cfg["vocab_size"])
        for rid, _ in rows:
            if rid not in plain:
                plain[rid] = plain_llama.forward(cfg, weights, sequences[rid], emulate_bf16=bf16)
        near(got, torch.stack([plain[rid][pos] for rid, pos in rows]).numpy(), dtype)
    engine.check_status()


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("kind", sorted(KINDS))
def test_captured_steps_forks_and_truncations(dtype, kind, tmp_path):
    """Captured decode steps of forked sequences over page ends, then back to earlier lengths: each step's logits are those of a prompt of
    the same tokens."""
    from nnis_b200 import LLM
    from nnis_b200.engine import SequenceStep
    llm = LLM(make_model(str(tmp_path), SHARED, 3), dtype=dtype, max_tokens=1 << 13, max_batch=8, **KINDS[kind])
    engine, step = llm.engine, llm.backend.step
    first = engine.acquire_slot()
    history = {first: tokens(1, 187)}
    engine.step([SequenceStep(first, history[first], [])])

    def check(logits):
        for row, (slot, fed) in enumerate(history.items()):
            alone = engine.acquire_slot()
            near(logits[row].cpu().numpy(), engine.step([SequenceStep(alone, fed, [len(fed) - 1])])[0].cpu().numpy(), dtype)
            engine.release_slot(alone)

    for turn in range(8):
        if turn in (1, 3):
            new = engine.fork(first)
            history[new] = list(history[first])
        if turn == 6:
            engine.truncate(first, 100)
            del history[first][100:]
        for i, slot in enumerate(history):
            history[slot].append(17 * turn + i)
        check(step([SequenceStep(slot, fed[-1:], [0]) for slot, fed in history.items()]).clone())
    snapshot = engine.snapshot(first)
    step([SequenceStep(first, [9], [0])])
    engine.restore(snapshot)
    engine.compact()
    for slot in history:
        history[slot].append(3)
    check(step([SequenceStep(slot, fed[-1:], [0]) for slot, fed in history.items()]).clone())
    for slot in history:
        engine.release_slot(slot)
    engine.cache.check()
    engine.check_status()


@pytest.mark.parametrize("kind", sorted(KINDS))
def test_recurring_prompt_steps_are_captured(kind, tmp_path):
    """A prompt shape that comes a second and a third time runs from a graph with scratch of its own for the pages read back."""
    from nnis_b200.engine import Engine, SequenceStep
    engine = Engine.from_dir(make_model(str(tmp_path), SHARED, 3), max_tokens=1 << 13, **KINDS[kind])
    for turn in range(4):
        got = []
        for chunk in ((0, 300), (300, 600)):  # (each shape recurs; the second reads back what the first has written)
            if chunk[0] == 0:
                slots = [engine.acquire_slot() for _ in range(2)]
            batch = [SequenceStep(s, tokens(20 + turn + i, 600)[chunk[0]:chunk[1]], [299]) for i, s in enumerate(slots)]
            got.append(engine.step(batch).cpu().numpy())
        if turn == 0:
            whole = engine.acquire_slot()
        for i, slot in enumerate(slots):
            engine.truncate(whole, 0)
            want = engine.step([SequenceStep(whole, tokens(20 + turn + i, 600), [299, 599])]).cpu().numpy()
            near(np.stack([got[0][i], got[1][i]]), want, "bfloat16")
            engine.release_slot(slot)
    engine.check_status()


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_few_tokens_after_a_long_context_read_the_codes(dtype, tmp_path, monkeypatch):
    """Drafted tokens attend over the codes row by row, longer chunks over pages read back: the same logits."""
    from nnis_b200.csrc import ops
    from nnis_b200.engine import Engine, SequenceStep
    engine = Engine.from_dir(make_model(str(tmp_path), SHARED, 3), dtype=dtype, max_tokens=1 << 13, cache_dtype="int8")
    calls = []
    for name in ("attention_int8", "read_pages_int8"):
        real = getattr(ops, name)
        monkeypatch.setattr(ops, name, lambda *a, _real=real, _name=name: (calls.append(_name), _real(*a))[1])
    slots = [engine.acquire_slot() for _ in range(2)]
    engine.step([SequenceStep(s, tokens(4 + i, 500 + i), []) for i, s in enumerate(slots)])
    assert calls == ["read_pages_int8"] * 2
    few = engine.step([SequenceStep(slots[0], tokens(6, 5), range(5)), SequenceStep(slots[1], tokens(7, 1), [0])]).cpu().numpy()
    assert calls[2:] == ["attention_int8"] * 2
    for s, n in zip(slots, (500, 501)):
        engine.truncate(s, n)
    many = engine.step([SequenceStep(slots[0], tokens(6, 5) + tokens(8, 70), range(5)), SequenceStep(slots[1], tokens(7, 1), [0])]).cpu().numpy()
    assert calls[4:] == ["read_pages_int8"] * 2
    near(few, many, dtype)


@pytest.mark.parametrize("kind", sorted(KINDS))
def test_generation(kind, tmp_path):
    """Greedy, sampled, behind a shared prompt, one token at a time and drafted: in float32 the tokens are the same whichever way."""
    from nnis_b200 import LLM, GenerationConfig, LookupDrafter, SamplingConfig
    llm = LLM(make_model(str(tmp_path), SHARED, 3), dtype="float32", max_tokens=1 << 13, max_batch=8, **KINDS[kind])
    document = tokens(2, 200)
    prompts = [document + [5 + i] for i in range(3)]
    want = [llm.generate([p], max_new_tokens=20, stop_token_ids=[])[0].token_ids for p in prompts]
    assert [r.token_ids for r in llm.generate(prompts, max_new_tokens=20, stop_token_ids=[])] == want
    assert [r.token_ids for r in llm.generate(prompts, max_new_tokens=20, stop_token_ids=[], share_prefix=True)] == want
    session = llm.new_session()
    assert list(session.generate(prompts[0], GenerationConfig(20))) == want[0]
    drafted = llm.new_session()
    assert list(drafted.generate_drafted(prompts[1], GenerationConfig(20), LookupDrafter(), drafts=4)) == want[1]
    policy = SamplingConfig(seed=7, temperature=0.8, top_k=40, top_p=0.95)
    sampled = [llm.generate([p], max_new_tokens=9, sampling=policy, stop_token_ids=[])[0].token_ids for p in prompts]
    assert [r.token_ids for r in llm.generate(prompts, max_new_tokens=9, sampling=policy, stop_token_ids=[])] == sampled


def test_the_cache_takes_the_bytes_it_says(tmp_path):
    from nnis_b200.engine import Engine
    made = make_model(str(tmp_path), SHARED, 3)
    wide, narrow = Engine.from_dir(made, max_tokens=1 << 12), Engine.from_dir(made, max_tokens=1 << 12, **KINDS["both"])
    layers, heads, d = 2, 2, 64
    assert wide.cache.kv_bytes_per_token() == layers * heads * d * 4 and narrow.cache.kv_bytes_per_token() == layers * heads * (d * 2 + 8)
    assert narrow.memory()["kv_bytes"] * 128 == wide.memory()["kv_bytes"] * 68
    assert narrow.memory()["weights_bytes_per_step"] < 0.75 * wide.memory()["weights_bytes_per_step"]


def test_the_command_line(tmp_path, capsys):
    from nnis_b200.cli.main import parse_args, run
    made = make_model(str(tmp_path), SHARED, 3)
    import io
    out = io.StringIO()
    assert run(parse_args(["generate", "--model", made, "--prompt-ids", "1,2,3", "--max-new-tokens", "4", "--cache-dtype", "int8",
                           "--weight-dtype", "int8"]), out) == 0
    assert out.getvalue().strip()


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_drafted_steps_are_captured(dtype, tmp_path, monkeypatch):
    """Over an 8-bit cache a sequence's drafted tokens run as a replayed step, a row each; the logits are those of a prompt of the same
    tokens."""
    from nnis_b200 import LLM, GenerationConfig, LookupDrafter
    from nnis_b200.engine import SequenceStep
    from nnis_b200.engine.decode import GraphDecoder
    llm = LLM(make_model(str(tmp_path), SHARED, 3), dtype=dtype, max_tokens=1 << 13, max_batch=4, cache_dtype="int8")
    launched, launch = [], GraphDecoder.launch
    monkeypatch.setattr(GraphDecoder, "launch", lambda self: (launched.append(self.rows), launch(self))[1])
    engine, backend = llm.engine, llm.backend
    slot, fed = engine.acquire_slot(), tokens(30, 122)
    engine.step([SequenceStep(slot, fed, [])])
    for turn, count in enumerate((5, 5, 3, 8, 1, 5)):  # (over the end of a page)
        drafted = tokens(40 + turn, count)
        got = backend.drafted_logits(slot, drafted, True).cpu().numpy()
        alone = engine.acquire_slot()
        want = engine.step([SequenceStep(alone, fed + drafted, list(range(len(fed), len(fed) + count)))]).cpu().numpy()
        engine.release_slot(alone)
        near(got, want, dtype)
        kept = max(1, count - turn % 3)  # some are rejected
        fed = fed + drafted[:kept]
        engine.truncate(slot, len(fed))
    assert len(launched) == 6 and set(launched) == {1, 4, 8}
    engine.release_slot(slot)
    phrase = tokens(50, 12) * 6
    want = llm.generate([phrase], max_new_tokens=40, stop_token_ids=[])[0].token_ids
    before = len(launched)
    got = list(llm.new_session().generate_drafted(phrase, GenerationConfig(40), LookupDrafter(), drafts=4))
    assert len(launched) > before
    if dtype == "float32":
        assert got == want
    engine.check_status()


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("config", ["A", "D", "E"])
def test_prompts_beside_single_tokens(dtype, config, tmp_path, monkeypatch):
    """A step of two prompts among sequences that bring one token or a few, which attend over the codes while the prompts' pages are read back:
    logits as of the same tokens step by step; run by run and replayed.  No more pages are read back than the prompts have."""
    from nnis_b200.csrc import ops
    from nnis_b200.engine import Engine, SequenceStep
    monkeypatch.setattr(ops, "INT8_READ_BACK", 0)
    engine = Engine.from_dir(make_model(str(tmp_path), {**MODELS[config], "max_position_embeddings": 2048}, 3), dtype=dtype, max_tokens=1 << 14,
                             cache_dtype="int8")
    read, real = [], ops.read_pages_int8
    monkeypatch.setattr(ops, "read_pages_int8", lambda *a: (read.append(a[6].shape[0]), real(*a))[1])
    vocab = engine.spec.vocab_size
    held, new = [700, 1, 0, 300, 90, 650], [1, 3, 150, 1, 130, 5]
    history = [[t % vocab for t in tokens(60 + i, a + 4 * b)] for i, (a, b) in enumerate(zip(held, new))]
    slots = [engine.acquire_slot() for _ in held]
    for s, h, n in zip(slots, history, held):
        if n:
            engine.step([SequenceStep(s, h[:n], [])])
    want = []
    for h, n, c in zip(history, held, new):
        alone = engine.acquire_slot()
        want.append(engine.step([SequenceStep(alone, h[:n + c], list(range(n, n + c)))]).cpu().numpy())
        engine.release_slot(alone)
    for turn in range(4):  # (captured in the second, replayed from the third on)
        read.clear()
        got = engine.step([SequenceStep(s, h[n:n + c], list(range(c))) for s, h, n, c in zip(slots, history, held, new)]).cpu().numpy()
        assert set(read) <= {3 + 4}
        near(got, np.concatenate(want), dtype)
        for s, n in zip(slots, held):
            engine.truncate(s, n)
    engine.check_status()


@pytest.mark.parametrize("from_dir", [True, False])
def test_loading_in_8_bits_takes_less_than_the_16_bit_weights(from_dir, tmp_path):
    """Matrices that would not fit in 16 bits may be held in 8: at no time are there 16-bit tensors of more than a block beside the codes."""
    from nnis_b200.config import read_config
    from nnis_b200.engine import Engine
    made = make_model(str(tmp_path), {**SHARED, "hidden_size": 768, "intermediate_size": 3000, "num_hidden_layers": 8, "head_dim": 64,
                                      "num_attention_heads": 12, "num_key_value_heads": 4}, 3)
    kept = load_plain_weights(made, True)
    whole = 2 * sum(t.numel() for t in kept.values())
    block = 2 * sum(t.numel() for name, t in kept.items() if ".layers.0." in name)
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    if from_dir:
        engine = Engine.from_dir(made, max_tokens=64, weight_dtype="int8")
    else:
        engine = Engine.from_spec(read_config(made).to_spec(), {n: t.to(torch.bfloat16) for n, t in kept.items()}, max_tokens=64, weight_dtype="int8")
    peak = torch.cuda.max_memory_allocated() - before
    tables = engine.model.embedding.table.numel() * 2 * (1 if engine.model.head.weight is engine.model.embedding.table else 2)
    # codes and scales, the tables, a block's tensors and what they are joined to; a page of cache and small things
    assert peak < (whole - tables) // 2 * 1.02 + tables + 2 * block + (4 << 20) < 0.9 * whole
