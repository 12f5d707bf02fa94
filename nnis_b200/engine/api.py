"""The Python entry point.

``LLM`` loads a model folder (the model class comes from config.json) and
generates for batches of prompts; ``InferenceSession`` is NNIS's one-sequence
surface - ``prefill``, ``decode_one``, ``generate``, ``generate_sampled``,
``reset`` (crates/nnis-model/src/runtime.rs:745-899,
crates/nnis-model/src/sampling.rs:216-255) - on a slot of the shared cache.
NNIS's own Python entry is a process wrapper around its binary with the options
``model_dir``, ``tokenizer_file``, ``prompt``, ``device_ordinal``,
``max_new_tokens`` (tools/nnis_hub_hf_generate.py:189-231); the same names are
used here in process.
"""
from __future__ import annotations

import contextlib
import warnings
from typing import Callable, Dict, List, Optional, Sequence, Union

import numpy as np
import torch

from ..sampling import SamplingConfig
from ..sampling import device as device_sampling
from ..cache import PAGE_SIZE
from ..csrc import ops
from .decode import GraphDecoder
from .engine import Engine, SequenceStep, StepError
from .sharing import BatchUnits, rooms_of
from .generate import (DEFAULT_MAX_NEW_TOKENS, GenerationConfig, GenerationRequest,
                       GenerationResult, Generator, StreamControl)

Prompt = Union[str, Sequence[int]]

MAX_SHARED_DECODERS = 8  # captured steps kept for batches whose sequences share pages
DRAFTED_ROWS = 64  # tokens of one sequence that a captured step takes, however few sequences a batch may hold


class EngineBackend:
    """What the generation loop needs of an engine."""

    def __init__(self, engine: Engine, max_rows: int = 64, pipeline: bool = True,
                 max_step_tokens: int = 16384):
        self.engine = engine
        self.max_rows = max_rows
        # most tokens of one prompt step; longer batches of prompts run in portions
        self.max_step_tokens = max_step_tokens
        # True: all-greedy batches keep tokens on the device and the host reads
        # picks one step late.  False: every step's tokens come from the host.
        self.pipeline = pipeline
        self._decoders = {}
        self._uncaptured = set()  # keys of decoders whose capture has failed for a session
        self._views = {}
        self._shared = BatchUnits(engine)
        self._drafted: Dict[int, BatchUnits] = {}  # by number of tokens
        self._pinned = None
        self._picked = None
        self._picked_for = None
        self._pick_host = None
        self._pick_np = None
        self.h2d_bytes = 0  # counted from the tensors copied, for measurements
        self.d2h_bytes = 0
        parts = [p for b in engine.model.blocks for p in b.parts()]
        if not all(getattr(p, "device_only", True) for p in parts):
            self.decode_greedy = None  # a part loops on the host: no graph

    def acquire_slot(self) -> int:
        return self.engine.acquire_slot()

    def release_slot(self, slot: int) -> None:
        self.engine.release_slot(slot)

    def fork_slot(self, slot: int) -> int:
        return self.engine.fork(slot)

    def step(self, batch, need_logits: bool = True):
        """Logits [len(batch) wanted rows, vocab] (or None when ``need_logits`` is
        false and the step could pick on the device: ``greedy`` then has the
        picks).  Steps in which every sequence brings one token and wants its
        logits run as a CUDA graph whose inputs (tokens, positions, page tables)
        come from the host in one copy."""
        single = True
        for s in batch:
            want = s.want
            if len(s.tokens) != 1 or len(want) != 1 or want[0] != 0:
                single = False
                break
        if not single or self.decode_greedy is None or len(batch) > self.max_rows:
            self._picked = None
            return self.engine.step_in_portions(batch, self.max_step_tokens)
        vocab = self.engine.spec.vocab_size
        slots, tokens = [], []
        for s in batch:
            token = int(s.tokens[0])
            if not 0 <= token < vocab:
                raise StepError(f"slot {s.slot}: token {s.tokens[0]} is outside the vocabulary")
            slots.append(s.slot)
            tokens.append(token)
        dec = self._replay(slots, tokens, need_logits)
        n = len(batch)
        views = self._views.get((id(dec), n))
        if views is None:  # (slicing a tensor costs microseconds: once per decoder and row count)
            views = self._views[(id(dec), n)] = (dec.picked[:n], dec.logits[:n] if dec.logits is not None else None)
        self._picked = views[0]
        return views[1] if need_logits else None

    def _replay(self, slots: List[int], tokens: List[int], need_logits: bool,
                dec: Optional[GraphDecoder] = None) -> GraphDecoder:
        """One token per slot as a replay of the captured step (``dec``: its decoder, where the caller has it); its inputs go
        up in one copy."""
        cache = self.engine.cache
        positions = [cache.length(s) for s in slots]
        new_lengths = [p + 1 for p in positions]
        cache.reserve(slots, new_lengths)
        if dec is None:
            dec = self._shared_decoder(slots, positions, max(new_lengths), need_logits)
        self.h2d_bytes += dec.upload(tokens, positions, slots)
        dec.launch()
        cache.commit(slots, new_lengths)
        return dec

    def decode_logits(self, slot: int, token: int, again: bool) -> torch.Tensor:
        """Logits [vocab] of one sequence's next token.  A step of the SmolLM2-135M shape is 154 launches, 4.1 ms from
        Python one by one and 0.47 ms as a replay; to capture one takes 11 to 29 ms, what three to eight replays save, so the
        first tokens that a session decodes (``again`` False) capture nothing, and replay only where the graph is there
        already."""
        engine = self.engine
        key = self._decoder_key(1, engine.cache.length(slot) + 1, True)
        dec = self._decoders.get(key)
        if dec is None or dec.graph is None:
            capture = again and self.decode_greedy is not None and key not in self._uncaptured \
                and 0 <= token < engine.spec.vocab_size
            dec = self._captured(key) if capture else None
        if dec is None or not 0 <= token < engine.spec.vocab_size:
            return engine.step([SequenceStep(slot, [token], [0])])[0]  # (which says what is wrong with a token)
        return self._replay([slot], [token], True, dec).logits[0]

    def drafted_logits(self, slot: int, tokens: List[int], again: bool) -> torch.Tensor:
        """Logits [tokens, vocab] of one sequence's next tokens, a token and drafts after it.  From the third such step on
        (``again``) it is a captured step whose rows are the tokens: what a sequence of the SmolLM2-135M shape waits for is
        then 0.6 ms instead of the 8 of its launches from Python one by one."""
        engine, cache, n = self.engine, self.engine.cache, len(tokens)
        vocab = engine.spec.vocab_size
        if not again or self.decode_greedy is None or not engine.model.all_share or n > max(self.max_rows, DRAFTED_ROWS) \
                or not all(0 <= t < vocab for t in tokens):
            return engine.step([SequenceStep(slot, tokens, list(range(n)))], drafted=True)
        held = cache.length(slot)
        positions = list(range(held, held + n))
        cache.reserve([slot], [held + n])
        key = self._decoder_key(n, held + n, True)
        units = self._drafted.setdefault(n, BatchUnits(engine, drafted=True)).units([slot] * n, positions, key[0])
        dec = self._captured(key if units is None else (*key, rooms_of(units)))
        if dec is None:
            return engine.step([SequenceStep(slot, tokens, list(range(n)))], drafted=True)
        if units is not None:
            dec.plans.fill(units)
        self.h2d_bytes += dec.upload(tokens, positions, [slot] * n)
        dec.launch()
        cache.commit([slot], [held + n])
        return dec.logits[:n]

    def _captured(self, key) -> Optional[GraphDecoder]:
        """The decoder of this key with its graph, captured now if it has none.  Where that fails (no memory for its buffers,
        say) None, and it is not tried again."""
        if key in self._uncaptured:
            return None
        try:
            self._made(key).capture()
        except RuntimeError as error:
            self._decoders.pop(key, None)
            self._uncaptured.add(key)
            warnings.warn(f"a decode step of up to {key[1]} positions could not be captured and is launched kernel by "
                          f"kernel: {error}", RuntimeWarning)
            return None
        return self._decoders[key]

    def greedy(self, logits: Optional[torch.Tensor]) -> List[int]:
        if self._picked is not None:  # the graph has picked already
            n = self._picked.numel()
            self.d2h_bytes += n * 4
            if self._pick_host is None or self._pick_host.numel() < n:
                self._pick_host = torch.empty(max(n, self.max_rows), dtype=torch.int32, pin_memory=True)
                self._pick_np = self._pick_host.numpy()
            ops.copy_async(self._pick_host[:n], self._picked)
            ops.stream_synchronize()
            return self._pick_np[:n].tolist()
        out = self.engine.workspace.get("picked", (logits.shape[0],), torch.int32)
        device_sampling.greedy(logits, out)
        self.d2h_bytes += out.numel() * 4
        return out.tolist()

    def new_rng(self, seed: int) -> torch.Tensor:
        """A SplitMix64 state on the device (int64 [1]) for one request."""
        return device_sampling.seed_states([seed], self.engine.device)

    def sample_temperature(self, logits: torch.Tensor, rows: Sequence[int],
                           temperatures: Sequence[float], states: Sequence[torch.Tensor]) -> List[int]:
        """One seeded draw per named row of ``logits`` on the device; each row's
        generator state advances in place."""
        index = torch.tensor(list(rows), dtype=torch.long, device=logits.device)
        picked_rows = logits if len(rows) == logits.shape[0] and list(rows) == list(range(len(rows))) \
            else logits[index].contiguous()
        temps = torch.tensor([float(t) for t in temperatures], dtype=torch.float32, device=logits.device)
        state = torch.cat(list(states))
        out = torch.empty(len(rows), dtype=torch.int32, device=logits.device)
        device_sampling.temperature(picked_rows, temps, state, out)
        for s, new in zip(states, state.split(1)):
            s.copy_(new)
        self.d2h_bytes += out.numel() * 4
        return out.tolist()

    def host_rows(self, logits: torch.Tensor, rows: Sequence[int]) -> np.ndarray:
        if len(rows) == logits.shape[0]:
            return logits.cpu().numpy()
        index = torch.tensor(list(rows), dtype=torch.long, device=logits.device)
        return logits[index].cpu().numpy()


    # -- greedy decoding with the batch's state on the device -------------------
    def _decoder_key(self, rows: int, max_context: int, want_logits: bool):
        bucket = 1
        while bucket < rows:
            bucket *= 2
        pages = 4
        while pages * PAGE_SIZE < max_context:
            pages *= 2
        context = min(pages * PAGE_SIZE, self.engine.spec.max_positions)
        return bucket, context, want_logits

    def _decoder(self, rows: int, max_context: int, want_logits: bool = False, rooms: Optional[tuple] = None) -> GraphDecoder:
        key = self._decoder_key(rows, max_context, want_logits)
        return self._made(key if rooms is None else (*key, rooms))

    def _made(self, key) -> GraphDecoder:
        """The decoder of this key: (rows, positions, whether it gives logits) and, if sequences share pages, its plans' sizes."""
        if len(key) > 3:
            # (what sequences share takes many forms: of the steps captured for it the least recently used goes)
            shared = [k for k in self._decoders if len(k) > 3]
            if key in self._decoders:
                self._decoders[key] = self._decoders.pop(key)
            elif len(shared) >= MAX_SHARED_DECODERS:
                gone = self._decoders.pop(shared[0])
                self._views = {k: v for k, v in self._views.items() if k[0] != id(gone)}
        if key not in self._decoders:
            self._decoders[key] = GraphDecoder(self.engine, *key[:3], rooms=key[3] if len(key) > 3 else None)
        return self._decoders[key]

    def _shared_decoder(self, slots: Sequence[int], positions: Sequence[int], max_context: int, want_logits: bool = False,
                        ahead: Optional[int] = None) -> GraphDecoder:
        """The decoder of these sequences, whose pages have been reserved: one that reads what they share once, where that
        pays.  ``ahead``: pages that they will grow by before the caller asks again (None: it asks at every step)."""
        rows = self._decoder_key(len(slots), max_context, want_logits)[0]
        units = self._shared.units(slots, positions, rows, ahead)
        dec = self._decoder(len(slots), max_context, want_logits, rooms_of(units))
        if units is not None:
            dec.plans.fill(units)
        return dec

    def decode_greedy(self, rows, emit) -> None:
        """rows: (request, slot, next input token, its position, tokens still to
        pick).  Calls ``emit(request, token)`` for every pick in order; a False
        return means that sequence has ended (its slot is already given back)."""
        cache = self.engine.cache
        slots, positions = [r[1] for r in rows], [r[3] for r in rows]
        longest = max(pos + left + 1 for _, _, _, pos, left in rows)
        if cache.shares_pages():  # (the pages that they will write into, copied together)
            cache.reserve(slots, [p + 1 for p in positions])
            dec = self._shared_decoder(slots, positions, longest, ahead=max(left for *_, left in rows) // PAGE_SIZE + 1)
        else:
            dec = self._decoder(len(rows), longest)
        # (shared pages are read by the table of the first of their sequences, which stays as it is when that one ends)
        with cache.in_place() if dec.plans is not None else contextlib.nullcontext():
            self._greedy_steps(dec, rows, emit)

    def _greedy_steps(self, dec: GraphDecoder, rows, emit) -> None:
        """``decode_greedy`` by the given decoder."""
        cache = self.engine.cache
        live = {}
        for r, (i, slot, token, pos, left) in enumerate(rows):
            dec.set_row(r, slot, token, pos)
            live[r] = [i, slot, pos, left]
        for r in range(len(rows), dec.rows):
            dec.clear_row(r)
        if self._pinned is None or self._pinned.shape[1] < dec.rows:
            self._pinned = torch.empty((2, max(dec.rows, self.max_rows)), dtype=torch.int32,
                                       pin_memory=True)
        ended = set()
        pending = None
        turn = 0
        while live or pending is not None:
            launched = None
            if live:
                for r, (i, slot, pos, left) in live.items():
                    cache.reserve([slot], [pos + 1])
                    dec.sync_pages(r, slot)
                    cache.commit([slot], [pos + 1])
                dec.launch()
                buf = self._pinned[turn % 2]
                turn += 1
                launched = (dec.picks_to_host(buf[:dec.rows]), buf, {r: v[0] for r, v in live.items()})
                for r in list(live):
                    live[r][2] += 1
                    live[r][3] -= 1
                    if live[r][3] == 0:  # this step picked its last token
                        del live[r]
                        dec.clear_row(r)
            if pending is not None:
                event, buf, who = pending
                event.synchronize()
                for r, i in who.items():
                    if i in ended:
                        continue  # it had stopped before this step was read: the pick is dropped
                    if not emit(i, int(buf[r])):
                        ended.add(i)
                        if r in live:
                            del live[r]
                            dec.clear_row(r)
            pending = launched


def load_tokenizer(tokenizer_file: str):
    from tokenizers import Tokenizer
    return Tokenizer.from_file(tokenizer_file)


class LLM:
    def __init__(self, model_dir: str, dtype: str = "bfloat16", device_ordinal: int = 0,
                 device: Optional[str] = None, max_tokens: Optional[int] = None,
                 max_batch: int = 64, tokenizer_file: Optional[str] = None,
                 pipeline_decode: bool = True, device_sampling: bool = False,
                 max_step_tokens: int = 16384, cache_dtype: Optional[str] = None, weight_dtype: Optional[str] = None):
        """``cache_dtype="int8"``: keys and values are held in 8-bit codes with a scale for every position and head, half the bytes of
        bfloat16 to keep and to read.  ``weight_dtype="int8"``: the layers' matrices in 8-bit codes with a scale for each output
        channel, multiplied with each token's activations in 8-bit codes as whole numbers; embedding and head keep their type.
        Either, both or none; refused with a ValueError for models whose layers have no such form (``Llama`` has both)."""
        device = device if device is not None else f"cuda:{int(device_ordinal)}"
        self.max_batch = max_batch
        if max_tokens is None:
            max_tokens = 1 << 17
        self.engine = Engine.from_dir(model_dir, dtype=dtype, device=device, max_tokens=max_tokens,
                                      max_slots=max(max_batch, 1), cache_dtype=cache_dtype, weight_dtype=weight_dtype)
        self.spec = self.engine.spec
        self.tokenizer = load_tokenizer(tokenizer_file) if tokenizer_file else None
        self.backend = EngineBackend(self.engine, max_batch, pipeline_decode, max_step_tokens)
        self._generator = Generator(self.backend, self.spec.vocab_size,
                                    self.spec.max_positions, max_batch, max_tokens, device_sampling)

    # -- text ---------------------------------------------------------------
    def encode(self, text: str) -> List[int]:
        if self.tokenizer is None:
            raise ValueError("a text prompt needs a tokenizer (tokenizer_file=...)")
        # special tokens on, as NNIS's command line does (crates/nnis-cli/src/main.rs:1075-1090)
        return list(self.tokenizer.encode(text, add_special_tokens=True).ids)

    def decode(self, ids: Sequence[int]) -> str:
        if self.tokenizer is None:
            raise ValueError("decoding to text needs a tokenizer (tokenizer_file=...)")
        return self.tokenizer.decode(list(ids), skip_special_tokens=True)

    # -- generation ---------------------------------------------------------
    def generate(self, prompts: Sequence[Prompt], max_new_tokens: int = DEFAULT_MAX_NEW_TOKENS,
                 sampling: Union[None, SamplingConfig, Sequence[Optional[SamplingConfig]]] = None,
                 stop_token_ids: Optional[Sequence[int]] = None,
                 on_token: Optional[Callable[[int, int], Optional[StreamControl]]] = None,
                 share_prefix: bool = False) -> List[GenerationResult]:
        """Greedy unless ``sampling`` is given (one policy for all prompts or one
        per prompt).  ``stop_token_ids=None`` takes config.json's eos ids.
        ``on_token(prompt index, token)`` sees tokens as they are emitted and may return
        ``StreamControl.STOP`` to end that prompt's generation; the others go on.
        ``share_prefix``: prompts that begin with the same tokens (several samples of one
        prompt, questions behind one document) run those once and share their pages."""
        stops = tuple(self.spec.stop_token_ids if stop_token_ids is None else stop_token_ids)
        if sampling is None or isinstance(sampling, SamplingConfig):
            sampling = [sampling] * len(prompts)
        if len(sampling) != len(prompts):
            raise ValueError(f"{len(prompts)} prompts but {len(sampling)} sampling policies")
        gen = GenerationConfig(max_new_tokens=max_new_tokens, stop_token_ids=stops)
        requests = [GenerationRequest(self.encode(p) if isinstance(p, str) else list(p), gen, s)
                    for p, s in zip(prompts, sampling)]
        return self._generator.generate(requests, on_token, share_prefix)

    def new_session(self) -> "InferenceSession":
        return InferenceSession(self)


class InferenceSession:
    """One sequence on one slot; logits come back to the host as float32."""

    EAGER_TOKENS = 5  # that a session decodes before its step is captured (see ``EngineBackend.decode_logits``)

    def __init__(self, llm: LLM, slot: Optional[int] = None):
        self.llm = llm
        self.engine = llm.engine
        self.slot = self.engine.acquire_slot() if slot is None else slot
        self._decoded = 0  # tokens that this session has decoded one by one
        self._drafted = 0  # steps with drafts that it has run

    def position(self) -> int:
        return self.engine.cache.length(self.slot)

    def capacity(self) -> int:
        return self.engine.spec.max_positions

    def reset(self) -> None:
        self.engine.release_slot(self.slot)
        self.slot = self.engine.acquire_slot()

    def truncate(self, position: int) -> None:
        """Back to ``position`` tokens, as NNIS's sessions allow
        (crates/nnis-core/src/session.rs:430-445): the next ``decode_one`` follows them."""
        self.engine.truncate(self.slot, int(position))

    def snapshot(self):
        """Where the session is now, to come back to with ``restore`` after further
        tokens: the way back for a model whose layers keep state of fixed size, which
        cannot be truncated; for keys and values alone it is the same as ``truncate``."""
        return self.engine.snapshot(self.slot)

    def restore(self, snapshot) -> None:
        self.engine.restore(snapshot)

    def fork(self) -> "InferenceSession":
        """A second session that holds what this one does and goes on by itself: their pages are shared until one of
        them writes into them, states are copied."""
        return InferenceSession(self.llm, self.engine.fork(self.slot))

    def close(self) -> None:
        if self.slot is not None:
            self.engine.release_slot(self.slot)
            self.slot = None

    def prefill(self, input_ids: Sequence[int]) -> np.ndarray:
        """Resets, runs the prompt in one step, returns the last position's logits."""
        self.reset()
        ids = list(input_ids)
        if not ids:
            raise ValueError("the prompt is empty")
        logits = self.engine.step([SequenceStep(self.slot, ids, [len(ids) - 1])])
        return logits[0].cpu().numpy()

    def decode_one(self, token: int) -> np.ndarray:
        logits = self.llm.backend.decode_logits(self.slot, int(token), self._decoded >= self.EAGER_TOKENS)
        self._decoded += 1
        return logits.cpu().numpy()

    def generate(self, input_ids: Sequence[int], generation: GenerationConfig,
                 on_token: Optional[Callable[[int], Optional[StreamControl]]] = None,
                 keep_context: bool = False) -> List[int]:
        """Greedy generation on this session's own slot
        (crates/nnis-model/src/runtime.rs:796-899).  Like NNIS it starts from an empty
        session (``keep_context=True``: the prompt follows what the session holds) and
        executes every emitted token, the last one and a stop token too, so that
        afterwards ``position()`` is prompt + emitted tokens (runtime.rs:1264-1268) and
        ``decode_one`` goes on from there."""
        return self._generate(input_ids, generation, None, on_token, keep_context)

    def generate_sampled(self, input_ids: Sequence[int], generation: GenerationConfig,
                         sampling: SamplingConfig, keep_context: bool = False) -> List[int]:
        """crates/nnis-model/src/sampling.rs:216-255: seeded sampling on the host's
        policy, every emitted token executed."""
        return self._generate(input_ids, generation, sampling, None, keep_context)

    def generate_sampled_streaming(self, input_ids: Sequence[int], generation: GenerationConfig,
                                   sampling: SamplingConfig,
                                   on_token: Callable[[int], Optional[StreamControl]],
                                   keep_context: bool = False) -> List[int]:
        """crates/nnis-model/src/streaming.rs:25-72: ``on_token(token)`` is called for
        each emitted token once it has been executed; ``StreamControl.STOP`` ends the
        generation cleanly and leaves the session ready to go on."""
        return self._generate(input_ids, generation, sampling, on_token, keep_context)

    def generate_drafted(self, input_ids: Sequence[int], generation: GenerationConfig, drafter, drafts: int = 4,
                         sampling: Optional[SamplingConfig] = None,
                         on_token: Optional[Callable[[int], Optional[StreamControl]]] = None,
                         keep_context: bool = False) -> List[int]:
        """Generation with drafted tokens: ``drafter`` (``drafting.LookupDrafter``, ``drafting.SessionDrafter``) proposes up to
        ``drafts`` tokens, one step runs them all, and those stay that the model keeps.  Greedy unless ``sampling`` is
        given (a temperature and a seed; top-k and top-p are refused): tokens are distributed as ``generate_sampled``'s without
        the drafter, not the same for the same seed.  Every emitted token is executed, as in ``generate``; where a
        callback raises, the session holds no draft that it has not been shown."""
        if self.engine.cache.fixed_history():
            raise ValueError("drafted tokens that are refused are taken back: not for a model with state of fixed size or a window")
        if drafts < 1:
            raise ValueError(f"drafts must be positive; got {drafts}")
        if sampling is not None and (sampling.top_k is not None or sampling.top_p is not None):
            raise ValueError("drafted generation samples with a temperature only (no top_k, no top_p)")
        llm = getattr(drafter, "llm", None)
        there = torch.device(getattr(getattr(llm, "engine", None), "device", self.engine.device))
        if (there.index or 0) != (self.engine.device.index or 0):
            raise ValueError(f"the drafting model is on {there}, this one on {self.engine.device}")
        other = getattr(llm, "spec", None)
        if other is not None and other.vocab_size != self.engine.spec.vocab_size:
            raise ValueError(f"the drafting model has {other.vocab_size} tokens, this one {self.engine.spec.vocab_size}")
        if not keep_context:
            self.reset()
        prompt = [int(t) for t in input_ids]
        why = self.llm._generator.refusal(GenerationRequest(prompt, generation, sampling, slot=self.slot, start=self.position()))
        if why is not None:
            raise ValueError(why)
        drafter.begin()
        verifier = device_sampling.DraftVerifier(self.engine.device, self.engine.workspace, sampling)
        told, emitted, feed, proposed, logits_of = list(prompt), [], prompt, [], None
        while True:
            held = self.position()
            if proposed:
                logits = self.llm.backend.drafted_logits(self.slot, feed, self._drafted >= 2)
                self._drafted += 1
            elif len(feed) == 1 and emitted:
                logits = self.llm.backend.decode_logits(self.slot, feed[0], self._decoded >= self.EAGER_TOKENS).reshape(1, -1)
                self._decoded += 1
            else:
                logits = self.engine.step([SequenceStep(self.slot, feed, [len(feed) - 1])])
            fed, kept, shown = held + len(feed) - len(proposed), 0, 0  # the session's length without any draft
            try:
                kept, token = verifier.verify(logits, proposed, logits_of)
                new, ended = proposed[:kept] + [token], False
                for n, t in enumerate(new):
                    stop = on_token is not None and on_token(t) is StreamControl.STOP
                    emitted.append(t)
                    shown = n + 1
                    if stop or t in generation.stop_token_ids or len(emitted) >= generation.max_new_tokens:
                        new, ended = new[:n + 1], True
                        break
            except BaseException:  # (no draft stays that has not been emitted)
                self.truncate(fed + min(shown, kept))
                raise
            told += new
            # what stays of the step: what was fed before the drafts, and the drafts that were emitted
            stays = fed + min(len(new), kept)
            if stays < self.position():
                self.truncate(stays)
            if ended:
                if len(new) > kept:  # the last one came from the distribution: it is executed here
                    self.engine.step([SequenceStep(self.slot, [token], [])])
                return emitted
            room = min(drafts, generation.max_new_tokens - len(emitted) - 1)
            proposed, logits_of = drafter.propose(told, room, verifier.temperature) if room > 0 else ([], None)
            proposed = list(proposed)[:room]
            logits_of = logits_of[:len(proposed)] if proposed and logits_of is not None else None
            feed = [token, *proposed]

    def _generate(self, input_ids, generation, sampling, on_token, keep_context) -> List[int]:
        if not keep_context:
            self.reset()
        request = GenerationRequest(list(input_ids), generation, sampling, slot=self.slot,
                                    start=self.position())
        callback = None if on_token is None else (lambda _i, t: on_token(t))
        res = self.llm._generator.generate([request], callback)[0]
        if res.error is not None:
            raise ValueError(res.error)
        return res.token_ids
