"""Steps are captured while the collector has old graphs to free."""
import gc

import pytest
import torch

from helpers import make_model
from test_shared_sequences_gpu import SHARED, tokens

pytestmark = pytest.mark.gpu


class Cycle:
    """A graph that only the collector frees."""

    def __init__(self):
        self.graph, self.itself = torch.cuda.CUDAGraph(), self
        x = torch.zeros(8, device="cuda")
        with torch.cuda.graph(self.graph):
            x.add_(1.0)


def test_graphs_in_cycles_are_freed_after_a_capture(tmp_path):
    """A prompt step and decode steps captured with the collector at its keenest and such graphs left to it."""
    from nnis_b200 import LLM, GenerationConfig
    from nnis_b200.engine import SequenceStep
    llm = LLM(make_model(str(tmp_path), SHARED, 3), dtype="float32", max_tokens=1 << 13, max_batch=4)
    prompt, threshold = tokens(1, 300), gc.get_threshold()
    want = llm.generate([prompt], max_new_tokens=8, stop_token_ids=[])[0].token_ids
    try:
        for turn in range(3):
            gc.disable()
            for _ in range(4):
                Cycle()
            gc.set_threshold(1, 1, 1)
            gc.enable()
            llm.backend._decoders.clear()
            llm.engine._step_graphs.clear()
            got = llm.generate([prompt], max_new_tokens=8, stop_token_ids=[])[0]
            assert got.error is None and got.token_ids == want and gc.isenabled()
            s = llm.new_session()
            for _ in range(3):  # (the second time a prompt's shape is seen it is captured, then replayed)
                s.prefill(prompt)
            assert s.generate(prompt, GenerationConfig(8)) == want
            s.close()
    finally:
        gc.set_threshold(*threshold)
        gc.enable()
    gc.collect()
