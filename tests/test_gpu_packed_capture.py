"""Recording the packed decoder's step: on the decoder's own device, from any current stream, and more than one of them."""

import pytest
import torch

from dual_mod_public_b200 import DualModConfig
from dual_mod_public_b200.eval.packed_decode import PackedDecoder
from dual_mod_public_b200.models import DualModLM

pytestmark = pytest.mark.gpu
PROMPTS = [[5, 6, 7, 8], [9], list(range(3, 70))]


def decoder(rows=4, dev="cuda:0"):
    torch.manual_seed(0)
    m = DualModLM(DualModConfig(d_model=128, n_layers=2, n_heads=2, mlp_hidden_override=128, vocab_size=259, max_seq_len=128,
                                attn_mode="vanilla")).to(dev)
    return PackedDecoder(m, rows, 128)


def test_the_recording_stream_is_of_the_decoders_device(monkeypatch):
    seen, inner = [], torch.cuda.graph.__init__

    def init(self, graph, *a, stream=None, **k):
        seen.append((stream, torch.cuda.current_device()))
        inner(self, graph, *a, stream=stream, **k)
    monkeypatch.setattr(torch.cuda.graph, "__init__", init)
    dev = f"cuda:{torch.cuda.device_count() - 1}"                  # another than the current one, where there are several
    dec = decoder(dev=dev)
    want = dec.generate(PROMPTS, 8)
    assert dec.capture().generate(PROMPTS, 8) == want
    (stream, current), = seen
    assert stream is not None and stream.device == dec.dev and current == dec.dev.index


def test_two_recorded_decoders_in_turn_and_a_current_stream_of_their_own():
    want = decoder().generate(PROMPTS, 8)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        a, b = decoder().capture(), decoder(rows=6).capture()
        for dec in (a, b, a, b):
            assert dec.generate(PROMPTS, 8)[0] == want[0]
