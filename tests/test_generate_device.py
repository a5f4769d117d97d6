"""Generation by a model that is not on the current device: its streams, its captures."""
import contextlib

import pytest
import torch

from hyperattention_b200 import llm
from hyperattention_b200.llm import ChatGLM2ShapedDecoder, DecoderCache, chatglm2_config


class Counting(ChatGLM2ShapedDecoder):
    """Token t is followed by t + 1, whatever the cache holds."""

    def forward(self, input_ids, cache=None, counts=None):
        cache.length += input_ids.shape[1]
        return self._run(input_ids, None)

    def _run(self, input_ids, step):
        return torch.nn.functional.one_hot(input_ids + 1, 50).float()


def test_everything_runs_on_the_models_device(monkeypatch):
    """a machine of two devices, of which the other one is current: what is entered, and by which device's streams (the calls are recorded, nothing is launched)"""
    now, seen = ['other'], []

    @contextlib.contextmanager
    def device_of(t):
        assert t is model.transformer.output_layer.weight
        now.append('model')
        yield
        now.pop()

    class Stream:
        def __init__(self, device=None):
            self.device = now[-1] if device is None else device

        def synchronize(self):
            seen.append(('synchronize', self.device))

    class Graph:
        def replay(self):
            seen.append(('replay', now[-1]))
            ids.add_(1)

    first = Stream()                                         # of torch's own captures: the device of the first of them

    @contextlib.contextmanager
    def graph(g, pool=None, stream=None, **kw):
        nonlocal ids
        seen.append(('capture', (stream or first).device))
        copy = torch.Tensor.copy_
        with monkeypatch.context() as m:                     # a captured copy copies nothing
            def note(self, *a, **k):
                nonlocal ids
                ids = self
                return self
            m.setattr(torch.Tensor, 'copy_', note)
            yield
        assert torch.Tensor.copy_ is copy

    cfg = chatglm2_config(num_layers=2, hidden_size=64, num_attention_heads=2, kv_channels=64, ffn_hidden_size=64, padded_vocab_size=50)
    model, ids = Counting(cfg, dtype=torch.bfloat16), None
    monkeypatch.setattr(llm, '_CAPTURE_STREAMS', {}, raising=False)
    monkeypatch.setattr(llm, 'check_device_status', lambda d: seen.append(('check', now[-1])))
    for name, fake in dict(device_of=device_of, Stream=Stream, CUDAGraph=Graph, graph=graph, current_stream=lambda d=None: Stream(),
                           is_current_stream_capturing=lambda: False).items():
        monkeypatch.setattr(torch.cuda, name, fake)
    out = model.generate(torch.tensor([[3, 4], [8, 9]]), 6, cache=DecoderCache(cfg, 2, 16, device='cpu'))
    assert out.tolist() == [[5, 6, 7, 8, 9, 10], [10, 11, 12, 13, 14, 15]]
    assert [s[0] for s in seen] == ['synchronize', 'capture'] + 4 * ['replay'] + ['check']
    assert {s[1] for s in seen} == {'model'} and now == ['other']


@pytest.mark.gpu
@pytest.mark.skipif(torch.cuda.device_count() < 2, reason='needs two GPUs')
def test_on_the_second_device():
    cfg = chatglm2_config(num_layers=2, hidden_size=256, num_attention_heads=4, ffn_hidden_size=512, padded_vocab_size=1000)
    ids = torch.randint(0, 1000, (2, 20), generator=torch.Generator().manual_seed(0))
    outs = []
    for d in (0, 1):
        m = ChatGLM2ShapedDecoder(cfg, device='cpu', dtype=torch.bfloat16).to(f'cuda:{d}')
        outs.append(m.generate(ids.to(f'cuda:{d}'), 10).cpu())
    assert torch.equal(*outs)
