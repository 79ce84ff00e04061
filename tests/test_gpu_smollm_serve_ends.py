"""SmolBatchDecoder when a prompt does not get to its end: pages and places stay as they were, and the others' tokens what they are."""
import pytest
import torch

from conftest import announce
from test_gpu_smollm_serve import make
from torch_npu_smollm_serve import SmolBatchDecoder

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('end', [RuntimeError, KeyboardInterrupt, torch.OutOfMemoryError])
def test_a_prompt_that_is_broken_off(device, end, monkeypatch):
    announce('smollm serve broken off', end.__name__)
    stack, io, _, g = make(device, 'w8a16', capacity=32)
    ids = [torch.randint(0, 1000, (n,), generator=g).tolist() for n in (20, 9)]
    runs = []
    for broken in (False, True):
        decoder = SmolBatchDecoder(stack, io, batch=2, slots=32, page=16, pages=4, graph=False)
        decoder.admit(ids[0], steps=6)
        decoder.step()
        if broken:
            free, held, state = list(decoder._free), list(decoder._held), [t.clone() for t in (decoder.table, decoder.position, decoder.tokens)]

            def broken_off(*_):
                raise end()

            with monkeypatch.context() as m:
                m.setattr(decoder, '_prompt', broken_off)
                with pytest.raises(end):
                    decoder.admit(ids[1], steps=6)
            assert decoder._free == free and decoder._held == held
            assert all(torch.equal(a, b) for a, b in zip(state, (decoder.table, decoder.position, decoder.tokens)))
        place = decoder.admit(ids[1], steps=6)
        for _ in range(5):
            decoder.step()
        runs.append((decoder.tokens.tolist(), decoder.logits.clone(), place))
    assert runs[0][0] == runs[1][0] and torch.equal(runs[0][1], runs[1][1]) and runs[0][2] == runs[1][2]
