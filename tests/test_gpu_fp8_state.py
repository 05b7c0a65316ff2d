"""GPU checks of the 8-bit decoder's state: it loads a bf16 decoder's weights."""
import pytest
import torch

from src.decoder import Decoder, DecoderConfig
from src.gpu_cache import GPUCache

pytestmark = pytest.mark.gpu

SMALL = DecoderConfig(layers=2, hidden=192, q_heads=3, kv_heads=1, intermediate=336, vocab=500, init_std=0.1)


def _logits(model):
    cache = GPUCache(None, layers=SMALL.layers, heads=SMALL.kv_heads, max_tokens=64)
    return model(cache, ids=torch.arange(9, device='cuda')[None], logits=9)


@pytest.mark.parametrize('make', [lambda s: s, lambda s: {k: v.cpu() for k, v in s.items()},
                                  lambda s: {k: v.float() for k, v in s.items()}])
def test_a_bf16_state_is_quantised_as_its_own_weights_are(cuda, make):
    state = make(Decoder(SMALL, seed=1).state_dict())
    before = dict(state)
    model = Decoder(SMALL, seed=0, projections='fp8')
    model.load_state_dict(state)
    expected = Decoder(SMALL, seed=1, projections='fp8')
    assert set(state) == set(before) and all(state[k] is before[k] for k in before)  # the caller's is left alone
    mine, other = model.state_dict(), expected.state_dict()
    assert list(mine) == list(other)
    assert all(mine[k].dtype == other[k].dtype and torch.equal(mine[k].float(), other[k].float()) for k in mine)
    assert torch.equal(_logits(model), _logits(expected))


def test_a_state_under_a_prefix_and_one_that_does_not_fit(cuda):
    class Holder(torch.nn.Module):
        def __init__(self, **kw):
            super().__init__()
            self.decoder = Decoder(SMALL, **kw)

    holder = Holder(seed=0, projections='fp8')
    holder.load_state_dict(Holder(seed=1).state_dict())
    assert torch.equal(_logits(holder.decoder), _logits(Decoder(SMALL, seed=1, projections='fp8')))
    model = Decoder(SMALL, projections='fp8')
    before = _logits(model)
    state = Decoder(SMALL, seed=1).state_dict()
    state['gate_up.1'] = state['gate_up.1'][:-1]
    with pytest.raises(RuntimeError, match='gate_up.1'):
        model.load_state_dict(state)
    state = Decoder(SMALL, seed=0).state_dict()
    del state['down.0']
    with pytest.raises(RuntimeError, match='down.0'):
        model.load_state_dict(state)
    state['down.0'] = Decoder(SMALL, seed=0).state_dict()['down.0']
    model.load_state_dict(state)
    assert torch.equal(_logits(model), before)


def test_moves_and_casts_leave_codes_and_scales_as_they_are(cuda):
    """model.to(torch.bfloat16), model.float() and the like are for the other weights."""
    model = Decoder(SMALL, projections='fp8')
    before, held = _logits(model), {k: v.clone() for k, v in model.state_dict().items()}
    for cast in (lambda: model.to(torch.bfloat16), lambda: model.bfloat16(), lambda: model.to('cuda', torch.bfloat16),
                 lambda: model.cpu().cuda(), lambda: model.to(torch.float32).to(torch.bfloat16)):
        cast()
        now = model.state_dict()
        assert all(now[k].dtype == held[k].dtype and now[k].device == held[k].device for k in held)
        assert all(torch.equal(now[k].float(), held[k].float()) for k in held)
        assert torch.equal(_logits(model), before)
