"""QwenAttentionLayer over an 8-bit cache: the steps of CachedAttentionStep, and what it refuses."""
import pytest
import torch

from pluto_b200 import PlutoStatusError, _capi
from pluto_b200.layers import CachedAttentionStep, FullAttentionParameters, KeyValueCache, LayerHooks, QwenAttentionLayer

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hq,hkv,dim,rotary", [(24, 4, 256, 64), (10, 2, 128, 128), (4, 2, 36, 12)])
def test_layer_over_an_8_bit_cache(hq, hkv, dim, rotary):
    gen = torch.Generator(device="cuda").manual_seed(dim)
    rnd = lambda *s: torch.randn(*s, device="cuda", generator=gen)  # noqa: E731
    p = FullAttentionParameters(hq, hkv, dim, rotary, 5)
    q_norm, k_norm = rnd(dim) * 0.1, rnd(dim) * 0.1
    of_layer, of_steps = (KeyValueCache.Create(5, hkv, dim, dtype=torch.float8_e4m3fn) for _ in range(2))
    layer = QwenAttentionLayer.Create(p, q_norm, k_norm, 1, of_layer)
    for t in range(5):
        q, k, v = rnd(1, 2 * hq * dim).bfloat16(), rnd(1, hkv * dim).bfloat16(), rnd(1, hkv * dim).bfloat16()
        out = torch.empty(hq, dim, dtype=torch.bfloat16, device="cuda")
        CachedAttentionStep(p, of_steps, q.view(hq, 2, dim), k.view(hkv, dim), v.view(hkv, dim), q_norm, k_norm, out)
        if t == 3:   # probabilities are of the other storage types; nothing has moved then
            with pytest.raises(PlutoStatusError, match="8-bit"):
                layer.fwd([q, k, v], LayerHooks(attention_probabilities_hook=lambda *a: None))
            assert of_layer.position() == t
        result = layer.fwd([q, k, v])
        assert torch.equal(result.outputs[0].view(hq, dim), out) and of_layer.position() == t + 1
        with pytest.raises(PlutoStatusError, match="inference only"):
            layer.bwd([result.outputs[0]], result.state)
    with pytest.raises(PlutoStatusError, match="capacity"):
        layer.fwd([q, k, v])
    for name, rows in of_layer.pool().items():
        assert torch.equal(rows.view(torch.uint8), of_steps.pool()[name].view(torch.uint8))
    assert _capi.kernel_status() == 0
