"""What GraphedSamplingDecoder does with the settings that it is given, and with logits that leave nothing to draw."""
import math

import pytest
import torch
from test_sampling_decode import _model, _prompt

pytest.importorskip("transformers")


@pytest.mark.parametrize("settings", [dict(temperature=-0.1), dict(temperature=math.nan), dict(top_k=-1), dict(top_k=1.5),
                                      dict(top_k=math.inf), dict(top_p=1.01), dict(top_p=math.nan), dict(min_p=-0.1),
                                      dict(min_p=None)], ids=str)
def test_numbers_are_checked_before_anything_else(pkg, settings):
    with pytest.raises(ValueError, match=next(iter(settings))):
        pkg.GraphedSamplingDecoder(None, 1, 2, 64, **settings)


@pytest.mark.gpu
def test_settings_are_the_decoder_s_own(pkg, cuda):
    """Tensors that already have the step's shape and type are copied: writing to them later changes nothing."""
    model = _model(cuda)
    pkg.patch_model_with_fused_kernels(model, fuse_attention=True)
    given = dict(temperature=torch.full((2, 3), 0.7, device=cuda), top_k=torch.full((2, 3), 40, dtype=torch.int32, device=cuda),
                 top_p=torch.full((2, 3), 0.95, device=cuda), min_p=torch.full((2, 3), 0.01, device=cuda))
    dec = pkg.GraphedSamplingDecoder(model, 2, 3, 64, page_size=16, **given)
    ids = _prompt(cuda, 2, 20)
    u = torch.rand((2, 3, 20), generator=torch.Generator().manual_seed(7))
    want = dec.generate(ids, 20, uniform=u)
    given["temperature"].fill_(0.0)
    given["top_k"].fill_(1)
    given["top_p"].fill_(0.0)
    given["min_p"].fill_(1.0)
    assert torch.equal(dec.generate(ids, 20, uniform=u), want)


@pytest.mark.gpu
def test_limits_beyond_32_bits_are_none(pkg, cuda):
    model = _model(cuda)
    pkg.patch_model_with_fused_kernels(model, fuse_attention=True)
    ids = _prompt(cuda, 1, 20)
    u = torch.rand((1, 3, 10), generator=torch.Generator().manual_seed(9))
    out = [pkg.GraphedSamplingDecoder(model, 1, 3, 64, page_size=16, top_k=torch.tensor(k)).generate(ids, 10, uniform=u)
           for k in (0, 2 ** 32 + 1, -2 ** 32 + 1, 2 ** 31)]
    assert all(torch.equal(o, out[0]) for o in out)


@pytest.mark.gpu
@pytest.mark.parametrize("use_graph", [True, False])
def test_nothing_to_draw(pkg, cuda, use_graph):
    """Logits that are all NaN end a generation with an error, not with tokens; the next generation is as before."""
    model = _model(cuda)
    pkg.patch_model_with_fused_kernels(model, fuse_attention=True)
    dec = pkg.GraphedSamplingDecoder(model, 2, 3, 64, page_size=16, use_graph=use_graph)
    ids = _prompt(cuda, 2, 20)
    u = torch.rand((2, 3, 8), generator=torch.Generator().manual_seed(3))
    want = dec.generate(ids, 8, uniform=u)
    with torch.no_grad():
        held = model.model.norm.weight.clone()
        model.model.norm.weight.fill_(math.nan)
        for new in (1, 8):
            with pytest.raises(RuntimeError, match="draw"):
                dec.generate(ids, new, uniform=u[:, :, :new])
        model.model.norm.weight.copy_(held)
    assert torch.equal(dec.generate(ids, 8, uniform=u), want)
