"""GPU: convert_to_int8 refuses before it replaces anything."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def communicating():
    from tcfp_b200.nn import LayerHooks, TCFPLinear

    lin = TCFPLinear(64, 64, use_tensor_cores=True).to(DEV)
    lin._hooks = LayerHooks(out_hook=lambda y: None)
    return lin


@pytest.mark.parametrize("make,error,text", [
    (communicating, ValueError, "ranks"),
    (lambda: torch.nn.Linear(64, 64), RuntimeError, "CUDA"),
    (lambda: torch.nn.Linear(64, 64, device="meta"), RuntimeError, "CUDA"),
    (lambda: torch.nn.Linear(64, 64, device=DEV, dtype=torch.float16), ValueError, "out_dtype"),
    (lambda: torch.nn.Linear(64, 64, device=DEV, dtype=torch.float64), ValueError, "out_dtype"),
    (lambda: torch.nn.Linear(131072, 1, device=DEV), ValueError, "131071"),
])
def test_a_refused_layer_leaves_the_model_as_it_was(make, error, text):
    from tcfp_b200.nn import Int8Linear, convert_to_int8

    inner = torch.nn.Sequential(torch.nn.Linear(64, 64, device=DEV))
    model = torch.nn.Sequential(torch.nn.Linear(64, 64, device=DEV), inner, make())
    before = list(model.modules())
    with pytest.raises(error, match=text):
        convert_to_int8(model)
    after = list(model.modules())
    assert len(after) == len(before) and all(a is b for a, b in zip(after, before))
    model[2] = torch.nn.Linear(64, 48, device=DEV)
    convert_to_int8(model)
    assert sum(isinstance(m, Int8Linear) for m in model.modules()) == 3
    assert model(torch.randn(5, 64, device=DEV)).shape == (5, 48)
