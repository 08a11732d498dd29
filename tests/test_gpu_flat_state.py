"""engine.FlatState.load_state_dict: moments of another floating type are converted, 8-bit codes are not."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def make(optimizer):
    from discrete_dppm_graphs_amd import engine
    from discrete_dppm_graphs_amd.model.ppgn import Powerful
    torch.manual_seed(3)
    model = Powerful(num_layers=2, hidden=16, hidden_final=16, normalization="instance", adj_out=True, cat_output=True).cuda()
    return engine.FlatState(model, optimizer=optimizer)


@pytest.mark.parametrize("optimizer", ["adam", "adamw"])
@pytest.mark.parametrize("dtype", [torch.float64, torch.bfloat16])
def test_moments_of_another_type_are_converted(optimizer, dtype):
    state = make(optimizer)
    saved = state.state_dict()
    moments = {k: torch.rand(saved[k].shape, device="cuda").to(dtype) for k in ("exp_avg", "exp_avg_sq")}
    state.load_state_dict({**saved, **moments, "step": 7})
    held = state.state_dict()
    assert held["step"] == 7 and all(held[k].dtype == torch.float32 and torch.equal(held[k], v.float()) for k, v in moments.items())


def test_codes_are_not_converted():
    state = make("adamw8")
    saved = state.state_dict()
    for k in ("exp_avg", "exp_avg_root"):
        with pytest.raises(ValueError, match="moment size"):
            state.load_state_dict({**saved, k: saved[k].float()})
    state.load_state_dict(saved)
    state = make("adamw")
    saved = state.state_dict()
    with pytest.raises(ValueError, match="moment size"):
        state.load_state_dict({**saved, "exp_avg": saved["exp_avg"].to(torch.float8_e4m3fn)})
