"""FlatMuon's Newton-Schulz sequence is checked where the optimizer is made, on any device."""
import pytest

from distributed_tensorflow_amd.optim import FlatMuon
from distributed_tensorflow_amd.runtime.arena import ParamArena, ParamSpec


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_flat_muon_refuses_sequences_of_another_length(device):
    a = ParamArena([ParamSpec("w", (6, 4), "ones")], device, FlatMuon.slots)
    one = (1.5, -0.5, 0.0)
    for kw in (dict(ns_steps=0), dict(ns_steps=17), dict(ns_steps=3, ns_coeffs=(one, one)), dict(ns_coeffs=(1.5, -0.5)), dict(ns_steps=1, ns_coeffs=((1.5, -0.5),)),
               dict(ns_coeffs=(float("nan"), 0.0, 0.0)), dict(ns_coeffs=(9.0, 0.0, 0.0))):
        with pytest.raises(ValueError, match="steps|coeffs|coefficients"):
            FlatMuon(a, **kw)
    FlatMuon(a, ns_steps=2, ns_coeffs=(one, one)).step(0.1)
