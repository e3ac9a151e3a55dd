"""Attention and the policy loss through the host layer, on the CPU oracle."""
import pytest

import language_programs as programs
from maidenx_amd.tensor import MxError


@pytest.mark.parametrize("name", ["gradients", "seeds", "layouts", "gradient_layouts", "bf16_model", "nothing"])
def test_programs(mx_oracle, name):
    getattr(programs, "check_" + name)(mx_oracle)


@pytest.mark.parametrize("i", range(31))
def test_refusals(mx_oracle, i):
    call, kind = programs.refusals(mx_oracle)[i]
    with pytest.raises(MxError) as e:
        call()
    assert e.value.kind == kind


def test_every_refusal_is_run(mx_oracle):
    assert len(programs.refusals(mx_oracle)) == 31


def test_a_step_lowers_what_it_descends(mx_oracle):
    """Parameters move along the gradient: SGD's update is the parameter less 0.05 times the gradient of an untouched copy."""
    import numpy as np
    case = programs.Case()
    a, b = programs.Model(mx_oracle, case), programs.Model(mx_oracle, case)
    b.loss().backward()
    g = b.gradients()
    a.step()
    for n, p in a.parameters().items():
        np.testing.assert_allclose(p.numpy(), case.p[n] - np.float32(0.05) * g[n], rtol=2.0 ** -23, atol=2.0 ** -23 * np.abs(g[n]).max(), err_msg=n)
