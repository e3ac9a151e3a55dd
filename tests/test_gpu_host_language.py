"""Attention and the policy loss through the host layer on the HIP backend."""
import numpy as np
import pytest

import language_programs as programs
from maidenx_amd.tensor import MxError

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("i", range(31))
def test_refusals(mx_hip, i):
    call, kind = programs.refusals(mx_hip)[i]
    with pytest.raises(MxError) as e:
        call()
    assert e.value.kind == kind


@pytest.mark.parametrize("name", ["gradients", "seeds", "layouts", "gradient_layouts", "bf16_model", "nothing"])
def test_programs(mx_hip, name):
    getattr(programs, "check_" + name)(mx_hip)


def test_a_target_out_of_range_is_reported(mx_hip):
    mx = mx_hip
    one = mx.ones((3,))
    with pytest.raises(MxError) as e:
        mx.policy_loss(mx.zeros((3, 5)), mx.indices([0, 5, 1]), mx.zeros((3,)), one, one)
    assert e.value.kind == "Backend" and "out of bounds" in str(e.value)
    assert np.isfinite(mx.policy_loss(mx.zeros((3, 5)), mx.indices([0, 4, 1]), mx.zeros((3,)), one, one).item())


def train(mx, case, steps, graphs, adam=False):
    m = programs.Model(mx, case)
    adams = [mx.Adam(lr=0.01) for _ in m.modules] if adam else None
    mx.set_graph_replay(graphs)
    try:
        mx.run_steps(lambda: m.step(adams), steps)
    finally:
        mx.set_graph_replay(True)
    out = {n: p.numpy() for n, p in m.parameters().items()}
    assert all(np.isfinite(a).all() for a in out.values()) and not np.array_equal(out["wq"], case.p["wq"])
    return out, mx.last_train_replayed()


def test_recorded_steps_are_the_eager_ones(mx_hip):
    """Training steps of the whole model replayed from a recording leave the bits that the same steps leave eagerly."""
    case = programs.Case()
    eager, none = train(mx_hip, case, 64, False)
    recorded, some = train(mx_hip, case, 64, True)
    assert none == 0 and some > 0
    for n in eager:
        np.testing.assert_array_equal(eager[n], recorded[n], err_msg=n)


def test_adam_steps_repeat(mx_hip):
    """(Adam's step number is in its scalars: those steps are not recorded.)"""
    case = programs.Case()
    a, b = (train(mx_hip, case, 12, False, adam=True)[0] for _ in range(2))
    for n in a:
        np.testing.assert_array_equal(a[n], b[n], err_msg=n)
