"""The 64-bit forms that the GPU tests of the row operations over the vocabulary go by: gradients against differences, distributions
against their definitions; and what the host side refuses before anything reaches a device."""
import numpy as np
import pytest

import rust_trainer_b200 as rt
import vocab_reference as R
from rust_trainer_b200 import ops


@pytest.mark.parametrize("mode", ["renorm", "tail"])
@pytest.mark.parametrize("temperature", [1.0, 0.7, 2.0])
def test_distillation_gradient_is_the_losses_difference_quotient(mode, temperature):
    rng = np.random.default_rng(5)
    z = rng.standard_normal(23) * 2
    index = np.array([4, 9, 4, -1, 20, 0])  # one index twice, one empty place
    t = np.log(np.array([0.2, 0.1, 0.15, 0.3, 0.05, 0.08]))
    loss, grad, _ = R.distill(z, index, t, temperature, mode, 1.5)
    h = 1e-5
    for v in range(z.size):
        up, down = z.copy(), z.copy()
        up[v] += h
        down[v] -= h
        diff = (R.distill(up, index, t, temperature, mode, 1.5)[0] - R.distill(down, index, t, temperature, mode, 1.5)[0]) / (2 * h)
        # central differences: h^2 times a third derivative below 10 / T^3, and the losses' rounding over h
        assert abs(diff - 1.5 / temperature * grad[v]) < 1e-8
    assert np.isfinite(loss)


def test_a_student_that_has_the_teachers_probabilities_has_no_loss_and_no_gradient():
    rng = np.random.default_rng(6)
    z = rng.standard_normal(40)
    index, t, _ = R.top(z, 7, 1.3)
    loss, grad, _ = R.distill(z, index, t, 1.3, "tail")
    assert abs(loss) < 1e-14 and np.abs(grad).max() < 1e-14
    full, tf, _ = R.top(z, 40, 1.3)
    loss, grad, _ = R.distill(z, full, tf, 1.3, "renorm")
    assert abs(loss) < 1e-14 and np.abs(grad).max() < 1e-14


def test_verified_tokens_are_distributed_as_the_target_says():
    """Over an even grid of random numbers, accepted or redrawn, the first token has the target's distribution whatever drafted it."""
    p, q = np.array([[0.5, 0.2, 0.3, 0.0], [0.1, 0.2, 0.3, 0.4]]), np.array([[0.1, 0.6, 0.1, 0.2]])
    n = 100
    got = np.zeros(4)
    for d in range(4):
        for ua in (np.arange(n) + 0.5) / n:
            for us in (np.arange(n) + 0.5) / n:
                k, token = R.verify(p, q, [d], [ua], us)
                got[d if k else token] += q[0][d] / n**2
    assert np.abs(got - p[0]).max() < 2.0 / n  # a grid of n points resolves a probability to 1 / n, twice


def test_rows_without_anything():
    assert R.verify([[0.0, 0.0]], None, [], [], 0.3) == (0, -1)
    assert R.verify([[0.5, 0.5], [1.0, 0.0]], [[0.5, 0.5]], [1], [1.0], 0.7) == (0, 1)  # nothing left of p - q: p itself
    assert R.top([-np.inf] * 3, 2, 1.0)[0].tolist() == [0, 1]


class _NoDevice:
    """In a context's place: these refusals come before the library is called."""

    _h = None

    def check(self, st):
        raise AssertionError("reached the library")


def test_the_host_side_refuses_what_does_not_fit():
    c, z, i = _NoDevice(), np.zeros((2, 5), np.float32), np.zeros((2, 3), np.int32)
    for call in (lambda: ops.distill(c, z, i, np.zeros((2, 4), np.float32)), lambda: ops.distill(c, z, i[:1], np.zeros((1, 3), np.float32)),
                 lambda: ops.distill(c, z, i, np.zeros((2, 3), np.float32), weight=np.ones(3, np.float32)),
                 lambda: ops.distill(c, z, i, np.zeros((2, 3), np.float32), mode="forward"), lambda: ops.top_logits(c, z[0], 1),
                 lambda: ops.softmax(c, z[0]), lambda: ops.verify_draft(c, z, None, [1], [0, 1], [0.5], [0.5, 0.5]),
                 lambda: ops.verify_draft(c, z, None, [1], [0, 2], [0.5], [0.5]), lambda: ops.verify_draft(c, z, z, [1], [0, 1], [0.5], [0.5])):
        with pytest.raises(rt.RtError):
            call()


def test_every_entry_point_refuses_a_missing_context():
    L = rt.lib()
    assert L.rt_top_logits_dev(None, 16, 0, 1, 4, 4, 1.0, 1, 16, 16, None) == 7
    assert L.rt_distill_dev(None, 16, 0, 1, 4, 4, 1.0, 16, 16, 1, 0, None, 16, None, 0, 0, None) == 7
    assert L.rt_softmax_dev(None, 16, 0, 1, 4, 4, 1.0, 16, 0, 4) == 7
    assert L.rt_verify_draft_dev(None, 16, 4, None, 0, 0, 4, 16, 16, 1, 1, 16, 16, 16, 16) == 7
