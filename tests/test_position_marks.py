"""The mark of consecutive positions, by which attention with a relative position bias leaves the values unread, where no gradient is recorded."""
import pytest
import torch

from savanna_b200.models.rope import are_consecutive, consecutive_positions, mark_consecutive


@pytest.mark.parametrize("mode", [torch.inference_mode, torch.no_grad, torch.enable_grad])
def test_a_write_ends_the_mark(mode):
    with mode():
        p, q = consecutive_positions(5), consecutive_positions(5)
        assert are_consecutive(p) and torch.equal(p, torch.arange(5))
        p[0] = 7
        q.add_(2)
        assert not are_consecutive(p) and not are_consecutive(q)
    assert not are_consecutive(p)


def test_a_write_after_inference_mode_ends_the_mark():
    with torch.inference_mode():
        p = consecutive_positions(5)
    assert are_consecutive(p)
    p[0] = 7
    assert not are_consecutive(p)


def test_tensors_of_inference_mode_have_no_mark():
    with torch.inference_mode():
        p = mark_consecutive(torch.arange(4))
        assert not are_consecutive(p)
    assert not are_consecutive(p)
