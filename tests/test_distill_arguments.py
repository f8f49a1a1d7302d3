"""Distillation refuses temperatures whose square is not an ordinary number before it touches the device."""
import pytest

from test_operator_arguments import ANY, distill_args, hip, refused


@pytest.mark.parametrize("temperature", [1e-19, 1e-20, 1e-30, 1e-38])
def test_temperatures_whose_square_vanishes(temperature):
    refused(hip.bh_distill_forward(*distill_args(temperature=temperature), None, None, ANY), "temperature")
    refused(hip.bh_distill_loss_grad(*distill_args(temperature=temperature), None, None, ANY, 1 << 40), "temperature")
    refused(hip.bh_distill_backward(*distill_args(temperature=temperature), ANY, None, ANY, 1 << 40), "temperature")
