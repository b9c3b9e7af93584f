"""What is built, for which interpreter, and what does not need what."""
import re
from pathlib import Path

import torch

import ghost_flow_b200


def test_the_declared_pytorch_has_the_interface_that_operators_go_through():
    need = re.search(r'"torch>=([\d.]+)"', (Path(ghost_flow_b200.__file__).parents[1] / "pyproject.toml").read_text()).group(1)
    assert (2, 11) <= tuple(map(int, need.split("."))) <= tuple(map(int, torch.__version__.split(".")[:2]))
    assert hasattr(torch.Tensor, "__dlpack_c_exchange_api__")
