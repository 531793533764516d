"""Rows that more warps would share than a launch of gradients has."""
import pytest
import torch
from test_rotary_cpu import check, values

from powersgd_b200.ops import host, rotary
from powersgd_b200.ops.rotary import rotate_heads

pytestmark = pytest.mark.gpu


@pytest.fixture(params=["extension", "python"])
def form(request, monkeypatch):
    if request.param == "python":
        monkeypatch.setattr(rotary, "operators", None)
    else:
        assert host.operators is not None
    return request.param


@pytest.mark.parametrize("heads, keys, values_, size", [(3000, 1096, 0, 256), (1096, 3000, 0, 256), (2400, 1184, 8, 136), (2369, 1, 0, 256), (2050, 2040, 6, 200)])
@pytest.mark.parametrize("rows", [1, 2])
def test_queries_and_keys_share_the_warps_of_a_launch(form, rows, heads, keys, values_, size):
    """Each kind alone may take half of the warps and more; both together have to find room."""
    torch.empty(rows, heads + keys + values_, size, device="cuda").fill_(float("nan"))     # (what an output that is not written may hold)
    check(values(rows, heads + keys + values_, size, torch.float32, "cuda"), heads, keys, lengths=[rows])
