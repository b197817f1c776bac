"""CPU: the rule that cuts a step of attention over ordinary heads into pieces refuses what is no step, where it once went on for ever."""
import subprocess
import sys

import pytest

from omni_npu_amd import _host
from omni_npu_amd import kernels as K
from tests.conftest import ROOT

GOOD = (2, 1, 8, 2, 128, 2, 100)


@pytest.mark.parametrize("side", ["K.gqa_plan", "H.load().gqa_plan"])
def test_heads_of_no_values(side):
    """In a process of its own, which can be ended."""
    code = f"from omni_npu_amd import kernels as K, _host as H\ntry:\n    {side}(1, 1, 8, 2, 0, 2, 100)\nexcept ValueError:\n    print('refused')"
    done = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=120)
    assert done.stdout.strip() == "refused", done.stderr


@pytest.mark.parametrize("at,bad", [(0, 0), (1, 0), (2, 0), (2, 1), (3, 0), (4, -1), (5, 0), (0, -3), (1, -1), (3, -2)])
def test_what_is_no_step(at, bad):
    args = GOOD[:at] + (bad,) + GOOD[at + 1:]
    for plan in (K.gqa_plan, _host.load().gqa_plan):
        assert tuple(plan(*GOOD)) == K.gqa_plan(*GOOD)
        with pytest.raises(ValueError, match="gqa_plan"):
            plan(*args)


@pytest.mark.parametrize("dim", [1, 2, 15, 64, 256])
@pytest.mark.parametrize("longest", [0, 1, 5000])
def test_both_sides_agree_on_narrow_heads(dim, longest):
    assert K.gqa_plan(3, 2, 64, 64, dim, 1, longest) == tuple(_host.load().gqa_plan(3, 2, 64, 64, dim, 1, longest))


@pytest.mark.gpu
def test_a_call_over_heads_of_no_values_is_refused(dev):
    import torch
    z = lambda *s: torch.zeros(*s, dtype=torch.bfloat16, device=dev)
    with pytest.raises(ValueError, match="heads of 0 values"):
        K.gqa_decode(z(2, 8, 0), z(4, 16, 2, 0), z(4, 16, 2, 0), torch.zeros(2, 3, dtype=torch.int32, device=dev),
                     torch.ones(2, dtype=torch.int32, device=dev), 1.0, z(2, 8, 0))
