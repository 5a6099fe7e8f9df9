"""What importing the package leaves as it found it."""
import subprocess
import sys

CODE = """
import torch
from torch.overrides import is_tensor_like

def state():
    classes = (torch.ScriptObject, torch._C.ScriptModule, torch.ScriptModule, torch.Tensor, torch.nn.Module)
    names = [sorted(vars(c)) for c in classes]
    traced = torch.jit.trace(torch.nn.Linear(2, 2), torch.ones(1, 2))
    packed = torch.ops.prepacked.linear_clamp_prepack(torch.ones(2, 2), None)      # a script object of another library
    return names, [is_tensor_like(x) for x in (traced, traced._c, packed, torch.ones(1))]

before = state()
import gaudirt_b200
assert state() == before, (before, state())
assert before[1] == [False, False, False, True]
"""


def test_torch_classes_are_left_alone():
    run = subprocess.run([sys.executable, "-W", "ignore", "-c", CODE], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stderr
