"""zmoe.ops and zmoe.ep without the compiled module zmoe._ops, as with libzmoe.so
alone built."""
import os
import subprocess
import sys

PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "zipmoe-icml26_b200")


def test_import_without_the_compiled_module():
    code = """
import sys
sys.path.insert(0, %r)
sys.modules["zmoe._ops"] = None                         # the import system raises for it
import torch
import zmoe.ep
from zmoe import ops
for call in (lambda: ops.lora_plan(torch.zeros(3, dtype=torch.int32), 2), lambda: ops.permute_grad(None, None),
             lambda: ops.combine_grad(None, None, None, None, 0), lambda: ops.lora(*[None] * 6),
             lambda: ops.lora_grad(*[None] * 7)):
    try:
        call()
    except ImportError as e:
        assert "zmoe._ops is not built" in str(e)
    else:
        raise AssertionError("no error")
try:
    ops.permute(torch.zeros(3, 2, dtype=torch.int32), None, 4)
except ValueError as e:
    assert "topk_idx" in str(e)
print("ok")
""" % PKG
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stderr[-2000:]
