"""The calls that the GPU tests make reach every kernel of the experts' block that is compiled."""
import os
import re
import subprocess

import expert_forms as F
from launch_recorder import recorded  # noqa: F401

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LIBRARY = os.path.join(ROOT, "nvshmem_amd", "lib", "libnvshmem_amd.so")

CODE = """
sys.path.insert(0, os.path.join(%(root)r, "tests"))
import expert_forms as F
from nvshmem_amd import Runtime
rt = Runtime(npes=F.NPES, symmetric_size=4 << 30)
p = [rt.malloc(300 << 20) for _ in range(10)]
launches()
for kind in F.KINDS:
    for _, rows, dim, hidden in F.CALLS:
        size = (rows * F.MINE, F.MINE * F.NPES, dim, hidden)
        rt.moe_experts(kind, *p[:6], *size, pre=p[6])
        rt.moe_experts_grad(kind, *p, *size)
    for _, rows, dim, hidden, group in F.FOUR_BIT_CALLS:
        rt.moe_experts_w4(kind, *p[:8], rows * F.FOUR_BIT_MINE, F.FOUR_BIT_MINE * F.NPES, dim, hidden, group)
print("\\n".join("kernel " + l[0] for l in launches()))
"""


def test_every_kernel_is_launched(recorded):  # noqa: F811
    symbols = subprocess.run(["nm", LIBRARY], check=True, stdout=subprocess.PIPE, text=True).stdout
    compiled = set(re.findall(r"\s(_ZN\S*\d+expert_(?:tile|few)\w*_kernel\S+)", symbols))
    assert len(compiled) > 100
    launched = set(re.findall(r"^kernel (\S+)", recorded(CODE % {"root": ROOT}), re.M))
    assert not compiled - launched, sorted(compiled - launched)
