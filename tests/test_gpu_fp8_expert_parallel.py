"""GPU: 8-bit experts in the expert-parallel layer. One rank, whose exchanges go to itself: the same rows, sums in the
same order, so it is bit-equal to the single-GPU layer. A process group of its own process, so that no other test
finds one."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

CODE = """
import os, sys
import torch, torch.distributed as dist
from datetime import timedelta
from tilelang_b200 import moe, ops
torch.cuda.set_device(0)
dist.init_process_group("nccl", init_method="file://" + sys.argv[1], rank=0, world_size=1, timeout=timedelta(seconds=60),
                        device_id=torch.device("cuda", 0))
g = torch.Generator(device="cuda")
g.manual_seed(1)
randn = lambda *shape: torch.randn(*shape, device="cuda", generator=g)
for T, E, k, H, F, kind in ((1, 4, 2, 128, 128, torch.bfloat16), (70, 6, 3, 200, 80, torch.float16),
                            (900, 8, 2, 256, 256, torch.bfloat16), (0, 4, 2, 200, 80, torch.bfloat16)):
    mlp = moe.Fp8ExpertMLP(ops.quant_fp8_weight(randn(E, 2 * F, H) * H ** -0.5), ops.quant_fp8_weight(randn(E, H, F) * F ** -0.5))
    x, logits, d = randn(T, H).to(kind), randn(T, E).requires_grad_(), randn(T, H).to(kind)
    one = moe.moe_forward(x, logits, k, E, mlp)
    ep = moe.moe_forward_ep(x, logits, k, E, mlp)
    assert ep.shape == (T, H) and ep.dtype == kind and torch.equal(one, ep), (T, "values")
    d_one, = torch.autograd.grad(one, logits, d)
    d_ep, = torch.autograd.grad(ep, logits, d)
    assert torch.equal(d_one, d_ep), (T, "gradient of the router")
    with torch.no_grad():
        assert torch.equal(moe.moe_forward_ep(x.requires_grad_(), logits, k, E, mlp), ep)
    try:
        moe.moe_forward_ep(x, logits, k, E, mlp)
        raise SystemExit("a gradient of the tokens was not refused")
    except ValueError:
        pass
ops.check_status()
torch.cuda.synchronize()
dist.destroy_process_group()
print("EP_OK")
"""


def test_one_rank_is_the_single_gpu_layer(tmp_path):
    env = dict(os.environ, PYTHONPATH=ROOT)
    r = subprocess.run([sys.executable, "-c", CODE, str(tmp_path / "store")], env=env, cwd=ROOT, capture_output=True, text=True, timeout=240)
    assert r.returncode == 0 and "EP_OK" in r.stdout, r.stdout[-2000:] + r.stderr[-3000:]
