"""Run as a program in a fresh process: the first call of an operator happens under a graph
capture.  Prints "ok" when the status word reads as zero before any replay and keeps through
replays what other kernels report."""

import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from moe_inference_verify_microbench_b200 import ops  # noqa: E402

dev = torch.device("cuda", 0)
# memory that a later allocation may get is full of ones
junk = [torch.full((1 << 16,), -1, dtype=torch.int32, device=dev) for _ in range(64)]
del junk
x = torch.randn(9, 256, device=dev).bfloat16()
one = torch.ones(256, device=dev)
want = x.float() * torch.rsqrt(x.float().pow(2).mean(-1, keepdim=True) + 1e-6)
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    h, y = ops.block_norm(x, torch.zeros_like(x), one, one, 1e-6)
ops.check_status(dev)  # nothing has run
graph.replay()
ops.check_status(dev)
assert torch.equal(h, x) and (y.float() - want).abs().max() <= 2.0 ** -7 * want.abs().max()
# a report stays through a replay
bad = torch.tensor([0, 5, 3], device=dev)
ops.tiles_from_offsets(bad, 8)
graph.replay()
try:
    ops.check_status(dev)
except ops.MoEKernelError:
    print("ok")
