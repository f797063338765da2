"""Run the cases of perf/operators.py on graphvae.ops, 400 calls each (the clocks settle after some tens), for a
kernel trace:
rocprofv3 --kernel-trace --stats --output-format csv -d OUT -- python3 benchmarks/norm8_kernels.py [case,case]"""
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))
import perf.operators as cases  # noqa: E402

cases.own = True
only = sys.argv[1].split(",") if len(sys.argv) > 1 else None
for case in cases.listed():
    if only and case["name"] not in only:
        continue
    state = cases.prepare(dict(case), 1)
    for _ in range(400):
        cases.run(state)
    torch.cuda.synchronize()
    print(case["name"], flush=True)
    del state
    torch.cuda.empty_cache()
