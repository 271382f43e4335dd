"""The hand-off of a long row's bins in sample_scores (the workgroup that arrives last finds the border's step) under arrival skew.

Every workgroup adds its bins to the row's, waits for the adds' old values, and arrives; the last to arrive reads the bins and clears them for
the next selection.  UR_TEST=arrival_skew_us=k delays every arrival by (hash of the workgroup) % k microseconds, so that the last arriver
moves over the XCDs.  An add that is still under way at the arrival would be missing from the border, or be left over in the next one's bins:
sums are integers, so every process must draw the same entries."""
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

CHILD = r'''
import hashlib, sys, torch
sys.path.insert(0, %r)
from unirec_amd import ops
dev = torch.device("cuda:0")
h = hashlib.sha256()
g = torch.Generator(device=dev).manual_seed(1)
for dtype, B, N in ((torch.float32, 16, 200_003), (torch.bfloat16, 24, 150_001), (torch.float32, 3, 1_000_000)):
    for it in range(12):
        x = (torch.randn(B, N, device=dev, generator=g) * 2).to(dtype)
        u = torch.rand(B, 8, device=dev, generator=g)
        for kw in (dict(top_p=0.9), dict(top_k=5000), dict(top_k=20_000, top_p=0.7, temperature=1.5)):
            for t in ops.sample_scores(x, u, **kw):
                h.update(t.cpu().numpy().tobytes())
print("DIGEST", h.hexdigest())
''' % ROOT


def _run(**env):
    e = dict(os.environ)
    e.pop("UR_TEST", None)
    e.update({k: str(v) for k, v in env.items()})
    r = subprocess.run([sys.executable, "-c", CHILD], env=e, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]
    return [ln for ln in r.stdout.splitlines() if ln.startswith("DIGEST")][-1]


@pytest.mark.gpu
def test_bins_are_complete_under_arrival_skew():
    base = _run()
    assert _run(UR_TEST="arrival_skew_us=30") == base
    assert _run(UR_TEST="arrival_skew_us=200") == base
