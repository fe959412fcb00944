"""Masked selections (nd_select_mask_d) over batches of changing size, which share the
context's workspace of split rows: every row of every call gets the definition's id, and
its log-probability within the 1e-9 of the kernel's float32 terms below e^-20."""

import sys

import numpy as np
import pytest

from helpers import DeviceArray
from test_gpu_shared import choice_oracle

pytestmark = pytest.mark.gpu


def test_masked_selections_of_changing_batches(hip, rng):
    calls = []
    for rows, v in ((64, 32768), (40, 32768), (1, 32768), (8, 4096), (3, 8192), (96, 8192), (64, 4096),
                    (2, 65536)):
        logits = (rng.standard_normal((rows, v)) * 4).astype(np.float32)
        ok = rng.random((rows, v)) < 0.02
        ok[np.arange(rows), rng.integers(0, v, rows)] = True
        bits = np.packbits(ok, axis=1, bitorder="little").view(np.uint32)
        calls.append((rows, v, DeviceArray(logits), DeviceArray(bits),
                      [choice_oracle(logits[r], ok[r]) for r in range(rows)]))
    for turn in (calls, calls[::-1], calls):
        for rows, v, dl, dm, want in turn:
            print("[case] select mask", rows, v, file=sys.stderr, flush=True)
            ids, lps = DeviceArray(np.full(rows, 0x5A5A5A5A, np.uint32)), DeviceArray(np.full(rows, 1e300))
            hip._check(hip.lib.nd_select_mask_d(hip.ctx, dl.ptr, rows, v, dm.ptr, ids.ptr, lps.ptr, None))
            hip._check(hip.lib.nd_sync(hip.ctx))
            got = ids.read(), lps.read()
            for r, (pick, lp) in enumerate(want):
                assert got[0][r] == pick, (rows, v, r)
                assert abs(got[1][r] - lp) <= 1e-9 * max(1, abs(lp)), (rows, v, r)
            ids.free(), lps.free()
    for _, _, dl, dm, _ in calls:
        dl.free(), dm.free()
