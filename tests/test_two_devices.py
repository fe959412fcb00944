"""Calls made while another device than the context's is current, without a GPU: the
library's host code over a stand-in for the HIP runtime (two_devices.cpp).  Whatever an
entry allocates, launches or waits for is the context's device's, and the caller's
device is current again afterwards."""

import json
import os
import subprocess
import sys
from pathlib import Path

import pytest

HERE = Path(__file__).resolve().parent

CALLS = """
import ctypes as C, json, sys
import numpy as np
double = C.CDLL(sys.argv[1], mode=C.RTLD_GLOBAL)
double.double_events.restype = C.c_char_p
sys.path[:0] = sys.argv[2:]
from needle_hip import (HipBackend, HipKvCache, HipRows, HipSelector, HipSharedAttention,
                        Int8Matrix)
from needle_hip import lib as L
from needle_hip.models import DecoderGeometry, DecoderWeights, HipBatch, HipDecoder

hip = HipBackend(device=0)
lib = hip.lib
mat = hip.upload(Int8Matrix(np.ones((40, 128), np.int8), np.ones((40, 1), np.float32), 128))
prefix, own = HipKvCache(hip, 2, 8, 32), HipKvCache(hip, 2, 16, 32)
g = DecoderGeometry(layers=2, vocab=512)
batch = HipBatch(HipDecoder(hip, DecoderWeights(g, 3)), 2, 16)
device = C.c_void_p()
assert double.hipMalloc(C.byref(device), C.c_size_t(1 << 20)) == 0
d = device.value
x, q = np.ones((9, 128), np.float32), np.ones((2, 8, 64), np.float32)
y = np.empty((9, 40), np.float32)
held, seen = {}, {}


def call(name, f):
    double.hipSetDevice(1)
    double.double_clear()
    held[name] = f()
    now = C.c_int()
    double.hipGetDevice(C.byref(now))
    seen[name] = [double.double_events().decode().split(), now.value]


call("nd_rows_create", lambda: HipRows(hip, 9, 128))
rows = held["nd_rows_create"]
call("nd_rows_quantize_d", lambda: rows.quantize(d, 9))
call("nd_rows_read", rows.read)
call("nd_matmul_rows_d", lambda: rows.matmul(mat, d))
call("nd_matmul_w8a8", lambda: hip._check(lib.nd_matmul_w8a8(hip.ctx, mat, L.ptr(x), 9, L.ptr(y))))
call("nd_rows_free", rows.free)
call("nd_shared_create", lambda: HipSharedAttention(hip, 2, 8, 8))
shared = held["nd_shared_create"]
call("nd_shared_attention_d", lambda: shared.run(prefix, 9, own, d, 32, 1, d, d))
call("nd_shared_attention", lambda: shared.attention(prefix, 9, own, [3, 0], 1, q))
call("nd_shared_free", shared.free)
call("nd_selector_create", lambda: HipSelector(hip, 9))
selector = held["nd_selector_create"]
call("nd_select_adjusted_d", lambda: selector.run(d, 9, 128, d, d))
call("nd_select_adjusted", lambda: selector.select(x, repetition=np.ones(9)))
call("nd_selector_free", selector.free)
call("nd_batch_set_prefix", lambda: batch.set_prefix(prefix, 20))
call("nd_batch_set_adjust", lambda: batch.set_adjust(8, history=np.zeros((2, 5), np.uint32)))
call("nd_batch_free", batch.free)
print(json.dumps(seen))
"""


@pytest.fixture(scope="module")
def seen(tmp_path_factory):
    double = tmp_path_factory.mktemp("two_devices") / "two_devices.so"
    rocm = os.environ.get("ROCM_PATH", "/opt/rocm")
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-D__HIP_PLATFORM_AMD__",
                    f"-I{rocm}/include", str(HERE / "two_devices.cpp"), "-o", str(double)], check=True)
    done = subprocess.run([sys.executable, "-c", CALLS, str(double), str(HERE.parent),
                           str(HERE.parent / "needle.js_amd")], check=True, capture_output=True,
                          text=True, timeout=300)
    return json.loads(done.stdout.splitlines()[-1])


WAITS = ("nd_rows_read", "nd_rows_free", "nd_shared_free", "nd_selector_free", "nd_batch_set_prefix",
         "nd_batch_set_adjust", "nd_batch_free")
ENTRIES = ("nd_rows_create", "nd_rows_quantize_d", "nd_matmul_rows_d", "nd_matmul_w8a8",
           "nd_shared_create", "nd_shared_attention_d", "nd_shared_attention", "nd_selector_create",
           "nd_select_adjusted_d", "nd_select_adjusted") + WAITS


@pytest.mark.parametrize("entry", ENTRIES)
def test_entries_work_on_the_contexts_device(seen, entry):
    events, current = seen[entry]
    assert events and all(e.endswith(":0") for e in events), events
    assert current == 1
    assert ("synchronize:0" in events) == (entry in WAITS or entry == "nd_matmul_w8a8"), events
