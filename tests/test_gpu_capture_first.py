"""One call of any operator on a device readies all of them there: each may be captured in a CUDA graph before it has been called (GPU).

A process of its own for each operator that is called first.
"""

import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

CHILD = """
import ctypes
import sys
import torch
import qr_v2_b200_kernel_b200 as qr

first = sys.argv[1]
BF = torch.bfloat16
x = torch.randn(40, 256, device="cuda").to(BF)
w = torch.randn(300, 256, device="cuda").to(BF)
k = torch.randn(40, 2, 64, device="cuda").to(BF)
q = torch.randn(1, 4, 8, 64, device="cuda").to(BF)
many = torch.randn(40, 40, 32, 64, device="cuda").to(BF)
slots = torch.arange(40, device="cuda")
table = torch.arange(4, device="cuda").int()[None]
tables = table.repeat(40, 1)
n = torch.tensor([40], dtype=torch.int32, device="cuda")
ns = torch.full((40,), 40, dtype=torch.int32, device="cuda")
long = torch.randn(1100, 8, 64, device="cuda").to(BF)
lists = torch.arange(1100, device="cuda")
lists[64:] = -1
A = torch.randn(2, 64, 64, device="cuda")


def cached(make, write, read, attend):
    cache = make(4, 16, 2, 64)
    write(cache, k, k, slots)
    return attend(q, cache, table, n), read(cache, slots)[0]


def prompts():
    cache = qr.kv8_cache(4, 16, 8, 64)
    qr.kv8_write(cache, long, long, lists)
    return (qr.kv8_attention(many, cache, tables, ns),)


def linear(quantise, product, *tile):
    a, sa = quantise(x)
    b, sb = quantise(w, *tile)
    return product(a, sa, b, sb), product(a[:5], sa[:5], b, sb)


calls = {
    "qr": lambda: qr.custom_kernel(A),
    "int8": lambda: linear(qr.quantize_int8, qr.int8_linear),
    "fp8": lambda: linear(qr.quantize_fp8, qr.fp8_linear, 128),
    "kv4": lambda: cached(qr.kv4_cache, qr.kv4_write, qr.kv4_read, qr.kv4_attention),
    "kv8": lambda: cached(qr.kv8_cache, qr.kv8_write, qr.kv8_read, qr.kv8_attention),
    "prompts": prompts,
}
calls[first]()
torch.cuda.synchronize()
# A stream of a program's own, which waits for the default one (torch's do not): nothing may use that one during a capture.
made = ctypes.c_void_p()
assert ctypes.CDLL("libcudart.so.12").cudaStreamCreate(ctypes.byref(made)) == 0
stream = torch.cuda.ExternalStream(made.value)
for name, call in calls.items():
    if name == "qr":
        continue
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        got = call()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, call())), name
    graph.reset()
print("as one")
"""


@pytest.mark.parametrize("first", ["qr", "int8", "fp8", "kv4", "kv8"])
def test_a_call_of_one_operator_readies_the_others_for_capture(first):
    r = subprocess.run([sys.executable, "-c", CHILD, first], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "as one" in r.stdout, r.stderr[-2000:]
