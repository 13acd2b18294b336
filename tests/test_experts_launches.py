"""Which kernels the experts' products launch, without a GPU: the library runs against a stand-in for the HIP runtime that writes
launches down.  The GPU tests have to reach every kernel that there is, so that a refit of the rules cannot leave one untested."""

import ctypes
import itertools
import json
import re
import shutil
import subprocess
import sys

import pytest

import test_gpu_experts as gpu
from pplx_garden_amd.native import p2p_all_to_all as native
from test_experts_host import BF16, F8, F16

RUNTIME = """
#include <cstddef>
#include <cstdint>
#include <map>
#include <string>
struct dim3 { uint32_t x, y, z; };
static std::map<const void *, std::string> kernels;
static std::string names, record;
static dim3 grid, block;
static size_t shared;
static void *stream;
extern "C" {
int hipGetDevice(int *device) { *device = 0; return 0; }
int hipSetDevice(int) { return 0; }
int hipGetLastError() { return 0; }
int hipDeviceGetAttribute(int *value, int, int) { *value = 256; return 0; }
void **__hipRegisterFatBinary(const void *) { static void *module; return &module; }
void __hipUnregisterFatBinary(void **) {}
void __hipRegisterVar(void **, void *, char *, char *, int, size_t, int, int) {}
void __hipRegisterFunction(void **, const void *function, char *, const char *name, unsigned, void *, void *, void *, void *, int *) {
    kernels[function] = name;
    names += std::string(name) + " ";
}
int __hipPushCallConfiguration(dim3 g, dim3 b, size_t s, void *t) { grid = g; block = b; shared = s; stream = t; return 0; }
int __hipPopCallConfiguration(dim3 *g, dim3 *b, size_t *s, void **t) { *g = grid; *b = block; *s = shared; *t = stream; return 0; }
int hipLaunchKernel(const void *function, dim3, dim3, void **, size_t, void *) { record += kernels[function] + " "; return 0; }
const char *all_kernels() { return names.c_str(); }
const char *launched() { static std::string last; last.swap(record); record.clear(); return last.c_str(); }
}
"""

# (no torch in it: torch brings the real runtime)
CALLS = """
import ctypes, json, sys
runtime = ctypes.CDLL(sys.argv[1], ctypes.RTLD_GLOBAL)     # before the library: its calls of the runtime find these first
lib = ctypes.CDLL(sys.argv[2])
runtime.launched.restype = runtime.all_kernels.restype = ctypes.c_char_p
out = []
for name, args in json.load(sys.stdin):
    rc = getattr(lib, name)(ctypes.create_string_buffer(bytes.fromhex(args)), None)
    assert rc == 0, (name, rc)
    out.append(runtime.launched().decode().split())
json.dump([runtime.all_kernels().decode().split(), out], sys.stdout)
"""

TYPE = {"fp8": F8, "bf16": BF16, "f16": F16}
MODES, ENDS, TYPES = ("forward", "dx", "dW"), ("plain", "gated", "gated fp8", "parts"), ("fp8", "bf16", "f16")


def readable(name):
    """(type, mode, end, rows, columns, "once" or "") of a product's kernel, (type, "finish", end) of its second launch."""
    numbers = [int(n) for n in re.findall(r"L[ib](\d+)E", name)]
    if "product_kernel" in name:
        t, mode, end, rows, columns, once = *numbers[:5], numbers[-1]
        return TYPES[t], MODES[mode], ENDS[end], rows, columns, "once" if once else ""
    if "finish_kernel" in name:
        return TYPES[numbers[0]], "finish", ENDS[numbers[1]]
    return (TYPES[numbers[0]], "gate") if "gate_gradient_kernel" in name else None


@pytest.fixture(scope="module")
def launches(tmp_path_factory):
    compiler = shutil.which("g++") or shutil.which("c++")
    if compiler is None:
        pytest.skip("needs a C++ compiler")
    folder = tmp_path_factory.mktemp("runtime")
    (folder / "runtime.cpp").write_text(RUNTIME)
    subprocess.run([compiler, "-std=c++17", "-shared", "-fPIC", str(folder / "runtime.cpp"), "-o", str(folder / "runtime.so")], check=True)

    def run(calls):
        """All kernels of the experts' products, and those that each call launches."""
        text = json.dumps([(name, bytes(args).hex()) for name, args in calls])
        result = subprocess.run([sys.executable, "-c", CALLS, str(folder / "runtime.so"), str(native.library_path())], input=text,
                                capture_output=True, text=True, timeout=100)
        assert result.returncode == 0, result.stderr
        everything, launched = json.loads(result.stdout)
        return {r for r in map(readable, everything) if r is not None}, [[readable(k) for k in one] for one in launched]

    return run


def forward(call, type_, rows, experts, n, k, expected=0, projections=False):
    gated, fp8 = call == "gated", type_ == "fp8"
    size, width = 1 if fp8 else 2, 2 * n if gated else n
    stride = -(-k * size // 16) * 16
    return f"a2a_expert_{call}", native.A2AExpertArgs(
        struct_size=ctypes.sizeof(native.A2AExpertArgs), num_experts=experts, expert_padding=1, rows=rows, rows_per_expert=expected, n=n, k=k,
        in_dtype=TYPE[type_], out_dtype=(F8 if gated else BF16) if fp8 else TYPE[type_], num_tokens=0x1000, x=0x1000, x_stride=stride,
        x_scale=0x1000 if fp8 else None, weight_scale=0x1000 if fp8 else None, weight=0x1000, weight_stride=stride,
        weight_stride_expert=width * stride, out=0x1000, out_stride=2 * n, out_scale=0x1000 if fp8 and gated else None,
        projections=0x1000 if projections else None, projections_stride=4 * n, workspace=0x1000 if rows <= 512 else None,
        workspace_bytes=16 << 20)


def gradient(call, type_, rows, experts, n, k, wide=0, grad_x=True, grad_w=True):
    width = 2 * n if call == "gated" else n
    stride = 2 * (k + wide)
    return f"a2a_expert_{call}_grad", native.A2AExpertGradArgs(
        struct_size=ctypes.sizeof(native.A2AExpertGradArgs), num_experts=experts, expert_padding=1, rows=rows, n=n, k=k, dtype=TYPE[type_],
        num_tokens=0x1000, grad_out=0x1000, grad_out_stride=2 * n, projections=0x1000, projections_stride=2 * width,
        grad_projections=0x1000, grad_projections_stride=2 * width, x=0x1000, x_stride=2 * k, weight=0x1000, weight_stride=2 * k,
        weight_stride_expert=2 * width * k, grad_x=0x1000 if grad_x else None, grad_x_stride=2 * k, grad_weight=0x1000 if grad_w else None,
        grad_weight_stride=stride, grad_weight_stride_expert=width * stride)


def parameters(test):
    """Dictionaries of a test's parametrised arguments."""
    axes = []
    for mark in test.pytestmark:
        if mark.name == "parametrize":
            names = [n.strip() for n in mark.args[0].split(",")]
            axes.append([dict(zip(names, v if len(names) > 1 else [v])) for v in mark.args[1]])
    for together in itertools.product(*axes):
        yield {name: value for one in together for name, value in one.items()}


def buffer_of(kind):
    counts, padding, extra = gpu.ROWS[kind]
    return sum(-(-c // padding) * padding for c in counts) + extra, len(counts)


def calls_of_the_gpu_tests():
    for p in parameters(gpu.test_fp8_matmul):
        yield forward("matmul", "fp8", *buffer_of(p["kind"]), p["n"], p["k"], p["expected"])
    for p in parameters(gpu.test_fp8_gated):
        yield forward("gated", "fp8", *buffer_of(p["kind"]), p["n"], p["k"], p["expected"])
    for p in parameters(gpu.test_matmul_and_gated):
        yield forward("matmul", p["type_"], *buffer_of(p["kind"]), 2 * p["n"], p["k"], p["expected"])
        yield forward("gated", p["type_"], *buffer_of(p["kind"]), p["n"], p["k"], p["expected"], True)
    for p in parameters(gpu.test_few_rows_of_long_sums):
        yield forward("matmul", p["type_"], *buffer_of(p["kind"]), 2 * p["n"], p["k"])
        yield forward("gated", p["type_"], *buffer_of(p["kind"]), p["n"], p["k"])
    for p in parameters(gpu.test_every_tile_of_a_product):
        yield forward("matmul", p["type_"], *buffer_of(p["kind"]), p["n"], p["k"], p["expected"])
    for p in parameters(gpu.test_every_tile_of_a_gated_product):
        yield forward("gated", p["type_"], *buffer_of(p["kind"]), p["n"], p["k"], p["expected"])
    for p in parameters(gpu.test_weights_larger_than_the_caches):
        n, k = (2064 // 32 * 16, "gated") if p["gated"] else (2064, "matmul")
        yield forward(k, p["type_"], 562, 18, n, 8464 if p["type_"] == "fp8" else 4240, p["expected"])
    for p in parameters(gpu.test_gradients):
        yield gradient("gated", p["type_"], *buffer_of(p["kind"]), p["n"], p["k"], wide=8)
    for p in parameters(gpu.test_every_tile_of_the_gradients):
        yield gradient("matmul", p["type_"], sum(p["counts"]) + 2, len(p["counts"]), p["n"], p["k"], wide=8)
    for p in parameters(gpu.test_a_large_weights_gradient_whose_lines_two_tiles_share):
        yield gradient("matmul", p["type_"], sum(p["counts"]) + 2, len(p["counts"]), p["n"], p["k"], grad_x=False)


def test_the_gpu_tests_reach_every_kernel(launches):
    everything, launched = launches(calls_of_the_gpu_tests())
    reached = {kernel for one in launched for kernel in one}
    assert None not in reached and len(everything) > 60
    assert everything - reached == set()
