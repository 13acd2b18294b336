"""The experts' products without a GPU: what the C ABI refuses and says, what the Python calls check, and the 64-bit
definition that the GPU tests compare with."""

import ctypes
import re
import shutil
import subprocess
import sys
from pathlib import Path

import pytest
import torch

import experts_reference as ref
from pplx_garden_amd.kernels import experts
from pplx_garden_amd.native import p2p_all_to_all as native

HEADER = (Path(__file__).resolve().parent.parent / "include" / "a2a.h").read_text()
F8, F16, BF16, F32 = 9, 11, 12, 13


def test_struct_layouts_match_the_header():
    for struct, cname in ((native.A2AExpertArgs, "a2a_expert_args"), (native.A2AExpertGradArgs, "a2a_expert_grad_args")):
        body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (cname, cname), HEADER, flags=re.S).group(1)
        body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
        assert [f for f, _ in struct._fields_] == re.findall(r"(\w+)\s*;", body), cname
    assert ctypes.sizeof(native.A2AExpertArgs) == 10 * 4 + 22 * 8
    assert ctypes.sizeof(native.A2AExpertGradArgs) == 8 * 4 + 17 * 8


def forward(**over):
    a = dict(struct_size=ctypes.sizeof(native.A2AExpertArgs), device=0, num_experts=4, expert_padding=1, rows=32, rows_per_expert=0,
             n=64, k=128, in_dtype=BF16, out_dtype=BF16, num_tokens=0x1000, x=0x1000, x_stride=256, weight=0x1000, weight_stride=256,
             weight_stride_expert=64 * 256, out=0x1000, out_stride=128)
    a.update(over)
    return native.A2AExpertArgs(**a)


FP8 = dict(in_dtype=F8, x_scale=0x1000, weight_scale=0x1000)


@pytest.mark.parametrize("gated,over,code,needle", [
    (False, dict(struct_size=8), -1, "struct_size"),
    (False, dict(in_dtype=F32), -3, "in_dtype"),
    (False, dict(out_dtype=F32), -3, "out_dtype"),
    (False, dict(out_dtype=F8, **FP8), -3, "out_dtype"),
    (True, dict(out_dtype=BF16, **FP8), -3, "out_dtype"),
    (False, dict(num_experts=0), -3, "num_experts"),
    (False, dict(num_experts=1025), -3, "num_experts"),
    (False, dict(expert_padding=0), -1, "expert_padding"),
    (False, dict(rows=0x7FFFFFFF), -3, "too many rows"),
    (False, dict(num_tokens=None), -1, "one expert"),
    (False, dict(n=0), -3, "n 0"),
    (False, dict(n=12), -3, "multiple of 8"),
    (True, dict(n=24, out_dtype=F8, out_scale=0x1000, **FP8), -3, "multiple of 16"),
    (False, dict(k=0), -3, "k 0"),
    (False, dict(k=12), -3, "multiple of 16 bytes"),
    (False, dict(in_dtype=F8, out_dtype=BF16), -1, "scales"),
    (False, dict(x_scale=0x1000), -1, "scales"),
    (False, dict(out_scale=0x1000), -1, "out_scale"),
    (True, dict(out_dtype=F8, **FP8), -1, "out_scale"),
    (False, dict(projections=0x1000, projections_stride=256), -3, "projections"),
    (False, dict(x=None), -1, "null x"),
    (False, dict(x=0x1008), -3, "multiples of 16"),
    (False, dict(x_stride=264), -3, "multiples of 16"),
    (False, dict(x_stride=240), -1, "shorter"),
    (False, dict(x_stride=1 << 24), -3, "below"),
    (False, dict(weight=None), -1, "null weight"),
    (False, dict(weight_stride_expert=64 * 256 + 8), -3, "expert to expert"),
    (False, dict(weight_stride_expert=256), -1, "overlap"),
    (False, dict(n=1 << 21, weight_stride=2048, weight_stride_expert=1 << 33, out_stride=1 << 22), -3, "4 GiB"),
    (False, dict(out=None), -1, "null out"),
    (False, dict(out_stride=112), -1, "shorter"),
    (True, dict(projections=0x1000, projections_stride=128, weight_stride_expert=128 * 256), -1, "projections"),
])
def test_bad_products_are_refused_with_a_message(gated, over, code, needle):
    lib = native.load_library()
    call = lib.a2a_expert_gated if gated else lib.a2a_expert_matmul
    args = dict(weight_stride_expert=128 * 256) if gated else {}
    rc = call(ctypes.byref(forward(**{**args, **over})), None)
    text = lib.a2a_last_error(None).decode()
    assert rc == code and needle in text, (rc, text)
    assert call(None, None) == -1


def gradient(**over):
    a = dict(struct_size=ctypes.sizeof(native.A2AExpertGradArgs), device=0, num_experts=4, expert_padding=1, rows=32, n=64, k=128,
             dtype=BF16, num_tokens=0x1000, grad_out=0x1000, grad_out_stride=128, projections=0x1000, projections_stride=256,
             grad_projections=0x1000, grad_projections_stride=256, x=0x1000, x_stride=256, weight=0x1000, weight_stride=256,
             weight_stride_expert=128 * 256, grad_x=0x1000, grad_x_stride=256, grad_weight=0x1000, grad_weight_stride=256,
             grad_weight_stride_expert=128 * 256)
    a.update(over)
    return native.A2AExpertGradArgs(**a)


@pytest.mark.parametrize("over,code,needle", [
    (dict(struct_size=8), -1, "struct_size"),
    (dict(dtype=F8), -3, "dtype"),
    (dict(num_experts=0), -3, "num_experts"),
    (dict(n=4), -3, "multiple of 8"),
    (dict(k=4), -3, "multiple of 16 bytes"),
    (dict(grad_out=None), -1, "null grad_out"),
    (dict(projections=None), -1, "null projections"),
    (dict(grad_projections=None), -1, "null grad_projections"),
    (dict(grad_projections_stride=128), -1, "shorter"),
    (dict(x=None), -1, "null x"),
    (dict(weight=None), -1, "null weight"),
    (dict(grad_x_stride=128), -1, "shorter"),
    (dict(grad_weight_stride_expert=64 * 256), -1, "overlap"),
    (dict(grad_weight=0x1004), -3, "multiples of 16"),
])
def test_bad_gradients_are_refused_with_a_message(over, code, needle):
    lib = native.load_library()
    rc = lib.a2a_expert_gated_grad(ctypes.byref(gradient(**over)), None)
    text = lib.a2a_last_error(None).decode()
    assert rc == code and needle in text, (rc, text)
    assert lib.a2a_expert_matmul_grad(None, None) == -1 and lib.a2a_expert_gated_grad(None, None) == -1


def test_a_product_of_no_rows_launches_nothing():
    lib = native.load_library()
    assert lib.a2a_expert_matmul(ctypes.byref(forward(rows=0, x=None, out=None)), None) == 0


def test_a_workspace_that_is_not_aligned_is_refused():
    lib = native.load_library()
    rc = lib.a2a_expert_matmul(ctypes.byref(forward(workspace=0x1008, workspace_bytes=1 << 20)), None)
    text = lib.a2a_last_error(None).decode()
    assert rc == -3 and "workspace" in text, (rc, text)


@pytest.mark.parametrize("over,code,needle", [(dict(rows=1 << 25), -3, "too many rows"), (dict(expert_padding=1 << 31), -1, "expert_padding")])
def test_counts_that_would_not_add_up_in_32_bits_are_refused(over, code, needle):
    lib = native.load_library()
    rc = lib.a2a_expert_matmul(ctypes.byref(forward(**over)), None)
    text = lib.a2a_last_error(None).decode()
    assert rc == code and needle in text, (rc, text)


def test_calls_refuse_tensors_that_are_not_on_a_gpu():
    x, w = torch.zeros((4, 16)).bfloat16(), torch.zeros((2, 8, 16)).bfloat16()
    num = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(AssertionError, match="GPU"):
        experts.expert_matmul(torch.zeros((4, 8)).bfloat16(), x, w, num)
    with pytest.raises(AssertionError, match="dimensions"):
        experts.expert_matmul(torch.zeros((4, 8)).bfloat16(), x[0], w, num)
    with pytest.raises(TypeError, match="expert_x must be a torch.Tensor"):
        experts.expert_gated(torch.zeros((4, 4)).bfloat16(), None, w, num)
    with pytest.raises(ValueError, match="expert_padding"):
        experts.expert_matmul(torch.zeros((4, 8)).bfloat16(), x, w, num, expert_padding=0)
    with pytest.raises(AssertionError, match="GPU"):
        experts.expert_gated_grad(None, None, x, x, x, x, w, num)


def test_quantized_weights_stand_for_the_weights():
    torch.manual_seed(0)
    w = torch.randn((2, 200, 150)) * torch.tensor([1.0, 1e-9])[:, None, None]
    codes, scale = experts.quantize_weight(w)
    assert codes.shape == w.shape and scale.shape == (2, 2, 2)
    for e in range(2):
        back = ref.dequantize(codes[e], scale[e], 128)
        step = scale[e].double().repeat_interleave(128, 0)[:200].repeat_interleave(128, 1)[:, :150]
        assert ((back - w[e].double()).abs() <= w[e].double().abs() * 2.0 ** -4 + step * 2.0 ** -10).all()
    assert (scale[1] == torch.tensor(1e-4) / 448).all()


def test_the_reference_gradients_are_those_of_the_reference_forward():
    torch.manual_seed(1)
    g, u, dh = (torch.randn((5, 7), dtype=torch.float64) * 3 for _ in range(3))
    g.requires_grad_(), u.requires_grad_()
    (ref.silu(g) * u * dh).sum().backward()
    dg, du = ref.gate_gradient(dh, g.detach(), u.detach())
    assert torch.allclose(dg, g.grad, rtol=1e-12) and torch.allclose(du, u.grad, rtol=1e-12)


def test_ranges_of_experts():
    assert ref.ranges([3, 0, 5], 4, 20) == [(0, 3), (4, 0), (4, 5)]
    assert ref.ranges([3, 9, 5], 4, 10) == [(0, 3), (4, 6), (10, 0)]


def test_a_step_that_expects_less_than_a_row_an_expert_says_none():
    """tokens * topk // experts of a small step: taken (what the call then refuses is that there is no GPU)."""
    x, w, num = torch.zeros((4, 16)).bfloat16(), torch.zeros((2, 8, 16)).bfloat16(), torch.zeros(2, dtype=torch.int32)
    for expected in (0, 1, None):
        with pytest.raises(AssertionError, match="GPU"):
            experts.expert_matmul(torch.zeros((4, 8)).bfloat16(), x, w, num, tokens_per_expert=expected)
        with pytest.raises(AssertionError, match="GPU"):
            experts.expert_gated(torch.zeros((4, 4)).bfloat16(), x, w, num, tokens_per_expert=expected)
    for expected in (-1, 1 << 31):
        with pytest.raises(ValueError, match="tokens_per_expert"):
            experts.expert_matmul(torch.zeros((4, 8)).bfloat16(), x, w, num, tokens_per_expert=expected)


RUNTIME_WITHOUT_UNITS = """
extern "C" {
int hipGetDevice(int *device) { *device = 0; return 0; }
int hipSetDevice(int) { return 0; }
int hipDeviceGetAttribute(int *value, int, int) { *value = 0; return 0; }
}
"""

CALL_WITHOUT_UNITS = """
import ctypes, sys
sys.path[:0] = sys.argv[2:]
ctypes.CDLL(sys.argv[1], ctypes.RTLD_GLOBAL)     # before the library: its calls of the runtime find these first
import test_experts_host as t
lib = t.native.load_library()
for call, args in ((lib.a2a_expert_matmul, t.forward()), (lib.a2a_expert_matmul_grad, t.gradient())):
    print(call(ctypes.byref(args), None), lib.a2a_last_error(None).decode())
"""


def test_a_device_that_names_no_compute_units_is_an_error(tmp_path):
    """The runtime answers, but with 0 units: refused before anything is launched, with a code that is not success."""
    compiler = shutil.which("g++") or shutil.which("c++")
    if compiler is None:
        pytest.skip("needs a C++ compiler")
    (tmp_path / "runtime.cpp").write_text(RUNTIME_WITHOUT_UNITS)
    runtime = tmp_path / "runtime.so"
    subprocess.run([compiler, "-shared", "-fPIC", str(tmp_path / "runtime.cpp"), "-o", str(runtime)], check=True)
    here = Path(__file__).resolve().parent
    result = subprocess.run([sys.executable, "-c", CALL_WITHOUT_UNITS, str(runtime), str(here), str(here.parent / "pplx-garden_amd")],
                            check=True, capture_output=True, text=True, timeout=100)
    lines = result.stdout.splitlines()
    assert len(lines) == 2 and all(line.startswith("-3 ") and "compute units" in line for line in lines), lines
