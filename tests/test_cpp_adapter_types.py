"""Storage types that the C++ adapter's classes refuse to be compiled for: bfloat16 where a class has fp16
kernels only (its bits would be read as binary16), and matrices whose entries have another size than T."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
ROCM = os.path.dirname(os.path.dirname(os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")))
PROLOGUE = """#include "lbann_amd/adapter/lbnorm_layers.hpp"
struct my_bfloat16 { uint16_t bits; };
struct my_half { uint16_t bits; };
template <> struct lbnorm::storage_of<my_bfloat16> { static constexpr lbnorm::storage value = lbnorm::storage::bf16; };
using namespace lbnorm;
"""


def compiles(line):
    out = subprocess.run(["g++", "-std=c++17", "-fsyntax-only", "-D__HIP_PLATFORM_AMD__", "-I" + os.path.join(ROCM, "include"), "-I" + ROOT,
                          "-x", "c++", "-"], input=PROLOGUE + line + "\n", text=True, capture_output=True)
    return out.returncode == 0, out.stderr


def test_types_with_kernels_compile():
    lines = [f"template class lbnorm::{c}<device_matrix<{t}>>;" for c in ("softmax_layer", "log_softmax_layer")
             for t in ("float", "my_half")]
    lines += [f"template void lbnorm::cross_entropy_layer<device_matrix<{t}>>::{d}_compute();" for t in ("float", "my_half") for d in ("fp", "bp")]
    lines += [f"template class lbnorm::{c}<{t}>;" for c in ("layer_norm_layer", "batch_normalization_layer") for t in ("float", "my_half", "double")]
    lines += [f"template class lbnorm::{c}<{t}>;" for c in ("dropout_layer", "residual_norm_layer", "logits_adjust_layer")
              for t in ("float", "my_half", "bfloat16", "my_bfloat16")]
    ok, errors = compiles("\n".join(lines))
    assert ok, errors


@pytest.mark.parametrize("kind", ["bfloat16", "my_bfloat16"])
@pytest.mark.parametrize("line", ["softmax_layer<device_matrix<{}>> l;", "log_softmax_layer<device_matrix<{}>> l;",
                                  "cross_entropy_layer<device_matrix<{}>> l;", "layer_norm_layer<{}> l({{8}});",
                                  "layer_norm_layer<my_half, device_matrix<{}>> l({{8}});",
                                  "batch_normalization_layer<{}> l;", "batch_normalization_layer<my_half, device_matrix<{}>> l;"])
def test_bfloat16_where_there_is_fp16_only(line, kind):
    ok, errors = compiles(line.format(kind))
    assert not ok and "no bfloat16 kernels" in errors, errors


@pytest.mark.parametrize("line", ["dropout_layer<float, device_matrix<bfloat16>> l;", "residual_norm_layer<float, device_matrix<my_half>> l;",
                                  "logits_adjust_layer<bfloat16, device_matrix<float>> l;"])
def test_entries_of_another_size(line):
    ok, errors = compiles(line)
    assert not ok and "storage type of Mat's entries" in errors, errors
