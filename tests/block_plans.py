"""Plans of block and grouped products without a GPU, for the tests of what is
chosen and refused: tests/cpp/block_plan.cpp as a program of its own, so that a
plan that ends its process ends that one."""
import os
import subprocess

import einsum_ir_amd as eir

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(ROOT, "einsum_ir_amd")


def build(folder):
    exe = os.path.join(str(folder), "block_plan")
    subprocess.check_call(["g++", "-O1", "-std=c++17", "-Wall", "-I" + os.path.join(ROOT, "include"),
                           os.path.join(ROOT, "tests", "cpp", "block_plan.cpp"), "-o", exe,
                           "-L" + PKG, "-leinsum_ir_hip", "-Wl,-rpath," + PKG])
    return exe


def _list(values):
    return "-" if values is None else ",".join(str(int(v)) for v in values)


def f8_line(loops, left=eir.F8E4M3, scale=eir.FP32, out=eir.BF16):
    """A line for the program; loops: of contraction_f8_loops."""
    lists = [loops.get(k) for k in ("dim_types", "sizes", "strides_left", "strides_right", "strides_scale_left",
                                    "strides_scale_right", "strides_bias", "strides_out")]
    return " ".join(["f8"] + [_list(v) for v in lists] + [str(v) for v in (
        loops.get("block_left", 1), loops.get("block_right", 128), left, eir.F8E4M3, scale, out, eir.UNDEFINED_KTYPE)])


def grouped_line(loops, left=eir.BF16, scale=eir.FP32, out=eir.BF16):
    """The same of grouped_loops."""
    lists = [loops.get(k) for k in ("dim_types", "sizes", "strides_left", "strides_right", "strides_scale_left",
                                    "strides_scale_right", "strides_out")]
    right = left if left == eir.BF16 else eir.F8E4M3
    return " ".join(["grouped"] + [_list(v) for v in lists] + [str(v) for v in (
        loops["ragged"], loops.get("block_left", 1), loops.get("block_right", 128), left, right, scale, out)])


def describe(exe, lines, env=None):
    """What the program says of each line; env: added to the environment."""
    res = subprocess.run([exe], input="\n".join(lines) + "\n", capture_output=True, text=True, timeout=120,
                         env=None if env is None else dict(os.environ, **env))
    assert res.returncode == 0, f"ended with {res.returncode} after {res.stdout!r}"
    found = res.stdout.splitlines()
    assert len(found) == len(lines)
    return found
