"""Shapes and plans of the state-space operators: what they refuse, and their layout.  No GPU needed."""
import ctypes as C
import os
import subprocess

import pytest

from fastconv_amd import capi

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_struct_layouts_match_the_header(tmp_path):
    structs = {"fc_rms_norm_shape": capi.RmsNormShape, "fc_rms_norm_plan": capi.RmsNormPlan, "fc_int8_product_shape": capi.Int8ProductShape,
               "fc_int8_product_plan": capi.Int8ProductPlan, "fc_causal_conv_shape": capi.CausalConvShape, "fc_causal_conv_plan": capi.CausalConvPlan,
               "fc_selective_scan_shape": capi.SelectiveScanShape, "fc_selective_scan_plan": capi.SelectiveScanPlan}
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "fastconv_hip.h"', 'int main(void) {']
    for cname, ct in structs.items():
        lines.append('printf("%s sizeof %%zu\\n", sizeof(%s));' % (cname, cname))
        lines += ['printf("%s %s %%zu\\n", offsetof(%s, %s));' % (cname, f, cname, f) for f, _ in ct._fields_]
    lines.append('return 0;}')
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines))
    subprocess.check_call(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)])
    seen = 0
    for line in subprocess.check_output([str(exe)], text=True).splitlines():
        cname, field, value = line.split()
        assert (C.sizeof(structs[cname]) if field == "sizeof" else getattr(structs[cname], field).offset) == int(value), (cname, field)
        seen += 1
    assert seen == sum(len(ct._fields_) + 1 for ct in structs.values())


MAKERS = {"norm": ("fc_rms_norm_make_plan", capi.RmsNormPlan, lambda: capi.RmsNormShape.packed(10, 64, capi.BF16)),
          "product": ("fc_int8_product_make_plan", capi.Int8ProductPlan, lambda: capi.Int8ProductShape.packed(10, 64, 48, capi.BF16)),
          "conv": ("fc_causal_conv_make_plan", capi.CausalConvPlan, lambda: capi.CausalConvShape.packed(2, 100, 64, 4, capi.BF16)),
          "scan": ("fc_selective_scan_make_plan", capi.SelectiveScanPlan, lambda: capi.SelectiveScanShape.packed(2, 100, 64, 16, 2, capi.BF16))}


def make(which, **change):
    name, plan, shape = MAKERS[which]
    plan, shape = plan(), shape()
    for f, v in change.items():
        setattr(shape, f, v)
    return getattr(capi.load_cdll(), name)(C.byref(shape), C.byref(plan)), plan


@pytest.mark.parametrize("which,field,value,status", [
    ("norm", "rows", 0, -1), ("norm", "C", 0, -1), ("norm", "dtype", 3, -1), ("norm", "eps", -1e-6, -1), ("norm", "eps", float("nan"), -1),
    ("norm", "eps", float("inf"), -1), ("norm", "x_row", -1, -1), ("norm", "residual_row", -1, -1), ("norm", "sum_row", -1, -1), ("norm", "y_row", -1, -1),
    ("norm", "C", (1 << 20) + 1, -6), ("norm", "rows", (1 << 40) + 1, -6), ("norm", "C", 1 << 20, 0), ("norm", "rows", 1 << 40, 0),
    ("product", "M", 0, -1), ("product", "N", 0, -1), ("product", "K", 0, -1), ("product", "dtype", -1, -1), ("product", "x_row", -1, -1),
    ("product", "w_row", -1, -1), ("product", "y_row", -1, -1), ("product", "K", 131071, 0), ("product", "K", 131072, -6), ("product", "M", 1 << 31, -6),
    ("product", "M", 1 << 30, -6), ("conv", "B", 0, -1), ("conv", "T", 0, -1), ("conv", "C", 0, -1), ("conv", "taps", 1, -1), ("conv", "taps", 9, -6),
    ("conv", "dtype", 7, -1), ("conv", "act", 4, -1), ("conv", "act", capi.ACT_GELU, -6), ("conv", "act", capi.ACT_RELU, -6), ("conv", "x_batch", -1, -1),
    ("conv", "x_token", -1, -1), ("conv", "y_batch", -1, -1), ("conv", "y_token", -1, -1), ("conv", "T", 1 << 31, -6), ("conv", "B", 1 << 24, -6),
    ("scan", "B", 0, -1), ("scan", "T", 0, -1), ("scan", "D", 0, -1), ("scan", "N", 0, -1), ("scan", "G", 0, -1), ("scan", "G", 3, -1), ("scan", "dtype", 3, -1),
    ("scan", "x_token", -1, -1), ("scan", "delta_batch", -1, -1), ("scan", "z_token", -1, -1), ("scan", "b_group", -1, -1), ("scan", "c_token", -1, -1),
    ("scan", "y_batch", -1, -1), ("scan", "N", 64, 0), ("scan", "N", 65, -6), ("scan", "T", 1 << 31, -6), ("scan", "B", 1 << 20, -6)])
def test_shapes(which, field, value, status):
    assert make(which, **{field: value})[0] == status


def test_null_arguments_are_refused():
    lib = capi.load_cdll()
    for name, plan, shape in MAKERS.values():
        assert getattr(lib, name)(None, C.byref(plan())) == -1
        assert getattr(lib, name)(C.byref(shape()), None) == -1
    # calls without a context
    for name, nulls in (("fc_rms_norm", 7), ("fc_rms_norm_int8", 7), ("fc_rms_norm_backward", 9), ("fc_int8_product", 8), ("fc_causal_conv", 8),
                        ("fc_causal_conv_backward", 13), ("fc_selective_scan", 14), ("fc_selective_scan_backward", 23)):
        assert getattr(lib, name)(None, *([None] * nulls)) == -5, name
    assert lib.fc_quantize_rows(None, 1, 1, 0, None, 1, None, 1, None) == -5


def test_workspaces_hold_what_the_plans_say():
    for t in (1, 4, 5, 33, 1225, 16384):
        for d in (1, 64, 65, 2048):
            for n in (1, 4, 16, 17, 64):
                for b in (1, 3, 64):
                    wide, few = (t * d, d), (t * n, n, n)
                    strides = dict(zip(("x_batch", "x_token"), wide), b_batch=few[0], b_token=few[1], b_group=few[2])
                    rc, p = make("scan", B=b, T=t, D=d, N=n, G=1, **strides)
                    assert rc == 0
                    tiles = -(-t // 32)
                    assert p.tiles == (tiles if t > 4 else 0) and 1 <= p.segments <= tiles and 1 <= p.walks_backward <= tiles
                    assert p.ws_bytes == (4 * b * p.segments * d * (n + 1) if p.segments > 1 else 0)
                    assert p.ws_backward_bytes >= 4 * b * tiles * d * (2 * n + 1)


def test_every_part_has_work():
    """No walk, segment or part of a plan is empty."""
    for t in (1, 7, 8, 9, 63, 64, 65, 3136, 12544):
        for c in (1, 8, 63, 64, 2048):
            rc, p = make("conv", T=t, C=c, x_token=c, y_token=c, x_batch=t * c, y_batch=t * c)
            assert rc == 0
            for walks in (p.walks, p.walks_backward):
                walk = -(-t // walks)
                assert (walks - 1) * walk < t
        rc, p = make("scan", T=t)
        tiles = -(-t // 32)
        for parts in (p.segments, p.walks_backward):
            per = -(-tiles // parts)
            assert (parts - 1) * per < tiles


def test_only_the_first_walk_of_a_convolution_reaches_the_state():
    """The state after a sequence may be written over the one before it: the walks after the first begin a window or more behind its start."""
    for taps in range(2, 9):
        for t in list(range(1, 70)) + [1225, 12544]:
            for c in (1, 2, 65, 2048):
                rc, p = make("conv", T=t, C=c, taps=taps, x_token=c, y_token=c, x_batch=t * c, y_batch=t * c)
                assert rc == 0 and (p.walks == 1 or -(-t // p.walks) >= taps - 1), (taps, t, c)


@pytest.mark.parametrize("field,value,status", [("T", 1 << 30, 0), ("T", (1 << 30) + 1, -6), ("T", (1 << 31) - 1, -6), ("C", 1 << 23, 0), ("C", (1 << 23) + 1, -6)])
def test_convolutions_whose_counts_pass_32_bits(field, value, status):
    assert make("conv", **{field: value})[0] == status


@pytest.mark.parametrize("M,N,status", [(1, 1 << 26, 0), (1, 1 << 28, -6), (1, (1 << 31) - 1, -6), (64, 1 << 27, 0), (64, 1 << 29, -6), ((1 << 31) - 1, 1, -6),
                                        (1 << 28, 1, 0), (1 << 20, 1 << 15, 0)])
def test_products_whose_launch_passes_32_bits(M, N, status):
    assert make("product", M=M, N=N, K=16, x_row=16, w_row=16, y_row=N)[0] == status


def test_scans_whose_launch_or_tiles_pass_32_bits():
    for t, token, status in ((1, 1 << 40, 0), (2, (1 << 24) - 1, 0), (2, 1 << 24, -6), (4, 1 << 24, -6), (5, 1 << 24, -6), (100, (1 << 24) - 1, 0)):
        for field in ("x_token", "delta_token", "z_token", "b_token", "c_token", "y_token"):
            assert make("scan", T=t, **{field: token})[0] == status, (t, token, field)
    for d, n, status in ((1 << 20, 64, 0), (1 << 21, 64, -6), (1 << 23, 14, -6), (1 << 23, 13, 0)):
        assert make("scan", B=1, T=1, D=d, N=n, G=1)[0] == status, (d, n)
